// Eviction from the paged cache by accumulated attention weight (the weight per key is what
// attention_mass.cu adds up): which keys of a request stay, and their move to the front of its pages.
//
//   choose   of the n keys of a request, per kv head, `budget` stay: the first `keep_first`, the last
//            `keep_last`, and of the others those of the largest weights, of equal weights the lowest
//            index. kept[0 .. min(n, budget)) are their indices in ascending order, -1 behind. n <= budget: all stay.
//   compact  the rows of the kept keys move to the front, in their order: row i <- row kept[i], of keys,
//            values and weights alike. Rows from min(n, budget) on are left as they are.
//
// choose is a selection by digits: a weight becomes a 32-bit number of the same order (NaN above all
// numbers, -0 as 0, the protected keys above both, so one rule decides), and three passes over the row in shared memory find the budget-th
// largest, eleven, eleven and ten bits a pass, from counts per digit (with eight bits first the weights of a row, whose exponents differ little, fall into a handful
// of digits, and the counts are waited for: 24 us for 48 requests of 2,900 keys and 4 kv heads, now 13). Long rows are shared out over a cluster of blocks, whose
// counts are summed through distributed shared memory in the order of the ranks. Then each warp takes a run of neighbouring keys, counts
// what stays of it, and writes its indices behind those of the runs before. Nothing depends on timing.
//
// compact works in place: kept[i] >= i and kept ascends, so a row's source is never a place that an earlier row
// fills. A block owns a strip of the rows' bytes of one (request, kv head) and walks the places in ascending chunks: it
// reads a whole chunk before it writes it. What a later chunk reads lies behind everything that was written.
#include "common.cuh"

#include <cooperative_groups.h>

using namespace pae;
namespace cg = cooperative_groups;

namespace {

constexpr int CHOOSE_THREADS = 1024;
constexpr int CHOOSE_WARPS = CHOOSE_THREADS / 32;
static_assert(CHOOSE_WARPS == 32, "a warp scans the warps' sums; a thread stands for two digits");
constexpr int DIGITS = 2048;
constexpr int MOST_STAGED = 47 * 1024;      // of a row's keys in a block's shared memory
constexpr int COPIES = 2;                  // of the counts per digit, each fed by every other warp

// A number of the same order as the weight: negative numbers' bits are complemented, the others' get the sign bit. 0 stands behind all of them.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t bits = __float_as_uint(w == 0.f ? 0.f : w);
  return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

struct ChooseParams {
  const float* mass;        // [pages, kv_heads, page_size]
  const int* block_table;
  const int* kv_len;
  int* kept;                // [requests, kv_heads, budget]
  int table_width, kv_heads, page_size, budget, keep_first, keep_last, max_kv_len;
  int staged;               // keys per block that shared memory holds
  int fours;                // whether four neighbouring weights can be read at once
};

__global__ void __launch_bounds__(CHOOSE_THREADS, 2) choose_kernel(const ChooseParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t order[];       // [staged, rounded up to fours]: zeros behind the last
  __shared__ uint2 counts[COPIES][DIGITS / 2];
  __shared__ uint2 block_counts[2][DIGITS / 2];           // read by the other blocks of the cluster, which may be one pass behind
  __shared__ uint32_t scan[CHOOSE_WARPS];
  __shared__ uint32_t chosen[2];                          // the digit, and how many of the rest are still to be taken
  __shared__ uint32_t warp_above[CHOOSE_WARPS], warp_equal[CHOOSE_WARPS];
  __shared__ uint32_t block_above, block_equal;           // likewise
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int g = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  dependent_launch_prologue();

  const int n = min(p.kv_len[b], p.max_kv_len);
  int* kept = p.kept + ((size_t)b * p.kv_heads + g) * p.budget;
  if (n <= p.budget) {                                    // the same in every block of the cluster
    for (int i = rank * CHOOSE_THREADS + tid; i < p.budget; i += ranks * CHOOSE_THREADS) kept[i] = i < n ? i : -1;
    return;
  }
  const int share = ((n + ranks - 1) / ranks + 3) & ~3;
  const int begin = min(rank * share, n), mine = min(share, n - begin);
  const int* table = p.block_table + (size_t)b * p.table_width;
  auto look_up = [&](int i) -> uint32_t {
    const int j = begin + i;
    if (j < p.keep_first || j >= n - p.keep_last) return 0xFFFFFFFFu;
    const int page = checked_page(table[checked_table_index(j / p.page_size, p.table_width)]);
    return order_of(p.mass[((size_t)page * p.kv_heads + g) * p.page_size + j % p.page_size]);
  };
  const int staged = min(mine, p.staged);
  if (p.fours) {
    // Four neighbouring weights at a time, several times four under way.
    constexpr int DEPTH = 2;
    for (int i0 = tid * 4; i0 < staged; i0 += CHOOSE_THREADS * 4 * DEPTH) {
      float4 w[DEPTH];
      int pages[DEPTH];
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        const int i = i0 + u * CHOOSE_THREADS * 4;
        pages[u] = i < staged ? checked_page(table[checked_table_index((begin + i) / p.page_size, p.table_width)]) : 0;
      }
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        const int i = i0 + u * CHOOSE_THREADS * 4;
        if (i < staged) w[u] = *(const float4*)(p.mass + ((size_t)pages[u] * p.kv_heads + g) * p.page_size + (begin + i) % p.page_size);
      }
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        const int i = i0 + u * CHOOSE_THREADS * 4;
        const float four[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = begin + i + k;
          if (i + k < staged) order[i + k] = j < p.keep_first || j >= n - p.keep_last ? 0xFFFFFFFFu : order_of(four[k]);
        }
      }
    }
  } else {
    for (int i = tid; i < staged; i += CHOOSE_THREADS) order[i] = look_up(i);
  }
  if (tid < (-staged & 3)) order[staged + tid] = 0u;
  // Calls f(number) for the block's keys, four at a time from shared memory (with up to three zeros, which no weight is), the rest as they lie.
  auto for_each = [&](auto f) {
    for (int i = tid * 4; i < staged; i += CHOOSE_THREADS * 4) {
      const uint4 v = *(const uint4*)(order + i);
      f(v.x);
      f(v.y);
      f(v.z);
      f(v.w);
    }
    for (int i = staged + tid; i < mine; i += CHOOSE_THREADS) f(look_up(i));
  };

  // ---- the budget-th largest, digit by digit
  uint32_t prefix = 0, left = (uint32_t)p.budget;         // of the numbers that begin with `prefix`, the left-th largest
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), digits = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < COPIES * DIGITS / 2; i += CHOOSE_THREADS) (&counts[0][0])[i] = make_uint2(0, 0);
    __syncthreads();
    uint32_t* mine_counts = (uint32_t*)counts[warp & (COPIES - 1)];
    const int above_shift = pass == 1 ? 21 : 10;
    for_each([&](uint32_t v) {
      if (pass == 0 || (v >> above_shift) == prefix) atomicAdd(&mine_counts[(v >> shift) & (digits - 1)], 1u);
    });
    __syncthreads();
    // Thread t stands for digits 2 (1023 - t) and the one above: how many numbers have a larger digit, by a scan.
    const int pair = DIGITS / 2 - 1 - tid;
    uint2 sum = counts[0][pair];
#pragma unroll
    for (int c = 1; c < COPIES; ++c) {
      sum.x += counts[c][pair].x;
      sum.y += counts[c][pair].y;
    }
    if (ranks > 1) {
      block_counts[pass & 1][pair] = sum;
      cluster.sync();
      for (int r = 1; r < ranks; ++r) {
        const uint2 theirs = cluster.map_shared_rank(block_counts[pass & 1], (rank + r) % ranks)[pair];
        sum.x += theirs.x;
        sum.y += theirs.y;
      }
    }
    uint32_t inclusive = sum.x + sum.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, inclusive, o);
      if (lane >= o) inclusive += other;
    }
    if (lane == 31) scan[warp] = inclusive;
    __syncthreads();
    uint32_t totals = scan[lane];                         // of the warps, scanned by every warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, totals, o);
      if (lane >= o) totals += other;
    }
    const uint32_t earlier = __shfl_sync(0xffffffffu, totals, max(warp - 1, 0));
    const uint32_t before = (warp > 0 ? earlier : 0u) + inclusive - sum.x - sum.y;
    if (before < left && left <= before + sum.y) {        // one thread, one of its two digits
      chosen[0] = 2u * pair + 1u;
      chosen[1] = left - before;
    } else if (before + sum.y < left && left <= before + sum.y + sum.x) {
      chosen[0] = 2u * pair;
      chosen[1] = left - before - sum.y;
    }
    __syncthreads();
    prefix = pass == 0 ? chosen[0] : (prefix << (pass == 1 ? 11 : 10)) | chosen[0];
    left = chosen[1];
  }
  // All numbers above `prefix` stay, and of its equals the first `left`.

  // ---- the indices, in ascending order: a warp takes a run of keys
  const int run = (((mine + CHOOSE_WARPS - 1) / CHOOSE_WARPS) + 127) & ~127;
  const int first = min(warp * run, mine), last = min(first + run, mine);
  auto four_at = [&](int i) {              // of a lane; zeros behind the run
    if (i < staged && i < last) return *(const uint4*)(order + i);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (i < last) {
      v.x = look_up(i);
      if (i + 1 < last) v.y = look_up(i + 1);
      if (i + 2 < last) v.z = look_up(i + 2);
      if (i + 3 < last) v.w = look_up(i + 3);
    }
    return v;
  };
  uint32_t above = 0, equal = 0;
  for (int i = first + lane * 4; i < last; i += 128) {
    const uint4 v = four_at(i);
    above += (v.x > prefix) + (v.y > prefix) + (v.z > prefix) + (v.w > prefix);
    equal += (v.x == prefix) + (v.y == prefix) + (v.z == prefix) + (v.w == prefix);
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    warp_above[warp] = above;
    warp_equal[warp] = equal;
  }
  __syncthreads();
  const uint32_t all_above = warp_above[lane], all_equal = warp_equal[lane];
  if (ranks > 1) {
    if (warp == 0) {
      const uint32_t a = __reduce_add_sync(0xffffffffu, all_above), e = __reduce_add_sync(0xffffffffu, all_equal);
      if (lane == 0) {
        block_above = a;
        block_equal = e;
      }
    }
    cluster.sync();
  }
  uint32_t above_before = __reduce_add_sync(0xffffffffu, lane < warp ? all_above : 0u);
  uint32_t equal_before = __reduce_add_sync(0xffffffffu, lane < warp ? all_equal : 0u);
  for (int r = 0; r < rank; ++r) {
    above_before += *cluster.map_shared_rank(&block_above, r);
    equal_before += *cluster.map_shared_rank(&block_equal, r);
  }
  for (int i0 = first; i0 < last; i0 += 128) {
    const int i = i0 + lane * 4;
    const uint4 v = four_at(i);
    const uint32_t four[4] = {v.x, v.y, v.z, v.w};
    uint32_t count = 0;                      // above in the low half, equal in the high one: at most 128 of each
#pragma unroll
    for (int k = 0; k < 4; ++k) count += (four[k] > prefix ? 1u : 0u) + (four[k] == prefix ? 0x10000u : 0u);
    uint32_t inclusive = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, inclusive, o);
      if (lane >= o) inclusive += other;
    }
    uint32_t a = above_before + ((inclusive - count) & 0xFFFFu), e = equal_before + ((inclusive - count) >> 16);
    if (count != 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool is_equal = four[k] == prefix;
        if (four[k] > prefix || (is_equal && e < left)) kept[a + min(e, left)] = begin + i + k;
        a += four[k] > prefix;
        e += is_equal;
      }
    }
    const uint32_t all = __shfl_sync(0xffffffffu, inclusive, 31);
    above_before += all & 0xFFFFu;
    equal_before += all >> 16;
  }
  if (ranks > 1) cluster.sync();                          // no block leaves while its counts may be read
}

// ---------------------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------------------
constexpr int IN_FLIGHT = 8;               // rows' pieces that a thread reads before it writes
constexpr int MOST_ROWS = 2048;            // of a chunk

struct CompactParams {
  uint8_t* pools[3];        // keys, values, weights: [pages, kv_heads, page_size] rows of row_units[i] units
  int row_units[3];
  int strip_units[3], strips[3];
  const int* block_table;
  const int* kv_len;
  const int* kept;
  int table_width, kv_heads, page_size, budget;
};

// Where a chunk's rows come from and go to, as row numbers of the pool (pages * kv_heads * page_size of them, fewer than 2^31), found by one thread
// a row while the chunk before is on its way; -1: the row does not move. (With unsigned numbers and another mark, the kernel of 1,024 threads took a tenth more.)
template <int THREADS, typename Unit>
__device__ __forceinline__ void compact_strip(const CompactParams& p, int pool, int strip, int2 (*moves)[MOST_ROWS]) {
  const int g = blockIdx.y, b = blockIdx.z;
  const int n = min(p.kv_len[b], p.table_width * p.page_size);
  const int places = min(n, p.budget);
  const int* kept = p.kept + ((size_t)b * p.kv_heads + g) * p.budget;
  const int* table = p.block_table + (size_t)b * p.table_width;
  const int units = p.row_units[pool], width = min(p.strip_units[pool], units - strip * p.strip_units[pool]);
  const int rows_a_pass = min(THREADS / width, MOST_ROWS / IN_FLIGHT), chunk_rows = rows_a_pass * IN_FLIGHT;
  const int my_row = threadIdx.x / width, my_unit = strip * p.strip_units[pool] + threadIdx.x % width;
  Unit* base = (Unit*)p.pools[pool] + my_unit;
  auto row_of = [&](int i) {
    const int page = page_or_none(table, i / p.page_size, p.table_width);
    return page < 0 ? -1 : (page * p.kv_heads + g) * p.page_size + i % p.page_size;
  };
  auto find = [&](int chunk, int2* to) {
    for (int r = threadIdx.x; r < chunk_rows; r += THREADS) {
      const int i = chunk + r, from = i < places ? kept[i] : -1;
      int2 move = from > i && from < n ? make_int2(row_of(from), row_of(i)) : make_int2(-1, 0);
      if (move.y < 0) move.x = -1;
      to[r] = move;
    }
  };
  find(0, moves[0]);
  __syncthreads();
  for (int chunk = 0, turn = 0; chunk < places; chunk += chunk_rows, turn ^= 1) {
    Unit held[IN_FLIGHT];
    int to[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const int2 move = my_row < rows_a_pass ? moves[turn][u * rows_a_pass + my_row] : make_int2(-1, 0);
      to[u] = move.x >= 0 ? move.y : -1;
      if (move.x >= 0) held[u] = base[(size_t)move.x * units];
    }
    if (chunk + chunk_rows < places) find(chunk + chunk_rows, moves[turn ^ 1]);
    __syncthreads();                       // the whole chunk is read, and the next one's rows are found
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u)
      if (to[u] >= 0) base[(size_t)to[u] * units] = held[u];
  }
}

template <int THREADS, typename Unit>
__global__ void __launch_bounds__(THREADS) compact_kernel(const CompactParams p) {
  // The next kernel is not let go early: an attention that follows directly fetches keys of earlier tokens before it waits for
  // the kernel before it (common.cuh), and those are what is written here.
  dependent_launch_wait();
  __shared__ int2 moves[2][MOST_ROWS];
  int strip = blockIdx.x;
  if (strip < p.strips[0]) {
    compact_strip<THREADS, Unit>(p, 0, strip, moves);
  } else if ((strip -= p.strips[0]) < p.strips[1]) {
    compact_strip<THREADS, Unit>(p, 1, strip, moves);
  } else {
    compact_strip<THREADS, uint32_t>(p, 2, 0, moves);
  }
  __threadfence();
}

}  // namespace

PAE_DEFINE_LAST_ERROR()

PAE_EXPORT int pae_choose_kept(int* kept, const float* mass, const int* block_table, int table_width, const int* kv_len, int seqs, int kv_heads,
                               int page_size, int budget, int keep_first, int keep_last, int max_kv_len, void* stream) {
  if (seqs < 1 || kv_heads < 1) return 0;
  if (kv_heads > 65535 || seqs > 65535) return fail(1, "choose_kept: %d requests of %d kv heads, at most 65535 of each", seqs, kv_heads);
  // A cluster's barriers and counts cost some 2 us a pass: one block a row of up to 16,384 keys (9,000 keys, 2 rows: 12.3 us, in clusters of two 13.1, of four 16.4), more
  // where all of them still have an SM each (64,000 keys: 8 rows 27.0 us in two blocks, 21.4 in four; 48 rows 31.5 and 40.6), and as many as hold the row.
  int ranks = 1;
  while (ranks < 8 && max_kv_len > 16384 * ranks && (long long)seqs * kv_heads * ranks * 2 <= 148) ranks *= 2;
  while (ranks < 8 && max_kv_len > MOST_STAGED * ranks) ranks *= 2;
  ChooseParams p = {mass, block_table, kv_len, kept, table_width, kv_heads, page_size, budget, keep_first, keep_last, max_kv_len, 0, page_size % 4 == 0 && (uintptr_t)mass % 16 == 0};
  p.staged = min(MOST_STAGED, ((max_kv_len + ranks - 1) / ranks + 3) & ~3);      // fours, as a block's share is
  const size_t smem = (size_t)p.staged * 4;
  static DevicesSet devices;
  if (int code = raise_shared_memory(devices, choose_kernel, MOST_STAGED * 4, "choose_kept")) return code;
  if (ranks == 1) launch_kernel(choose_kernel, dim3(1, kv_heads, seqs), dim3(CHOOSE_THREADS), smem, (cudaStream_t)stream, p);
  else launch_kernel_cluster(choose_kernel, dim3(ranks, kv_heads, seqs), dim3(CHOOSE_THREADS), smem, (cudaStream_t)stream, ranks, p);
  return check_launch("choose_kept");
}

// `row_bytes` of keys, then of values (0: no values); their rows are units of `unit` bytes (16, 4 or 2).
PAE_EXPORT int pae_compact_kept(void* keys, void* values, float* mass, const int* block_table, int table_width, const int* kv_len, const int* kept,
                                int seqs, int kv_heads, int page_size, int budget, int key_bytes, int value_bytes, int unit, void* stream) {
  if (seqs < 1 || kv_heads < 1) return 0;
  if (kv_heads > 65535 || seqs > 65535) return fail(1, "compact_kept: %d requests of %d kv heads, at most 65535 of each", seqs, kv_heads);
  CompactParams p = {};
  p.pools[0] = (uint8_t*)keys;
  p.pools[1] = (uint8_t*)values;
  p.pools[2] = (uint8_t*)mass;
  p.block_table = block_table;
  p.kv_len = kv_len;
  p.kept = kept;
  p.table_width = table_width;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.budget = budget;
  const int bytes[3] = {key_bytes, values != nullptr ? value_bytes : 0, mass != nullptr ? 4 : 0};
  // A row's bytes in strips of 256: pieces of a row that are moved at different times cost the memory another row activation each. So blocks of 1,024
  // threads where blocks of 256 would leave too little under way, and narrower strips only for launches of few rows. us of a choice with its move, 8
  // kv heads of 128 and contexts of 50,000 to 64,000 (96 blocks of whole strips): 6 requests 143, never with 1,024 threads 191, with strips halved up to 148
  // blocks 162; 4 kv heads, 1,900 to 3,900: 48 requests 81, with 1,024 threads there too 90, 8 requests 25.3, without narrower strips 27.9; one
  // request, 2 kv heads, 640 keys: 10.3 and 11.2.
  const long long pairs = (long long)seqs * kv_heads;
  auto strips_of = [&](int bytes) { return pairs * ((key_bytes + bytes - 1) / bytes + (value_bytes + bytes - 1) / bytes); };
  int strip_bytes = 256;
  bool wide = strips_of(256) < 296;
  while (strip_bytes > 32 && strips_of(strip_bytes) < 74) strip_bytes /= 2;
  if (strip_bytes < 64) wide = false;
  int blocks = 0;
  for (int i = 0; i < 3; ++i) {
    p.row_units[i] = bytes[i] / (i < 2 ? unit : 4);
    p.strip_units[i] = min(i < 2 ? max(1, strip_bytes / unit) : 1, max(1, p.row_units[i]));
    p.strips[i] = (p.row_units[i] + p.strip_units[i] - 1) / p.strip_units[i];
    blocks += p.strips[i];
  }
  if (blocks == 0) return 0;
  const dim3 grid(blocks, kv_heads, seqs);
  const cudaStream_t s = (cudaStream_t)stream;
  if (unit == 16 && wide) launch_kernel(compact_kernel<1024, uint4>, grid, dim3(1024), 0, s, p);
  else if (unit == 16) launch_kernel(compact_kernel<256, uint4>, grid, dim3(256), 0, s, p);
  else if (unit == 4) launch_kernel(compact_kernel<256, uint32_t>, grid, dim3(256), 0, s, p);
  else launch_kernel(compact_kernel<256, uint16_t>, grid, dim3(256), 0, s, p);
  return check_launch("compact_kept");
}
