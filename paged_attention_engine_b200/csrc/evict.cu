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
// numbers, -0 as 0, the protected keys above both, so one rule decides), and four passes over the row in shared memory find the budget-th
// largest, eight bits a pass, from counts per digit. Long rows are shared out over a cluster of blocks, whose
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

constexpr int CHOOSE_THREADS = 512;
constexpr int CHOOSE_WARPS = CHOOSE_THREADS / 32;
constexpr int COPIES = 4;                  // of the counts per digit, each fed by every fourth warp

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
};

__global__ void __launch_bounds__(CHOOSE_THREADS) choose_kernel(const ChooseParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ uint32_t order[];                     // [staged]
  __shared__ uint32_t counts[COPIES][256];
  __shared__ uint32_t block_counts[256];                  // read by the other blocks of the cluster
  __shared__ uint32_t scan[8];
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
  const int share = (n + ranks - 1) / ranks;
  const int begin = min(rank * share, n), mine = min(share, n - begin);
  const int* table = p.block_table + (size_t)b * p.table_width;
  auto look_up = [&](int i) -> uint32_t {
    const int j = begin + i;
    if (j < p.keep_first || j >= n - p.keep_last) return 0xFFFFFFFFu;
    const int page = checked_page(table[checked_table_index(j / p.page_size, p.table_width)]);
    return order_of(p.mass[((size_t)page * p.kv_heads + g) * p.page_size + j % p.page_size]);
  };
  const int staged = min(mine, p.staged);
  for (int i = tid; i < staged; i += CHOOSE_THREADS) order[i] = look_up(i);
  auto at = [&](int i) { return i < staged ? order[i] : look_up(i); };

  // ---- the budget-th largest, digit by digit
  uint32_t prefix = 0, left = (uint32_t)p.budget;         // of the numbers that begin with `prefix`, the left-th largest
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < COPIES * 256; i += CHOOSE_THREADS) (&counts[0][0])[i] = 0;
    __syncthreads();
    for (int i = tid; i < mine; i += CHOOSE_THREADS) {
      const uint32_t v = at(i);
      if (shift == 24 || (v >> (shift + 8)) == prefix) atomicAdd(&counts[warp & (COPIES - 1)][(v >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t sum = 0;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) sum += counts[c][tid];
      block_counts[tid] = sum;
    }
    if (ranks > 1) cluster.sync(); else __syncthreads();
    // Thread t stands for digit 255 - t: how many numbers have a larger digit, by a scan.
    uint32_t count = 0, before = 0;
    if (tid < 256) {
      for (int r = 0; r < ranks; ++r) count += cluster.map_shared_rank(block_counts, r)[255 - tid];
      uint32_t inclusive = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += other;
      }
      if (lane == 31) scan[warp] = inclusive;
      before = inclusive - count;
    }
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < warp; ++w) before += scan[w];
      if (before < left && left <= before + count) {      // one thread
        chosen[0] = 255u - tid;
        chosen[1] = left - before;
      }
    }
    if (ranks > 1) cluster.sync(); else __syncthreads();  // nobody writes its counts again before all have read them
    prefix = (prefix << 8) | chosen[0];
    left = chosen[1];
  }
  // All numbers above `prefix` stay, and of its equals the first `left`.

  // ---- the indices, in ascending order: a warp takes a run of keys
  const int run = (((mine + CHOOSE_WARPS - 1) / CHOOSE_WARPS) + 31) & ~31;
  const int first = min(warp * run, mine), last = min(first + run, mine);
  uint32_t above = 0, equal = 0;
  for (int i = first + lane; i < last; i += 32) {
    const uint32_t v = at(i);
    above += v > prefix;
    equal += v == prefix;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    warp_above[warp] = above;
    warp_equal[warp] = equal;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t a = 0, e = 0;
    for (int w = 0; w < CHOOSE_WARPS; ++w) {
      a += warp_above[w];
      e += warp_equal[w];
    }
    block_above = a;
    block_equal = e;
  }
  if (ranks > 1) cluster.sync(); else __syncthreads();
  uint32_t above_before = 0, equal_before = 0;
  for (int r = 0; r < rank; ++r) {
    above_before += *cluster.map_shared_rank(&block_above, r);
    equal_before += *cluster.map_shared_rank(&block_equal, r);
  }
  for (int w = 0; w < warp; ++w) {
    above_before += warp_above[w];
    equal_before += warp_equal[w];
  }
  const uint32_t below_me = (1u << lane) - 1u;
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t v = i < last ? at(i) : 0u;
    const bool is_above = i < last && v > prefix, is_equal = i < last && v == prefix;
    const uint32_t a = __ballot_sync(0xffffffffu, is_above), e = __ballot_sync(0xffffffffu, is_equal);
    const uint32_t equals = equal_before + __popc(e & below_me);
    if (is_above || (is_equal && equals < left)) kept[above_before + __popc(a & below_me) + min(equals, left)] = begin + i;
    above_before += __popc(a);
    equal_before += __popc(e);
  }
  if (ranks > 1) cluster.sync();                          // no block leaves while its counts may be read
}

// ---------------------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------------------
constexpr int COMPACT_THREADS = 256;
constexpr int IN_FLIGHT = 8;               // rows' pieces that a thread reads before it writes

struct CompactParams {
  uint8_t* pools[3];        // keys, values, weights: [pages, kv_heads, page_size] rows of row_units[i] units
  int row_units[3];
  int strip_units[3], strips[3];
  const int* block_table;
  const int* kv_len;
  const int* kept;
  int table_width, kv_heads, page_size, budget;
};

template <typename Unit>
__device__ __forceinline__ void compact_strip(const CompactParams& p, int pool, int strip) {
  const int g = blockIdx.y, b = blockIdx.z;
  const int n = min(p.kv_len[b], p.table_width * p.page_size);
  const int places = min(n, p.budget);
  const int* kept = p.kept + ((size_t)b * p.kv_heads + g) * p.budget;
  const int* table = p.block_table + (size_t)b * p.table_width;
  const int units = p.row_units[pool], width = min(p.strip_units[pool], units - strip * p.strip_units[pool]);
  const int rows_a_pass = COMPACT_THREADS / width;
  const int my_row = threadIdx.x / width, my_unit = strip * p.strip_units[pool] + threadIdx.x % width;
  Unit* base = (Unit*)p.pools[pool];
  auto unit_at = [&](int i) {
    const int page = checked_page(table[checked_table_index(i / p.page_size, p.table_width)]);
    return base + (((size_t)page * p.kv_heads + g) * p.page_size + i % p.page_size) * units + my_unit;
  };
  for (int chunk = 0; chunk < places; chunk += rows_a_pass * IN_FLIGHT) {
    Unit held[IN_FLIGHT];
    bool moves[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const int i = chunk + u * rows_a_pass + my_row;
      const int from = my_row < rows_a_pass && i < places ? kept[i] : -1;
      moves[u] = from > i && from < n;
      if (moves[u]) held[u] = *unit_at(from);
    }
    __syncthreads();                       // the whole chunk is read
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u)
      if (moves[u]) *unit_at(chunk + u * rows_a_pass + my_row) = held[u];
  }
}

template <typename Unit>
__global__ void __launch_bounds__(COMPACT_THREADS) compact_kernel(const CompactParams p) {
  // The next kernel is not let go early: an attention that follows directly fetches keys of earlier tokens before it waits for
  // the kernel before it (common.cuh), and those are what is written here.
  dependent_launch_wait();
  int strip = blockIdx.x;
  if (strip < p.strips[0]) {
    compact_strip<Unit>(p, 0, strip);
  } else if ((strip -= p.strips[0]) < p.strips[1]) {
    compact_strip<Unit>(p, 1, strip);
  } else {
    compact_strip<uint32_t>(p, 2, 0);
  }
  __threadfence();
}

}  // namespace

PAE_DEFINE_LAST_ERROR()

PAE_EXPORT int pae_choose_kept(int* kept, const float* mass, const int* block_table, int table_width, const int* kv_len, int seqs, int kv_heads,
                               int page_size, int budget, int keep_first, int keep_last, int max_kv_len, void* stream) {
  if (seqs < 1 || kv_heads < 1) return 0;
  if (kv_heads > 65535 || seqs > 65535) return fail(1, "choose_kept: %d requests of %d kv heads, at most 65535 of each", seqs, kv_heads);
  int ranks = 1;
  while (ranks < 8 && (long long)seqs * kv_heads * ranks < 148 && max_kv_len > 2048 * ranks) ranks *= 2;
  while (ranks < 8 && max_kv_len > 16384 * ranks) ranks *= 2;
  ChooseParams p = {mass, block_table, kv_len, kept, table_width, kv_heads, page_size, budget, keep_first, keep_last, max_kv_len, 0};
  p.staged = min(48 * 1024, (max_kv_len + ranks - 1) / ranks);
  const size_t smem = (size_t)p.staged * 4;
  static DevicesSet devices;
  if (int code = raise_shared_memory(devices, choose_kernel, 48 * 1024 * 4, "choose_kept")) return code;
  launch_kernel_cluster(choose_kernel, dim3(ranks, kv_heads, seqs), dim3(CHOOSE_THREADS), smem, (cudaStream_t)stream, ranks, p);
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
  int blocks = 0;
  for (int i = 0; i < 3; ++i) {
    p.row_units[i] = bytes[i] / (i < 2 ? unit : 4);
    p.strip_units[i] = min(i < 2 ? max(1, 64 / unit) : 1, max(1, p.row_units[i]));
    p.strips[i] = (p.row_units[i] + p.strip_units[i] - 1) / p.strip_units[i];
    blocks += p.strips[i];
  }
  if (blocks == 0) return 0;
  const dim3 grid(blocks, kv_heads, seqs), threads(COMPACT_THREADS);
  if (unit == 16) launch_kernel(compact_kernel<uint4>, grid, threads, 0, (cudaStream_t)stream, p);
  else if (unit == 4) launch_kernel(compact_kernel<uint32_t>, grid, threads, 0, (cudaStream_t)stream, p);
  else launch_kernel(compact_kernel<uint16_t>, grid, threads, 0, (cudaStream_t)stream, p);
  return check_launch("compact_kept");
}
