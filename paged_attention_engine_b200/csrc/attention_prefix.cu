// Attention of a step whose requests share the first keys of their contexts: groups of consecutive requests, each group with one run of
// shared keys that lies once in the pages, and behind it every request's own keys.
//
//   out[t, h] = (sum over shared keys j of e_j v_j + sum over own keys j <= position(t) of e_j v_j) / (sum of all e_j),
//   e_j = exp(scale q . k_j - m), m the largest of the row's scaled scores
//
// A softmax over two sets of keys is the two sets' (maximum, sum, unnormalised output) brought to one maximum and added, so the
// shared keys are taken for all rows (token, query head of the kv head) of a group at once: they are read once a
// group and not once a request, and there are enough rows to fill the tensor cores. The own keys go the same way, with the rows of one
// request. One launch and a merge:
//
//   slices   a block takes up to 128 rows x a slice of shared keys, or of a request's own, 64 keys a tile, as the paired prefill attention works
//            (attention_tcgen05.cu), which see for the roles and the references that may lie behind the maxima: keys and values by TMA,
//            both products as tcgen05.mma, scores, probabilities and output in tensor memory. Softmax warps without a row take no part, so that over
//            own keys, which few rows read, a tile costs little more than its bytes.
//   merge    a row's slices, shared and own, in their order.
//
// The same kernel without shared keys is the attention of paged_attention_mass for steps of few tokens: it leaves its scores besides (4 bytes for each token, query
// head and key, where keys and values are 4 * head size bytes for each kv head and key; in rows as long as the longest context, whatever the request's own, so a
// launch takes as many of the step's requests as a bound on its scratch allows), and further blocks of the merge turn them into
// weights once a row's maximum and sum are known, and add them up per key (attention_mass.cu says what is computed).
//
// Other types and sizes than those of the tensor-core kernel take the same slices of 16 rows on CUDA cores (any_slices_kernel).
//
// Scores are scaled in float32, maxima, sums and outputs are float32; probabilities are rounded to bfloat16 for the second
// product, as the value operand is, and the result once. Every wait on an mbarrier is bounded and reports through `error`.
#include <cfloat>

#include "attention_mma.cuh"
#include "attention_pages.cuh"

using namespace pae;
using namespace pae_tcgen05;

namespace {

constexpr int ROWS = 128;                // of a block
constexpr int BKEYS = 64;                // keys per tile
constexpr int THREADS = 192;             // TMA warp, MMA warp, four softmax warps (one thread per row)
constexpr int SOFTMAX_WARPS = 4;
constexpr int KV_STAGES = 2;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float REFERENCE_SLACK = 8.f;   // as the paired prefill attention
constexpr float REFERENCE_LIMIT = 256.f;

struct Params {
  const __nv_bfloat16* qkv;     // [tokens, heads + 2 kv_heads, D]
  const __nv_bfloat16* keys;    // [pages, kv_heads, page_size, D]
  const __nv_bfloat16* values;
  const int* block_table;
  const int* q_start;
  const int* q_pos0;
  const int* kv_len;
  const int* prefix_len;        // [requests], alike in a group
  const int* group_start;       // [groups + 1]
  float* part_out;              // [tokens, heads, slots, D]
  float* part_max;              // [tokens, heads, slots], units of log2
  float* part_sum;
  int table_width, heads, kv_heads, page_size, max_prefix;
  int shared_blocks, row_tiles, shared_slices, shared_keys;      // keys per slice of the shared ones, a multiple of BKEYS
  int own_row_tiles, own_slices, own_keys;                       // likewise of the own ones
  int slots;                    // slices of a row at most: shared ones, then own ones
  int box;                      // own slices start on multiples of it
  int max_tokens;               // of a request
  int part_tokens;              // that the scratch holds where it holds scores
  float* scores;                // [tokens, heads, span], not scaled, of own keys; token 0 is the first request's first
  int span;
  float scale_log2, slack;
  int* error;
};

enum Bar : int {
  Q_FULL = 0, O_FULL = 1, S_FULL = 2, P_READY = 4, O_REST = 6,
  K_FULL = 7, K_EMPTY = K_FULL + KV_STAGES, V_FULL = K_EMPTY + KV_STAGES, V_EMPTY = V_FULL + KV_STAGES, NUM_BARS = V_EMPTY + KV_STAGES
};

template <int D>
struct Layout {
  static constexpr int HALVES = D / 64;
  static constexpr int Q_HALF_BYTES = ROWS * 128;
  static constexpr int KV_HALF_BYTES = BKEYS * 128;
  static constexpr int Q_BYTES = HALVES * Q_HALF_BYTES;
  static constexpr int KV_BYTES = HALVES * KV_HALF_BYTES;
  static constexpr int Q_OFFSET = 0;
  static constexpr int K_OFFSET = Q_BYTES;
  static constexpr int V_OFFSET = K_OFFSET + KV_STAGES * KV_BYTES;
  static constexpr int BAR_OFFSET = V_OFFSET + KV_STAGES * KV_BYTES;
  static constexpr size_t SMEM_BYTES = (size_t)BAR_OFFSET + 256 + 1024;    // wherever the block's memory begins, the tiles begin on 1024 bytes
  static_assert(8 * NUM_BARS + 8 <= 256 && 2 * (SMEM_BYTES + 1024) <= 228 * 1024, "two blocks fit an SM");
  static constexpr int S_COLUMNS = BKEYS;
  static constexpr int O_COLUMN = 2 * S_COLUMNS;
  static constexpr int TMEM_COLUMNS = 256;
};

// The pages of a run of keys from `begin` (where a box of rows starts) to `end`, for a converged warp: the table is read 32 boxes at a time, one
// load ahead of need.
struct PageRun {
  const int* table;
  int begin, box_rows, shift, last, width, lane;
  int held, ahead, window;                 // entries of boxes window * 32 + lane, and of the next 32
  __device__ __forceinline__ int entry(int box) const {
    return checked_page(table[checked_table_index(min((begin + box * box_rows) >> shift, last), width)]);     // behind the end any page will do
  }
  __device__ __forceinline__ void start(const int* t, int b, int e, int rows, int page_size, int w, int l) {
    table = t, begin = b, box_rows = rows, width = w, lane = l, window = 0;
    shift = 31 - __clz(page_size);         // page sizes are powers of two
    last = (e - 1) >> shift;
    held = entry(lane);
    ahead = entry(32 + lane);
  }
  // Box `lane` of tile t (all lanes call; tiles in ascending order, at most 32 boxes behind the furthest).
  __device__ __forceinline__ int page(int t, int boxes) {
    const int box = t * boxes + lane;
    const int first = __shfl_sync(0xffffffffu, box, 0);
    if (first >= (window + 1) * 32) {
      held = ahead;
      ++window;
      ahead = entry((window + 1) * 32 + lane);
    }
    return __shfl_sync(0xffffffffu, held, box & 31);
  }
};
// Where the own keys of a tile of TILE_ROWS rows begin and end; their slices start at `base`, where a box of rows does.
struct OwnSpan {
  int first, base, end;
};
template <int TILE_ROWS>
__device__ __forceinline__ OwnSpan own_span(const Params& p, int shared, int kv_len, int pos0, int tokens, int groups, int row_tile) {
  OwnSpan s;
  s.first = shared;
  s.base = shared / p.box * p.box;
  s.end = min(kv_len, pos0 + min((row_tile * TILE_ROWS + TILE_ROWS - 1) / groups, tokens - 1) + 1);
  return s;
}

// Of a launch that keeps scores: the tokens of a request, and whether they have room in the scratch (they do unless a request before brought more
// than `max_tokens`).
__device__ __forceinline__ int tokens_of(const Params& p, int b) { return min(p.q_start[b + 1] - p.q_start[b], p.max_tokens); }
__device__ __forceinline__ bool in_part(const Params& p, int token0, int tokens) { return token0 - p.q_start[0] + tokens <= p.part_tokens; }

// What a block works on: rows row0 .. row0 + rows - 1 (token, head of kv head g) behind `first_token`, keys begin .. end - 1 by the table of
// request b. Row r sees those from `first` on that stand at or before pos0 + its token's index.
struct Work {
  int b, g, first_token, row0, rows, begin, end, first, pos0, slot;
};
constexpr int EVERY_KEY = 1 << 30;       // pos0 of rows behind all keys
template <int TILE_ROWS, bool SCORES>
__device__ __forceinline__ Work find_work(const Params& p, int index) {
  const int groups = p.heads / p.kv_heads;
  Work w = {0, 0, 0, 0, 0, 0, 0, 0, EVERY_KEY, 0};
  if (index < p.shared_blocks) {
    // The row tiles of a kv head and a slice are neighbours: they read the same keys.
    const int row_tile = index % p.row_tiles;
    index /= p.row_tiles;
    w.g = index % p.kv_heads;
    index /= p.kv_heads;
    w.slot = index % p.shared_slices;
    const int group = index / p.shared_slices;
    w.b = p.group_start[group];
    const int b_end = p.group_start[group + 1];
    if (w.b >= b_end) return w;
    w.first_token = p.q_start[w.b];
    w.row0 = row_tile * TILE_ROWS;
    w.rows = min(TILE_ROWS, (p.q_start[b_end] - w.first_token) * groups - w.row0);
    w.begin = w.slot * p.shared_keys;
    w.end = min(min(p.prefix_len[w.b], p.max_prefix), w.begin + p.shared_keys);
    return w;
  }
  index -= p.shared_blocks;
  const int slice = index % p.own_slices;
  index /= p.own_slices;
  const int row_tile = index % p.own_row_tiles;
  index /= p.own_row_tiles;
  w.g = index % p.kv_heads;
  w.b = index / p.kv_heads;
  w.first_token = p.q_start[w.b];
  const int tokens = SCORES ? tokens_of(p, w.b) : p.q_start[w.b + 1] - w.first_token, shared = p.max_prefix > 0 ? min(p.prefix_len[w.b], p.max_prefix) : 0;
  if (SCORES && !in_part(p, w.first_token, tokens)) return w;
  w.pos0 = p.q_pos0[w.b];
  const OwnSpan span = own_span<TILE_ROWS>(p, shared, p.kv_len[w.b], w.pos0, tokens, groups, row_tile);
  if (span.end <= span.first) return w;
  w.row0 = row_tile * TILE_ROWS;
  w.rows = min(TILE_ROWS, tokens * groups - w.row0);
  w.first = shared;
  w.begin = span.base + slice * p.own_keys;
  w.end = min(span.end, w.begin + p.own_keys);
  w.slot = (shared + p.shared_keys - 1) / p.shared_keys + slice;
  return w;
}

template <int D, bool SCORES>
__global__ void __launch_bounds__(THREADS, 2) prefix_kernel(const __grid_constant__ PageMaps maps, const Params p) {
  using L = Layout<D>;
  extern __shared__ uint8_t raw_smem[];
  const uint32_t raw = smem_u32(raw_smem);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* generic_base = raw_smem + (base - raw);
  const uint32_t bars = base + L::BAR_OFFSET;
  volatile uint32_t* tmem_holder = (volatile uint32_t*)(generic_base + L::BAR_OFFSET + 8 * NUM_BARS);
  volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
  auto bar = [&](int which, int i = 0) { return bars + 8u * (which + i); };
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const Work work = find_work<ROWS, SCORES>(p, blockIdx.x);
  const bool working = work.rows > 0 && work.begin < work.end;      // the same in every thread
  const int rows = work.rows, kv_begin = work.begin, kv_end = work.end, g = work.g, groups = p.heads / p.kv_heads;
  const int n_tiles = (kv_end - kv_begin + BKEYS - 1) / BKEYS;
  const int row_warps = (rows + 31) / 32;              // the softmax warps that have rows

  const int box_rows = min(p.page_size, BKEYS);
  PageRun pages;                                       // of the producer; the table was on the device before the step's first kernel began
  if (warp == 0 && working) pages.start(p.block_table + (size_t)work.b * p.table_width, kv_begin, kv_end, box_rows, p.page_size, p.table_width, lane);
  if (threadIdx.x == 0 && working) {
    mbar_init(bar(Q_FULL), SOFTMAX_WARPS * 32);
    for (int i = 0; i < KV_STAGES; ++i) {
      mbar_init(bar(K_FULL, i), 1);
      mbar_init(bar(K_EMPTY, i), 1);
      mbar_init(bar(V_FULL, i), 1);
      mbar_init(bar(V_EMPTY, i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S_FULL, i), 1);
      mbar_init(bar(P_READY, i), row_warps);
    }
    mbar_init(bar(O_REST), 1);
    mbar_init(bar(O_FULL), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1 && working) {
    tmem_alloc(smem_u32((const void*)tmem_holder), L::TMEM_COLUMNS);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  dependent_launch_trigger();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  dependent_launch_wait();
  if (!working) return;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: lane i brings box i of a tile
    const int boxes = BKEYS / box_rows;
    auto page_of = [&](int t) { return t < n_tiles ? pages.page(t, boxes) : 0; };
    auto load = [&](bool values, int t, int page) {
      const int stage = t % KV_STAGES;
      const uint32_t full = bar(values ? V_FULL : K_FULL, stage);
      if (t >= KV_STAGES && !mbar_wait_warp(bar(values ? V_EMPTY : K_EMPTY, stage), (t / KV_STAGES - 1) & 1, abort_flag, p.error, values ? 10 : 1))
        return false;
      if (lane == 0) mbar_expect_tx(full, L::KV_BYTES);
      __syncwarp();
      load_pages<D>(maps, values, base + (values ? L::V_OFFSET : L::K_OFFSET) + stage * L::KV_BYTES, full, BKEYS, box_rows, lane, g, page,
                    (kv_begin + t * BKEYS + lane * box_rows) & (p.page_size - 1));
      return true;
    };
    int page0 = page_of(0), page1 = page_of(1), page2 = page_of(2);               // of tiles t, t + 1, t + 2
    bool ok = load(false, 0, page0);
    int keys_issued = 1, values_issued = 0;
    if (n_tiles > 1) {
      ok = ok && load(false, 1, page1);
      keys_issued = 2;
    }
    for (int t = 0; t < n_tiles && ok; ++t) {
      const int page3 = page_of(t + 3);
      if (!(ok = load(true, t, page0))) break;
      values_issued = t + 1;
      if (t + 2 < n_tiles) {
        if (!(ok = load(false, t + 2, page2))) break;
        keys_issued = t + 3;
      }
      page0 = page1;
      page1 = page2;
      page2 = page3;
    }
    if (lane == 0 && *abort_flag) {      // copies that were issued still write into this block's shared memory
      for (int t = max(0, keys_issued - KV_STAGES); t < keys_issued; ++t)
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(bar(K_FULL, t % KV_STAGES), (t / KV_STAGES) & 1); ++w) __nanosleep(64);
      for (int t = max(0, values_issued - KV_STAGES); t < values_issued; ++t)
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(bar(V_FULL, t % KV_STAGES), (t / KV_STAGES) & 1); ++w) __nanosleep(64);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = instruction_descriptor(ROWS, BKEYS, false);
    constexpr uint32_t idesc_o = instruction_descriptor(ROWS, D, true);
    const uint64_t q_first = smem_descriptor(base + L::Q_OFFSET), k_first = smem_descriptor(base + L::K_OFFSET);
    const uint64_t v_first = mn_major_descriptor(base + L::V_OFFSET, box_rows * 128);
    bool ok = mbar_wait_warp(bar(Q_FULL), 0, abort_flag, p.error, 2);
    auto issue_scores = [&](int t) {
      const int st = t & 1, stage = t % KV_STAGES;
      ok = ok && mbar_wait_warp(bar(K_FULL, stage), (t / KV_STAGES) & 1, abort_flag, p.error, 3);
      // These scores go where the probabilities of tile t - 2 lay.
      if (t >= 2) ok = ok && mbar_wait_warp(bar(O_REST), (t - 2) & 1, abort_flag, p.error, 4);
      if (!ok) return;
      tcgen05_fence_after();
      const uint64_t keys = further(k_first, stage * L::KV_BYTES);
      if (leader) {
#pragma unroll
        for (int half = 0; half < L::HALVES; ++half)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem_base + st * L::S_COLUMNS, further(q_first, half * L::Q_HALF_BYTES + k * 32),
                      further(keys, half * L::KV_HALF_BYTES + k * 32), idesc_s, (half > 0 || k > 0) ? 1u : 0u);
        tcgen05_commit(bar(S_FULL, st));
        tcgen05_commit(bar(K_EMPTY, stage));
      }
      __syncwarp();
    };
    issue_scores(0);
    for (int t = 0; t < n_tiles && ok; ++t) {
      if (t + 1 < n_tiles) issue_scores(t + 1);
      const int stage = t % KV_STAGES;
      ok = ok && mbar_wait_warp(bar(V_FULL, stage), (t / KV_STAGES) & 1, abort_flag, p.error, 5);
      if (ok && kv_begin + (t + 1) * BKEYS > kv_end)
        clear_values<D>(generic_base + L::V_OFFSET + stage * L::KV_BYTES, kv_end - kv_begin - t * BKEYS, BKEYS, box_rows, lane);
      ok = ok && mbar_wait_warp(bar(P_READY, t & 1), (t >> 1) & 1, abort_flag, p.error, 6);
      if (!ok) break;
      tcgen05_fence_after();
      const uint64_t values = further(v_first, stage * L::KV_BYTES);
      if (leader) {
#pragma unroll
        for (int k = 0; k < BKEYS / 16; ++k)
          umma_bf16_tmem_a(tmem_base + L::O_COLUMN, tmem_base + (t & 1) * L::S_COLUMNS + k * 8, further(values, value_step<D>(k, box_rows)), idesc_o,
                           (t > 0 || k > 0) ? 1u : 0u);
        tcgen05_commit(bar(O_REST));
        tcgen05_commit(bar(V_EMPTY, stage));
        if (t + 1 == n_tiles) tcgen05_commit(bar(O_FULL));
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax, one thread per row
    const int quadrant = warp & 3;
    const int r = quadrant * 32 + lane;                       // row of the tile, lane of tensor memory
    const uint32_t lane_base = tmem_base + ((uint32_t)(quadrant * 32) << 16);
    const int row = work.row0 + r;
    const size_t token = (size_t)(work.first_token + row / groups);
    const int head = g * groups + row % groups;
    // Beside scores the parts of one launch's requests are kept, which may be some of the step's (the weights' scratch has a bound).
    const size_t part_row = (token - (SCORES ? p.q_start[0] : 0)) * p.heads + head;
    const int row_end = min(kv_end, work.pos0 + row / groups + 1);               // the keys before it are visible to the row
    const int all_see = min(kv_end, work.pos0 + work.row0 / groups + 1);         // those before it to every row
    {
      // The warp brings its rows' queries, neighbouring lanes a row's, into the operand's swizzled layout; rows behind the last are zeros.
      constexpr int CHUNKS = D / 8, ROWS_A_PASS = 32 / CHUNKS;
      const int query = (int)token * (p.heads + 2 * p.kv_heads) + head, chunk = lane % CHUNKS;
      uint4 held[32 / ROWS_A_PASS];
#pragma unroll
      for (int i = 0; i < 32 / ROWS_A_PASS; ++i) {
        const int mine = i * ROWS_A_PASS + lane / CHUNKS, from = __shfl_sync(0xffffffffu, query, mine);
        held[i] = quadrant * 32 + mine < rows ? ((const uint4*)(p.qkv + (size_t)from * D))[chunk] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 32 / ROWS_A_PASS; ++i) {
        const int mine = quadrant * 32 + i * ROWS_A_PASS + lane / CHUNKS;
        *(uint4*)(generic_base + L::Q_OFFSET + (chunk >> 3) * L::Q_HALF_BYTES + mine * 128 + (((chunk & 7) ^ (mine & 7)) << 4)) = held[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(bar(Q_FULL));
    }
    float reference = -FLT_MAX, row_sum = 0.f;                // the reference in units of log2, scaled
    bool ok = true;
    for (int t = 0; t < (quadrant < row_warps ? n_tiles : 0); ++t) {
      const int st = t & 1;
      ok = ok && mbar_wait(bar(S_FULL, st), (t >> 1) & 1, abort_flag, p.error, 8);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      const int key0 = kv_begin + t * BKEYS, lo = work.first - key0, hi = r < rows ? row_end - key0 : 0;
      const bool unmasked = lo <= 0 && key0 + BKEYS <= all_see;      // else the row sees the tile's keys lo .. hi - 1
      uint32_t packed[BKEYS / 2];
      uint64_t sum01, sum23, factor2, offset2;
      auto begin = [&] {
        const float offset = reference != -FLT_MAX ? -reference : 0.f;     // without one the visible scores are -infinity or no number: 0 or no number
        factor2 = pack2(p.scale_log2, p.scale_log2);
        offset2 = pack2(offset, offset);
        sum01 = sum23 = 0;
      };
      auto take = [&](const float* s, int i, auto counts) {   // s: the scores of keys i .. i + 3
        float e[4];
        unpack2(fma2(pack2(s[0], s[1]), factor2, offset2), e[0], e[1]);
        unpack2(fma2(pack2(s[2], s[3]), factor2, offset2), e[2], e[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = counts(i + j) ? fast_exp2(e[j]) : 0.f;
        sum01 = add2(sum01, pack2(e[0], e[1]));
        sum23 = add2(sum23, pack2(e[2], e[3]));
        const __nv_bfloat162 h01 = __floats2bfloat162_rn(e[0], e[1]), h23 = __floats2bfloat162_rn(e[2], e[3]);
        packed[i / 2] = *(const uint32_t*)&h01;
        packed[i / 2 + 1] = *(const uint32_t*)&h23;
      };
      auto take32 = [&](const float* s, int first) {
        if (unmasked) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) take(s + i, first + i, [](int) { return true; });
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) take(s + i, first + i, [&](int key) { return key >= lo && key < hi; });
        }
      };
      auto tile_sum = [&] {
        float sums[4];
        unpack2(sum01, sums[0], sums[1]);
        unpack2(sum23, sums[2], sums[3]);
        return (sums[0] + sums[1]) + (sums[2] + sums[3]);
      };
      const uint32_t scores = lane_base + st * L::S_COLUMNS;
      auto leave = [&](const float* s, int first, int count) {
        if constexpr (SCORES) {
          if (r < rows) {
            float* to = p.scores + part_row * p.span + key0 + first;
#pragma unroll
            for (int i = 0; i < count; i += 4) *(float4*)(to + i) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
          }
        }
      };
      bool taken = false, left = false;
      float slack = p.slack;
      if (p.slack > 0.f && !__any_sync(0xffffffffu, r < rows && reference == -FLT_MAX)) {
        // Against the references as they are; should a sum come out above REFERENCE_LIMIT (or not a number), the tile is taken again below.
        float s[32], behind[32];
        tmem_ask32(scores, s);
        tmem_arrived(s);
        tmem_ask32(scores + 32, behind);
        begin();
        take32(s, 0);
        tmem_arrived(behind);
        take32(behind, 32);
        leave(s, 0, 32);
        leave(behind, 32, 32);
        left = true;
        const float sum = tile_sum();
        taken = __all_sync(0xffffffffu, sum <= REFERENCE_LIMIT);
        if (taken) row_sum += sum;
        else slack = 0.f;
      }
      if (!taken) {
        float s[BKEYS];
        tmem_load64(scores, s);
        if (!left) leave(s, 0, BKEYS);
        float m4[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
        if (unmasked) {
#pragma unroll
          for (int i = 0; i < BKEYS; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i]);
        } else {
#pragma unroll
          for (int i = 0; i < BKEYS; ++i) m4[i & 3] = fmaxf(m4[i & 3], i >= lo && i < hi ? s[i] : -FLT_MAX);
        }
        float tile_max = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (tile_max != -FLT_MAX) tile_max *= p.scale_log2;        // the scale is positive: max(s) scales with it
        const bool moves = tile_max > reference + slack || (reference == -FLT_MAX && tile_max != -FLT_MAX);
        if (__any_sync(0xffffffffu, moves)) {
          const float shrink = !moves ? 1.f : (reference == -FLT_MAX ? 0.f : fast_exp2(reference - tile_max));
          if (moves) {
            reference = tile_max;
            row_sum *= shrink;
          }
          if (t >= 1) {
            ok = mbar_wait(bar(O_REST), (t - 1) & 1, abort_flag, p.error, 7);      // the product of the tile before has completed
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tcgen05_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              float o[32];
              uint32_t back[32];
              tmem_load32(lane_base + L::O_COLUMN + c, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) back[i] = __float_as_uint(o[i] * shrink);
              tmem_store32(lane_base + L::O_COLUMN + c, back);
            }
          }
        }
        begin();
        take32(s, 0);
        take32(s + 32, 32);
        row_sum += tile_sum();
      }
      tmem_store32(scores, packed);      // over the scores, which are in registers
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(P_READY, st));
    }
    ok = __all_sync(0xffffffffu, ok);
    if (ok && quadrant < row_warps) {
      ok = mbar_wait(bar(O_FULL), 0, abort_flag, p.error, 9);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tcgen05_fence_after();
        // Through shared memory, where keys and values lay (every product has read them): a row leaves as one run of bytes.
        const uint32_t at = (uint32_t)(part_row * p.slots + work.slot);
        float* mine = (float*)(generic_base + L::K_OFFSET) + quadrant * 32 * D;      // [32][D], 16-byte chunk c of row r at c ^ (r & 7)
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_load32(lane_base + L::O_COLUMN + c, o);
#pragma unroll
          for (int j = 0; j < 32; j += 4) *(float4*)(mine + lane * D + ((((c + j) >> 2) ^ (lane & 7)) << 2)) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
        __syncwarp();
        constexpr int CHUNKS = D / 4, ROWS_A_PASS = 32 / CHUNKS;
        const int chunk = lane % CHUNKS;
#pragma unroll 8
        for (int i = 0; i < 32; i += ROWS_A_PASS) {
          const int from = i + lane / CHUNKS;
          const uint32_t to = __shfl_sync(0xffffffffu, at, from);
          if (quadrant * 32 + from < rows) *(float4*)(p.part_out + (size_t)to * D + chunk * 4) = *(const float4*)(mine + from * D + ((chunk ^ (from & 7)) << 2));
        }
        if (r < rows) {
          p.part_max[at] = reference;
          p.part_sum[at] = row_sum;
        }
      }
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLUMNS);
  }
}

// The slices of token i of a request and head r of a kv head: shared ones, then own ones.
template <int TILE_ROWS>
__device__ __forceinline__ int slices_of(const Params& p, int shared, int kv_len, int pos0, int tokens, int i, int r) {
  const int groups = p.heads / p.kv_heads;
  const OwnSpan span = own_span<TILE_ROWS>(p, shared, kv_len, pos0, tokens, groups, (i * groups + r) / TILE_ROWS);
  const int own = span.end > span.first ? (span.end - span.base + p.own_keys - 1) / p.own_keys : 0;
  return min((shared + p.shared_keys - 1) / p.shared_keys + own, p.slots);
}

template <int D, int DEPTH>
__global__ void __launch_bounds__(pae_attention::MERGE_WARPS * 32) prefix_merge_kernel(__nv_bfloat16* __restrict__ out, const Params p) {
  dependent_launch_trigger();
  extern __shared__ float weights[];          // [slots], then [MERGE_WARPS][D]
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  const int groups = p.heads / p.kv_heads, token0 = p.q_start[b], tokens = p.q_start[b + 1] - token0;
  const int shared = min(p.prefix_len[b], p.max_prefix), kv_len = p.kv_len[b], pos0 = p.q_pos0[b];
  dependent_launch_wait();
  if (i >= tokens) return;
  const int slices = slices_of<ROWS>(p, shared, kv_len, pos0, tokens, i, h % groups);
  const size_t row = (size_t)(token0 + i) * p.heads + h, at = row * p.slots;
  pae_attention::merge_parts<D, DEPTH>(out + row * D, p.part_out + at * D, p.part_max + at, p.part_sum + at, slices, p.slots, weights);
}

template <int N>
__device__ __forceinline__ void load_floats(float (&to)[N], const float* from) {       // of a boundary of N floats
  if constexpr (N == 4) {
    const float4 v = *(const float4*)from;
    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
  } else {
    const float2 v = *(const float2*)from;
    to[0] = v.x, to[1] = v.y;
  }
}

// A row's merge by one warp. The first slices' outputs are asked for together with the maxima and sums that weigh them.
template <int D, int DEPTH>
__device__ __forceinline__ void merge_row(__nv_bfloat16* __restrict__ out, const Params& p, size_t at, int slices, int lane) {
  constexpr int PER_LANE = D / 32;
  static_assert(32 % DEPTH == 0, "a lane holds the weight of one of 32 slices");
  const float* maxima = p.part_max + at;
  const float* sums = p.part_sum + at;
  const float* outputs = p.part_out + at * D + lane * PER_LANE;
  const float my_max = lane < slices ? maxima[lane] : -FLT_MAX, my_sum = lane < slices ? sums[lane] : 0.f;
  float part[DEPTH][PER_LANE];
  auto ask = [&](int s0) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (s0 + u < slices) load_floats(part[u], outputs + (size_t)(s0 + u) * D);
  };
  ask(0);
  float top = my_max, total = 0.f;
  for (int s = lane + 32; s < slices; s += 32) top = fmaxf(top, maxima[s]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane < slices) total = my_sum * exp2f(my_max - top);
  for (int s = lane + 32; s < slices; s += 32) total += sums[s] * exp2f(maxima[s] - top);
  total = warp_sum(total);
  float acc[PER_LANE];
#pragma unroll
  for (int j = 0; j < PER_LANE; ++j) acc[j] = 0.f;
  for (int s0 = 0; s0 < slices; s0 += 32) {
    const float weight = s0 + lane < slices ? exp2f((s0 == 0 ? my_max : maxima[s0 + lane]) - top) : 0.f;
    for (int k = 0; k < min(32, slices - s0); k += DEPTH) {
      if (s0 + k > 0) ask(s0 + k);
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        const float w = __shfl_sync(0xffffffffu, weight, k + u);
        if (s0 + k + u < slices) {
#pragma unroll
          for (int j = 0; j < PER_LANE; ++j) acc[j] += part[u][j] * w;
        }
      }
    }
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int j = 0; j < PER_LANE; j += 2) *(__nv_bfloat162*)(out + lane * PER_LANE + j) = __floats2bfloat162_rn(acc[j] * inv, acc[j + 1] * inv);
}

// The same by one warp a row, for launches of so many rows that warps are there for all SMs.
template <int D, int DEPTH>
__global__ void __launch_bounds__(128) prefix_merge_rows_kernel(__nv_bfloat16* __restrict__ out, const Params p) {
  dependent_launch_trigger();
  const int h = blockIdx.x * 4 + (threadIdx.x >> 5), i = blockIdx.y, b = blockIdx.z;
  const int groups = p.heads / p.kv_heads, token0 = p.q_start[b], tokens = p.q_start[b + 1] - token0;
  const int shared = min(p.prefix_len[b], p.max_prefix), kv_len = p.kv_len[b], pos0 = p.q_pos0[b];
  dependent_launch_wait();
  if (i >= tokens || h >= p.heads) return;
  const size_t row = (size_t)(token0 + i) * p.heads + h;
  merge_row<D, DEPTH>(out + row * D, p, row * p.slots, slices_of<ROWS>(p, shared, kv_len, pos0, tokens, i, h % groups), threadIdx.x & 31);
}

// ---------------------------------------------------------------------------------------
// attention weights added up per key
// ---------------------------------------------------------------------------------------
struct MassParams {
  float* mass;                  // [pages, kv_heads, page_size]
  const int* slots;             // [tokens] or null: a request whose first slot is negative pads the step
  int keep_first, row_blocks, chunks;
};
constexpr int MASS_CHUNK = 512;          // keys per block of 128 threads, four a thread
constexpr int MASS_ROWS = 32;            // rows at a time

// Blocks 0 .. row_blocks - 1 of a request merge its rows (a block each, or a warp each where WARPS); the others add the weights of a chunk of one kv head's keys.
template <int D, bool WARPS, int DEPTH>
__global__ void __launch_bounds__(128) mass_merge_kernel(__nv_bfloat16* __restrict__ out, const Params p, const MassParams m) {
  dependent_launch_trigger();
  extern __shared__ float weights[];     // [slots], then [MERGE_WARPS][D]
  __shared__ float logarithm[MASS_ROWS];
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.heads / p.kv_heads, token0 = p.q_start[b], part0 = token0 - p.q_start[0], tokens = tokens_of(p, b), n = p.kv_len[b], pos0 = p.q_pos0[b];
  dependent_launch_wait();
  if ((int)blockIdx.x < m.row_blocks) {
    const int index = WARPS ? (int)blockIdx.x * 4 + warp : (int)blockIdx.x, i = index / p.heads, h = index % p.heads;
    if (i >= tokens || !in_part(p, token0, tokens)) return;
    const int slices = slices_of<ROWS>(p, 0, n, pos0, tokens, i, h % groups);
    const size_t at = ((size_t)(part0 + i) * p.heads + h) * p.slots;
    __nv_bfloat16* to = out + ((size_t)(token0 + i) * p.heads + h) * D;
    if constexpr (WARPS) merge_row<D, DEPTH>(to, p, at, slices, lane);
    else pae_attention::merge_parts<D, DEPTH>(to, p.part_out + at * D, p.part_max + at, p.part_sum + at, slices, p.slots, weights);
    return;
  }
  const int g = ((int)blockIdx.x - m.row_blocks) / m.chunks, key0 = (((int)blockIdx.x - m.row_blocks) % m.chunks) * MASS_CHUNK;
  const int last = min(min(n, pos0 + tokens), p.span), rows = tokens * groups;
  if (rows <= 0 || !in_part(p, token0, tokens) || key0 >= last || key0 + MASS_CHUNK <= m.keep_first || (m.slots != nullptr && m.slots[token0] < 0)) return;
  const int j0 = key0 + threadIdx.x * 4;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < rows; first += MASS_ROWS) {
    __syncthreads();
    for (int u = warp; u < min(MASS_ROWS, rows - first); u += 4) {
      const int i = (first + u) / groups, r = (first + u) % groups;
      const int slices = slices_of<ROWS>(p, 0, n, pos0, tokens, i, r);
      const size_t at = ((size_t)(part0 + i) * p.heads + g * groups + r) * p.slots;
      float top = -FLT_MAX, total = 0.f;
      for (int s = lane; s < slices; s += 32) top = fmaxf(top, p.part_max[at + s]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      for (int s = lane; s < slices; s += 32) total += p.part_sum[at + s] * exp2f(p.part_max[at + s] - top);
      total = warp_sum(total);
      if (lane == 0) logarithm[u] = total == 0.f ? INFINITY : top + log2f(total);      // of a row without a key the weights are 0
    }
    __syncthreads();
    if (j0 < last) {
      const int count = min(MASS_ROWS, rows - first);
#pragma unroll 4
      for (int u = 0; u < count; ++u) {
        const int i = (first + u) / groups, seen = pos0 + i;
        const float4 s = *(const float4*)(p.scores + ((size_t)(part0 + i) * p.heads + g * groups + (first + u) % groups) * p.span + j0);
        const float l = logarithm[u];
        if (j0 <= seen) w[0] += exp2f(fmaf(s.x, p.scale_log2, -l));
        if (j0 + 1 <= seen) w[1] += exp2f(fmaf(s.y, p.scale_log2, -l));
        if (j0 + 2 <= seen) w[2] += exp2f(fmaf(s.z, p.scale_log2, -l));
        if (j0 + 3 <= seen) w[3] += exp2f(fmaf(s.w, p.scale_log2, -l));
      }
    }
  }
  for (int k = 0; k < 4; ++k) {
    const int j = j0 + k;
    if (j < m.keep_first || j >= last) continue;
    const int page = page_or_none(p.block_table + (size_t)b * p.table_width, j / p.page_size, p.table_width);
    if (page < 0) continue;
    float* to = m.mass + ((size_t)page * p.kv_heads + g) * p.page_size + j % p.page_size;
    *to = (j >= pos0 ? 0.f : *to) + w[k];
  }
}

// ---------------------------------------------------------------------------------------
// any type and head size, on CUDA cores
// ---------------------------------------------------------------------------------------
constexpr int ANY_ROWS = 16;
constexpr int ANY_THREADS = 128;
constexpr int AT_ONCE = 8;               // pieces of keys and of values that a thread asks for before it waits for any

// The operands and the result in their type; the Params' own pointers to them are not used.
template <typename T>
struct AnyOperands {
  const T* qkv;
  const T* keys;
  const T* values;
  T* out;
  int d;                        // a multiple of 4 up to 256
};

__device__ __forceinline__ float4 load4(const float* from) { return *(const float4*)from; }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* from) {
  const uint2 v = *(const uint2*)from;
  const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)&v.x), b = __bfloat1622float2(*(const __nv_bfloat162*)&v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void fma4(float4& acc, float w, const float4& v) {
  acc.x = fmaf(w, v.x, acc.x);
  acc.y = fmaf(w, v.y, acc.y);
  acc.z = fmaf(w, v.z, acc.z);
  acc.w = fmaf(w, v.w, acc.w);
}

// 64 keys a tile: scores by one thread per key and half of the rows, the running softmax by a warp per row, the output by one thread per four channels and
// a share of the keys; the shares are added in their order.
template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) any_slices_kernel(const AnyOperands<T> x, const Params p) {
  extern __shared__ __align__(16) float any_smem[];
  __shared__ float weight[BKEYS][ANY_ROWS], top_of[ANY_ROWS], sum_of[ANY_ROWS], shrink_of[ANY_ROWS];
  dependent_launch_prologue();
  const Work work = find_work<ANY_ROWS, false>(p, blockIdx.x);
  if (work.rows <= 0 || work.begin >= work.end) return;
  const int rows = work.rows, groups = p.heads / p.kv_heads, units = x.d / 4, stride = x.d + 4, tid = threadIdx.x;
  float* q = any_smem;                                   // [ANY_ROWS][d]
  float* k = q + ANY_ROWS * x.d;                         // [BKEYS][stride]: eight rows' 16 bytes fall into different banks
  float* v = k + BKEYS * stride;                         // [BKEYS][d]
  auto token_of = [&](int r) { return work.first_token + (work.row0 + r) / groups; };
  auto head_of = [&](int r) { return work.g * groups + (work.row0 + r) % groups; };
  for (int i = tid; i < rows * units; i += ANY_THREADS) {
    const int r = i / units, c = (i % units) * 4;
    *(float4*)(q + r * x.d + c) = load4(x.qkv + ((size_t)token_of(r) * (p.heads + 2 * p.kv_heads) + head_of(r)) * x.d + c);
  }
  if (tid < ANY_ROWS) {
    top_of[tid] = -FLT_MAX;
    sum_of[tid] = 0.f;
  }
  const int key = tid % BKEYS, half = tid / BKEYS;
  const int shares = ANY_THREADS / units, unit = tid % units, share = tid / units;      // threads behind the last share have no part in the output
  float4 acc[ANY_ROWS];
#pragma unroll
  for (int r = 0; r < ANY_ROWS; ++r) acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int* table = p.block_table + (size_t)work.b * p.table_width;
  for (int key0 = work.begin; key0 < work.end; key0 += BKEYS) {
    const int count = min(BKEYS, work.end - key0);
    __syncthreads();                                     // the tile before is read
    for (int i0 = tid; i0 < BKEYS * units; i0 += ANY_THREADS * AT_ONCE) {
      float4 kv[AT_ONCE], vv[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * ANY_THREADS, row = i / units, c = (i % units) * 4, j = key0 + row;
        kv[u] = vv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < count && j >= work.first) {
          const int page = checked_page(table[checked_table_index(j / p.page_size, p.table_width)]);
          const size_t at = (((size_t)page * p.kv_heads + work.g) * p.page_size + j % p.page_size) * x.d + c;
          kv[u] = load4(x.keys + at);
          vv[u] = load4(x.values + at);
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * ANY_THREADS, row = i / units, c = (i % units) * 4;
        if (row < BKEYS) {
          *(float4*)(k + row * stride + c) = kv[u];
          *(float4*)(v + row * x.d + c) = vv[u];
        }
      }
    }
    __syncthreads();
    {
      float s[ANY_ROWS / 2];                             // of the key with rows half, half + 2, ...
#pragma unroll
      for (int i = 0; i < ANY_ROWS / 2; ++i) s[i] = 0.f;
      for (int c = 0; c < x.d; c += 4) {
        const float4 kv = *(const float4*)(k + key * stride + c);
#pragma unroll
        for (int i = 0; i < ANY_ROWS / 2; ++i)
          if (half + 2 * i < rows) {
            const float4 qv = *(const float4*)(q + (half + 2 * i) * x.d + c);
            s[i] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, s[i]))));
          }
      }
      const int j = key0 + key;
#pragma unroll
      for (int i = 0; i < ANY_ROWS / 2; ++i) {
        const int r = half + 2 * i;
        if (r < rows) weight[key][r] = key < count && j >= work.first && j <= work.pos0 + (work.row0 + r) / groups ? s[i] * p.scale_log2 : -FLT_MAX;
      }
    }
    __syncthreads();
    // A warp per row: the running maximum and sum, and the scores become weights.
    for (int r = tid >> 5; r < rows; r += ANY_THREADS / 32) {
      const int lane = tid & 31;
      const float s0 = weight[lane][r], s1 = weight[lane + 32][r];
      float top = fmaxf(s0, s1);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float before = top_of[r], higher = fmaxf(before, top);
      const float e0 = s0 == -FLT_MAX ? 0.f : exp2f(s0 - higher), e1 = s1 == -FLT_MAX ? 0.f : exp2f(s1 - higher);
      weight[lane][r] = e0;
      weight[lane + 32][r] = e1;
      const float sum = warp_sum(e0 + e1);
      __syncwarp();
      if (lane == 0) {
        const float shrink = before == -FLT_MAX ? 1.f : exp2f(before - higher);      // without a key all is 0, or not a number
        sum_of[r] = sum_of[r] * shrink + sum;
        top_of[r] = higher;
        shrink_of[r] = shrink;
      }
    }
    __syncthreads();
    if (share < shares) {
#pragma unroll
      for (int r = 0; r < ANY_ROWS; ++r)
        if (r < rows) {
          const float shrink = shrink_of[r];
          acc[r].x *= shrink;
          acc[r].y *= shrink;
          acc[r].z *= shrink;
          acc[r].w *= shrink;
        }
      for (int j = share; j < count; j += shares) {
        const float4 vv = *(const float4*)(v + j * x.d + unit * 4);
#pragma unroll
        for (int r = 0; r < ANY_ROWS; r += 4)
          if (r < rows) {
            const float4 w = *(const float4*)&weight[j][r];
            fma4(acc[r], w.x, vv);
            if (r + 1 < rows) fma4(acc[r + 1], w.y, vv);
            if (r + 2 < rows) fma4(acc[r + 2], w.z, vv);
            if (r + 3 < rows) fma4(acc[r + 3], w.w, vv);
          }
      }
    }
  }
  __syncthreads();
  float* sums = k;                                       // [shares][rows][d], over the tiles' memory
  if (share < shares) {
#pragma unroll
    for (int r = 0; r < ANY_ROWS; ++r)
      if (r < rows) *(float4*)(sums + ((size_t)share * rows + r) * x.d + unit * 4) = acc[r];
  }
  __syncthreads();
  auto at = [&](int r) { return ((size_t)token_of(r) * p.heads + head_of(r)) * p.slots + work.slot; };
  for (int i = tid; i < rows * units; i += ANY_THREADS) {
    const int r = i / units, c = (i % units) * 4;
    float4 total = *(const float4*)(sums + r * x.d + c);
    for (int s = 1; s < shares; ++s) fma4(total, 1.f, *(const float4*)(sums + ((size_t)s * rows + r) * x.d + c));
    *(float4*)(p.part_out + at(r) * x.d + c) = total;
  }
  if (tid < rows) {
    p.part_max[at(tid)] = top_of[tid];
    p.part_sum[at(tid)] = sum_of[tid];
  }
}

template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) any_merge_kernel(const AnyOperands<T> x, const Params p) {
  dependent_launch_prologue();
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int groups = p.heads / p.kv_heads, token0 = p.q_start[b], tokens = p.q_start[b + 1] - token0;
  if (i >= tokens) return;
  const int slices = slices_of<ANY_ROWS>(p, p.max_prefix > 0 ? min(p.prefix_len[b], p.max_prefix) : 0, p.kv_len[b], p.q_pos0[b], tokens, i, h % groups);
  const size_t row = (size_t)(token0 + i) * p.heads + h, at = row * p.slots;
  float top = -FLT_MAX, total = 0.f;
  for (int s = lane; s < slices; s += 32) top = fmaxf(top, p.part_max[at + s]);           // every warp works them out for itself
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  for (int s = lane; s < slices; s += 32) total += p.part_sum[at + s] * exp2f(p.part_max[at + s] - top);
  total = warp_sum(total);
  const float inverse = total > 0.f ? 1.f / total : 0.f;
  for (int c = threadIdx.x; c < x.d; c += ANY_THREADS) {
    float sum = 0.f;
#pragma unroll 8
    for (int s = 0; s < slices; ++s) sum = fmaf(exp2f(p.part_max[at + s] - top), p.part_out[(at + s) * x.d + c], sum);
    x.out[row * x.d + c] = from_float<T>(sum * inverse);
  }
}

// ---------------------------------------------------------------------------------------
// how the keys are cut
// ---------------------------------------------------------------------------------------
struct Cut {
  int row_tiles, shared_slices, shared_keys, own_row_tiles, own_slices, own_keys, slots;
  long long shared_blocks, own_blocks;
};
// Two blocks share an SM (three of the CUDA-core kernel). Own keys are cut into as many slices as fill a wave, of one tile at least and OWN_TILES at most. The shared keys' blocks fill
// that share of one wave that their tiles are of all tiles (a request's own keys taken as half of the longest's), half of it at least: what is left
// goes to the own blocks, which wait for memory while the others compute. 64 requests, 8,000 shared and 20 to 700 own keys, 28 heads over 4 of
// 128, us a pass, captured, with the merge, in turn: 36.8 with the wave full of shared blocks, 36.0 with three quarters, 31.9 with half (32.5 by the rule), with 3,000 to
// 5,000 own keys 122.6, 120.1 and 113.0 (112.1), 180 requests 71.2, 72.5 and 75.7 (73.2); 24 requests of five tokens, 30,011 shared and 100 to 900 own keys, 40 heads over 8:
// 100.9, 111.7 and 142.2 (98.8). With 4 and 32 tiles at most in place of 12, in another call: 64 requests 35.4 and 30.3 (30.4), with the longer own keys 146 and 101 (107), 180
// requests 88.6 and 69.8 (69.8), the 24 of five tokens 99.0 and 94.1 (95.1); the weights of 48 requests of five tokens over 300 to
// 6,000 keys, 28 heads over 4, whose slices follow the same rule, 193 and 158 (149).
constexpr int OWN_TILES = 12;
Cut cut_keys(int seqs, int groups, int heads, int kv_heads, int box, int max_q_len, int max_prefix, int max_own, int max_group_tokens, bool any) {
  const int share = heads / kv_heads, wave = (any ? 3 : 2) * pae_attention::multiprocessors(), rows = any ? ANY_ROWS : ROWS;
  Cut c;
  c.row_tiles = (int)(((long long)max_group_tokens * share + rows - 1) / rows);
  c.own_row_tiles = (int)(((long long)max_q_len * share + rows - 1) / rows);
  const long long pairs = (long long)seqs * kv_heads * c.own_row_tiles;
  const int own_tiles = (max_own + box - 1 + BKEYS - 1) / BKEYS;     // a span may begin inside a box
  long long most = wave / pairs;
  if (most < (own_tiles + OWN_TILES - 1) / OWN_TILES) most = (own_tiles + OWN_TILES - 1) / OWN_TILES;
  if (most > own_tiles) most = own_tiles;
  if (most < 1) most = 1;
  c.own_keys = own_tiles > 0 ? (int)((own_tiles + most - 1) / most) * BKEYS : BKEYS;
  c.own_slices = own_tiles > 0 ? (own_tiles * BKEYS + c.own_keys - 1) / c.own_keys : 1;
  c.own_blocks = pairs * c.own_slices;
  const long long per_slice = (long long)groups * kv_heads * c.row_tiles;
  const int tiles = (max_prefix + BKEYS - 1) / BKEYS;
  const double shared_work = (double)per_slice * tiles, own_work = 0.5 * pairs * own_tiles;
  const double blocks = wave * fmax(0.5, shared_work / fmax(1.0, shared_work + own_work));
  long long slices = (long long)(blocks / per_slice + 0.5);
  while (slices > 1 && slices * per_slice > wave) --slices;
  const int least = any ? 1 : 2;                         // tiles of a shared slice
  if (slices > (tiles + least - 1) / least) slices = (tiles + least - 1) / least;
  if (slices < 1) slices = 1;
  const int slice_tiles = tiles > 0 ? (int)((tiles + slices - 1) / slices) : 1;
  c.shared_keys = slice_tiles * BKEYS;
  c.shared_slices = tiles > 0 ? (tiles + slice_tiles - 1) / slice_tiles : 0;
  c.shared_blocks = per_slice * c.shared_slices;
  c.slots = c.shared_slices + c.own_slices;
  return c;
}

// Whether the merge of so many rows, a warp each, asks for 16 slices of a row at once: the registers leave an SM some 20 warps then, which have to hold all rows.
// us a pass, captured, with 8 and 16 at once: 28 heads of 64 requests (1,792 rows) 32.0 and 30.3; 40 heads of 24 requests of five tokens 95.1 and 95.7, 28 heads of 180
// requests 69.8 and 70.5. mass_merge_kernel's rows, 4 and 16 at once: 28 heads of 16 requests of up to five tokens 76.5 and 68.1, of 48 of five 149 and 163.
bool rows_in_flight(long long rows) { return rows <= 16LL * pae_attention::multiprocessors(); }

template <int D>
int launch(const Params& p, void* out, long long pages, int blocks, int seqs, int max_q_len, cudaStream_t s) {
  PageMaps maps;
  if (int err = encode_page_maps(&maps, p.keys, p.values, pages, p.kv_heads, p.page_size, D, BKEYS)) return err;
  static DevicesSet devices;
  if (int err = raise_shared_memory(devices, prefix_kernel<D, false>, Layout<D>::SMEM_BYTES, "paged_attention_prefix")) return err;
  launch_kernel(prefix_kernel<D, false>, dim3(blocks), dim3(THREADS), Layout<D>::SMEM_BYTES, s, maps, p);
  if (int err = check_launch("paged_attention_prefix")) return err;
  // A warp a row where the rows fill the SMs with warps, a block a row below that. us a pass, captured, with warps and with blocks: 12 heads of 4 requests
  // 7.4 and 7.6, 28 heads of 64 30.4 and 35.1, 14 heads of 123 18.2 and 19.8; the rows of mass_merge_kernel, 28 heads of 48 requests of five tokens, 149 and 201, of 4 38.1 and 39.9.
  const long long rows = (long long)p.heads * max_q_len * seqs;
  if (rows >= 8LL * pae_attention::multiprocessors()) {
    const auto merge = rows_in_flight(rows) ? prefix_merge_rows_kernel<D, 16> : prefix_merge_rows_kernel<D, 8>;
    launch_kernel(merge, dim3((p.heads + 3) / 4, max_q_len, seqs), dim3(128), 0, s, (__nv_bfloat16*)out, p);
    return check_launch("paged_attention_prefix");
  }
  const auto merge = pae_attention::merge_in_few_registers(p.heads * max_q_len, seqs, p.slots) ? prefix_merge_kernel<D, 8> : prefix_merge_kernel<D, 24>;
  launch_kernel(merge, dim3(p.heads, max_q_len, seqs), dim3(pae_attention::MERGE_WARPS * 32),
                (p.slots + pae_attention::MERGE_WARPS * D) * sizeof(float), s, (__nv_bfloat16*)out, p);
  return check_launch("paged_attention_prefix");
}

template <int D, bool WARPS, int DEPTH>
int launch_mass(const Params& p, const MassParams& m, void* out, long long pages, int blocks, int seqs, cudaStream_t s) {
  PageMaps maps;
  if (int err = encode_page_maps(&maps, p.keys, p.values, pages, p.kv_heads, p.page_size, D, BKEYS)) return err;
  static DevicesSet devices;
  if (int err = raise_shared_memory(devices, prefix_kernel<D, true>, Layout<D>::SMEM_BYTES, "paged_attention_mass")) return err;
  launch_kernel(prefix_kernel<D, true>, dim3(blocks), dim3(THREADS), Layout<D>::SMEM_BYTES, s, maps, p);
  if (int err = check_launch("paged_attention_mass")) return err;
  launch_kernel(mass_merge_kernel<D, WARPS, DEPTH>, dim3(m.row_blocks + p.kv_heads * m.chunks, seqs), dim3(128),
                WARPS ? 0 : (p.slots + pae_attention::MERGE_WARPS * D) * sizeof(float), s, (__nv_bfloat16*)out, p, m);
  return check_launch("paged_attention_mass");
}

template <typename T>
int launch_any(const AnyOperands<T>& x, const Params& p, int blocks, int seqs, int max_q_len, cudaStream_t s) {
  const size_t tiles = (size_t)BKEYS * (2 * x.d + 4), shares = (size_t)(ANY_THREADS / (x.d / 4)) * ANY_ROWS * x.d;
  const size_t bytes = ((size_t)ANY_ROWS * x.d + (tiles > shares ? tiles : shares)) * sizeof(float);
  static DevicesSet devices;
  if (int err = raise_shared_memory(devices, any_slices_kernel<T>, 160 * 1024, "paged_attention_prefix")) return err;
  launch_kernel(any_slices_kernel<T>, dim3(blocks), dim3(ANY_THREADS), bytes, s, x, p);
  if (int err = check_launch("paged_attention_prefix")) return err;
  launch_kernel(any_merge_kernel<T>, dim3(p.heads, max_q_len, seqs), dim3(ANY_THREADS), 0, s, x, p);
  return check_launch("paged_attention_prefix");
}

int box_of(int page_size, bool any) { return any ? 1 : (page_size < BKEYS ? page_size : BKEYS); }

// What the kernels are told of a step, but for its operands.
int set_up(Params* to, long long* blocks, const int* block_table, int table_width, const int* q_start, const int* q_pos0, const int* kv_len, const int* prefix_len,
           const int* group_start, int tokens, int seqs, int groups, int heads, int kv_heads, int d, int page_size, int max_q_len, int max_prefix, int max_own,
           int max_group_tokens, float scale, float* scratch, bool any) {
  if (seqs > 65535 || max_q_len > 65535) return fail(3, "paged_attention_prefix: %d requests of up to %d tokens exceed one launch", seqs, max_q_len);
  if ((uintptr_t)scratch & 15) return fail(2, "paged_attention_prefix: the scratch does not start on a 16-byte boundary");
  const Cut c = cut_keys(seqs, groups, heads, kv_heads, box_of(page_size, any), max_q_len, max_prefix, max_own, max_group_tokens, any);
  if ((size_t)(c.slots + pae_attention::MERGE_WARPS * d) * sizeof(float) > 40 * 1024 || c.shared_blocks + c.own_blocks > 0x7fffffffll ||
      (long long)tokens * heads * c.slots > 0xffffffffll)
    return fail(3, "paged_attention_prefix: %d slices a row, %lld + %lld blocks exceed one launch", c.slots, c.shared_blocks, c.own_blocks);
  Params p = {};
  p.block_table = block_table;
  p.q_start = q_start;
  p.q_pos0 = q_pos0;
  p.kv_len = kv_len;
  p.prefix_len = prefix_len;
  p.group_start = group_start;
  const size_t rows = (size_t)tokens * heads * c.slots;
  p.part_out = scratch;
  p.part_max = scratch + rows * d;
  p.part_sum = p.part_max + rows;
  p.table_width = table_width;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.max_prefix = max_prefix;
  p.shared_blocks = (int)c.shared_blocks;
  p.row_tiles = c.row_tiles;
  p.shared_slices = c.shared_slices;
  p.shared_keys = c.shared_keys;
  p.own_row_tiles = c.own_row_tiles;
  p.own_slices = c.own_slices;
  p.own_keys = c.own_keys;
  p.slots = c.slots;
  p.box = box_of(page_size, any);
  p.max_tokens = max_q_len;
  p.scale_log2 = scale * LOG2E;
  p.slack = REFERENCE_SLACK;
  *to = p;
  *blocks = c.shared_blocks + c.own_blocks;
  return 0;
}

}  // namespace

PAE_DEFINE_LAST_ERROR()

PAE_EXPORT int pae_attention_prefix_supports(int heads, int kv_heads, int d, int page_size) {
  return (d == 64 || d == 128) && (page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128) && kv_heads >= 1 && heads % kv_heads == 0;
}

// Floats of scratch that pae_paged_attention_prefix (any = 0) or pae_paged_attention_prefix_any (any = 1) needs for the same sizes.
PAE_EXPORT long long pae_attention_prefix_floats(int tokens, int seqs, int groups, int heads, int kv_heads, int d, int page_size, int max_q_len, int max_prefix,
                                                 int max_own, int max_group_tokens, int any) {
  const Cut c = cut_keys(seqs, groups, heads, kv_heads, box_of(page_size, any), max_q_len, max_prefix, max_own, max_group_tokens, any);
  return (long long)tokens * heads * c.slots * (d + 2);
}

PAE_EXPORT int pae_paged_attention_prefix(void* out, const void* qkv, const void* keys, const void* values, long long pages, const int* block_table,
                                          int table_width, const int* q_start, const int* q_pos0, const int* kv_len, const int* prefix_len,
                                          const int* group_start, int tokens, int seqs, int groups, int heads, int kv_heads, int d, int page_size,
                                          int max_q_len, int max_prefix, int max_own, int max_group_tokens, float scale, float* scratch, int* error,
                                          void* stream) {
  if (tokens == 0 || seqs == 0) return 0;
  if (!pae_attention_prefix_supports(heads, kv_heads, d, page_size))
    return fail(2, "paged_attention_prefix: head_dim %d with pages of %d is not taken (64 or 128; 16, 32, 64 or 128)", d, page_size);
  if ((((uintptr_t)qkv | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) & 15) != 0)
    return fail(2, "paged_attention_prefix: an operand does not start on a 16-byte boundary");
  Params p;
  long long blocks;
  if (int err = set_up(&p, &blocks, block_table, table_width, q_start, q_pos0, kv_len, prefix_len, group_start, tokens, seqs, groups, heads, kv_heads, d, page_size,
                       max_q_len, max_prefix, max_own, max_group_tokens, scale, scratch, false))
    return err;
  p.qkv = (const __nv_bfloat16*)qkv;
  p.keys = (const __nv_bfloat16*)keys;
  p.values = (const __nv_bfloat16*)values;
  p.error = error;
  if (d == 64) return launch<64>(p, out, pages, (int)blocks, seqs, max_q_len, (cudaStream_t)stream);
  return launch<128>(p, out, pages, (int)blocks, seqs, max_q_len, (cudaStream_t)stream);
}

// The same on CUDA cores: dtype 0 float32, 1 bfloat16; head sizes that are multiples of 4 up to 256, pages of any size. max_prefix 0: nothing is shared, and
// prefix_len and group_start are not read.
PAE_EXPORT int pae_paged_attention_prefix_any(void* out, const void* qkv, const void* keys, const void* values, const int* block_table, int table_width,
                                              const int* q_start, const int* q_pos0, const int* kv_len, const int* prefix_len, const int* group_start, int tokens,
                                              int seqs, int groups, int heads, int kv_heads, int d, int page_size, int max_q_len, int max_prefix, int max_own,
                                              int max_group_tokens, float scale, int dtype, float* scratch, void* stream) {
  if (tokens == 0 || seqs == 0) return 0;
  if (d < 4 || d > 256 || d % 4) return fail(2, "paged_attention_prefix: head_dim %d is not a multiple of 4 up to 256", d);
  if (kv_heads < 1 || heads % kv_heads) return fail(2, "paged_attention_prefix: %d heads over %d kv heads", heads, kv_heads);
  if (((uintptr_t)qkv | (uintptr_t)keys | (uintptr_t)values) & (dtype == kF32 ? 15 : 7))
    return fail(2, "paged_attention_prefix: an operand does not start on a boundary of four elements");
  Params p;
  long long blocks;
  if (int err = set_up(&p, &blocks, block_table, table_width, q_start, q_pos0, kv_len, prefix_len, group_start, tokens, seqs, groups, heads, kv_heads, d, page_size,
                       max_q_len, max_prefix, max_own, max_group_tokens, scale, scratch, true))
    return err;
  if (dtype == kF32) return launch_any<float>({(const float*)qkv, (const float*)keys, (const float*)values, (float*)out, d}, p, (int)blocks, seqs, max_q_len, (cudaStream_t)stream);
  return launch_any<__nv_bfloat16>({(const __nv_bfloat16*)qkv, (const __nv_bfloat16*)keys, (const __nv_bfloat16*)values, (__nv_bfloat16*)out, d}, p, (int)blocks, seqs,
                                   max_q_len, (cudaStream_t)stream);
}

// Floats of scratch that pae_paged_attention_few_mass needs; `tokens`: what the requests bring at most.
PAE_EXPORT long long pae_attention_few_mass_floats(int tokens, int seqs, int heads, int kv_heads, int d, int page_size, int max_q_len, int max_kv_len) {
  const Cut c = cut_keys(seqs, 1, heads, kv_heads, box_of(page_size, false), max_q_len, 0, max_kv_len, max_q_len, false);
  return (long long)tokens * heads * (c.slots * (d + 2) + (long long)c.own_slices * c.own_keys);
}

// Attention of consecutive requests that bring few tokens, and the weights of their keys: those that block_table, q_start, q_pos0 and kv_len begin with (q_start
// counts tokens of the whole step, as qkv, out and `slots` do); `slots` and `keep_first` as pae_paged_attention_any_mass (attention_mass.cu) takes them.
PAE_EXPORT int pae_paged_attention_few_mass(void* out, const void* qkv, const void* keys, const void* values, float* mass, long long pages, const int* block_table,
                                            int table_width, const int* q_start, const int* q_pos0, const int* kv_len, const int* slots, int tokens, int seqs,
                                            int heads, int kv_heads, int d, int page_size, int max_q_len, int max_kv_len, float scale, int keep_first,
                                            float* scratch, int* error, void* stream) {
  if (tokens == 0 || seqs == 0 || max_kv_len < 1) return 0;
  if (!pae_attention_prefix_supports(heads, kv_heads, d, page_size))
    return fail(2, "paged_attention_mass: head_dim %d with pages of %d is not taken (64 or 128; 16, 32, 64 or 128)", d, page_size);
  if ((((uintptr_t)qkv | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) & 15) != 0)
    return fail(2, "paged_attention_mass: an operand does not start on a 16-byte boundary");
  Params p;
  long long blocks;
  if (int err = set_up(&p, &blocks, block_table, table_width, q_start, q_pos0, kv_len, nullptr, nullptr, tokens, seqs, 1, heads, kv_heads, d, page_size, max_q_len, 0,
                       max_kv_len, max_q_len, scale, scratch, false))
    return err;
  p.qkv = (const __nv_bfloat16*)qkv;
  p.keys = (const __nv_bfloat16*)keys;
  p.values = (const __nv_bfloat16*)values;
  p.error = error;
  p.span = p.own_slices * p.own_keys;
  p.scores = scratch;                                    // rows of a multiple of 64 floats
  p.part_tokens = tokens;
  p.part_out = scratch + (size_t)tokens * heads * p.span;
  p.part_max = p.part_out + (size_t)tokens * heads * p.slots * d;
  p.part_sum = p.part_max + (size_t)tokens * heads * p.slots;
  const int rows = heads * max_q_len;
  const bool warps = (long long)rows * seqs >= 8LL * pae_attention::multiprocessors(), deep = rows_in_flight((long long)rows * seqs);
  const MassParams m = {mass, slots, keep_first, warps ? (rows + 3) / 4 : rows, (p.span + MASS_CHUNK - 1) / MASS_CHUNK};
  const cudaStream_t s = (cudaStream_t)stream;
  const auto run = d == 64 ? (!warps ? launch_mass<64, false, 24> : deep ? launch_mass<64, true, 16> : launch_mass<64, true, 4>)
                           : (!warps ? launch_mass<128, false, 24> : deep ? launch_mass<128, true, 16> : launch_mass<128, true, 4>);
  return run(p, m, out, pages, (int)blocks, seqs, s);
}
