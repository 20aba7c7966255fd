// The attention weights of prompt portions, added up per key (attention_mass.cu says what is computed), on the fifth-generation
// tensor cores. The attention itself ran before (attention_tcgen05.cu) and left of every row r = (token, query head) the logarithm l_r
// of its softmax's denominator, in units of log2, so that a weight is one exponential:
//
//   w[g, j] = sum over the rows of kv head g that see key j of 2^(scale_log2 q_r . k_j - l_r)
//
// The sum runs over rows, so the keys are the MMA's rows: a block owns 128 keys of one (request, kv head), which it loads once, and
// walks a chunk of the request's query rows, 128 / (heads per kv head) tokens a tile:
//
//   warp 0      TMA: the keys once, by their pages; per tile one box of heads x tokens x 64 channels for each half of the head dimension
//   warp 1      MMA: scores [128 keys x 128 rows] = K . Q^T into one of two buffers in tensor memory
//   warps 2-9   two threads per key, each for half of a tile's rows: 64 scores, 64 exponentials, one sum. No shuffles, no second product.
//   warp 10     the rows' l_r, negated, into shared memory beside the scores' buffers; -infinity where a tile's rows end
//
// The rows are cut into chunks so that many blocks of nearly one length are there (a causal mask makes late key tiles short); their sums
// are added in the chunks' order by a second kernel, which writes the mass. Two blocks share an SM. The exponentials, 16 a clock and SM, bound it at 1,024 clocks a
// tile of 128 x 128, the operands of the MMA in shared memory at 565; three portions of 700 to 1,500 tokens over 1,500 to 2,900 keys, 28
// heads over 4 of 128, take some 100 us of a pass's 230 (108 alone, with cold caches), the attention the rest, the exponentials' pipe half busy. One thread a key, blocks of 256 keys alone on an SM, and three to
// five stages of queries took the same time.
#include <cfloat>
#include <climits>

#include "attention_pages.cuh"

using namespace pae;
using namespace pae_tcgen05;

namespace {

constexpr int KEYS = 128;               // per block: the MMA's rows
constexpr int TILE = 128;               // query rows per tile: its columns
constexpr int STAGES = 2;
constexpr int THREADS = 352;
constexpr int SUM_WARPS = 8;
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  __nv_bfloat16* out;           // [tokens, heads, d]
  float* mass;                  // [pages, kv_heads, page_size]
  float* part;                  // [chunks, requests, kv_heads, span]
  const float* lse;             // [tokens, heads], units of log2
  const int* block_table;
  const int* q_start;
  const int* q_pos0;
  const int* kv_len;
  const int* slots;             // [tokens] or null: a request whose first slot is negative pads the step
  int table_width, heads, kv_heads, d, page_size, keep_first;
  int tile_tokens, chunk_tiles, span, seqs;
  int least;                    // tokens of the requests that are taken: 2 where the kernel of single tokens takes the others, else 1
  float scale_log2;
  int* error;
};

template <int D>
struct Layout {
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = KEYS * 128;
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
  static constexpr int K_OFFSET = 0;
  static constexpr int Q_OFFSET = TILE_BYTES;                         // two stages
  static constexpr int LSE_OFFSET = Q_OFFSET + STAGES * TILE_BYTES;   // [2][TILE] floats
  static constexpr int BAR_OFFSET = LSE_OFFSET + 2 * TILE * 4;
  static constexpr size_t SMEM_BYTES = (size_t)BAR_OFFSET + 256 + 1024;
  static constexpr int TMEM_COLUMNS = 2 * TILE;
};

enum Bar : int { K_FULL = 0, Q_FULL = 1, Q_EMPTY = 3, S_FULL = 5, S_EMPTY = 7, L_FULL = 9, L_EMPTY = 11, NUM_BARS = 13 };

// Which tiles of query rows a block takes: those of its chunk that see its keys.
struct Tiles {
  int tokens, pos0, first, last;
};
__device__ __forceinline__ Tiles tiles_of(const Params& p, int b, int key0, int chunk) {
  Tiles t;
  const int start = p.q_start[b];
  t.tokens = p.q_start[b + 1] - start;
  t.pos0 = p.q_pos0[b];
  const int all = (t.tokens + p.tile_tokens - 1) / p.tile_tokens;
  t.first = max(chunk * p.chunk_tiles, max(0, key0 - t.pos0) / p.tile_tokens);
  t.last = min((chunk + 1) * p.chunk_tiles, all);
  if (t.tokens < p.least || key0 >= min(p.kv_len[b], t.pos0 + t.tokens) || key0 + KEYS <= p.keep_first || (p.slots != nullptr && p.slots[start] < 0)) t.last = t.first;
  return t;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2) column_sums_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ PageMaps maps,
                                                                 const Params p) {
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
  // The last chunks' rows see the most keys: their blocks go first, the shorter ones fill in behind them.
  const int g = blockIdx.y % p.kv_heads, b = blockIdx.y / p.kv_heads, chunk = gridDim.z - 1 - blockIdx.z, key0 = blockIdx.x * KEYS;
  const Tiles tiles = tiles_of(p, b, key0, chunk);
  const bool working = tiles.first < tiles.last;       // the same in every thread
  const int n_tiles = tiles.last - tiles.first;
  const int first_token = p.q_start[b];
  const int kv_end = min(p.kv_len[b], tiles.pos0 + tiles.tokens);
  const int groups = p.heads / p.kv_heads, tile_rows = p.tile_tokens * groups;

  if (threadIdx.x == 0 && working) {
    mbar_init(bar(K_FULL), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(Q_FULL, i), 1);
      mbar_init(bar(Q_EMPTY, i), 1);
      mbar_init(bar(S_FULL, i), 1);
      mbar_init(bar(S_EMPTY, i), SUM_WARPS);
      mbar_init(bar(L_FULL, i), 32);
      mbar_init(bar(L_EMPTY, i), SUM_WARPS);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1 && working) {
    tmem_alloc(smem_u32((const void*)tmem_holder), L::TMEM_COLUMNS);
    tmem_relinquish();
  }
  // Rows of a stage that no box fills are zeros: their scores are masked, but they are computed.
  for (int i = working ? threadIdx.x : INT_MAX; i < (TILE - tile_rows) * (D / 8) * STAGES; i += THREADS) {
    const int stage = i / ((TILE - tile_rows) * (D / 8)), rest = i % ((TILE - tile_rows) * (D / 8));
    const int row = tile_rows + rest / (D / 8), c = rest % (D / 8);
    *(uint4*)(generic_base + L::Q_OFFSET + stage * L::TILE_BYTES + (c >> 3) * L::HALF_BYTES + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tcgen05_fence_before();
  __syncthreads();
  dependent_launch_trigger();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  dependent_launch_wait();
  if (!working) return;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const int* table = p.block_table + (size_t)b * p.table_width;
    const int box_rows = min(p.page_size, KEYS), last_page = (kv_end - 1) / p.page_size;
    const int page = lane < KEYS / box_rows ? checked_page(table[checked_table_index(min((key0 + lane * box_rows) / p.page_size, last_page), p.table_width)]) : 0;
    if (lane == 0) mbar_expect_tx(bar(K_FULL), L::TILE_BYTES);
    __syncwarp();
    load_pages<D>(maps, false, base + L::K_OFFSET, bar(K_FULL), KEYS, box_rows, lane, g, page, 0);
    int issued = 0;
    for (int t = 0; t < n_tiles; ++t) {
      const int st = t % STAGES;
      if (t >= STAGES && !mbar_wait_warp(bar(Q_EMPTY, st), (t / STAGES - 1) & 1, abort_flag, p.error, 1)) break;
      if (lane == 0) {
        mbar_expect_tx(bar(Q_FULL, st), (uint32_t)(tile_rows * 128 * L::HALVES));
#pragma unroll
        for (int half = 0; half < L::HALVES; ++half)
          asm volatile(
              "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
              ::"r"(base + L::Q_OFFSET + st * L::TILE_BYTES + half * L::HALF_BYTES), "l"(&map_q), "r"(bar(Q_FULL, st)), "r"(half * 64), "r"(g * groups),
                "r"(first_token + (tiles.first + t) * p.tile_tokens)
              : "memory");
      }
      __syncwarp();
      issued = t + 1;
    }
    if (lane == 0 && *abort_flag) {      // copies that were issued still write into this block's shared memory
      for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(bar(K_FULL), 0); ++w) __nanosleep(64);
      for (int t = max(0, issued - STAGES); t < issued; ++t)
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(bar(Q_FULL, t % STAGES), (t / STAGES) & 1); ++w) __nanosleep(64);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    constexpr uint32_t idesc = instruction_descriptor(KEYS, TILE, false);
    const uint64_t k_first = smem_descriptor(base + L::K_OFFSET), q_first = smem_descriptor(base + L::Q_OFFSET);
    bool ok = mbar_wait_warp(bar(K_FULL), 0, abort_flag, p.error, 2);
    for (int t = 0; t < n_tiles && ok; ++t) {
      const int st = t % STAGES;
      ok = ok && mbar_wait_warp(bar(Q_FULL, st), (t / STAGES) & 1, abort_flag, p.error, 3);
      if (t >= 2) ok = ok && mbar_wait_warp(bar(S_EMPTY, t & 1), ((t >> 1) - 1) & 1, abort_flag, p.error, 4);
      if (!ok) break;
      tcgen05_fence_after();
      const uint64_t queries = further(q_first, st * L::TILE_BYTES);
      if (leader) {
#pragma unroll
        for (int half = 0; half < L::HALVES; ++half)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tmem_base + (t & 1) * TILE, further(k_first, half * L::HALF_BYTES + k * 32), further(queries, half * L::HALF_BYTES + k * 32), idesc,
                      (half > 0 || k > 0) ? 1u : 0u);
        tcgen05_commit(bar(S_FULL, t & 1));
        tcgen05_commit(bar(Q_EMPTY, st));
      }
      __syncwarp();
    }
  } else if (warp == 2 + SUM_WARPS) {
    // ------------------------------------------------------------------ the rows' logarithms
    for (int t = 0; t < n_tiles; ++t) {
      const int token0 = (tiles.first + t) * p.tile_tokens, rows = min(p.tile_tokens, tiles.tokens - token0) * groups;
      float v[TILE / 32];
#pragma unroll
      for (int i = 0; i < TILE / 32; ++i) {
        const int row = i * 32 + lane;
        v[i] = row < rows ? -p.lse[(size_t)(first_token + token0 + row / groups) * p.heads + g * groups + row % groups] : -INFINITY;
      }
      if (t >= 2 && !mbar_wait_warp(bar(L_EMPTY, t & 1), ((t >> 1) - 1) & 1, abort_flag, p.error, 5)) break;
      float* to = (float*)(generic_base + L::LSE_OFFSET) + (t & 1) * TILE;
#pragma unroll
      for (int i = 0; i < TILE / 32; ++i) to[i * 32 + lane] = v[i];
      mbar_arrive(bar(L_FULL, t & 1));
    }
  } else {
    // ------------------------------------------------------------------ two threads per key
    const int quadrant = warp & 3, r = quadrant * 32 + lane, side = (warp - 2) >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quadrant * 32) << 16);
    const int j = key0 + r;
    uint64_t sum01 = 0, sum23 = 0;
    const uint64_t factor2 = pack2(p.scale_log2, p.scale_log2);
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int token0 = (tiles.first + t) * p.tile_tokens;
      ok = ok && mbar_wait(bar(L_FULL, t & 1), (t >> 1) & 1, abort_flag, p.error, 6);
      ok = ok && mbar_wait(bar(S_FULL, t & 1), (t >> 1) & 1, abort_flag, p.error, 7);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      // The tile's first `until` rows are the request's; of them the key is seen from row `from` on.
      const int until = min(p.tile_tokens, tiles.tokens - token0) * groups, from = max(0, j - tiles.pos0 - token0) * groups;
      // (Rows that no box fills score 0 against an l_r of infinity: their weight is 0 without a mask.)
      const bool all = until == tile_rows && key0 + KEYS - 1 <= tiles.pos0 + token0;
      const ulonglong2* negated = (const ulonglong2*)(generic_base + L::LSE_OFFSET + (t & 1) * TILE * 4);
      const int column = side * (TILE / 2);
      const uint32_t scores = lane_base + (t & 1) * TILE + column;
      auto add = [&](const float (&s)[32], int c, auto counts) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const ulonglong2 l = negated[(column + c + i) / 4];
          float e[4];
          unpack2(fma2(pack2(s[i], s[i + 1]), factor2, l.x), e[0], e[1]);
          unpack2(fma2(pack2(s[i + 2], s[i + 3]), factor2, l.y), e[2], e[3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) e[k] = counts(column + c + i + k) ? fast_exp2(e[k]) : 0.f;
          sum01 = add2(sum01, pack2(e[0], e[1]));
          sum23 = add2(sum23, pack2(e[2], e[3]));
        }
      };
      float s[32], behind[32];
      tmem_ask32(scores, s);
      tmem_arrived(s);
      tmem_ask32(scores + 32, behind);
      if (all) {
        add(s, 0, [](int) { return true; });
        tmem_arrived(behind);
        add(behind, 32, [](int) { return true; });
      } else {
        auto seen = [&](int row) { return row >= from && row < until; };
        add(s, 0, seen);
        tmem_arrived(behind);
        add(behind, 32, seen);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(S_EMPTY, t & 1));
        mbar_arrive(bar(L_EMPTY, t & 1));
      }
    }
    float e[4];
    unpack2(sum01, e[0], e[1]);
    unpack2(sum23, e[2], e[3]);
    const float sum = (e[0] + e[1]) + (e[2] + e[3]);
    float* halves = (float*)(generic_base + L::K_OFFSET);       // the second halves' sums, where the keys lay: every product has read them
    if (side == 1) halves[r] = sum;
    asm volatile("bar.sync 1, 256;" ::: "memory");              // the sum warps
    if (ok && side == 0 && j < p.span) p.part[(((size_t)chunk * p.seqs + b) * p.kv_heads + g) * p.span + j] = sum + halves[r];
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLUMNS);
  }
}

__global__ void __launch_bounds__(KEYS) add_chunks_kernel(const Params p, int chunks) {
  dependent_launch_prologue();
  const int g = blockIdx.y, b = blockIdx.z, key0 = blockIdx.x * KEYS, j = key0 + threadIdx.x;
  Tiles tiles = tiles_of(p, b, key0, 0);
  const int n = min(p.kv_len[b], tiles.pos0 + tiles.tokens);
  if (n <= 0 && key0 == 0 && tiles.tokens >= p.least) {      // a request without keys: the attention leaves its rows as they were
    const int pieces = p.heads / p.kv_heads * p.d / 8;                                // of 16 bytes, of a token's heads of g
    uint4* out = (uint4*)(p.out + (size_t)p.q_start[b] * p.heads * p.d) + g * pieces;
    for (int i = threadIdx.x; i < tiles.tokens * pieces; i += KEYS) out[(size_t)(i / pieces) * p.kv_heads * pieces + i % pieces] = make_uint4(0, 0, 0, 0);
  }
  if (j < p.keep_first || j >= min(n, p.span) || tiles.tokens < p.least || (p.slots != nullptr && p.slots[p.q_start[b]] < 0)) return;
  float w = 0.f;
  for (int c = 0; c < chunks; ++c) {
    tiles = tiles_of(p, b, key0, c);
    if (tiles.first < tiles.last) w += p.part[(((size_t)c * p.seqs + b) * p.kv_heads + g) * p.span + j];
  }
  const int page = page_or_none(p.block_table + (size_t)b * p.table_width, j / p.page_size, p.table_width);
  if (page < 0) return;
  float* to = p.mass + ((size_t)page * p.kv_heads + g) * p.page_size + j % p.page_size;
  *to = (j >= tiles.pos0 ? 0.f : *to) + w;
}

// Tiles per chunk: so many that some four times as many blocks are there as run at once, of eight tiles at least.
int tiles_a_chunk(int seqs, int kv_heads, int max_q_len, int max_kv_len, int tile_tokens) {
  const long long blocks = (long long)seqs * kv_heads * ((max_kv_len + KEYS - 1) / KEYS);
  const int tiles = (max_q_len + tile_tokens - 1) / tile_tokens;
  long long chunks = (8 * 148 + blocks - 1) / blocks;
  if (chunks > (tiles + 7) / 8) chunks = (tiles + 7) / 8;
  if (chunks < 1) chunks = 1;
  return (int)((tiles + chunks - 1) / chunks);
}
int chunk_count(int seqs, int kv_heads, int max_q_len, int max_kv_len, int tile_tokens) {
  const int tiles = (max_q_len + tile_tokens - 1) / tile_tokens, each = tiles_a_chunk(seqs, kv_heads, max_q_len, max_kv_len, tile_tokens);
  return (tiles + each - 1) / each;
}

template <int D>
int launch(const Params& p, const void* qkv, const void* keys, long long pages, int tokens, int chunks, cudaStream_t s) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return fail(101, "attention_mass: the driver does not export cuTensorMapEncodeTiled");
  CUtensorMap map_q;
  const int share = p.heads / p.kv_heads, all = p.heads + 2 * p.kv_heads;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)all, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)all * D * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)share, (cuuint32_t)p.tile_tokens};
  const cuuint32_t element_strides[3] = {1, 1, 1};
  if (encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(qkv), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(102, "attention_mass: cuTensorMapEncodeTiled failed for %d tokens of %d heads of %d", tokens, all, D);
  PageMaps maps;
  if (int err = encode_page_maps(&maps, keys, keys, pages, p.kv_heads, p.page_size, D, KEYS)) return err;
  static DevicesSet devices;
  if (int err = raise_shared_memory(devices, column_sums_kernel<D>, Layout<D>::SMEM_BYTES, "attention_mass")) return err;
  const int key_tiles = (p.span + KEYS - 1) / KEYS;
  launch_kernel(column_sums_kernel<D>, dim3(key_tiles, p.kv_heads * p.seqs, chunks), dim3(THREADS), Layout<D>::SMEM_BYTES, s, map_q, maps, p);
  if (int err = check_launch("attention_mass")) return err;
  launch_kernel(add_chunks_kernel, dim3(key_tiles, p.kv_heads, p.seqs), dim3(KEYS), 0, s, p, chunks);
  return check_launch("attention_mass");
}

}  // namespace

PAE_DEFINE_LAST_ERROR()

PAE_EXPORT int pae_attention_mass_prompt_supports(int heads, int kv_heads, int d, int page_size) {
  return (d == 64 || d == 128) && (page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128) && kv_heads >= 1 && heads % kv_heads == 0 &&
         heads / kv_heads <= TILE;
}

// Floats of scratch that pae_attention_mass_prompt needs for the same sizes.
PAE_EXPORT long long pae_attention_mass_prompt_floats(int seqs, int heads, int kv_heads, int max_q_len, int max_kv_len) {
  return (long long)chunk_count(seqs, kv_heads, max_q_len, max_kv_len, TILE / (heads / kv_heads)) * seqs * kv_heads * max_kv_len;
}

// Adds the weights of the requests that bring `least` (1 or 2) tokens and more. `lse` [tokens, heads] is what the attention left of their rows,
// `out` its result, in which the rows of requests without keys become zeros.
PAE_EXPORT int pae_attention_mass_prompt(void* out, float* mass, const void* qkv, const void* keys, long long pages, const float* lse, const int* block_table,
                                         int table_width, const int* q_start, const int* q_pos0, const int* kv_len, const int* slots, int tokens, int seqs,
                                         int max_q_len, int max_kv_len, int heads, int kv_heads, int d, int page_size, float scale, int keep_first,
                                         int least, float* scratch, int* error, void* stream) {
  if (tokens == 0 || seqs == 0 || max_kv_len < 1) return 0;
  if (!pae_attention_mass_prompt_supports(heads, kv_heads, d, page_size))
    return fail(2, "attention_mass: %d heads over %d of head_dim %d with pages of %d are not taken", heads, kv_heads, d, page_size);
  if (((uintptr_t)qkv | (uintptr_t)keys) & 15) return fail(2, "attention_mass: an operand does not start on a 16-byte boundary");
  Params p = {};
  p.out = (__nv_bfloat16*)out;
  p.d = d;
  p.mass = mass;
  p.part = scratch;
  p.lse = lse;
  p.block_table = block_table;
  p.q_start = q_start;
  p.q_pos0 = q_pos0;
  p.kv_len = kv_len;
  p.slots = slots;
  p.table_width = table_width;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.keep_first = keep_first;
  p.tile_tokens = TILE / (heads / kv_heads);
  p.chunk_tiles = tiles_a_chunk(seqs, kv_heads, max_q_len, max_kv_len, p.tile_tokens);
  p.span = max_kv_len;
  p.seqs = seqs;
  p.least = least;
  p.scale_log2 = scale * LOG2E;
  p.error = error;
  const int chunks = chunk_count(seqs, kv_heads, max_q_len, max_kv_len, p.tile_tokens);
  if ((long long)kv_heads * seqs > 65535 || chunks > 65535) return fail(3, "attention_mass: %d requests of %d kv heads, %d chunks exceed one launch", seqs, kv_heads, chunks);
  if (d == 64) return launch<64>(p, qkv, keys, pages, tokens, chunks, (cudaStream_t)stream);
  return launch<128>(p, qkv, keys, pages, tokens, chunks, (cudaStream_t)stream);
}
