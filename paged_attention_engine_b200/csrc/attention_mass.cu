// The attention weight that a step's queries give to the cached keys, added up per key: what an eviction
// goes by (evict.cu). Of request b, kv head g and key j
//
//   w[b, g, j] = sum over the step's tokens t of b at or behind j, and the query heads h of g, of
//                exp(s_thj - max_k s_thk) / sum_k exp(s_thk - max_k s_thk),   s = scale q . k
//   mass[page(b, j), g, place(b, j)] = (j is a key of this step ? 0 : mass) + w,    j >= keep_first
//
// in float32 throughout: scores, maxima, sums, weights. (The output of the bfloat16 kernels is paged_attention's: there the probabilities, but not the weights, are
// rounded to bfloat16 for the second product on tensor cores.) Requests that only pad a step (slot -1) add nothing.
// No atomics: a key's sum is one thread's, in the order of the rows.
//
//   slices, merge   steps of single tokens in bfloat16 (head sizes 32, 64, 128): the sliced decode attention of attention_mma.cuh,
//                   which leaves the scaled scores beside its partial outputs (4 bytes for each query head and key, where the keys and values
//                   are 4 * head size bytes for each kv head and key), and one kernel that merges the slices and, in further blocks,
//                   turns the scores into weights once a row's maximum and sum are known.
//   slices, merge   the same on CUDA cores for single tokens of any other type and head size that is a multiple of 4 up to 256 (up to 16 query
//                   heads a kv head): a block takes 64 keys a tile, one thread per key and half of the rows for the scores, one per four channels and a share
//                   of the keys for the output.
//   stats, columns  every other step: the rows' maxima and sums over runs of keys, then per tile of keys and chunk of rows the
//                   weights, from scores that are computed again, and the chunks' sums in their order. CUDA cores, any type and head size that is a multiple of 4 up to 256. (Steps of several tokens in
//                   bfloat16, and of more than 16 query heads a kv head, go to attention_prefix.cu and attention_mass_prompt.cu where those take their sizes.)
#include "attention_mma.cuh"

using namespace pae;
using namespace pae_attention;

namespace {

struct MassParams {
  float* mass;                  // [pages, kv_heads, page_size]
  const int* block_table;
  const int* q_start;
  const int* kv_len;
  const int* slots;             // [tokens] or null: a request whose first slot is negative pads the step
  int table_width, heads, kv_heads, page_size, keep_first;
};

__device__ __forceinline__ bool pads(const MassParams& m, int token) { return m.slots != nullptr && m.slots[token] < 0; }

// mass = (mass, or 0 for a key that starts from nothing) + w.
__device__ __forceinline__ void add_mass(const MassParams& m, int b, int g, int j, bool fresh, float w) {
  const int page = page_or_none(m.block_table + (size_t)b * m.table_width, j / m.page_size, m.table_width);
  if (page < 0) return;
  float* to = m.mass + ((size_t)page * m.kv_heads + g) * m.page_size + j % m.page_size;
  *to = (fresh ? 0.f : *to) + w;
}

// The weights of the step's keys start from nothing: for a step whose attention adds none. A block a request.
__global__ void __launch_bounds__(128) start_keys_kernel(const MassParams m, const int* __restrict__ q_pos0) {
  dependent_launch_prologue();
  const int b = blockIdx.x, token0 = m.q_start[b], tokens = m.q_start[b + 1] - token0;
  if (tokens < 1 || pads(m, token0)) return;
  const int first = q_pos0[b], count = min(tokens, m.kv_len[b] - first);
  for (int i = threadIdx.x; i < count * m.kv_heads; i += 128) add_mass(m, b, i / count, first + i % count, true, 0.f);
}

// ---------------------------------------------------------------------------------------
// single tokens, bfloat16
// ---------------------------------------------------------------------------------------
// As decode_slices_kernel, which see; the scaled scores (units of log2) go to `scores` [request, head, span].
template <int D>
__global__ void __launch_bounds__(SLICE_WARPS * 32) mass_slices_kernel(const DecodeParams p, float* __restrict__ scores, int span) {
  dependent_launch_trigger();
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.x * SLICE_WARPS + warp;
  const int g = blockIdx.y, b = blockIdx.z;
  const int token = p.q_start[b], kv_len = p.kv_len[b];
  const int begin = slice * p.slice_keys, end = min(kv_len, begin + p.slice_keys);
  const int groups = p.heads / p.kv_heads;
  if (p.q_start[b + 1] - token != 1 || slice >= p.max_slices || begin >= kv_len) {
    dependent_launch_wait();
    return;
  }
  const int row_elems = (p.heads + 2 * p.kv_heads) * D;
  constexpr int TILE_BYTES = TILE_KEYS * D * 2;
  const uint32_t mine = smem_u32(smem + warp * SLICE_STAGES * 2 * TILE_BYTES);
  const int* table = p.block_table + (size_t)b * p.table_width;
  auto fetch = [&](int stage, int key0) {
    const int page = checked_page(table[checked_table_index(key0 / p.page_size, p.table_width)]);
    const size_t row0 = ((size_t)page * p.kv_heads + g) * p.page_size + key0 % p.page_size;
    const uint32_t k_dst = mine + stage * 2 * TILE_BYTES;
#pragma unroll
    for (int i = lane; i < TILE_KEYS * D / 8; i += 32) {
      const int row = i / (D / 8), c = i % (D / 8);
      const int off = TileLayout<D>::offset_bytes(row, c);
      cp_async16(k_dst + off, p.keys + (row0 + row) * D + c * 8);
      cp_async16_or_zeros(k_dst + TILE_BYTES + off, p.values + (row0 + row) * D + c * 8, key0 + row < end);
    }
  };
  const int tiles = (end - begin + TILE_KEYS - 1) / TILE_KEYS;
  int early = 0;                         // tiles of earlier tokens only are asked for before the wait
  while (early < SLICE_STAGES - 1 && early < tiles && begin + (early + 1) * TILE_KEYS <= kv_len - 1) {
    fetch(early, begin + early * TILE_KEYS);
    cp_async_commit();
    ++early;
  }
  dependent_launch_wait();
  uint32_t q[D / 16][4];
  load_query_fragments<D>(q, [&](int r) -> const __nv_bfloat16* {
    return r < groups ? p.qkv + (size_t)token * row_elems + (size_t)(g * groups + r) * D : nullptr;
  });
  for (int i = early; i < SLICE_STAGES - 1; ++i) {
    if (i < tiles) fetch(i, begin + i * TILE_KEYS);
    cp_async_commit();
  }
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float row_max[2] = {-FLT_MAX, -FLT_MAX}, row_sum[2] = {0.f, 0.f};
  float* row_scores = scores + ((size_t)b * p.heads + g * groups + (lane >> 2)) * span + (lane & 3) * 2;
  for (int t = 0; t < tiles; ++t) {
    const int ahead = t + SLICE_STAGES - 1;
    if (ahead < tiles) fetch(ahead % SLICE_STAGES, begin + ahead * TILE_KEYS);
    cp_async_commit();
    cp_async_wait<SLICE_STAGES - 1>();
    __syncwarp();
    const uint32_t k_tile = mine + (t % SLICE_STAGES) * 2 * TILE_BYTES;
    const int key0 = begin + t * TILE_KEYS;
    float s[2][4];
    scores_16_keys<D>(s, q, k_tile, 0);
    // The span is a whole number of tiles, so keys behind the last are written too; nobody reads them.
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if ((lane >> 2) + half * 8 < groups) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *(float2*)(row_scores + (size_t)half * 8 * span + key0 + i * 8) =
              make_float2(s[i][half * 2] * p.scale_log2, s[i][half * 2 + 1] * p.scale_log2);
      }
    uint32_t pa[4];
    softmax_step<D>(s, row_max, row_sum, o, pa, p.scale_log2, key0 + TILE_KEYS <= end, [&](int, int key) { return key0 + key < end; });
    accumulate_16_keys<D>(o, pa, k_tile + TILE_BYTES, 0);
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = (lane >> 2) + half * 8;
    if (r >= groups) continue;
    const size_t at = ((size_t)b * p.heads + g * groups + r) * p.max_slices + slice;
    float* out = p.part_out + at * D;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) *(float2*)(out + n * 8 + (lane & 3) * 2) = make_float2(o[n][half * 2], o[n][half * 2 + 1]);
    if ((lane & 3) == 0) {
      p.part_max[at] = row_max[half];
      p.part_sum[at] = row_sum[half];
    }
  }
}

constexpr int MASS_CHUNK = 512;          // keys per block of 128 threads, four a thread

// The weights of keys key0 .. key0 + MASS_CHUNK - 1 of (request b, kv head g), from the scores and the slices' maxima and sums.
__device__ __forceinline__ void add_chunk(const MassParams& m, const float* __restrict__ part_max, const float* __restrict__ part_sum, const float* __restrict__ scores, int b,
                                          int g, int key0, int token, int n_kv, int slices, int slice_keys, int max_slices, int span, float* top_of, float* inverse_of) {
  const int last = min(n_kv, slices * slice_keys);
  if (key0 >= last || key0 + MASS_CHUNK <= m.keep_first || pads(m, token)) return;
  const int groups = m.heads / m.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < groups; r += MERGE_WARPS) {
    const size_t at = ((size_t)b * m.heads + g * groups + r) * max_slices;
    float top = -FLT_MAX, total = 0.f;
    for (int s = lane; s < slices; s += 32) top = fmaxf(top, part_max[at + s]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int s = lane; s < slices; s += 32) total += part_sum[at + s] * exp2f(part_max[at + s] - top);
    total = warp_sum(total);
    if (lane == 0) {
      top_of[r] = top;
      inverse_of[r] = total == 0.f ? 0.f : 1.f / total;          // NaN for all keys of a row whose sum is NaN
    }
  }
  __syncthreads();
  const int j0 = key0 + threadIdx.x * 4;
  if (j0 >= last) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  const float* from = scores + ((size_t)b * m.heads + g * groups) * span + j0;
  for (int r = 0; r < groups; ++r) {
    const float4 s = *(const float4*)(from + (size_t)r * span);
    const float top = top_of[r], inverse = inverse_of[r];
    w[0] += exp2f(s.x - top) * inverse;
    w[1] += exp2f(s.y - top) * inverse;
    w[2] += exp2f(s.z - top) * inverse;
    w[3] += exp2f(s.w - top) * inverse;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = j0 + i;
    if (j < m.keep_first || j >= last) continue;
    add_mass(m, b, g, j, j == n_kv - 1, w[i]);
  }
}

// Blocks 0 .. heads - 1 of a request merge the slices of a head; the others add the weights of a chunk of one kv head's keys.

template <int D, int DEPTH>
__global__ void __launch_bounds__(MERGE_WARPS * 32) mass_merge_kernel(__nv_bfloat16* __restrict__ out, const DecodeParams p, const MassParams m,
                                                                      const float* __restrict__ scores, int span, int chunks) {
  dependent_launch_trigger();
  extern __shared__ float weights[];     // [max_slices], then [MERGE_WARPS][D]
  __shared__ float top_of[16], inverse_of[16];
  const int b = blockIdx.y;
  const int token = p.q_start[b], n_kv = p.kv_len[b];
  const bool single = p.q_start[b + 1] - token == 1;
  dependent_launch_wait();
  if (!single) return;
  const int slices = min(p.max_slices, (n_kv + p.slice_keys - 1) / p.slice_keys);
  if ((int)blockIdx.x < p.heads) {
    const int h = blockIdx.x;
    const size_t at = ((size_t)b * p.heads + h) * p.max_slices;
    merge_parts<D, DEPTH>(out + ((size_t)token * p.heads + h) * D, p.part_out + at * D, p.part_max + at, p.part_sum + at, slices, p.max_slices, weights);
    return;
  }
  add_chunk(m, p.part_max, p.part_sum, scores, b, ((int)blockIdx.x - p.heads) / chunks, (((int)blockIdx.x - p.heads) % chunks) * MASS_CHUNK, token, n_kv, slices,
            p.slice_keys, p.max_slices, span, top_of, inverse_of);
}

// ---------------------------------------------------------------------------------------
// single tokens, any type
// ---------------------------------------------------------------------------------------
constexpr int ANY_KEYS = 64;
constexpr int ANY_THREADS = 128;
constexpr int AT_ONCE = 8;               // pieces of keys and of values that a thread asks for before it waits for any
constexpr int ANY_ROWS = 16;

template <typename T>
struct AnyParams {
  MassParams m;
  const T* qkv;
  const T* keys;
  const T* values;
  T* out;
  float* scores;                // [requests, heads, span]
  float* part_out;              // [requests, heads, slices, d]
  float* part_max;
  float* part_sum;
  int d, slice_keys, max_slices, span;
  float scale_log2;
};

// Four neighbouring elements as float32 (a row starts on a multiple of four elements).
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

template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) any_slices_kernel(const AnyParams<T> p) {
  extern __shared__ __align__(16) float any_smem[];
  __shared__ float weight[ANY_KEYS][ANY_ROWS], top_of[ANY_ROWS], sum_of[ANY_ROWS], shrink_of[ANY_ROWS];
  dependent_launch_prologue();
  const int slice = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int token = p.m.q_start[b], n = p.m.kv_len[b], begin = slice * p.slice_keys, end = min(n, begin + p.slice_keys);
  if (p.m.q_start[b + 1] - token != 1 || begin >= end) return;
  const int groups = p.m.heads / p.m.kv_heads, units = p.d / 4, stride = p.d + 4, tid = threadIdx.x;
  float* q = any_smem;                                   // [groups][d]
  float* k = q + ANY_ROWS * p.d;                         // [ANY_KEYS][stride]: a quarter-warp's 16-byte reads of eight rows fall into different banks
  float* v = k + ANY_KEYS * stride;                      // [ANY_KEYS][d]
  const T* query = p.qkv + (size_t)token * (p.m.heads + 2 * p.m.kv_heads) * p.d + (size_t)g * groups * p.d;
  for (int i = tid; i < groups * units; i += ANY_THREADS) *(float4*)(q + i * 4) = load4(query + i * 4);
  if (tid < ANY_ROWS) {
    top_of[tid] = -FLT_MAX;
    sum_of[tid] = 0.f;
  }
  const int key = tid % ANY_KEYS, half = tid / ANY_KEYS;
  const int shares = ANY_THREADS / units, unit = tid % units, share = tid / units;      // threads behind the last share have no part in the output
  float4 acc[ANY_ROWS];
#pragma unroll
  for (int r = 0; r < ANY_ROWS; ++r) acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  float* row_scores = p.scores + ((size_t)b * p.m.heads + g * groups) * p.span;
  for (int key0 = begin; key0 < end; key0 += ANY_KEYS) {
    const int count = min(ANY_KEYS, end - key0);
    __syncthreads();                                     // the tile before is read
    for (int i0 = tid; i0 < ANY_KEYS * units; i0 += ANY_THREADS * AT_ONCE) {
      float4 kv[AT_ONCE], vv[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * ANY_THREADS, row = i / units, c = (i % units) * 4;
        kv[u] = vv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < count) {
          const int j = key0 + row, page = checked_page(p.m.block_table[(size_t)b * p.m.table_width + checked_table_index(j / p.m.page_size, p.m.table_width)]);
          const size_t at = (((size_t)page * p.m.kv_heads + g) * p.m.page_size + j % p.m.page_size) * p.d + c;
          kv[u] = load4(p.keys + at);
          vv[u] = load4(p.values + at);
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * ANY_THREADS, row = i / units, c = (i % units) * 4;
        if (row < ANY_KEYS) {
          *(float4*)(k + row * stride + c) = kv[u];
          *(float4*)(v + row * p.d + c) = vv[u];
        }
      }
    }
    __syncthreads();
    {
      float s[ANY_ROWS / 2];                             // of the key with rows half, half + 2, ...
#pragma unroll
      for (int i = 0; i < ANY_ROWS / 2; ++i) s[i] = 0.f;
      for (int c = 0; c < p.d; c += 4) {
        const float4 kv = *(const float4*)(k + key * stride + c);
#pragma unroll
        for (int i = 0; i < ANY_ROWS / 2; ++i)
          if (half + 2 * i < groups) {
            const float4 qv = *(const float4*)(q + (half + 2 * i) * p.d + c);
            s[i] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, s[i]))));
          }
      }
#pragma unroll
      for (int i = 0; i < ANY_ROWS / 2; ++i)
        if (half + 2 * i < groups) {
          const float score = key < count ? s[i] * p.scale_log2 : -FLT_MAX;
          weight[key][half + 2 * i] = score;
          if (key < count) row_scores[(size_t)(half + 2 * i) * p.span + key0 + key] = score;
        }
    }
    __syncthreads();
    // A warp per row: the running maximum and sum, and the scores become weights.
    for (int r = tid >> 5; r < groups; r += ANY_THREADS / 32) {
      const int lane = tid & 31;
      const float s0 = weight[lane][r], s1 = weight[lane + 32][r];
      float top = fmaxf(s0, s1);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float before = top_of[r], higher = fmaxf(before, top);
      const float e0 = lane < count ? exp2f(s0 - higher) : 0.f, e1 = lane + 32 < count ? exp2f(s1 - higher) : 0.f;
      weight[lane][r] = e0;
      weight[lane + 32][r] = e1;
      const float sum = warp_sum(e0 + e1);
      __syncwarp();
      if (lane == 0) {
        const float shrink = before == -FLT_MAX ? 0.f : exp2f(before - higher);
        sum_of[r] = sum_of[r] * shrink + sum;
        top_of[r] = higher;
        shrink_of[r] = shrink;
      }
    }
    __syncthreads();
    if (share < shares) {
#pragma unroll
      for (int r = 0; r < ANY_ROWS; ++r)
        if (r < groups) {
          const float shrink = shrink_of[r];
          acc[r].x *= shrink;
          acc[r].y *= shrink;
          acc[r].z *= shrink;
          acc[r].w *= shrink;
        }
      for (int j = share; j < count; j += shares) {
        const float4 vv = *(const float4*)(v + j * p.d + unit * 4);
#pragma unroll
        for (int r = 0; r < ANY_ROWS; r += 4)
          if (r < groups) {
            const float4 w = *(const float4*)&weight[j][r];
            fma4(acc[r], w.x, vv);
            if (r + 1 < groups) fma4(acc[r + 1], w.y, vv);
            if (r + 2 < groups) fma4(acc[r + 2], w.z, vv);
            if (r + 3 < groups) fma4(acc[r + 3], w.w, vv);
          }
      }
    }
  }
  // ---- the shares of the keys, added in their order, over the tiles' memory
  __syncthreads();
  float* sums = k;                                       // [shares][groups][d]
  if (share < shares) {
#pragma unroll
    for (int r = 0; r < ANY_ROWS; ++r)
      if (r < groups) *(float4*)(sums + ((size_t)share * groups + r) * p.d + unit * 4) = acc[r];
  }
  __syncthreads();
  const size_t first = ((size_t)b * p.m.heads + g * groups) * p.max_slices + slice;
  for (int i = tid; i < groups * units; i += ANY_THREADS) {
    const int r = i / units, c = (i % units) * 4;
    float4 total = *(const float4*)(sums + r * p.d + c);
    for (int s = 1; s < shares; ++s) fma4(total, 1.f, *(const float4*)(sums + ((size_t)s * groups + r) * p.d + c));
    *(float4*)(p.part_out + (first + (size_t)r * p.max_slices) * p.d + c) = total;
  }
  if (tid < groups) {
    p.part_max[first + (size_t)tid * p.max_slices] = top_of[tid];
    p.part_sum[first + (size_t)tid * p.max_slices] = sum_of[tid];
  }
}

template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) any_merge_kernel(const AnyParams<T> p, int chunks) {
  __shared__ float top_of[ANY_ROWS], inverse_of[ANY_ROWS];
  dependent_launch_prologue();
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int token = p.m.q_start[b], n = p.m.kv_len[b];
  if (p.m.q_start[b + 1] - token != 1) return;
  const int slices = min(p.max_slices, (n + p.slice_keys - 1) / p.slice_keys);
  if ((int)blockIdx.x >= p.m.heads) {
    add_chunk(p.m, p.part_max, p.part_sum, p.scores, b, ((int)blockIdx.x - p.m.heads) / chunks, (((int)blockIdx.x - p.m.heads) % chunks) * MASS_CHUNK, token, n, slices,
              p.slice_keys, p.max_slices, p.span, top_of, inverse_of);
    return;
  }
  const size_t at = ((size_t)b * p.m.heads + blockIdx.x) * p.max_slices;
  float top = -FLT_MAX, total = 0.f;
  for (int s = lane; s < slices; s += 32) top = fmaxf(top, p.part_max[at + s]);           // every warp works them out for itself
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  for (int s = lane; s < slices; s += 32) total += p.part_sum[at + s] * exp2f(p.part_max[at + s] - top);
  total = warp_sum(total);
  const float inverse = total > 0.f ? 1.f / total : 0.f;
  for (int c = tid; c < p.d; c += ANY_THREADS) {
    float sum = 0.f;
#pragma unroll 8
    for (int s = 0; s < slices; ++s) sum = fmaf(exp2f(p.part_max[at + s] - top), p.part_out[(at + s) * p.d + c], sum);
    p.out[((size_t)token * p.m.heads + blockIdx.x) * p.d + c] = from_float<T>(sum * inverse);
  }
}

// ---------------------------------------------------------------------------------------
// every other step
// ---------------------------------------------------------------------------------------
// Tiles of 16 rows (token, head of a kv head) x 64 keys; a thread has one key and eight of the rows.
constexpr int ROWS = 16;
constexpr int MOST_RUNS = 16;            // of keys, that a request's maxima and sums are taken over

template <typename T>
struct RowParams {
  MassParams m;
  const T* qkv;                 // [tokens, (heads + 2 kv_heads) * d]
  const T* keys;                // [pages, kv_heads, page_size, d]
  const int* q_pos0;
  float* part_max;              // [runs, tokens * heads], in units of log2
  float* part_sum;
  float* part;                  // [chunks, requests, kv_heads, span]
  int d, runs, run_keys, row_tiles, chunk_tiles, span, seqs;
  long long rows;               // tokens * heads
  float scale_log2;
};

// Rows 0 .. rows - 1 of a tile, row r from row_ptr(r) (null: zeros), `stride` floats each.
template <typename T, typename RowPtr>
__device__ __forceinline__ void load_tile(float* tile, int rows, int d, int stride, RowPtr row_ptr) {
  const int units = d / 4;
  for (int i0 = threadIdx.x; i0 < rows * units; i0 += ANY_THREADS * AT_ONCE) {
    float4 v[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * ANY_THREADS;
      const T* from = i < rows * units ? row_ptr(i / units) : nullptr;
      v[u] = from != nullptr ? load4(from + (i % units) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u * ANY_THREADS;
      if (i < rows * units) *(float4*)(tile + (i / units) * stride + (i % units) * 4) = v[u];
    }
  }
}

// The scores of this thread's key with rows half, half + 2, ... of the tile, scaled, in units of log2.
__device__ __forceinline__ void eight_scores(float (&s)[ROWS / 2], const float* q_tile, const float* k_tile, int d, int stride, float scale_log2) {
  const float* k = k_tile + (threadIdx.x % ANY_KEYS) * stride;
  const float* q = q_tile + (threadIdx.x / ANY_KEYS) * stride;
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) s[i] = 0.f;
  for (int c = 0; c < d; c += 4) {
    const float4 kv = *(const float4*)(k + c);
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i) {
      const float4 qv = *(const float4*)(q + 2 * i * stride + c);
      s[i] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, s[i]))));
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) s[i] *= scale_log2;
}

template <typename T>
__device__ __forceinline__ const T* key_row(const RowParams<T>& p, int b, int g, int j) {
  const int page = checked_page(p.m.block_table[(size_t)b * p.m.table_width + checked_table_index(j / p.m.page_size, p.m.table_width)]);
  return p.keys + (((size_t)page * p.m.kv_heads + g) * p.m.page_size + j % p.m.page_size) * p.d;
}
template <typename T>
__device__ __forceinline__ const T* query_row(const RowParams<T>& p, int token0, int g, int groups, int i) {
  return p.qkv + ((size_t)(token0 + i / groups) * (p.m.heads + 2 * p.m.kv_heads) + g * groups + i % groups) * p.d;
}
// How many keys some row of the tile that begins with row0 sees.
__device__ __forceinline__ int seen_by(int row0, int count, int groups, int pos0, int n) { return min(n, pos0 + (min(row0 + ROWS, count) - 1) / groups + 1); }

template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) row_stats_kernel(const RowParams<T> p) {
  extern __shared__ __align__(16) float shared[];
  __shared__ float tops[2][2][ROWS / 2], sums[2][2][ROWS / 2];       // [half of the keys][parity of the row][row / 2]
  dependent_launch_prologue();
  const int tile = blockIdx.x % p.row_tiles, run = blockIdx.x / p.row_tiles, g = blockIdx.y, b = blockIdx.z;
  const int groups = p.m.heads / p.m.kv_heads, token0 = p.m.q_start[b];
  const int count = (p.m.q_start[b + 1] - token0) * groups;
  const int row0 = tile * ROWS;
  if (row0 >= count || pads(p.m, token0)) return;
  const int pos0 = p.q_pos0[b], visible = seen_by(row0, count, groups, pos0, p.m.kv_len[b]);
  const int begin = run * p.run_keys, end = min(visible, begin + p.run_keys);
  const int stride = p.d + 4, key = threadIdx.x % ANY_KEYS, half = threadIdx.x / ANY_KEYS, lane = threadIdx.x & 31;
  float* q_tile = shared;
  float* k_tile = shared + ROWS * stride;
  load_tile<T>(q_tile, ROWS, p.d, stride, [&](int r) -> const T* { return row0 + r < count ? query_row(p, token0, g, groups, row0 + r) : nullptr; });
  float top[ROWS / 2], sum[ROWS / 2];
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    top[i] = -FLT_MAX;
    sum[i] = 0.f;
  }
  for (int key0 = begin; key0 < end; key0 += ANY_KEYS) {
    __syncthreads();
    load_tile<T>(k_tile, ANY_KEYS, p.d, stride, [&](int r) -> const T* { return key0 + r < end ? key_row(p, b, g, key0 + r) : nullptr; });
    __syncthreads();
    float s[ROWS / 2];
    eight_scores(s, q_tile, k_tile, p.d, stride, p.scale_log2);
    const int j = key0 + key;
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i) {
      if (j >= end || j > pos0 + (row0 + half + 2 * i) / groups) continue;
      const float higher = fmaxf(top[i], s[i]);
      sum[i] = (top[i] == -FLT_MAX ? sum[i] : sum[i] * exp2f(top[i] - higher)) + exp2f(s[i] - higher);
      top[i] = higher;
    }
  }
  const int part = key / 32;                 // this warp's half of the tile's keys
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    float both = top[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) both = fmaxf(both, __shfl_xor_sync(0xffffffffu, both, o));
    const float total = warp_sum(top[i] == -FLT_MAX ? sum[i] : sum[i] * exp2f(top[i] - both));
    if (lane == 0) {
      tops[part][half][i] = both;
      sums[part][half][i] = total;
    }
  }
  __syncthreads();
  const int r = threadIdx.x;
  if (r < ROWS && row0 + r < count) {
    const float a = tops[0][r & 1][r >> 1], c = tops[1][r & 1][r >> 1], both = fmaxf(a, c);
    const float total = (a == -FLT_MAX ? sums[0][r & 1][r >> 1] : sums[0][r & 1][r >> 1] * exp2f(a - both)) +
                        (c == -FLT_MAX ? sums[1][r & 1][r >> 1] : sums[1][r & 1][r >> 1] * exp2f(c - both));
    const int i = row0 + r;
    const size_t at = (size_t)run * p.rows + (size_t)(token0 + i / groups) * p.m.heads + g * groups + i % groups;
    p.part_max[at] = both;
    p.part_sum[at] = total;
  }
}

// Which row tiles a block of any_column_sums_kernel takes: those of its chunk that see its keys. Empty: first >= last.
struct ChunkTiles {
  int first, last, pos0, tokens, n;
};
template <typename T>
__device__ __forceinline__ ChunkTiles chunk_tiles(const RowParams<T>& p, int b, int key0, int chunk) {
  ChunkTiles t;
  const int groups = p.m.heads / p.m.kv_heads, token0 = p.m.q_start[b];
  t.tokens = p.m.q_start[b + 1] - token0;
  t.pos0 = p.q_pos0[b];
  t.n = min(p.m.kv_len[b], t.pos0 + t.tokens);
  const int all = (t.tokens * groups + ROWS - 1) / ROWS;
  t.first = max(chunk * p.chunk_tiles, max(0, key0 - t.pos0) * groups / ROWS);
  t.last = min((chunk + 1) * p.chunk_tiles, all);
  if (t.tokens < 1 || key0 >= t.n || key0 + ANY_KEYS <= p.m.keep_first || pads(p.m, token0)) t.last = t.first;
  return t;
}

template <typename T>
__global__ void __launch_bounds__(ANY_THREADS) any_column_sums_kernel(const RowParams<T> p) {
  extern __shared__ __align__(16) float shared[];
  __shared__ float logarithm[ROWS], halves[ANY_KEYS];
  dependent_launch_prologue();
  const int g = blockIdx.y % p.m.kv_heads, chunk = blockIdx.y / p.m.kv_heads, b = blockIdx.z, key0 = blockIdx.x * ANY_KEYS;
  const ChunkTiles tiles = chunk_tiles(p, b, key0, chunk);
  if (tiles.first >= tiles.last) return;
  const int groups = p.m.heads / p.m.kv_heads, token0 = p.m.q_start[b], count = tiles.tokens * groups;
  const int stride = p.d + 4, key = threadIdx.x % ANY_KEYS, half = threadIdx.x / ANY_KEYS, j = key0 + key;
  float* q_tile = shared;
  float* k_tile = shared + ROWS * stride;
  load_tile<T>(k_tile, ANY_KEYS, p.d, stride, [&](int r) -> const T* { return key0 + r < tiles.n ? key_row(p, b, g, key0 + r) : nullptr; });
  float sum = 0.f;
  for (int tile = tiles.first; tile < tiles.last; ++tile) {
    const int row0 = tile * ROWS;
    __syncthreads();
    load_tile<T>(q_tile, ROWS, p.d, stride, [&](int r) -> const T* { return row0 + r < count ? query_row(p, token0, g, groups, row0 + r) : nullptr; });
    if (threadIdx.x < ROWS && row0 + (int)threadIdx.x < count) {
      const int i = row0 + threadIdx.x;
      const size_t at = (size_t)(token0 + i / groups) * p.m.heads + g * groups + i % groups;
      const int runs = min(p.runs, (seen_by(row0, count, groups, tiles.pos0, p.m.kv_len[b]) + p.run_keys - 1) / p.run_keys);      // only these left something
      float top = -FLT_MAX, total = 0.f;
      for (int k = 0; k < runs; ++k) top = fmaxf(top, p.part_max[(size_t)k * p.rows + at]);
      for (int k = 0; k < runs; ++k) total += p.part_sum[(size_t)k * p.rows + at] * exp2f(p.part_max[(size_t)k * p.rows + at] - top);
      logarithm[threadIdx.x] = total == 0.f ? INFINITY : top + log2f(total);
    }
    __syncthreads();
    float s[ROWS / 2];
    eight_scores(s, q_tile, k_tile, p.d, stride, p.scale_log2);
#pragma unroll
    for (int i = 0; i < ROWS / 2; ++i) {
      const int r = row0 + half + 2 * i;
      if (r < count && j <= tiles.pos0 + r / groups) sum += exp2f(s[i] - logarithm[half + 2 * i]);
    }
  }
  if (half == 1) halves[key] = sum;
  __syncthreads();
  if (half == 0 && j < p.span) p.part[(((size_t)chunk * p.seqs + b) * p.m.kv_heads + g) * p.span + j] = sum + halves[key];
}

// The chunks' sums in their order, into the mass.
template <typename T>
__global__ void __launch_bounds__(ANY_KEYS) add_chunks_kernel(const RowParams<T> p, int chunks) {
  dependent_launch_prologue();
  const int g = blockIdx.y, b = blockIdx.z, key0 = blockIdx.x * ANY_KEYS, j = key0 + threadIdx.x;
  ChunkTiles tiles = chunk_tiles(p, b, key0, 0);
  if (j < p.m.keep_first || j >= min(tiles.n, p.span) || tiles.tokens < 1 || pads(p.m, p.m.q_start[b])) return;
  float w = 0.f;
  for (int c = 0; c < chunks; ++c) {
    tiles = chunk_tiles(p, b, key0, c);
    if (tiles.first < tiles.last) w += p.part[(((size_t)c * p.seqs + b) * p.m.kv_heads + g) * p.span + j];
  }
  add_mass(p.m, b, g, j, j >= tiles.pos0, w);
}

template <int D>
int launch_decode_mass(const DecodeParams& p, const MassParams& m, __nv_bfloat16* out, float* scores, int span, int seqs, cudaStream_t s) {
  const size_t bytes = slices_smem_bytes(D);
  if (int err = allow_smem(mass_slices_kernel<D>, bytes, "paged_attention_mass")) return err;
  launch_kernel(mass_slices_kernel<D>, dim3((p.max_slices + SLICE_WARPS - 1) / SLICE_WARPS, p.kv_heads, seqs), dim3(SLICE_WARPS * 32), bytes, s, p, scores, span);
  if (int err = check_launch("paged_attention_mass")) return err;
  const int chunks = (span + MASS_CHUNK - 1) / MASS_CHUNK;
  const auto merge = merge_in_few_registers(p.heads, seqs, p.max_slices) ? mass_merge_kernel<D, 8> : mass_merge_kernel<D, MERGE_DEPTH>;
  launch_kernel(merge, dim3(p.heads + p.kv_heads * chunks, seqs), dim3(MERGE_WARPS * 32), (p.max_slices + MERGE_WARPS * D) * sizeof(float), s, out, p, m, scores,
                span, chunks);
  return check_launch("paged_attention_mass");
}

// How a step's rows and keys are cut: the stats into runs of keys, the columns into chunks of rows, until some 600 blocks are there.
struct RowCut {
  int row_tiles, runs, run_keys, chunk_tiles, chunks;
};
RowCut cut_rows(int seqs, int heads, int kv_heads, int max_q_len, int max_kv_len) {
  RowCut c;
  const long long pairs = (long long)seqs * kv_heads;
  const int key_tiles = (max_kv_len + ANY_KEYS - 1) / ANY_KEYS;
  c.row_tiles = (int)(((long long)max_q_len * (heads / kv_heads) + ROWS - 1) / ROWS);
  long long runs = 592 / (pairs * c.row_tiles), chunks = 592 / (pairs * key_tiles);
  if (runs > MOST_RUNS) runs = MOST_RUNS;
  if (runs > key_tiles) runs = key_tiles;
  if (runs < 1) runs = 1;
  c.run_keys = (int)((key_tiles + runs - 1) / runs) * ANY_KEYS;
  c.runs = (max_kv_len + c.run_keys - 1) / c.run_keys;
  if (chunks > (c.row_tiles + 1) / 2) chunks = (c.row_tiles + 1) / 2;
  if (chunks < 1) chunks = 1;
  c.chunk_tiles = (int)((c.row_tiles + chunks - 1) / chunks);
  c.chunks = (c.row_tiles + c.chunk_tiles - 1) / c.chunk_tiles;
  return c;
}

template <typename T>
int launch_rows(RowParams<T> p, const RowCut& c, int max_kv_len, cudaStream_t s) {
  const size_t bytes = (size_t)(ROWS + ANY_KEYS) * (p.d + 4) * sizeof(float);
  static DevicesSet stats_devices, column_devices;
  if (int err = raise_shared_memory(stats_devices, row_stats_kernel<T>, (ROWS + ANY_KEYS) * 260 * sizeof(float), "attention_mass")) return err;
  if (int err = raise_shared_memory(column_devices, any_column_sums_kernel<T>, (ROWS + ANY_KEYS) * 260 * sizeof(float), "attention_mass")) return err;
  const int key_tiles = (max_kv_len + ANY_KEYS - 1) / ANY_KEYS;
  launch_kernel(row_stats_kernel<T>, dim3(c.row_tiles * c.runs, p.m.kv_heads, p.seqs), dim3(ANY_THREADS), bytes, s, p);
  if (int err = check_launch("attention_mass")) return err;
  launch_kernel(any_column_sums_kernel<T>, dim3(key_tiles, p.m.kv_heads * c.chunks, p.seqs), dim3(ANY_THREADS), bytes, s, p);
  if (int err = check_launch("attention_mass")) return err;
  launch_kernel(add_chunks_kernel<T>, dim3(key_tiles, p.m.kv_heads, p.seqs), dim3(ANY_KEYS), 0, s, p, c.chunks);
  return check_launch("attention_mass");
}

template <typename T>
int launch_any(AnyParams<T> p, int seqs, cudaStream_t s) {
  const int groups = p.m.heads / p.m.kv_heads;
  size_t tiles = (size_t)ANY_KEYS * (2 * p.d + 4), shares = (size_t)(ANY_THREADS / (p.d / 4)) * groups * p.d;
  const size_t bytes = ((size_t)ANY_ROWS * p.d + (tiles > shares ? tiles : shares)) * sizeof(float);
  static DevicesSet devices;
  if (int err = raise_shared_memory(devices, any_slices_kernel<T>, 160 * 1024, "paged_attention_mass")) return err;
  launch_kernel(any_slices_kernel<T>, dim3(p.max_slices, p.m.kv_heads, seqs), dim3(ANY_THREADS), bytes, s, p);
  if (int err = check_launch("paged_attention_mass")) return err;
  const int chunks = (p.span + MASS_CHUNK - 1) / MASS_CHUNK;
  launch_kernel(any_merge_kernel<T>, dim3(p.m.heads + p.m.kv_heads * chunks, seqs), dim3(ANY_THREADS), 0, s, p, chunks);
  return check_launch("paged_attention_mass");
}

}  // namespace

PAE_DEFINE_LAST_ERROR()

// mass of this step's keys = 0, of requests whose first slot is not negative (slots null: of all).
PAE_EXPORT int pae_start_mass(float* mass, const int* block_table, int table_width, const int* q_start, const int* q_pos0, const int* kv_len, const int* slots, int seqs,
                              int kv_heads, int page_size, void* stream) {
  if (seqs < 1) return 0;
  const MassParams m = {mass, block_table, q_start, kv_len, slots, table_width, kv_heads, kv_heads, page_size, 0};
  launch_kernel(start_keys_kernel, dim3(seqs), dim3(128), 0, (cudaStream_t)stream, m, q_pos0);
  return check_launch("start_mass");
}

// Floats of scratch for a step of single tokens in bfloat16, cut into slices (as pae_paged_attention_decode).
PAE_EXPORT long long pae_decode_mass_floats(int seqs, int heads, int d, int slice_keys, int max_slices) {
  return decode_scratch_floats(seqs, heads, d, max_slices) + (long long)seqs * heads * slice_keys * max_slices;
}

// Requests that bring exactly one token: out as pae_paged_attention_decode without a window, and the weights of their keys. Others are skipped.
PAE_EXPORT int pae_paged_attention_decode_mass(void* out, const void* qkv, const void* keys, const void* values, float* mass, const int* block_table,
                                               int table_width, const int* q_start, const int* kv_len, const int* slots, int seqs, int heads, int kv_heads,
                                               int d, int page_size, float scale, int keep_first, int slice_keys, int max_slices, float* scratch,
                                               void* stream) {
  if (seqs == 0) return 0;
  if (int err = check_sizes("paged_attention_mass", heads, kv_heads, d, page_size, seqs)) return err;
  if (heads / kv_heads > 16) return fail(2, "paged_attention_mass: %d query heads per kv head are more than 16", heads / kv_heads);
  if (slice_keys < 16 || slice_keys % 16 || max_slices < 1) return fail(2, "paged_attention_mass: slices of %d keys x %d", slice_keys, max_slices);
  if ((size_t)(max_slices + MERGE_WARPS * d) * sizeof(float) > 40 * 1024) return fail(2, "paged_attention_mass: %d slices are more than the merge takes", max_slices);
  if ((uintptr_t)scratch & 15) return fail(2, "paged_attention_mass: the scratch does not start on a 16-byte boundary");
  DecodeParams p{};
  p.qkv = (const __nv_bfloat16*)qkv;
  p.keys = (const __nv_bfloat16*)keys;
  p.values = (const __nv_bfloat16*)values;
  p.block_table = block_table;
  p.q_start = q_start;
  p.kv_len = kv_len;
  const size_t rows = (size_t)seqs * heads * max_slices;
  const int span = slice_keys * max_slices;
  float* scores = scratch;                                       // rows of a multiple of 16 floats: aligned
  p.part_out = scratch + (size_t)seqs * heads * span;
  p.part_max = p.part_out + rows * d;
  p.part_sum = p.part_max + rows;
  p.table_width = table_width;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.slice_keys = slice_keys;
  p.max_slices = max_slices;
  p.scale_log2 = scale * LOG2E;
  const MassParams m = {mass, block_table, q_start, kv_len, slots, table_width, heads, kv_heads, page_size, keep_first};
  const cudaStream_t s = (cudaStream_t)stream;
  if (d == 32) return launch_decode_mass<32>(p, m, (__nv_bfloat16*)out, scores, span, seqs, s);
  if (d == 64) return launch_decode_mass<64>(p, m, (__nv_bfloat16*)out, scores, span, seqs, s);
  return launch_decode_mass<128>(p, m, (__nv_bfloat16*)out, scores, span, seqs, s);
}

// Steps of single tokens on CUDA cores (dtype 0 float32, 1 bfloat16): out and weights; requests of several tokens are skipped. `slice_keys` is a
// multiple of 64; scratch as pae_decode_mass_floats.
PAE_EXPORT int pae_paged_attention_any_mass(void* out, const void* qkv, const void* keys, const void* values, float* mass, const int* block_table, int table_width,
                                            const int* q_start, const int* kv_len, const int* slots, int seqs, int heads, int kv_heads, int d, int page_size,
                                            float scale, int keep_first, int slice_keys, int max_slices, int dtype, float* scratch, void* stream) {
  if (seqs == 0) return 0;
  if (d < 4 || d > 256 || d % 4) return fail(2, "paged_attention_mass: head_dim %d is not a multiple of 4 up to 256", d);
  if (kv_heads < 1 || heads % kv_heads || heads / kv_heads > ANY_ROWS) return fail(2, "paged_attention_mass: %d heads over %d kv heads", heads, kv_heads);
  if (slice_keys < ANY_KEYS || slice_keys % ANY_KEYS || max_slices < 1) return fail(2, "paged_attention_mass: slices of %d keys x %d", slice_keys, max_slices);
  if (kv_heads > 65535 || seqs > 65535) return fail(1, "paged_attention_mass: %d requests of %d kv heads, at most 65535 of each", seqs, kv_heads);
  const int align = dtype == kF32 ? 15 : 7;
  if ((((uintptr_t)qkv | (uintptr_t)keys | (uintptr_t)values) & align) || ((uintptr_t)scratch & 15))
    return fail(2, "paged_attention_mass: an operand does not start on a boundary of four elements");
  const MassParams m = {mass, block_table, q_start, kv_len, slots, table_width, heads, kv_heads, page_size, keep_first};
  const int span = slice_keys * max_slices;
  const size_t rows = (size_t)seqs * heads * max_slices;
  float* scores = scratch;
  float* part_out = scratch + (size_t)seqs * heads * span;
  const float scale_log2 = scale * LOG2E;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == kF32)
    return launch_any<float>({m, (const float*)qkv, (const float*)keys, (const float*)values, (float*)out, scores, part_out, part_out + rows * d,
                              part_out + rows * (d + 1), d, slice_keys, max_slices, span, scale_log2}, seqs, s);
  return launch_any<__nv_bfloat16>({m, (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)keys, (const __nv_bfloat16*)values, (__nv_bfloat16*)out, scores, part_out,
                                    part_out + rows * d, part_out + rows * (d + 1), d, slice_keys, max_slices, span, scale_log2}, seqs, s);
}

// Floats of scratch for pae_attention_mass_rows.
PAE_EXPORT long long pae_attention_mass_floats(int tokens, int seqs, int heads, int kv_heads, int max_q_len, int max_kv_len) {
  if (seqs < 1 || max_q_len < 1 || max_kv_len < 1) return 1;
  const RowCut c = cut_rows(seqs, heads, kv_heads, max_q_len, max_kv_len);
  return 2ll * c.runs * tokens * heads + (long long)c.chunks * seqs * kv_heads * max_kv_len;
}

// The weights of any step's keys, whatever its rows, type (0 float32, 1 bfloat16) and head size (a multiple of 4 up to 256); the attention's output is not computed.
PAE_EXPORT int pae_attention_mass_rows(float* mass, const void* qkv, const void* keys, const int* block_table, int table_width, const int* q_start,
                                       const int* q_pos0, const int* kv_len, const int* slots, int tokens, int seqs, int max_q_len, int max_kv_len, int heads,
                                       int kv_heads, int d, int page_size, float scale, int keep_first, int dtype, float* scratch, void* stream) {
  if (seqs < 1 || tokens < 1 || max_q_len < 1 || max_kv_len < 1) return 0;
  if (d < 4 || d > 256 || d % 4) return fail(2, "paged_attention_mass: head_dim %d is not a multiple of 4 up to 256", d);
  if (((uintptr_t)qkv | (uintptr_t)keys) & (dtype == kF32 ? 15 : 7)) return fail(2, "paged_attention_mass: an operand does not start on a boundary of four elements");
  const RowCut c = cut_rows(seqs, heads, kv_heads, max_q_len, max_kv_len);
  if ((long long)kv_heads * c.chunks > 65535 || seqs > 65535 || (long long)c.row_tiles * c.runs > 0x7fffffffll)
    return fail(1, "paged_attention_mass: %d requests of %d kv heads x %d chunks exceed one launch", seqs, kv_heads, c.chunks);
  const MassParams m = {mass, block_table, q_start, kv_len, slots, table_width, heads, kv_heads, page_size, keep_first};
  const long long rows = (long long)tokens * heads;
  float* part_sum = scratch + c.runs * rows;
  float* part = part_sum + c.runs * rows;
  const float scale_log2 = scale * LOG2E;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == kF32)
    return launch_rows<float>({m, (const float*)qkv, (const float*)keys, q_pos0, scratch, part_sum, part, d, c.runs, c.run_keys, c.row_tiles, c.chunk_tiles, max_kv_len, seqs,
                               rows, scale_log2}, c, max_kv_len, s);
  return launch_rows<__nv_bfloat16>({m, (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)keys, q_pos0, scratch, part_sum, part, d, c.runs, c.run_keys, c.row_tiles,
                                     c.chunk_tiles, max_kv_len, seqs, rows, scale_log2}, c, max_kv_len, s);
}
