// What the attention kernels on tcgen05 share beside tcgen05.cuh: tiles of keys and values straight from the pages of the cache by TMA,
// the second product's operands (values as they lie, probabilities in tensor memory), and loads and stores of tensor memory.
#pragma once

#include <mutex>
#include <unordered_map>

#include "tcgen05.cuh"

namespace pae_tcgen05 {

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A box of keys or values: coordinates in a pool seen as [pages][kv heads][D / 64][rows of a page][64].
__device__ __forceinline__ void tma_load_pages(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int half, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(row), "r"(half), "r"(head), "r"(page)
      : "memory");
}
// How keys and values come into shared memory. What the TMA unit takes is time per box, not bytes: with a box a page and half of
// a row, 16 boxes of 2 KB for 64 keys of a page size of 16, it set the pace of the paired kernel (8,192 tokens, 12 heads of 128: 235 us against
// 177 with pages of 64; now 173 with either, 1,190 TFLOP/s, and a tenth more where no two pages follow one another). So the pages of a tile that follow one another in the pool, as a prompt's pages mostly do, come as ONE box per half
// of the keys and one of the values; others come a box each (and half, of the keys). The values lie [page][half][row][64] (the
// halves' distance is the descriptor's leading byte offset), the keys [half][page][row][64].
struct PageMaps {
  CUtensorMap key, value;                // a page (or the rows of it that a tile covers)
  CUtensorMap key_run, value_run;        // the pages of a tile
};
// Tile of `rows` keys, `rows_a_box` of them a box, by a converged warp: lane i brings the box at `row` of `page`, or lane 0 all of them.
template <int D>
__device__ __forceinline__ void load_pages(const PageMaps& maps, bool values, uint32_t dst, uint32_t full, int rows, int rows_a_box, int lane, int head,
                                           int page, int row) {
  constexpr int HALVES = D / 64;
  const int boxes = rows / rows_a_box;
  const int first = __shfl_sync(0xffffffffu, page, 0);
  if (boxes > 1 && __all_sync(0xffffffffu, lane >= boxes || page == first + lane)) {
    if (lane == 0) {
      if (values) {
        tma_load_pages(dst, &maps.value_run, full, 0, 0, head, page);
      } else {
#pragma unroll
        for (int half = 0; half < HALVES; ++half) tma_load_pages(dst + half * rows * 128, &maps.key_run, full, 0, half, head, page);
      }
    }
  } else if (lane < boxes) {
    if (values) {
      tma_load_pages(dst + lane * rows_a_box * 128 * HALVES, &maps.value, full, row, 0, head, page);
    } else {
#pragma unroll
      for (int half = 0; half < HALVES; ++half) tma_load_pages(dst + half * rows * 128 + lane * rows_a_box * 128, &maps.key, full, row, half, head, page);
    }
  }
}
// Where the 16 keys of step k of the second product lie among a tile's values (a box has 16, 32, 64 or 128 rows).
template <int D>
__device__ __forceinline__ uint32_t value_step(int k, int rows_a_box) {
  const int row = k * 16;
  return (uint32_t)(row + (D / 64 - 1) * (row & -rows_a_box)) * 128;
}
// Rows `from` .. `rows` - 1 of a tile of values become zeros, by a converged warp, before the tensor core reads them: they lie behind the
// last visible key, and a probability of 0 times what a page holds there is 0 only for a number.
template <int D>
__device__ __forceinline__ void clear_values(uint8_t* tile, int from, int rows, int rows_a_box, int lane) {
  constexpr int CHUNKS = D / 8;
  const int chunk = lane % CHUNKS, in_box = rows_a_box - 1;          // boxes have 16, 32, 64 or 128 rows
  uint8_t* to = tile + chunk / 8 * rows_a_box * 128 + chunk % 8 * 16;
#pragma unroll 4
  for (int row = from + lane / CHUNKS; row < rows; row += 32 / CHUNKS)
    *(uint4*)(to + ((row & ~in_box) * (D / 64) + (row & in_box)) * 128) = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
// 32 consecutive float32 columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tmem_load32(uint32_t address, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// MN-major operand with 128-byte swizzle: a 128-byte row holds 64 consecutive MN elements of
// one K index; 8 consecutive K indices are 8 rows (1024 bytes, the stride byte offset); the
// next 64 MN elements lie `mn_group_bytes` further (the leading byte offset).
__device__ __forceinline__ uint64_t mn_major_descriptor(uint32_t address, uint32_t mn_group_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((address & 0x3FFFFu) >> 4);
  d |= (uint64_t)((mn_group_bytes >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// The descriptor of the place `bytes` (a multiple of 16) further: shared memory ends below 256 KB, so nothing carries out of the address
// field.
__device__ __forceinline__ uint64_t further(uint64_t descriptor, uint32_t bytes) {
  return (descriptor & 0xFFFFFFFF00000000ull) | (uint32_t)((uint32_t)descriptor + (bytes >> 4));
}
// float32 accumulator, bfloat16 operands, A K-major; B K-major or MN-major (bit 16).
__host__ __device__ constexpr uint32_t instruction_descriptor(int m, int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// 64 consecutive float32 columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tmem_load64(uint32_t address, float* v) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(address)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 columns that are there after `tmem_arrived` of the same variables.
__device__ __forceinline__ void tmem_ask32(uint32_t address, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void tmem_arrived(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
// 32 columns written (the whole warp calls it).
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
      "tcgen05.wait::st.sync.aligned;"
      ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]^T: a lane of A is a row, a column holds two neighbouring bfloat16 of K.
__device__ __forceinline__ void umma_bf16_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Two floats side by side: one instruction for both, each rounded as the single one rounds.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// ---------------------------------------------------------------------------------------
// Host side: the maps of a pool
// ---------------------------------------------------------------------------------------
// A pool [pages, kv_heads, page_size, d] as boxes of `rows` rows of `halves` halves of `run` pages, 128-byte swizzle.
inline int page_map(CUtensorMap* out, const void* ptr, long long pages, int kv_heads, int page_size, int d, int rows, int halves, int run) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return fail(101, "paged_attention_tcgen05: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t dims[5] = {64, (cuuint64_t)page_size, (cuuint64_t)(d / 64), (cuuint64_t)kv_heads, (cuuint64_t)pages};
  const cuuint64_t strides[4] = {(cuuint64_t)d * 2, 128, (cuuint64_t)page_size * d * 2, (cuuint64_t)kv_heads * page_size * d * 2};
  const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)halves, 1, (cuuint32_t)run};
  const cuuint32_t element_strides[5] = {1, 1, 1, 1, 1};
  CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(ptr), dims, strides, box, element_strides,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(102, "paged_attention_tcgen05: cuTensorMapEncodeTiled failed with %d for pages of %d", (int)r, page_size);
  return 0;
}
// What brings tiles of `tile_keys` keys.
inline int encode_page_maps(PageMaps* out, const void* keys, const void* values, long long pages, int kv_heads, int page_size, int d, int tile_keys) {
  const int rows = page_size < tile_keys ? page_size : tile_keys, run = tile_keys / rows, halves = d / 64;
  if (int err = page_map(&out->key, keys, pages, kv_heads, page_size, d, rows, 1, 1)) return err;
  if (int err = page_map(&out->value, values, pages, kv_heads, page_size, d, rows, halves, 1)) return err;
  if (int err = page_map(&out->key_run, keys, pages, kv_heads, page_size, d, rows, 1, run)) return err;
  return page_map(&out->value_run, values, pages, kv_heads, page_size, d, rows, halves, run);
}
// The same, kept. A pool's maps say where it lies and how it is laid out, nothing of what it holds; they are kept
// (encoding four takes a microsecond and more of every launch).
struct PageMapsKey {
  const void *keys, *values;
  long long pages;
  int kv_heads, page_size, d, tile_keys;
  bool operator==(const PageMapsKey& o) const {
    return keys == o.keys && values == o.values && pages == o.pages && kv_heads == o.kv_heads && page_size == o.page_size && d == o.d && tile_keys == o.tile_keys;
  }
};
struct PageMapsKeyHash {
  size_t operator()(const PageMapsKey& key) const {
    size_t h = (size_t)key.keys;
    h = h * 1000003u ^ (size_t)key.values;
    h = h * 1000003u ^ (size_t)key.pages;
    h = h * 1000003u ^ (size_t)(key.kv_heads * 4096 + key.page_size);
    return h * 1000003u ^ (size_t)(key.d * 4096 + key.tile_keys);
  }
};
inline int page_maps(PageMaps* out, const void* keys, const void* values, long long pages, int kv_heads, int page_size, int d, int tile_keys) {
  static std::mutex mutex;
  static std::unordered_map<PageMapsKey, PageMaps, PageMapsKeyHash> cache;
  const PageMapsKey key{keys, values, pages, kv_heads, page_size, d, tile_keys};
  std::lock_guard<std::mutex> guard(mutex);
  auto found = cache.find(key);
  if (found != cache.end()) {
    *out = found->second;
    return 0;
  }
  if (int err = encode_page_maps(out, keys, values, pages, kv_heads, page_size, d, tile_keys)) return err;
  if (cache.size() > 1024) cache.clear();
  cache.emplace(key, *out);
  return 0;
}

}  // namespace pae_tcgen05
