// What the kernels of attention over the 8-bit cache share: arguments, conversions, launches.
#pragma once
#include "kv8.cuh"
#include "sm100.cuh"

namespace kv8 {

struct Attn {
  const void* q; long long ldq;
  void* out; long long ldo;
  const uint8_t* k_pages; const uint8_t* v_pages; const float* k_scales; const float* v_scales;
  int n_pages, page_size, heads, kv_heads, hd, window;
  const int* block_table; int bt_stride;
  Step step;
  int parts;                         // CTAs of a cluster
  int page_shift;                    // log2 of the page size, where that is a power of two
  int few;                           // a launch's requests: of more than `few` rows (tcgen05), of `few` at most (mma.sync)
  float scale_log2;                  // scale * log2(e)
  int* status;
};

constexpr int STATUS_TIMEOUT = 40;   // (and the three behind it) a bounded wait ran out

__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ex2(float x) {                // relative error 2^-22; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Bytes 0, 1 (2, 3) of a word as two f16.
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// 0xff in the bytes that are NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 255u; }
// log2 of a power of two (the sign does not matter)
__device__ __forceinline__ float log2_of(float scale) { return (float)((int)((__float_as_uint(scale) >> 23) & 0xffu) - 127); }

// The pool of pages [rows, hd] as a tensor map whose copies are groups of sixteen rows.
static bool group_map(CUtensorMap* map, const void* pages, long long rows, int hd, CUtensorMapSwizzle swizzle) {
  const TensorMapFn fn = tensor_map_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd};
  const cuuint32_t box[2] = {(cuuint32_t)hd, 16}, step[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pages), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many clusters of `parts` CTAs of a kernel the GPU holds at a time (a cluster lies within a part of the chip, so not all SMs can
// be had).  A property of the kernel and the chip: asked once.
template <typename K>
static int clusters_at_a_time(K kernel, int parts, int threads, size_t smem) {
  struct Known { const void* kernel; int parts; size_t smem; int clusters; };
  static thread_local Known known[128];
  static thread_local int n_known = 0;
  for (int i = 0; i < n_known; ++i)
    if (known[i].kernel == (const void*)kernel && known[i].parts == parts && known[i].smem == smem) return known[i].clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(parts * 148));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (n_known < 128) known[n_known++] = {(const void*)kernel, parts, smem, n};
  return n;
}

// Launches `kernel` over the tiles, their kv heads and parts (x in this order, parts fastest: the tiles with the most keys of
// every head start first), a tile's parts as a cluster.
template <typename K, typename... Maps>
static int launch_parts(K kernel, Attn p, int parts, long long tiles, int threads, size_t smem, cudaStream_t stream, const Maps&... maps) {
  p.parts = parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.kv_heads * parts));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (gb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (parts > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)parts;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  GB_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps..., p));
  return GB_OK;
}

}  // namespace kv8
