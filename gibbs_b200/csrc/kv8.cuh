// What the kernels of the 8-bit paged cache share: its numbers, its scales and how a launch finds its work.
//
// Keys and values lie in pages [n_pages, kv_heads, page_size, head_dim] of e4m3 numbers, with one scale for each (page, kv
// head) in float32 [n_pages, kv_heads]: an entry stands for number * |scale|.  A scale is a power of two, the smallest 2^e
// with -64 <= e under which the largest magnitude among the page's rows is at most 448, and e <= 50.  So
//   - dividing by a scale is exact, and what is rounded is rounded once, to half a step of e4m3 (2^-4 of the value, or 2^-10
//     of the scale below 2^-6): a power of two loses nothing against any other scale, since e4m3 is a floating format;
//   - when a page's next row asks for a larger scale, the rows it holds are divided by a power of two, which changes only
//     numbers that fall below 2^-6.
// What is not finite, or above 448 * 2^50 (5e17), is stored as NaN, does not count for the scale, and makes the scale's sign
// NEGATIVE: kernels take the careful way through such a page, and pay nothing for NaN anywhere else.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "gb_plan_op.h"

#define GB_OP(name) GB_API int name(const GbPlanCtx* ctx, const long long* a, const double* f, int flags)

namespace kv8 {

enum { STATUS_BAD_PAGE_WRITE = 1, STATUS_BAD_PAGE_READ = 2 };

constexpr int MIN_EXP = -64, MAX_EXP = 50;
constexpr float LARGEST = 448.f * 1125899906842624.f;          // 448 * 2^50

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The smallest scale that holds `amax` (finite, not negative).  448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return pow2(e < MIN_EXP ? MIN_EXP : e);
}
// 1 / scale of a power of two within the exponents above, by its exponent alone.  (Of 0, a scale nobody set or no page: 2^127, which only
// weights of 0 meet.)
__device__ __forceinline__ float inverse(float scale) {
  const int bits = __float_as_int(scale);
  return __int_as_float((254 << 23) - (bits & 0x7f800000));
}
__device__ __forceinline__ bool holdable(float x) { return fabsf(x) <= LARGEST; }     // (false for NaN)

// Two e4m3 numbers (lo in the low byte), rounded to nearest even; NaN for what the cache does not hold.
__device__ __forceinline__ unsigned short pack2(float lo, float hi, float inv) {
  lo = holdable(lo) ? lo * inv : __int_as_float(0x7fffffff);
  hi = holdable(hi) ? hi * inv : __int_as_float(0x7fffffff);
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack2(unsigned short v) {
  unsigned h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  float2 r;
  asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(h));
  return r;
}
__device__ __forceinline__ uint2 pack8(const float* v, float inv) {
  uint2 r;
  r.x = (unsigned)pack2(v[0], v[1], inv) | (unsigned)pack2(v[2], v[3], inv) << 16;
  r.y = (unsigned)pack2(v[4], v[5], inv) | (unsigned)pack2(v[6], v[7], inv) << 16;
  return r;
}
__device__ __forceinline__ void unpack8(uint2 w, float* v) {
  const float2 a = unpack2((unsigned short)w.x), b = unpack2((unsigned short)(w.x >> 16));
  const float2 c = unpack2((unsigned short)w.y), d = unpack2((unsigned short)(w.y >> 16));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
// Eight numbers of a page whose scale has grown: number * ratio (a power of two, 1 at most), rounded again.
__device__ __forceinline__ uint2 again8(uint2 w, float ratio) {
  float v[8];
  unpack8(w, v);
  return pack8(v, ratio);
}

// cos and sin of position * frequency.  The product and its remainder are taken in 64 bits: a 32-bit product is off by
// 2^-24 of itself, 5e-4 of a turn at position 8,000.
__device__ __forceinline__ float2 turn(int pos, float freq) {
  const double t = (double)pos * (double)freq;
  const double r = t - rint(t * 0.15915494309189535) * 6.283185307179586;
  float s, c;
  sincosf((float)r, &s, &c);
  return make_float2(c, s);
}

// The step, as the operations find it among its symbols.
struct Step {
  const int* q_start; const int* q_len; const int* start_pos;
  int n_tokens, n_requests, max_q, max_ctx, one_each;
};
static inline Step step_of(const GbPlanCtx* ctx) {
  Step s;
  s.q_start = reinterpret_cast<const int*>(ctx->sym[GB_SYM_PORTION_START]);
  s.q_len = reinterpret_cast<const int*>(ctx->sym[GB_SYM_PORTION_LENGTH]);
  s.start_pos = reinterpret_cast<const int*>(ctx->sym[GB_SYM_LENGTH_BEFORE]);
  s.n_tokens = (int)ctx->sym[GB_SYM_TOKENS];
  s.n_requests = (int)ctx->sym[GB_SYM_REQUESTS];
  s.max_q = (int)ctx->sym[GB_SYM_MAX_PORTION];
  s.max_ctx = (int)ctx->sym[GB_SYM_MAX_CONTEXT];
  s.one_each = (int)ctx->sym[GB_SYM_ONE_EACH];
  return s;
}

// An entry of a block table, for kernels that look at it later: one that is not a page's id is as large as no pool (and never -1,
// which stands for keys that nobody sees).
__device__ __forceinline__ int page_id(const int* entry) { return (int)min((unsigned)*entry, 0x7fffffffu); }

// A request of a step: its place, how many tokens it brings, how many it holds, and where in the step its tokens begin.
struct Request {
  int r, n, before, start;
};
// Piece `index` of a launch over pieces of requests, `count(n, before)` for a request: which request (r -1: none) and which of its
// pieces.  A whole warp looks at 32 requests at a time, all that is known of them in one trip; every lane gets the answer.  With
// `last_first` the requests are taken from the last to the first.
template <typename Count>
__device__ __forceinline__ Request find_piece(int index, const Step& step, bool last_first, Count count, int& piece) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < step.n_requests; base += 32) {
    const int i = base + lane, r = last_first ? step.n_requests - 1 - i : i;
    int n = 0, before = 0, start = 0, upto = 0;
    if (i < step.n_requests) {
      n = step.q_len[r];
      before = step.start_pos[r];
      start = step.q_start[r];
      upto = count(n, before);
    }
    const int mine = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned have = __ballot_sync(0xffffffffu, index < upto);
    if (have) {
      const int who = __ffs(have) - 1;
      piece = index - __shfl_sync(0xffffffffu, upto - mine, who);
      return {__shfl_sync(0xffffffffu, r, who), __shfl_sync(0xffffffffu, n, who), __shfl_sync(0xffffffffu, before, who),
              __shfl_sync(0xffffffffu, start, who)};
    }
    index -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return {-1, 0, 0, 0};
}

// Before a block without work leaves: the first one of a launch waits like those that work, so that a launch all of whose blocks leave
// still ends behind the kernel in front (what comes next waits for this launch alone).
__device__ __forceinline__ void leave() {
  if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
}

// The driver's cuTensorMapEncodeTiled (null where there is none).
typedef CUresult (*TensorMapFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapFn tensor_map_fn() {
  static const TensorMapFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess;
    return found ? (TensorMapFn)p : (TensorMapFn) nullptr;
  }();
  return fn;
}

}  // namespace kv8
