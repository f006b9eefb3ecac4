// Storing a step's keys and values in the 8-bit paged cache (kv8.cuh): a norm per head (optional) and the rotation of q and
// k, q into rows of its own, k and v into their pages under the pages' scales.
//
//   q, k: x = R(pos) (y / sqrt(mean y^2 + eps) * gain)      v: x = y        (y: the row's values, 32-bit from here on)
//   page: s' = max(s of the rows it holds, the smallest scale for its new rows); old rows * s / s', new rows x / s', rounded
//
// The formulas of norm and rotation are those of attention.cu (MisterTK/gibbs arch/lib/transformer.json5:22-24, 55-58,
// src/graph/cpu.rs:632-697); the angle is taken in 64 bits (kv8::turn).
//
// The unit of work is (request, page it writes to, head): all new rows of a page and head are brought together, because they
// share a scale.  Nothing outside those rows is touched, and no two units touch the same bytes.
//
// a0 rows [q heads | k heads | v heads], a1 their stride, a2 dtype, a3 q out [tokens, heads * hd], a4 q gain, a5 k gain (or
// 0), a6 rotary table (rotary_dim / 2 frequencies and a factor; or 0), a7 rotary_dim, a8 adjacent pairs, a9 k pages, a10 v
// pages, a11 k scales, a12 v scales (a9..a12 0: only q is worked on), a13 pages, a14 page size, a15 heads, a16 kv heads, a17
// hd, a18 block table, a19 its stride; f0 eps.  The step's requests come from its symbols.  With GB_OP_TAKES_PARTIALS the
// rows may be the partial tiles of the product in front.
#include "kv8.cuh"

namespace {

using namespace kv8;

struct Store {
  const void* rows; long long ld;
  const float* part; int splits; const float* part_bias; long long part_stride;   // splits > 0: partial tiles instead of rows
  void* q_out;
  const float* q_gain; const float* k_gain; const float* rotary;
  int rotary_dim, adjacent;
  uint8_t* k_pages; uint8_t* v_pages; float* k_scales; float* v_scales;
  int n_pages, page_size, heads, kv_heads, hd;
  const int* block_table; int bt_stride;
  Step step;
  float eps;
  int* status;
  int write;
};

// Entry `col` of row `row` of [q | k | v].
template <typename T>
__device__ __forceinline__ float entry(const Store& p, int row, int col) {
  if (p.splits > 0) {
    float v = 0.f;
    for (int s = 0; s < p.splits; ++s) v += ldcg_now(p.part + (size_t)s * p.part_stride + (size_t)row * p.ld + col);
    if (p.part_bias) v += p.part_bias[col];
    return to_f32(from_f32<T>(v));                            // rounded where the product's own sum would have been
  }
  return to_f32(reinterpret_cast<const T*>(p.rows)[(size_t)row * p.ld + col]);
}

// Any type, head size, page size and rotation: a warp takes a unit's rows one after the other, twice (once for the largest
// magnitude, once to store).  Bound by that chain: 2,048 tokens of 32 / 8 heads of 64 in bfloat16 take 66 us here and 9 below.
template <typename T>
__global__ void __launch_bounds__(128) kv8_store_any_kernel(const Store p) {
  extern __shared__ float rows_of[];                          // [4 warps][hd]
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int seg = 0;
  const Request q = find_piece((int)blockIdx.x, p.step, false, [&](int n, int before) {
    return n > 0 ? (before + n - 1) / p.page_size - before / p.page_size + 1 : 0;
  }, seg);
  const int r = q.r;
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  const int slot = (int)blockIdx.y * 4 + warp;
  if (r < 0 || slot >= slots) return leave();
  const int before = q.before, end = before + q.n;
  const int block = before / p.page_size + seg;
  const int from = max(before, block * p.page_size), to = min(end, (block + 1) * p.page_size);      // positions of the unit
  const int row0 = q.start + (from - before);
  const int hd = p.hd;
  const bool is_q = slot < p.heads, is_k = !is_q && slot < p.heads + p.kv_heads;
  const int kvh = is_q ? 0 : (slot - p.heads) % p.kv_heads;
  int page = 0;
  if (!is_q) page = p.block_table[(size_t)r * p.bt_stride + block];
  pdl_wait();
  if (!is_q && (page < 0 || page >= p.n_pages)) {
    if (lane == 0) atomicExch(p.status, STATUS_BAD_PAGE_WRITE);
    return;
  }
  const float* gain = is_q ? p.q_gain : is_k ? p.k_gain : nullptr;
  const int half = ((is_q || is_k) && p.rotary) ? p.rotary_dim / 2 : 0;
  const float factor = half ? p.rotary[half] : 1.f;
  float* x = rows_of + (size_t)warp * hd;
  // row `i` of the unit, finished, in x
  auto row = [&](int i) {
    __syncwarp();
    float ss = 0.f;
    for (int d = lane; d < hd; d += 32) {
      const float v = entry<T>(p, row0 + i, slot * hd + d);
      x[d] = v;
      ss += v * v;
    }
    __syncwarp();
    if (gain) {
      const float scale = 1.0f / sqrtf(warp_sum(ss) / (float)hd + p.eps);
      for (int d = lane; d < hd; d += 32) x[d] = x[d] * scale * gain[d];
      __syncwarp();
    }
    for (int j = lane; j < half; j += 32) {
      const int i0 = p.adjacent ? 2 * j : j, i1 = p.adjacent ? 2 * j + 1 : j + half;
      const float2 t = turn(from + i, p.rotary[j]);
      const float c = t.x * factor, s = t.y * factor, u = x[i0], v = x[i1];
      x[i0] = u * c - v * s;
      x[i1] = u * s + v * c;
    }
    __syncwarp();
  };
  const int n = to - from;
  if (is_q) {
    for (int i = 0; i < n; ++i) {
      row(i);
      T* dst = reinterpret_cast<T*>(p.q_out) + ((size_t)(row0 + i) * p.heads + slot) * hd;
      for (int d = lane; d < hd; d += 32) dst[d] = from_f32<T>(x[d]);
    }
    return;
  }
  float amax = 0.f;
  int bad = 0;
  for (int i = 0; i < n; ++i) {
    row(i);
    for (int d = lane; d < hd; d += 32) {
      if (holdable(x[d])) amax = fmaxf(amax, fabsf(x[d]));
      else bad = 1;
    }
  }
  amax = warp_max(amax);
  bad = __any_sync(0xffffffffu, bad);
  const int held = from - block * p.page_size;                // rows that the page holds already
  float* scale_at = (is_k ? p.k_scales : p.v_scales) + (size_t)page * p.kv_heads + kvh;
  uint8_t* dst = (is_k ? p.k_pages : p.v_pages) + ((size_t)page * p.kv_heads + kvh) * p.page_size * hd;
  const float was = held > 0 ? *scale_at : 0.f;
  const float now = fmaxf(fabsf(was), scale_for(amax)), inv = inverse(now);
  if (held > 0 && fabsf(was) < now) {
    const float ratio = fabsf(was) * inv;
    for (int i = lane; i < held * hd / 2; i += 32) {
      unsigned short* at = reinterpret_cast<unsigned short*>(dst) + i;
      const float2 v = unpack2(*at);
      *at = pack2(v.x, v.y, ratio);
    }
  }
  for (int i = 0; i < n; ++i) {
    row(i);
    unsigned short* at = reinterpret_cast<unsigned short*>(dst + (size_t)(held + i) * hd);
    for (int d = lane; d < hd / 2; d += 32) at[d] = pack2(x[2 * d], x[2 * d + 1], inv);
  }
  __syncwarp();
  if (lane == 0) *scale_at = (bad || signbit(was)) ? -now : now;
}

template <typename T>
int launch_any(const Store& p, long long segments, cudaStream_t stream) {
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  gb_launch(kv8_store_any_kernel<T>, dim3((unsigned)segments, (slots + 3) / 4), dim3(128), (size_t)4 * p.hd * sizeof(float),
            stream, p);
  return GB_OK;
}

// ---------------------------------------------------------------- heads of 64 or 128, the rotation over the whole head (or none)
// HD / 8 threads share a row, and a thread has the pairs that the rotation turns: entries 4 s .. 4 s + 3 and the four HD / 2 further,
// so that nothing is exchanged but the sum of squares.
template <typename T>
__device__ __forceinline__ void load4(const T* src, float* v) {
  if constexpr (sizeof(T) == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(src);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
    v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const float4 a = *reinterpret_cast<const float4*>(src);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* dst, const float* v) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
// Columns col .. col + 3 and col + HD / 2 .. of a row.
template <typename T, int HD>
__device__ __forceinline__ void load8(const Store& p, int row, int col, float* v) {
  if (p.splits > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    const float* src = p.part + (size_t)row * p.ld + col;
    for (int s = 0; s < p.splits; ++s, src += p.part_stride) {
      const float4 a = ldcg_now(reinterpret_cast<const float4*>(src)), b = ldcg_now(reinterpret_cast<const float4*>(src + HD / 2));
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p.part_bias) v[e] += p.part_bias[col + e + (e < 4 ? 0 : HD / 2 - 4)];
      v[e] = to_f32(from_f32<T>(v[e]));                        // rounded where the product's own sum would have been
    }
    return;
  }
  const T* src = reinterpret_cast<const T*>(p.rows) + (size_t)row * p.ld + col;
  load4<T>(src, v);
  load4<T>(src + HD / 2, v + 4);
}
// Norm (gain: this thread's eight) and rotation (cs: cos and sin of this thread's four pairs, or null) of a row whose eight values
// v this thread has.  All lanes of the warp take part.
template <int HD>
__device__ __forceinline__ void norm_rotate(float* v, const float* gain, bool norm, float eps, const float2* cs) {
  constexpr int TPR = HD / 8;
  if (norm) {                                                  // (the same for the threads of a row)
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
    const unsigned row = TPR == 8 ? 0xffu << (threadIdx.x & 24) : 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(row, ss, o);
    const float scale = rsqrtf(ss * (1.f / HD) + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= scale * gain[e];
  }
  if (cs != nullptr) {
    const float4 a = reinterpret_cast<const float4*>(cs)[0], b = reinterpret_cast<const float4*>(cs)[1];
    const float c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = v[e], hi = v[e + 4];
      v[e] = lo * c[e] - hi * s[e];
      v[e + 4] = lo * s[e] + hi * c[e];
    }
  }
}
// The largest magnitude among a thread's eight (and `amax`).  A sum of squares says in one comparison that all is finite and far
// below what a page holds; only where it does not, the values are looked at one by one.
__device__ __forceinline__ void magnitude8(const float* v, float& amax, bool& bad) {
  float ss = 0.f, top = amax;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    ss = fmaf(v[e], v[e], ss);
    top = fmaxf(top, fabsf(v[e]));
  }
  if (ss <= 1e30f) {
    amax = top;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (holdable(v[e])) amax = fmaxf(amax, fabsf(v[e]));
    else bad = true;
  }
}
// Four numbers; `bad`: some value of the page is not one that it holds.
__device__ __forceinline__ uint32_t pack4(const float* v, float inv, bool bad) {
  if (bad) return (uint32_t)pack2(v[0], v[1], inv) | (uint32_t)pack2(v[2], v[3], inv) << 16;
  unsigned short a, b;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(v[1] * inv), "f"(v[0] * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(v[3] * inv), "f"(v[2] * inv));
  return (uint32_t)a | (uint32_t)b << 16;
}

// Steps in which every request brings one token: a row is a unit, and 256 / HD of a block's 128 threads' rows make a warp's.  What
// the step's metadata and the tables give (position, page, angles, gains) is worked out before the wait for the product in front.
// Bound by the chain of trips: 1.9 us a launch in a chain of them, at 8 tokens of 32 / 8 heads of 64 in bfloat16.
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv8_store_rows_kernel(const Store p) {
  constexpr int TPR = HD / 8, SLOTS = 128 / TPR;
  __shared__ __align__(16) float2 cs[HD / 2];
  pdl_trigger();
  const int r = blockIdx.x, sub = threadIdx.x % TPR, slot = (int)blockIdx.y * SLOTS + threadIdx.x / TPR;
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  const bool active = slot < slots;
  const bool is_q = slot < p.heads, is_k = !is_q && slot < p.heads + p.kv_heads;
  const int pos = p.step.start_pos[r], row = p.step.q_start[r];
  if (p.step.q_len[r] <= 0) return leave();                    // (the whole block)
  int page = -1;
  if (active && !is_q) page = p.block_table[(size_t)r * p.bt_stride + pos / p.page_size];
  const int held = pos % p.page_size;                          // rows that the page holds already
  if (p.rotary)
    for (int j = threadIdx.x; j < HD / 2; j += 128) {
      const float2 t = turn(pos, p.rotary[j]);
      cs[j] = make_float2(t.x * p.rotary[HD / 2], t.y * p.rotary[HD / 2]);
    }
  const float* gain_at = is_q ? p.q_gain : is_k ? p.k_gain : nullptr;
  const bool norm = active && gain_at != nullptr;
  float gain[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    gain[e] = norm ? gain_at[sub * 4 + e + (e < 4 ? 0 : HD / 2 - 4)] : 1.f;
    gb_pin(gain[e]);
  }
  gb_pin(page);
  pdl_wait();
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float was = 0.f;
  const int kvh = active && !is_q ? (slot - p.heads) % p.kv_heads : 0;
  const bool there = page >= 0 && page < p.n_pages;
  float* scale_at = (is_k ? p.k_scales : p.v_scales) + (there ? (size_t)page * p.kv_heads + kvh : 0);
  if (active) load8<T, HD>(p, row, slot * HD + sub * 4, v);
  if (there && held > 0) was = *scale_at;
  __syncthreads();                                             // the angles
  norm_rotate<HD>(v, gain, norm, p.eps, active && (is_q || is_k) && p.rotary ? cs + sub * 4 : nullptr);
  float amax = 0.f;
  bool bad = false;
  magnitude8(v, amax, bad);
#pragma unroll
  for (int o = TPR / 2; o > 0; o >>= 1) {
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad ? 1 : 0, o) != 0;
  }
  if (!active) return;
  if (is_q) {
    T* q = reinterpret_cast<T*>(p.q_out) + ((size_t)row * p.heads + slot) * HD + sub * 4;
    store4<T>(q, v);
    store4<T>(q + HD / 2, v + 4);
    return;
  }
  if (!there) {
    if (sub == 0) atomicExch(p.status, STATUS_BAD_PAGE_WRITE);
    return;
  }
  uint8_t* dst = (is_k ? p.k_pages : p.v_pages) + ((size_t)page * p.kv_heads + kvh) * p.page_size * HD;
  const float now = fmaxf(fabsf(was), scale_for(amax)), inv = inverse(now);
  if (held > 0 && fabsf(was) < now) {
    const float ratio = fabsf(was) * inv;
#pragma unroll 4
    for (int i = 0; i < held; ++i) {
      uint2* at = reinterpret_cast<uint2*>(dst + (size_t)i * HD + sub * 8);
      *at = again8(*at, ratio);
    }
  }
  uint32_t* at = reinterpret_cast<uint32_t*>(dst + (size_t)held * HD + sub * 4);
  at[0] = pack4(v, inv, bad);
  at[HD / 8] = pack4(v + 4, inv, bad);
  if (sub == 0) *scale_at = (bad || signbit(was)) ? -now : now;
}

// Portions: a block has one page that a request writes to, and runs over a share of its heads.  A unit (a page's new rows of one
// head) is held in registers by page_size / 16 warps, sixteen rows each, from the load to the store, so a row is read once; its
// angles are worked out once a block into shared memory.  Bound by a block's chain (rows, norm, the page's maximum, store) more than
// by memory: 2,048 tokens of 32 / 8 heads of 64 in bfloat16 9.2 us, 2.5 TB/s of the 23 MB that go in and out; 1,100 tokens of 16 / 2 heads of 128 in
// 32 bits 8.1 us, 2.5 TB/s.
template <typename T, int HD>
__global__ void __launch_bounds__(256, HD == 64 ? 3 : 2) kv8_store_pages_kernel(const Store p, int per_block) {
  constexpr int TPR = HD / 8, RPP = 32 / TPR, PASSES = 16 / RPP;       // threads of a row, rows of a pass, passes of sixteen rows
  extern __shared__ __align__(16) float2 cs_all[];                     // [new rows][HD / 2]
  __shared__ float top_of[8];
  __shared__ int bad_of[8];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % TPR;
  int seg = 0;
  const Request q = find_piece((int)blockIdx.x, p.step, false, [&](int n, int before) {
    return n > 0 ? (before + n - 1) / p.page_size - before / p.page_size + 1 : 0;
  }, seg);
  const int r = q.r;
  if (r < 0) return leave();
  const int before = q.before, end = before + q.n;
  const int block = before / p.page_size + seg, base = block * p.page_size;
  const int from = max(before, base) - base, to = min(end, base + p.page_size) - base;      // new rows of the page
  const int row0 = q.start + base - before;                   // batch row of the page's row 0 (if it were new)
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  const int wpu = p.page_size / 16, wu = warp % wpu, units = 8 / wpu;
  int page = -1;
  if (p.write) page = p.block_table[(size_t)r * p.bt_stride + block];
  const bool there = page >= 0 && page < p.n_pages;
  if (p.rotary)
    for (int i = threadIdx.x; i < (to - from) * (HD / 2); i += 256) {
      const float2 t = turn(base + from + i / (HD / 2), p.rotary[i % (HD / 2)]);
      cs_all[i] = make_float2(t.x * p.rotary[HD / 2], t.y * p.rotary[HD / 2]);
    }
  pdl_wait();
  __syncthreads();
  if (p.write && !there && threadIdx.x == 0) atomicExch(p.status, STATUS_BAD_PAGE_WRITE);
  const int slot_end = min(slots, (int)(blockIdx.y + 1) * per_block);
  for (int slot0 = (int)blockIdx.y * per_block; slot0 < slot_end; slot0 += units) {
    const int slot = slot0 + warp / wpu;
    const bool is_q = slot < p.heads, is_k = !is_q && slot < p.heads + p.kv_heads;
    const bool active = slot < slot_end && (is_q || there);
    const int kvh = is_q ? 0 : (slot - p.heads) % p.kv_heads;
    const float* gain_at = is_q ? p.q_gain : is_k ? p.k_gain : nullptr;
    float v[PASSES][8];
    bool mine[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int o = 16 * wu + i * RPP + lane / TPR;             // row of the page
      mine[i] = active && o >= from && o < to;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (mine[i]) load8<T, HD>(p, row0 + o, slot * HD + sub * 4, v[i]);
    }
    float gain[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) gain[e] = gain_at ? gain_at[sub * 4 + e + (e < 4 ? 0 : HD / 2 - 4)] : 1.f;
    float was = 0.f;
    float* scale_at = (is_k ? p.k_scales : p.v_scales) + (there && !is_q ? (size_t)page * p.kv_heads + kvh : 0);
    if (active && !is_q && from > 0) was = *scale_at;
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int o = 16 * wu + i * RPP + lane / TPR;
      norm_rotate<HD>(v[i], gain, gain_at != nullptr, p.eps,
                      (is_q || is_k) && p.rotary ? cs_all + (mine[i] ? o - from : 0) * (HD / 2) + sub * 4 : nullptr);
      if (is_q) {
        if (mine[i]) {
          T* q = reinterpret_cast<T*>(p.q_out) + ((size_t)(row0 + o) * p.heads + slot) * HD + sub * 4;
          store4<T>(q, v[i]);
          store4<T>(q + HD / 2, v[i] + 4);
        }
      } else if (mine[i]) {
        magnitude8(v[i], amax, bad);
      }
    }
    // the page's largest magnitude, over the warps that hold it
    amax = warp_max(amax);
    bad = __any_sync(0xffffffffu, bad);
    if (wpu > 1) {
      if (lane == 0) {
        top_of[warp] = amax;
        bad_of[warp] = bad ? 1 : 0;
      }
      __syncthreads();
      for (int i = 0; i < wpu; ++i) {
        amax = fmaxf(amax, top_of[warp - wu + i]);
        bad |= bad_of[warp - wu + i] != 0;
      }
      __syncthreads();
    }
    if (!active || is_q) continue;
    uint8_t* dst = (is_k ? p.k_pages : p.v_pages) + ((size_t)page * p.kv_heads + kvh) * p.page_size * HD;
    const float now = fmaxf(fabsf(was), scale_for(amax)), inv = inverse(now);
    const bool grown = from > 0 && fabsf(was) < now;
    const float ratio = fabsf(was) * inv;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int o = 16 * wu + i * RPP + lane / TPR;
      if (mine[i]) {
        uint32_t* at = reinterpret_cast<uint32_t*>(dst + o * HD + sub * 4);
        at[0] = pack4(v[i], inv, bad);
        at[HD / 8] = pack4(v[i] + 4, inv, bad);
      } else if (grown && o < from) {
        uint2* at = reinterpret_cast<uint2*>(dst + o * HD + sub * 8);
        *at = again8(*at, ratio);
      }
    }
    // (every warp of the unit has read the old scale: they met above, or there is only this one)
    if (wu == 0 && lane == 0) *scale_at = (bad || signbit(was)) ? -now : now;
  }
}

template <typename T, int HD>
int launch_fast(const Store& p, long long segments, cudaStream_t stream) {
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  if (p.step.one_each) {
    constexpr int SLOTS = 128 / (HD / 8);
    gb_launch(kv8_store_rows_kernel<T, HD>, dim3(p.step.n_requests, (slots + SLOTS - 1) / SLOTS), dim3(128), 0, stream, p);
    return GB_OK;
  }
  // heads of a block: whole rounds of its warps, as many as leave four blocks for every SM (2,048 tokens of 32 / 8 heads of 64, us with
  // one, two, four, eight: 12.2, 9.1, 9.2, 10.6; a portion of one page has no other blocks than these)
  const int units = 8 / (p.page_size / 16), rounds = (slots + units - 1) / units;
  long long shares = (4 * 148 + segments - 1) / segments;
  if (shares > rounds) shares = rounds;
  const int per_block = units * (int)((rounds + shares - 1) / shares);
  const size_t smem = p.rotary ? (size_t)p.page_size * (HD / 2) * sizeof(float2) : 0;
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_store_pages_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * (HD / 2) * 8));
    attr_set = true;
  }
  gb_launch(kv8_store_pages_kernel<T, HD>, dim3((unsigned)segments, (slots + per_block - 1) / per_block), dim3(256), smem, stream, p, per_block);
  return GB_OK;
}

// Whether the kernels above take a call: what they hold in registers, and sixteen bytes at a time.
bool fast(const Store& p, int dtype) {
  const int wpu = p.page_size / 16;
  const uintptr_t size = dtype == GB_BF16 ? 2 : 4;
  return (p.hd == 64 || p.hd == 128) && (p.rotary == nullptr || (p.rotary_dim == p.hd && !p.adjacent)) &&
         (p.step.one_each || (p.page_size % 16 == 0 && (wpu == 1 || wpu == 2 || wpu == 4 || wpu == 8))) &&
         (((uintptr_t)p.rows | (uintptr_t)p.part | (uintptr_t)p.q_out) & 15) == 0 && (p.ld * size) % 16 == 0;
}

}  // namespace

GB_OP(gb_op_kv8_store) {
  Store p;
  p.step = step_of(ctx);
  if (p.step.n_tokens <= 0 || p.step.n_requests <= 0) return 0;
  p.rows = reinterpret_cast<const void*>(a[0]);
  p.ld = a[1];
  const int dtype = (int)a[2];
  p.q_out = reinterpret_cast<void*>(a[3]);
  p.q_gain = reinterpret_cast<const float*>(a[4]);
  p.k_gain = reinterpret_cast<const float*>(a[5]);
  p.rotary = reinterpret_cast<const float*>(a[6]);
  p.rotary_dim = (int)a[7];
  p.adjacent = (int)a[8];
  p.k_pages = reinterpret_cast<uint8_t*>(a[9]);
  p.v_pages = reinterpret_cast<uint8_t*>(a[10]);
  p.k_scales = reinterpret_cast<float*>(a[11]);
  p.v_scales = reinterpret_cast<float*>(a[12]);
  p.n_pages = (int)a[13];
  p.page_size = (int)a[14];
  p.heads = (int)a[15];
  p.kv_heads = (int)a[16];
  p.hd = (int)a[17];
  p.block_table = reinterpret_cast<const int*>(a[18]);
  p.bt_stride = (int)a[19];
  p.eps = (float)f[0];
  p.status = ctx->status;
  p.write = p.k_pages != nullptr;
  p.part = ctx->part;
  p.splits = (flags & GB_OP_TAKES_PARTIALS) && ctx->part != nullptr ? ctx->part_splits : 0;
  p.part_bias = ctx->part_bias;
  p.part_stride = 0;
  if (p.heads <= 0 || p.kv_heads <= 0 || p.hd <= 0 || p.hd % 8 != 0 || p.hd > 256 || p.page_size <= 0 ||
      (long long)p.page_size * p.hd > 0x7fffffff)
    GB_FAIL(GB_ERR_ARG, "kv8_store: %d heads, %d kv heads, head_dim %d, pages of %d: head sizes are multiples of 8 up to 256, a page's rows of a head fewer than 2^31 entries",
            p.heads, p.kv_heads, p.hd, p.page_size);
  if (dtype != GB_F32 && dtype != GB_BF16) GB_FAIL(GB_ERR_ARG, "kv8_store: rows are float32 or bfloat16");
  if (p.rotary != nullptr && (p.rotary_dim < 0 || p.rotary_dim > p.hd || p.rotary_dim % 2 != 0))
    GB_FAIL(GB_ERR_ARG, "kv8_store: a rotation over %d of %d entries", p.rotary_dim, p.hd);
  if (p.splits > 0) {
    p.ld = (long long)(p.heads + (p.write ? 2 * p.kv_heads : 0)) * p.hd;     // the product's own columns
    p.part_stride = (long long)p.step.n_tokens * p.ld;
  }
  // upper bound of the pages written to: sum_r (pages of its tokens + 1 for beginning inside one)
  const long long segments = p.step.one_each ? p.step.n_requests
                                             : (long long)p.step.n_tokens / p.page_size + 2ll * p.step.n_requests;
  int rc;
  if (fast(p, dtype))
    rc = p.hd == 64 ? (dtype == GB_F32 ? launch_fast<float, 64>(p, segments, ctx->stream) : launch_fast<bf16, 64>(p, segments, ctx->stream))
                    : (dtype == GB_F32 ? launch_fast<float, 128>(p, segments, ctx->stream) : launch_fast<bf16, 128>(p, segments, ctx->stream));
  else
    rc = dtype == GB_F32 ? launch_any<float>(p, segments, ctx->stream) : launch_any<bf16>(p, segments, ctx->stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_store");
  return 1;
}
