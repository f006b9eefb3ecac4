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
// magnitude, once to store).
template <typename T>
__global__ void __launch_bounds__(128) kv8_store_any_kernel(const Store p) {
  extern __shared__ float rows_of[];                          // [4 warps][hd]
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int seg = 0;
  const int r = find_piece((int)blockIdx.x, p.step.n_requests, false, [&](int i) {
    const int n = p.step.q_len[i], b = p.step.start_pos[i];
    return n > 0 ? (b + n - 1) / p.page_size - b / p.page_size + 1 : 0;
  }, seg);
  const int slots = p.heads + (p.write ? 2 * p.kv_heads : 0);
  const int slot = (int)blockIdx.y * 4 + warp;
  if (r < 0 || slot >= slots) return;
  const int before = p.step.start_pos[r], end = before + p.step.q_len[r];
  const int block = before / p.page_size + seg;
  const int from = max(before, block * p.page_size), to = min(end, (block + 1) * p.page_size);      // positions of the unit
  const int row0 = p.step.q_start[r] + (from - before);
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
  if (p.heads <= 0 || p.kv_heads <= 0 || p.hd <= 0 || p.hd % 8 != 0 || p.hd > 256 || p.page_size <= 0)
    GB_FAIL(GB_ERR_ARG, "kv8_store: %d heads, %d kv heads, head_dim %d, pages of %d: head sizes are multiples of 8 up to 256",
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
  int rc = dtype == GB_F32 ? launch_any<float>(p, segments, ctx->stream) : launch_any<bf16>(p, segments, ctx->stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_store");
  return 1;
}
