// Causal grouped-query attention over the 8-bit paged cache (kv8.cuh), for a ragged batch of prompt portions and single
// tokens: out = softmax(scale * q K^T over the visible keys) V, keys j <= pos (and j > pos - window), query head h on kv head
// h / (heads / kv_heads) (MisterTK/gibbs src/graph/cpu.rs:826-951, on entries number * |scale|).
//
// A tile is up to RT consecutive (token, query head of the kv head's group) rows of one request, which all read the same
// keys; its visible keys are cut into chunks that the warps of a CTA, and the CTAs of a cluster, take in turn, each with its
// own running maximum, sum and output in 32 bits.  The states are joined in shared memory, and across the cluster through
// distributed shared memory: there is no workspace, and the order of the sums is fixed by the sizes of the launch.
//
// a0 q rows, a1 their stride, a2 dtype (of q and out), a3 out, a4 its stride, a5 k pages, a6 v pages, a7 k scales, a8 v
// scales, a9 pages, a10 page size, a11 heads, a12 kv heads, a13 hd, a14 block table, a15 its stride, a16 window (0: none);
// f0 scale (of any sign, finite).  The step's requests come from its symbols.
#include "kv8_attention.cuh"

namespace {

using namespace kv8;

// Rows of a request (its tokens times the heads of a kv head's group) up to which 256-row tiles are not worth their time, which does not
// depend on the rows.  32 / 8 heads of 64, 4,000 keys, us by tiles of few rows / by 256 rows: at 48 rows 1 request 20 / 25, 8 48 / 52,
// 32 135 / 159; at 64 rows 20 / 25, 55 / 52, 176 / 159; at 32 rows 18 / 25, 43 / 52, 92 / 159.
constexpr int FEW = 48;
constexpr int MAX_PARTS = 16;        // CTAs of a cluster that share a tile's keys, at most (8 is the portable limit)

// A tile's request, rows and keys.
struct Tile {
  int r, row0, rows;                 // rows row0 .. row0 + rows - 1 of the request's (token, head of the group) rows
  int lo, hi;                        // keys lo .. hi - 1 are visible to some row
  int qstart, start, group;
  __device__ __forceinline__ int pos(int row) const { return start + (row0 + row) / group; }
};

template <int RT>
__device__ __forceinline__ bool find_tile(const Attn& p, int index, Tile& t) {
  t.group = p.heads / p.kv_heads;
  int tile = 0;
  Request q;
  if (p.step.one_each && t.group <= RT) {                      // (a tile a request: nothing to look for)
    q.r = p.step.n_requests - 1 - index;
    q.n = p.step.q_len[q.r];
    q.before = p.step.start_pos[q.r];
    q.start = p.step.q_start[q.r];
  } else {
    q = find_piece(index, p.step, true,
                   [&](int n, int) {
                     const int rows = n * t.group;
                     return rows > p.few ? 0 : (rows + RT - 1) / RT;
                   }, tile);
  }
  if (q.r < 0 || q.n <= 0) return false;
  const int qlen = q.n;
  t.r = q.r;
  t.qstart = q.start;
  t.start = q.before;
  const int tiles = (qlen * t.group + RT - 1) / RT;
  t.row0 = (tiles - 1 - tile) * RT;                            // the tiles with the most keys first
  t.rows = min(RT, qlen * t.group - t.row0);
  t.hi = t.pos(t.rows - 1) + 1;
  const int first = t.pos(0);
  t.lo = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
  return true;
}

__device__ __forceinline__ float ld_cluster(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}

// Joins the states of the CTA's NW warps (and of the cluster's CTAs) and stores the rows: m and l [NW][RT], o [NW][RT][hd]
// (unnormalised, under 2^m).  Sums run in the order of the warps, then of the CTAs.  All threads of the CTA come here.
template <typename T, int RT, int NW>
__device__ __forceinline__ void join(const Attn& p, const Tile& t, int kvh, int part, int parts, float* m, float* l, float* o) {
  const int hd = p.hd;
  __syncthreads();
  float* cm = m + NW * RT;                                     // [RT] of the CTA
  float* cl = cm + RT;
  // weights of the warps, in place of their maxima (a sum is NaN where a row sees a NaN: it stays so under a weight of 0)
  for (int r = threadIdx.x; r < t.rows; r += blockDim.x) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < NW; ++w) top = fmaxf(top, m[w * RT + r]);
    for (int w = 0; w < NW; ++w) {
      const float f = m[w * RT + r] == -INFINITY ? 0.f : exp2f(m[w * RT + r] - top);
      m[w * RT + r] = f;
      sum = fmaf(f, l[w * RT + r], sum);
    }
    cm[r] = top;
    cl[r] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows * hd; i += blockDim.x) {
    const int r = i / hd, d = i - r * hd;
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) acc = fmaf(m[w * RT + r], o[((size_t)w * RT + r) * hd + d], acc);
    if (parts == 1) {
      const int tok = (t.row0 + r) / t.group, g = (t.row0 + r) - tok * t.group;
      reinterpret_cast<T*>(p.out)[(size_t)(t.qstart + tok) * p.ldo + (size_t)(kvh * t.group + g) * hd + d] =
          from_f32<T>(cl[r] != 0.f ? acc / cl[r] : 0.f);
    } else {
      o[(size_t)r * hd + d] = acc;                             // (warp 0's place, read by this thread only)
    }
  }
  if (parts == 1) return;
  sm100::cluster_sync_all();
  const int total = t.rows * hd, end = (int)((long long)total * (part + 1) / parts);
  for (int i = (int)((long long)total * part / parts) + threadIdx.x; i < end; i += blockDim.x) {
    const int r = i / hd, d = i - r * hd;
    float top = -INFINITY, sum = 0.f, acc = 0.f, zm[MAX_PARTS];
#pragma unroll
    for (int z = 0; z < MAX_PARTS; ++z) {
      zm[z] = z < parts ? ld_cluster(cm + r, z) : -INFINITY;
      top = fmaxf(top, zm[z]);
    }
#pragma unroll
    for (int z = 0; z < MAX_PARTS; ++z) {
      if (z >= parts) continue;
      const float f = zm[z] == -INFINITY ? 0.f : exp2f(zm[z] - top);
      sum = fmaf(f, ld_cluster(cl + r, z), sum);
      acc = fmaf(f, ld_cluster(o + (size_t)r * hd + d, z), acc);
    }
    const int tok = (t.row0 + r) / t.group, g = (t.row0 + r) - tok * t.group;
    reinterpret_cast<T*>(p.out)[(size_t)(t.qstart + tok) * p.ldo + (size_t)(kvh * t.group + g) * hd + d] = from_f32<T>(sum != 0.f ? acc / sum : 0.f);
  }
  sm100::cluster_sync_all();                                   // nobody leaves while another CTA reads its share
}

// ---------------------------------------------------------------- any type, head size and page size
// A warp takes chunks of 32 keys: for the scores a lane has a key, for the output it has pairs of columns.  Bound by the trips of a chunk
// (page, scales, a key's bytes piece by piece): 9 requests of 2,000 keys, 24 / 8 heads of 48 in 32 bits, 45 us.
template <typename T, int NP>
__global__ void __launch_bounds__(128) kv8_attention_any_kernel(const Attn p) {
  constexpr int RT = 4, NW = 4;
  extern __shared__ __align__(16) float sm[];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.hd;
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;
  Tile t;
  if (!find_tile<RT>(p, unit / p.kv_heads, t)) return leave();  // (the same for every CTA of a cluster)
  const int c_lo = t.lo / 32, chunks = (t.hi + 31) / 32 - c_lo;
  const int parts = max(1, min(p.parts, (chunks + NW - 1) / NW));
  if (part >= parts) return;                                   // (a thread that has left counts as arrived at the cluster's barriers)
  float* q = sm;                                               // [RT][hd]
  float* m_s = q + RT * hd;                                    // [NW + 1][RT], [RT] sums of the CTA
  float* l_s = m_s + (NW + 2) * RT;                            // [NW][RT]
  float* o_s = l_s + NW * RT;                                  // [NW][RT][hd]
  float4* pw = reinterpret_cast<float4*>(o_s + NW * RT * hd) + warp * 32;                              // [32] weights of a key
  long long* at = reinterpret_cast<long long*>(reinterpret_cast<float4*>(o_s + NW * RT * hd) + NW * 32) + warp * 32;
  pdl_wait();
  for (int i = threadIdx.x; i < RT * hd; i += blockDim.x) {
    const int r = i / hd, d = i - r * hd;
    float v = 0.f;
    if (r < t.rows) {
      const int tok = (t.row0 + r) / t.group, g = (t.row0 + r) - tok * t.group;
      v = to_f32(reinterpret_cast<const T*>(p.q)[(size_t)(t.qstart + tok) * p.ldq + (size_t)(kvh * t.group + g) * hd + d]);
    }
    q[i] = v;
  }
  __syncthreads();
  const int* bt = p.block_table + (size_t)t.r * p.bt_stride;
  float m[RT], l[RT], o[RT][NP][2];
  int pos[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    pos[r] = r < t.rows ? t.pos(r) : -1;                       // (a row that does not exist sees nothing)
#pragma unroll
    for (int i = 0; i < NP; ++i) o[r][i][0] = o[r][i][1] = 0.f;
  }
  for (int c = part * NW + warp; c < chunks; c += parts * NW) {
    const int j = (c_lo + c) * 32 + lane;
    long long row = -1;
    float ks = 0.f, vs = 0.f;
    if (j >= t.lo && j < t.hi) {
      const int page = bt[j / p.page_size];
      if (page >= 0 && page < p.n_pages) {
        const size_t ph = (size_t)page * p.kv_heads + kvh;
        row = ((long long)ph * p.page_size + j % p.page_size) * hd;
        ks = fabsf(p.k_scales[ph]) * p.scale_log2;
        vs = fabsf(p.v_scales[ph]);
      } else {
        atomicExch(p.status, STATUS_BAD_PAGE_READ);
      }
    }
    float s[RT] = {0.f, 0.f, 0.f, 0.f};
    if (row >= 0) {
      const uint2* kp = reinterpret_cast<const uint2*>(p.k_pages + row);
      for (int d = 0; d < hd; d += 8) {
        float k[8];
        unpack8(kp[d / 8], k);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float4 a = *reinterpret_cast<const float4*>(q + r * hd + d), b = *reinterpret_cast<const float4*>(q + r * hd + d + 4);
          s[r] = fmaf(a.x, k[0], s[r]); s[r] = fmaf(a.y, k[1], s[r]); s[r] = fmaf(a.z, k[2], s[r]); s[r] = fmaf(a.w, k[3], s[r]);
          s[r] = fmaf(b.x, k[4], s[r]); s[r] = fmaf(b.y, k[5], s[r]); s[r] = fmaf(b.z, k[6], s[r]); s[r] = fmaf(b.w, k[7], s[r]);
        }
      }
    }
    float w[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const bool seen = row >= 0 && j <= pos[r] && (p.window <= 0 || j + p.window > pos[r]);
      const float v = seen ? s[r] * ks : -INFINITY;
      const float top = fmaxf(m[r], warp_max(v));
      const float use = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[r] - use);                    // (0 when nothing was seen before)
      const float e = seen ? exp2f(v - use) : 0.f;
      l[r] = l[r] * corr + e;
      m[r] = top;
      w[r] = seen ? e * vs : -1.f;                             // -1: this row does not see the key, whatever its value is
      if (corr != 1.f) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          o[r][i][0] *= corr;
          o[r][i][1] *= corr;
        }
      }
    }
    __syncwarp();
    pw[lane] = make_float4(w[0], w[1], w[2], w[3]);
    at[lane] = row;
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const long long vr = at[i];
      if (vr < 0) continue;
      const float4 a = pw[i];
      const float wr[RT] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int d = 2 * (lane + 32 * n);
        if (d >= hd) continue;
        const float2 v = unpack2(*reinterpret_cast<const unsigned short*>(p.v_pages + vr + d));
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (!(wr[r] < 0.f)) {
            o[r][n][0] = fmaf(wr[r], v.x, o[r][n][0]);
            o[r][n][1] = fmaf(wr[r], v.y, o[r][n][1]);
          }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float sum = warp_sum(l[r]);
    if (lane == 0) {
      m_s[warp * RT + r] = m[r];
      l_s[warp * RT + r] = sum;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int d = 2 * (lane + 32 * n);
      if (d < hd) *reinterpret_cast<float2*>(o_s + ((size_t)warp * RT + r) * hd + d) = make_float2(o[r][n][0], o[r][n][1]);
    }
  }
  join<T, RT, NW>(p, t, kvh, part, parts, m_s, l_s, o_s);
}

// ---------------------------------------------------------------- heads of 32, 64 or 128 in 32-bit arithmetic
// The 32-bit path (and bfloat16 heads that the kernels below do not take).  Tiles of 4 rows; a warp takes chunks of 32 keys.  HD / 8
// lanes share a key, eight bytes each, of K and of V alike, so all loads of a chunk are whole lines and go out together.  A lane's
// partial scores of its keys are added and handed out in one go (each step exchanges half of them), and end as the scores of ONE key
// in every lane; weights go back through shared memory.  Bound by a chunk's chain (loads, conversions, sums over lanes, softmax) with
// three warps a scheduler: 64 requests of 2,048 keys, 32 / 8 heads of 64, 97 us, 11 TFLOP/s; nine requests of 1 to 4,002 keys, 24 / 8 heads,
// 14.1 us; a prompt of 2,048 tokens 893 us, 19 TFLOP/s (with pairs of FMAs, whose operands have to be moved together, 1,020).
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv8_attention_rows_kernel(const Attn p) {
  constexpr int RT = 4, NW = 4, LPR = HD / 8, KG = 32 / LPR, KEYS = 32 / KG;       // lanes of a key, keys at a time, keys of a lane
  extern __shared__ __align__(16) float sm[];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, db = lane % LPR, kg = lane / LPR;
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;
  Tile t;
  if (!find_tile<RT>(p, unit / p.kv_heads, t)) return leave();  // (the same for every CTA of a cluster)
  const int c_lo = t.lo / 32, chunks = (t.hi + 31) / 32 - c_lo;
  const int parts = max(1, min(p.parts, (chunks + NW - 1) / NW));
  if (part >= parts) return;                                   // (a thread that has left counts as arrived at the cluster's barriers)
  float* m_s = sm;                                             // [NW + 1][RT], [RT] sums of the CTA
  float* l_s = m_s + (NW + 2) * RT;                            // [NW][RT]
  float* o_s = l_s + NW * RT;                                  // [NW][RT][HD]
  float4* pw = reinterpret_cast<float4*>(o_s + NW * RT * HD) + warp * 32;          // [32] weights of a key
  pdl_wait();
  float q[RT][8], o[RT][8], m[RT], l[RT];
  int pos[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    pos[r] = r < t.rows ? t.pos(r) : -1;                       // (a row that does not exist sees nothing)
    const int tok = (t.row0 + r) / t.group, g = (t.row0 + r) - tok * t.group;
    const T* src = reinterpret_cast<const T*>(p.q) + (size_t)(t.qstart + tok) * p.ldq + (size_t)(kvh * t.group + g) * HD + db * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[r][e] = r < t.rows ? to_f32(src[e]) : 0.f;
      o[r][e] = 0.f;
    }
  }
  const int* bt = p.block_table + (size_t)t.r * p.bt_stride;
  // The key whose scores end in this lane: at step `b` of the hand-out (LPR / 2, ..., 1) a lane keeps the upper half of its keys where
  // the bit of its place is set.
  int own = 0;
#pragma unroll
  for (int b = LPR / 2, half = KEYS / 2; b > 0; b >>= 1, half >>= 1) own += (db & b) ? half : 0;
  const int own_key = own * KG + kg;                           // of a chunk: a lane's keys are kg, kg + KG, ...
  // lane = key of a chunk.  What a chunk needs before its loads is asked for ahead: its page's id two chunks ahead, the page's scales
  // one ahead, so that a chunk waits for one trip and not for three.
  const int stride = parts * NW;
  auto page_of = [&](int c) {                                  // -1: not visible to any row
    const int j = (c_lo + c) * 32 + lane;
    return (c >= chunks || j < t.lo || j >= t.hi) ? -1 : page_id(bt + j / p.page_size);
  };
  long long row_next;
  float ks_next, vs_next;
  auto look_up = [&](int c, int page) {
    row_next = -1;
    ks_next = vs_next = 0.f;
    if (page < 0) return;
    if (page >= p.n_pages) {
      atomicExch(p.status, STATUS_BAD_PAGE_READ);
      return;
    }
    const size_t ph = (size_t)page * p.kv_heads + kvh;
    row_next = ((long long)ph * p.page_size + ((c_lo + c) * 32 + lane) % p.page_size) * HD;
    ks_next = p.k_scales[ph];
    vs_next = p.v_scales[ph];
  };
  look_up(part * NW + warp, page_of(part * NW + warp));
  int page_next = page_of(part * NW + warp + stride);
  for (int c = part * NW + warp; c < chunks; c += stride) {
    const long long row = row_next;
    const float ks = fabsf(ks_next) * p.scale_log2, vs = fabsf(vs_next);       // vs 0: no such key
    uint2 kw[KEYS], vw[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const long long at = __shfl_sync(0xffffffffu, row, i * KG + kg);
      kw[i] = vw[i] = make_uint2(0u, 0u);
      if (at >= 0) {
        kw[i] = *reinterpret_cast<const uint2*>(p.k_pages + at + db * 8);
        vw[i] = *reinterpret_cast<const uint2*>(p.v_pages + at + db * 8);
      }
    }
    look_up(c + stride, page_next);
    page_next = page_of(c + 2 * stride);
    float s[KEYS][RT];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      float k[8];
      unpack8(kw[i], k);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        s[i][r] = q[r][0] * k[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) s[i][r] = fmaf(q[r][e], k[e], s[i][r]);
      }
    }
#pragma unroll
    for (int b = LPR / 2, half = KEYS / 2; b > 0; b >>= 1, half >>= 1) {
      const bool upper = (db & b) != 0;
#pragma unroll
      for (int i = 0; i < half; ++i)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float keep = upper ? s[i + half][r] : s[i][r], give = upper ? s[i][r] : s[i + half][r];
          s[i][r] = keep + __shfl_xor_sync(0xffffffffu, give, b);
        }
    }
    // this lane's key: its page's scales, and whether there is one, from the lane that looked it up
    const float ks_own = __shfl_sync(0xffffffffu, ks, own_key), vs_own = __shfl_sync(0xffffffffu, vs, own_key);
    const int j_own = (c_lo + c) * 32 + own_key;
    const bool there = vs_own != 0.f;
    float w[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const bool seen = there && j_own <= pos[r] && (p.window <= 0 || j_own + p.window > pos[r]);
      const float v = seen ? s[0][r] * ks_own : -INFINITY;
      const float top = fmaxf(m[r], warp_max(v));
      const float use = top == -INFINITY ? 0.f : top;
      const float corr = exp2f(m[r] - use);                    // (0 when nothing was seen before)
      const float e = seen ? exp2f(v - use) : 0.f;
      l[r] = l[r] * corr + e;
      m[r] = top;
      w[r] = seen ? e * vs_own : -1.f;                         // -1: this row does not see the key, whatever its value is
      if (corr != 1.f) {
#pragma unroll
        for (int d = 0; d < 8; ++d) o[r][d] *= corr;
      }
    }
    __syncwarp();
    pw[own_key] = make_float4(w[0], w[1], w[2], w[3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const float4 a = pw[i * KG + kg];
      const float wr[RT] = {a.x, a.y, a.z, a.w};
      float v[8];
      unpack8(vw[i], v);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        if (!(wr[r] < 0.f)) {
#pragma unroll
          for (int d = 0; d < 8; ++d) o[r][d] = fmaf(wr[r], v[d], o[r][d]);
        }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float sum = warp_sum(l[r]);
    if (lane == 0) {
      m_s[warp * RT + r] = m[r];
      l_s[warp * RT + r] = sum;
    }
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int x = LPR; x < 32; x <<= 1) o[r][d] += __shfl_xor_sync(0xffffffffu, o[r][d], x);
    if (kg == 0) {
      float4* at = reinterpret_cast<float4*>(o_s + ((size_t)warp * RT + r) * HD + db * 8);
      at[0] = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
      at[1] = make_float4(o[r][4], o[r][5], o[r][6], o[r][7]);
    }
  }
  join<T, RT, NW>(p, t, kvh, part, parts, m_s, l_s, o_s);
}

// ---------------------------------------------------------------- bfloat16 rows on mma.sync
// Tiles of 8 NB rows.  K and V stay in 8 bits until they are operands: a lane reads the bytes of its mma fragments and turns two
// of them at a time into f16, which holds every e4m3 number exactly.  The products are S^T = K Q^T and O^T = V^T P^T: keys (and columns
// of the output) are the 16 rows of an mma and the few query rows its 8 columns, so that a decoded token of a group of eight
// heads or fewer wastes little.  Which entry of a head stands at which place of the contraction is free as long as q and K
// agree, and so is which column of the output has which place: they are chosen such that a lane (g, t) = (lane / 4, lane % 4)
//   - holds hd/4 contiguous bytes of the keys in places g and g + 8 of sixteen, and of q;
//   - holds hd/8 contiguous bytes (columns g hd/8 ...) of the values in places 2t, 2t+1, 2t+8, 2t+9.
// f16 has no room for the scales, so they go elsewhere, where powers of two are exact and cost nothing:
//   - q's row is multiplied by the power of two that brings its largest magnitude to 2^14 (what is below 2^-28 of that loses
//     bits; nothing of a bfloat16 above it does), and the scores by its inverse and the page's scale, in 32 bits;
//   - the page's scale of V goes into the exponent: with x_j = score_j + log2(scale_j) the output is
//     sum_j 2^(x_j - M) n_j / sum_j 2^(x_j - M) / scale_j, n the stored numbers and M the running maximum of the x.  The weights
//     w = 2^(x - M + 12) lie below 2^15 and are rounded to f16 (2^-11 of a weight; below 2^-40 of the largest contribution it is
//     gone, where a 32-bit sum would not see it either); their sum is of the unrounded ones, in 32 bits.
// K and V come by TMA, sixteen keys (a group, which lies in one page) a copy, into a ring of SLOTS slots per warp: no barrier but
// the warp's own, and a copy costs an instruction instead of one for every lane and piece.  The rows are swizzled (128-byte
// rows by the 16-byte piece XOR row, 64-byte rows by piece XOR row / 2) and the keys of a group take the places pi(0..15) of the
// products: with these every fragment is read without a bank conflict.
// Bound by memory and by how evenly the CTAs lie on the SMs: 64 requests of 2,112 keys, 32 / 8 heads of 64, 30.3 us, 4.6 TB/s of the
// cache's 139 MB; 4 requests of 30,000 to 32,768 keys, 32 / 8 heads of 128, 47.3 us, 5.4 TB/s; one request of 2,048 keys 7.3 us, by its trips.
template <int HD, int WARPS> struct Mma {
  static constexpr int NW = WARPS;
  static constexpr int NG = 2;                                 // groups of a slot, taken together
  static constexpr int SLOTS = HD <= 64 ? 3 : 2;
  static constexpr int CTAS = WARPS > 4 ? 1 : HD <= 64 ? 4 : 3;        // on an SM: by shared memory, and registers capped to that
  static constexpr int CK = 16 * NG;                           // keys of a chunk
  static constexpr int KB = HD / 4, VB = HD / 8;               // bytes of a lane's piece of a key, of a value
  static constexpr int GROUP = 16 * HD;                        // bytes of a group's keys
  static constexpr int SLOT = 2 * NG * GROUP;
  static constexpr int RING = NW * SLOTS * SLOT;
  static constexpr int join(int rt) { return ((2 * NW + 2) * rt + NW * rt * HD) * 4; }
  static constexpr int smem(int rt) { return (RING > join(rt) ? RING : join(rt)) + 1024; }
};

// Where in a group of sixteen rows of HD bytes (a multiple of 1024 bytes from 0) byte x (a multiple of 4) of row r lies.
template <int HD> __device__ __forceinline__ int place(int r, int x) {
  return r * HD + (HD == 128 ? x ^ ((r & 7) << 4) : x ^ (((r >> 1) & 3) << 4));
}
// The key of a group that takes place g (0..7; 8 + g likewise): even places have rows 0, 1, 4, 5, odd ones 3, 2, 7, 6.
__device__ __forceinline__ int key_at(int g) { return (g & 1) ? ((g & 4) | (3 - ((g >> 1) & 1))) : ((g & 4) | ((g >> 1) & 1)); }

// BYTES (a multiple of 8) from byte x of row r of a group.
template <int HD, int BYTES>
__device__ __forceinline__ void read_bytes(const uint8_t* group, int r, int x, uint32_t* w) {
  if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(group + place<HD>(r, x));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(group + place<HD>(r, x + 16 * i));
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // an 8 x 8 matrix of 16-bit entries, two neighbours a lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int HD, int NB, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, NB == 1 ? Mma<HD, WARPS>::CTAS : 1)
kv8_attention_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Attn p) {
  using C = Mma<HD, WARPS>;
  constexpr int RT = 8 * NB, NW = C::NW, NG = C::NG, CK = C::CK, KW = C::KB / 4, VW = C::VB / 4, SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[NW][SLOTS];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;
  Tile t;
  const bool found = find_tile<RT>(p, unit / p.kv_heads, t);   // (the same for every CTA of a cluster)
  const int c_lo = found ? t.lo / CK : 0, chunks = found ? (t.hi + CK - 1) / CK - c_lo : 0;
  const int parts = max(1, min(p.parts, (chunks + NW - 1) / NW));
  if (!found || part >= parts) return leave();                 // (a thread that has left counts as arrived at the cluster's barriers)
  const int* bt = p.block_table + (size_t)t.r * p.bt_stride;
  const int stride = parts * NW, first = part * NW + warp;
  const int mine = first < chunks ? (chunks - 1 - first) / stride + 1 : 0;           // chunks of this warp
  if (lane == 0) {
    for (int s = 0; s < SLOTS; ++s) sm100::mbar_init(&full[warp][s], 1);
    sm100::fence_barrier_init();
    sm100::tma_prefetch_desc(&map_k);
    sm100::tma_prefetch_desc(&map_v);
  }
  __syncwarp();

  // The warp's groups are numbered n = 0, 1, ... (chunk n / NG).  Lane i holds what belongs to group 32 b + i: the row of its
  // first key in the pool (ABSENT where nothing of it is visible: no page has it, and none of its keys counts), and the page's scales.
  constexpr int NONE = -1;                                     // (a page)
  constexpr int ABSENT = -16;                                  // (a group: sixteen rows in front of the pool, which a copy fills with zeros)
  auto page_of = [&](int n) {
    const int c = first + (n / NG) * stride, j = (c_lo + c) * CK + (n % NG) * 16;
    return (c >= chunks || j >= t.hi || j + 15 < t.lo) ? NONE : page_id(bt + (j >> p.page_shift));
  };
  auto checked = [&](int page) {                               // (apart from the lookup, so that its trip is not waited for there)
    if (page < p.n_pages) return page;
    atomicExch(p.status, STATUS_BAD_PAGE_READ);
    return NONE;
  };
  auto row_of = [&](int n, int page) {
    const int j = (c_lo + first + (n / NG) * stride) * CK + (n % NG) * 16;
    return page == NONE ? ABSENT : (((page * p.kv_heads + kvh) << p.page_shift) | (j & (p.page_size - 1)));
  };
  // Requests run SLOTS chunks ahead of the products: `row` is of the 32 groups that are being requested, `ks`, `vs` of the 32 that
  // are being worked on, `ks_next`, `vs_next` of the former where they differ, `page_ahead` of the 32 behind those.
  int page = page_of(lane), page_ahead = page_of(32 + lane);
  page = checked(page);
  int row = row_of(lane, page);
  float ks_own = 0.f, vs_own = 0.f, ks_next = 0.f, vs_next = 0.f, lv_own = 0.f, inv_own = 0.f;
  auto scales_of = [&](int page_, float& ks, float& vs) {      // (0: no page)
    ks = vs = 0.f;
    if (page_ != NONE) {
      ks = p.k_scales[(size_t)page_ * p.kv_heads + kvh];
      vs = p.v_scales[(size_t)page_ * p.kv_heads + kvh];
    }
  };
  uint8_t* ring = smem + warp * SLOTS * C::SLOT;
  // Requests the groups of the warp's chunk i.  A group without a page comes as zeros: its weights are 0, and 0 times what a page of
  // another request holds need not be 0.
  auto request = [&](int i, int slot) {
    int at[NG];
#pragma unroll
    for (int y = 0; y < NG; ++y) at[y] = __shfl_sync(0xffffffffu, row, (i * NG + y) & 31);
    if (lane == 0) {
      uint8_t* dst = ring + slot * C::SLOT;
      sm100::mbar_arrive_expect_tx(&full[warp][slot], C::SLOT);
#pragma unroll
      for (int y = 0; y < NG; ++y) {
        sm100::tma_load_2d(dst + y * C::GROUP, &map_k, 0, at[y], &full[warp][slot]);
        sm100::tma_load_2d(dst + (NG + y) * C::GROUP, &map_v, 0, at[y], &full[warp][slot]);
      }
    }
  };
  gb_pin(row);
  gb_pin(page_ahead);
  pdl_wait();
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
    if (i < mine) request(i, i);
  scales_of(page, ks_own, vs_own);
  lv_own = log2_of(vs_own);
  inv_own = inverse(vs_own);

  // q: row g of each block, entries t4 * KB ... + KB, under its power of two.  In the lane's columns of S^T and O^T stand rows
  // 2t and 2t + 1 of each block.
  uint32_t qb[NB][HD / 16][2];
  int rpos[NB][2];
  float factor[NB][2];                                         // scale * log2(e) / the row's power of two
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int row = 8 * b + g;
    uint32_t w[HD / 8];
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) w[x] = 0u;
    if (row < t.rows) {
      const int tok = (t.row0 + row) / t.group, h = (t.row0 + row) - tok * t.group;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.q) + (size_t)(t.qstart + tok) * p.ldq +
                                                        (size_t)(kvh * t.group + h) * HD + t4 * C::KB);
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) {
        const uint4 u = src[x];
        w[4 * x] = u.x; w[4 * x + 1] = u.y; w[4 * x + 2] = u.z; w[4 * x + 3] = u.w;
      }
    }
    uint32_t top = 0u;                                         // largest magnitude: bits of a bfloat16 compare like a number's
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) top = max(top, max(w[x] & 0x7fffu, (w[x] >> 16) & 0x7fffu));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(127, max((int)(top >> 7) - 127, -112));  // (a row of zeros, or one that is not finite, under any power)
    const float up = pow2(min(14 - e, 126)), back = p.scale_log2 * pow2(max(e - 14, -126));
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t v = w[2 * kk + y];
        qb[b][kk][y] = pack_f16(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xffff0000u) * up);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      factor[b][r] = __shfl_sync(0xffffffffu, back, (2 * t4 + r) * 4);
      const int at = 8 * b + 2 * t4 + r;
      rpos[b][r] = at < t.rows ? t.pos(at) : -1;               // (a row that does not exist sees nothing)
    }
  }

  // use: what is taken off a row's x: its maximum in use, minus 12 (0 and minus 12 before it has seen anything)
  float m[NB][2], use[NB][2], l[NB][2], o[NB][HD / 16][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b][0] = m[b][1] = -INFINITY;
    use[b][0] = use[b][1] = -12.f;
    l[b][0] = l[b][1] = 0.f;
#pragma unroll
    for (int n = 0; n < HD / 16; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[b][n][i] = 0.f;
  }
  const int pos_first = t.pos(0), pos_last = t.pos(t.rows - 1);
  const int key_g = key_at(g), key_0 = key_at(2 * t4), key_1 = key_at(2 * t4 + 1);
  bool alive = true;
  uint32_t marked = __ballot_sync(0xffffffffu, vs_own < 0.f);  // which of the 32 groups lie in pages with NaN among their values

  int slot = 0, phase = 0;
  for (int i = 0; i < mine; ++i) {
    const int n0 = i * NG;
    if (!__all_sync(0xffffffffu, sm100::mbar_wait(&full[warp][slot], phase))) {
      alive = false;
      break;
    }
    const uint8_t* kt = ring + slot * C::SLOT;
    const uint8_t* vt = kt + NG * C::GROUP;
    const int j_chunk = (c_lo + first + i * stride) * CK;
    float s[NB][NG][4], inv[NG];
    const bool careful = (marked >> (n0 & 31)) & ((1u << NG) - 1);     // some page of the chunk has NaN among its values
#pragma unroll
    for (int y = 0; y < NG; ++y) {
      const float ks = __shfl_sync(0xffffffffu, ks_own, (n0 + y) & 31), lv = __shfl_sync(0xffffffffu, lv_own, (n0 + y) & 31);
      inv[y] = __shfl_sync(0xffffffffu, inv_own, (n0 + y) & 31);
      uint32_t w[2][KW];
#pragma unroll
      for (int h = 0; h < 2; ++h) read_bytes<HD, C::KB>(kt + y * C::GROUP, key_g + 8 * h, t4 * C::KB, w[h]);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[b][y][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t a[4];
        to_f16(w[0][kk], a[0], a[2]);
        to_f16(w[1][kk], a[1], a[3]);
#pragma unroll
        for (int b = 0; b < NB; ++b) mma_f16(s[b][y], a, qb[b][kk][0], qb[b][kk][1]);
      }
      // x = score + log2(scale of V), -inf where a row does not see the key
      const int j0 = j_chunk + 16 * y;
      const bool full_ = ks != 0.f && j0 + 15 <= pos_first && (p.window <= 0 || j0 + p.window > pos_last);
      const float kf = fabsf(ks);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float f0 = factor[b][0] * kf, f1 = factor[b][1] * kf;
        s[b][y][0] = fmaf(s[b][y][0], f0, lv);
        s[b][y][1] = fmaf(s[b][y][1], f1, lv);
        s[b][y][2] = fmaf(s[b][y][2], f0, lv);
        s[b][y][3] = fmaf(s[b][y][3], f1, lv);
        if (!full_) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + key_g + 8 * (e >> 1), pos = rpos[b][e & 1];
            const bool seen = ks != 0.f && j <= pos && (p.window <= 0 || j + p.window > pos);
            s[b][y][e] = seen ? s[b][y][e] : -INFINITY;
          }
        }
      }
    }
    // The maximum in use follows a row's only when it would fall behind by more than 2^3: a weight stays below 2^15.
    bool grow = false;
    float top[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[b][r] = fmaxf(s[b][0][r], s[b][0][r + 2]);
#pragma unroll
        for (int y = 1; y < NG; ++y) top[b][r] = fmaxf(top[b][r], fmaxf(s[b][y][r], s[b][y][r + 2]));
        grow |= top[b][r] > m[b][r] + 3.f;                     // (m -inf: anything seen)
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top_r = top[b][r];
#pragma unroll
          for (int x = 4; x < 32; x *= 2) top_r = fmaxf(top_r, __shfl_xor_sync(0xffffffffu, top_r, x));
          if (top_r > m[b][r]) {
            const float corr = ex2(m[b][r] - top_r);           // 0 when nothing was seen before
            m[b][r] = top_r;
            use[b][r] = top_r - 12.f;
            l[b][r] *= corr;
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
              o[b][n][r] *= corr;
              o[b][n][r + 2] *= corr;
            }
          }
        }
    }
#pragma unroll
    for (int y = 0; y < NG; ++y) {
      uint32_t pb[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float e0 = ex2(s[b][y][0] - use[b][0]), e1 = ex2(s[b][y][1] - use[b][1]);
        const float e2 = ex2(s[b][y][2] - use[b][0]), e3 = ex2(s[b][y][3] - use[b][1]);
        l[b][0] = fmaf(e0 + e2, inv[y], l[b][0]);
        l[b][1] = fmaf(e1 + e3, inv[y], l[b][1]);
        pb[b][0] = transposed(pack_f16(e0, e1));               // places 0..7 of the group, then 8..15
        pb[b][1] = transposed(pack_f16(e2, e3));
      }
      uint32_t v[4][VW];                                       // places 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int h = 0; h < 4; ++h) read_bytes<HD, C::VB>(vt + y * C::GROUP, ((h & 1) ? key_1 : key_0) + 4 * (h & 2), g * C::VB, v[h]);
      const int j0 = j_chunk + 16 * y;
      if (j0 + 16 > t.hi) {                                    // rows behind the context hold anything: 0 * NaN is not 0
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (j0 + ((h & 1) ? key_1 : key_0) + 4 * (h & 2) >= t.hi) {
#pragma unroll
            for (int w = 0; w < VW; ++w) v[h][w] = 0u;
          }
      }
      if (careful) {
        // A NaN reaches the rows that see its key and no other: the numbers go in as 0, and (columns of a key that are NaN)
        // times (rows that see the key) tells where the output is NaN.
        uint32_t see[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            see[b][h] = transposed(pack_f16(s[b][y][2 * h] == -INFINITY ? 0.f : 1.f, s[b][y][2 * h + 1] == -INFINITY ? 0.f : 1.f));
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t bad[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            bad[h] = nan_bytes(v[h][w]);
            v[h][w] &= ~bad[h];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __byte_perm(bad[0], bad[1], h ? 0x7362 : 0x5140), hi = __byte_perm(bad[2], bad[3], h ? 0x7362 : 0x5140);
            uint32_t a[4];                                     // 1 (f16) where a number is NaN
            a[0] = __byte_perm(lo, 0u, 0x1404) & 0x3c003c00u;
            a[1] = __byte_perm(lo, 0u, 0x3424) & 0x3c003c00u;
            a[2] = __byte_perm(hi, 0u, 0x1404) & 0x3c003c00u;
            a[3] = __byte_perm(hi, 0u, 0x3424) & 0x3c003c00u;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              float n[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(n, a, see[b][0], see[b][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n[e] > 0.f) o[b][2 * w + h][e] = __int_as_float(0x7fffffff);
            }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4];
          to_f16(__byte_perm(v[0][w], v[1][w], h ? 0x7362 : 0x5140), a[0], a[1]);
          to_f16(__byte_perm(v[2][w], v[3][w], h ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
          for (int b = 0; b < NB; ++b) mma_f16(o[b][2 * w + h], a, pb[b][0], pb[b][1]);
        }
    }
    __syncwarp();                                              // every lane has read the slot
    const int ahead = i + SLOTS;
    if (ahead < mine) {
      if (((ahead * NG) & 31) == 0) {
        const int next = checked(page_ahead);
        row = row_of(ahead * NG + lane, next);
        scales_of(next, ks_next, vs_next);
        page_ahead = page_of(ahead * NG + 32 + lane);
      }
      request(ahead, slot);
    }
    if (++slot == SLOTS) slot = 0, phase ^= 1;
    if (((n0 + NG) & 31) == 0) {
      ks_own = ks_next;
      vs_own = vs_next;
      lv_own = log2_of(vs_own);
      inv_own = inverse(vs_own);
      marked = __ballot_sync(0xffffffffu, vs_own < 0.f);
    }
  }
  pdl_trigger();       // (not earlier: CTAs of the next kernel beside these would leave its others unevenly spread over the SMs)
  if (!alive) {
    if (lane == 0) atomicExch(p.status, STATUS_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);          // copies still in flight land before the memory is used again
  }
  __syncthreads();                                             // the rings are no longer read
  float* m_s = reinterpret_cast<float*>(smem);                 // [NW + 1][RT], [RT] sums of the CTA
  float* l_s = m_s + (NW + 2) * RT;                            // [NW][RT]
  float* o_s = l_s + NW * RT;                                  // [NW][RT][HD]
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int x = 4; x < 32; x *= 2) l[b][r] += __shfl_xor_sync(0xffffffffu, l[b][r], x);
      const int row = 8 * b + 2 * t4 + r;
      if (row >= t.rows) continue;
      if (g == 0) {
        m_s[warp * RT + row] = m[b][r];
        l_s[warp * RT + row] = l[b][r];
      }
      float* at = o_s + ((size_t)warp * RT + row) * HD + g * C::VB;
#pragma unroll
      for (int n = 0; n < HD / 16; n += 2)
        *reinterpret_cast<float4*>(at + 2 * n) = make_float4(o[b][n][r], o[b][n][r + 2], o[b][n + 1][r], o[b][n + 1][r + 2]);
    }
  join<bf16, RT, NW>(p, t, kvh, part, parts, m_s, l_s, o_s);
}

// ---------------------------------------------------------------- launches
// How many CTAs share a tile's keys, a chunk for every warp at least: as many as make no more than `over` times what the chip holds.
template <typename K>
int parts_that_fit(K kernel, int over, long long ctas, long long chunks, int warps, size_t smem) {
  int parts = 1;
  for (int x = 2; x <= MAX_PARTS && chunks > (long long)(x - 1) * warps; ++x)
    if (ctas <= (long long)over * clusters_at_a_time(kernel, x, 32 * warps, smem)) parts = x;
  return parts;
}

template <typename T, int NP>
int launch_any(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  constexpr int RT = 4, NW = 4;
  const size_t smem = (size_t)(RT * p.hd + (2 * NW + 2) * RT + NW * RT * p.hd) * 4 + NW * 32 * (16 + 8);
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_any_kernel<T, NP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set = true;
  }
  // (Once what the chip holds.  24 / 8 heads of 256, us with once / twice: nine requests of 2,000 keys 209 / 285, of 1 to 4,002 304 / 205; of 48:
  // 45 / 53 and 71 / 46.)
  const int parts = parts_that_fit(kv8_attention_any_kernel<T, NP>, 1, tiles * p.kv_heads, (keys + 31) / 32, NW, smem);
  return launch_parts(kv8_attention_any_kernel<T, NP>, p, parts, tiles, 32 * NW, smem, stream);
}
template <typename T, int HD>
int launch_rows(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  constexpr int RT = 4, NW = 4, SMEM = ((2 * NW + 2) * RT + NW * RT * HD) * 4 + NW * 32 * 16;
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_rows_kernel<T, HD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set = true;
  }
  // (Twice what the chip holds: requests of a step differ in length, and the CTAs of short ones leave at once.  24 / 8 heads of 64, us with
  // once / twice: nine requests of 1 to 4,002 keys 28 / 23, eight of 100 to 8,000 37 / 33; nine of 2,000 25 / 31.)
  const int parts = parts_that_fit(kv8_attention_rows_kernel<T, HD>, 2, tiles * p.kv_heads, (keys + 31) / 32, NW, SMEM);
  return launch_parts(kv8_attention_rows_kernel<T, HD>, p, parts, tiles, 32 * NW, SMEM, stream);
}
template <typename T>
int dispatch_any(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  switch (p.hd) {
    case 32: return launch_rows<T, 32>(p, tiles, keys, stream);
    case 64: return launch_rows<T, 64>(p, tiles, keys, stream);
    case 128: return launch_rows<T, 128>(p, tiles, keys, stream);
  }
  switch ((p.hd + 63) / 64) {
    case 1: return launch_any<T, 1>(p, tiles, keys, stream);
    case 2: return launch_any<T, 2>(p, tiles, keys, stream);
    case 3: return launch_any<T, 3>(p, tiles, keys, stream);
    default: return launch_any<T, 4>(p, tiles, keys, stream);
  }
}

// Few tiles (a launch of few requests, tiles of 8 rows): one CTA of many warps for an SM, and a tile's keys shared by a cluster of
// them, as many as the chip holds at a time.  (Clusters of four-warp CTAs come to lie three or four on an SM and leave others empty: 4 requests of 32,000
// keys, 32 / 8 heads of 128, 55 us against 48.)  Many tiles: CTAs of four warps, several on an SM, so that one's beginning and end lie
// beside the others' work.  2,000 keys, 32 / 8 heads of 64, us by many warps / by four: 16 requests 20 / 29, 24 requests 31 / 25, 64 requests
// 57 / 43; with heads of 128 29 / 31, 41 / 36, 76 / 82.
template <int HD, int NB, int WARPS>
int launch_mma_of(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  using C = Mma<HD, WARPS>;
  constexpr int SMEM = C::smem(8 * NB);
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_mma_kernel<HD, NB, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_mma_kernel<HD, NB, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set = true;
  }
  CUtensorMap mk, mv;
  const long long rows = (long long)p.n_pages * p.kv_heads * p.page_size;
  constexpr CUtensorMapSwizzle SWIZZLE = HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (!group_map(&mk, p.k_pages, rows, HD, SWIZZLE) || !group_map(&mv, p.v_pages, rows, HD, SWIZZLE))
    GB_FAIL(GB_ERR_CUDA, "kv8_attention: cuTensorMapEncodeTiled failed (%lld rows of %d)", rows, HD);
  const long long chunks = (keys + C::CK - 1) / C::CK, ctas = tiles * p.kv_heads;
  int parts = 1;
  if (C::CTAS == 1)
    parts = parts_that_fit(kv8_attention_mma_kernel<HD, NB, WARPS>, 1, ctas, chunks, C::NW, SMEM);
  else if (NB == 1)
    while (parts < MAX_PARTS && ctas * parts * 2 <= 148 * C::CTAS && chunks >= (long long)parts * 2 * C::NW) parts *= 2;
  return launch_parts(kv8_attention_mma_kernel<HD, NB, WARPS>, p, parts, tiles, 32 * C::NW, SMEM, stream, mk, mv);
}
template <int HD>
int launch_mma(const Attn& p, bool rows16, long long tiles, long long keys, cudaStream_t stream) {
  if (rows16) return launch_mma_of<HD, 2, 4>(p, tiles, keys, stream);
  return tiles * p.kv_heads <= 148 ? launch_mma_of<HD, 1, HD == 64 ? 16 : 12>(p, tiles, keys, stream)
                                   : launch_mma_of<HD, 1, 4>(p, tiles, keys, stream);
}

}  // namespace

int kv8_attention_tcgen05(const kv8::Attn& p, cudaStream_t stream);      // kv8_attention_tcgen05.cu

GB_OP(gb_op_kv8_attention) {
  (void)flags;
  Attn p;
  p.step = step_of(ctx);
  if (p.step.n_tokens <= 0 || p.step.n_requests <= 0) return 0;
  p.q = reinterpret_cast<const void*>(a[0]);
  p.ldq = a[1];
  const int dtype = (int)a[2];
  p.out = reinterpret_cast<void*>(a[3]);
  p.ldo = a[4];
  p.k_pages = reinterpret_cast<const uint8_t*>(a[5]);
  p.v_pages = reinterpret_cast<const uint8_t*>(a[6]);
  p.k_scales = reinterpret_cast<const float*>(a[7]);
  p.v_scales = reinterpret_cast<const float*>(a[8]);
  p.n_pages = (int)a[9];
  p.page_size = (int)a[10];
  p.heads = (int)a[11];
  p.kv_heads = (int)a[12];
  p.hd = (int)a[13];
  p.block_table = reinterpret_cast<const int*>(a[14]);
  p.bt_stride = (int)a[15];
  p.window = a[16] > 0x3fffffff ? 0 : (int)a[16];               // (one that no context reaches is none, and sums with it stay in 32 bits)
  p.scale_log2 = (float)(f[0] * 1.4426950408889634);
  p.status = ctx->status;
  if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads != 0 || p.hd <= 0 || p.hd % 8 != 0 || p.hd > 256 || p.page_size <= 0 ||
      (long long)p.page_size * p.hd > 0x7fffffff)
    GB_FAIL(GB_ERR_ARG, "kv8_attention: %d heads, %d kv heads, head_dim %d, pages of %d: head sizes are multiples of 8 up to 256, a page's rows of a head fewer than 2^31 entries",
            p.heads, p.kv_heads, p.hd, p.page_size);
  if (dtype != GB_F32 && dtype != GB_BF16) GB_FAIL(GB_ERR_ARG, "kv8_attention: q and out are float32 or bfloat16");
  if (!isfinite(p.scale_log2)) GB_FAIL(GB_ERR_ARG, "kv8_attention: a scale of %g", f[0]);
  const int group = p.heads / p.kv_heads;
  p.page_shift = 0;
  while ((1 << p.page_shift) < p.page_size) ++p.page_shift;
  const bool mma = dtype == GB_BF16 && (p.hd == 64 || p.hd == 128) && p.page_size >= 16 &&
                   (1 << p.page_shift) == p.page_size && (long long)p.n_pages * p.kv_heads * p.page_size < 0x7fffffff &&
                   p.ldq % 8 == 0 && ((uintptr_t)p.q & 15) == 0;
  // Requests of more than FEW rows go to tcgen05, which takes 256 rows at a time; they have to lie on 16-byte boundaries.
  const bool wide = mma && (long long)p.step.max_q * group > FEW && group <= 64 && p.ldo % 8 == 0 && ((uintptr_t)p.out & 15) == 0;
  p.few = 0x7fffffff;
  // Where no request can have few rows (the shortest brings at least what the longest leave of the step's tokens) there is nothing for the
  // launch in front, which would be waited for: 8 requests of 16 tokens over 2,000 keys, 32 / 8 heads of 64, 32 us without it and 34
  // with it, two of 16 over 4,000 keys with heads of 128 33 and 40.
  const long long shortest = p.step.n_tokens - (p.step.n_requests - 1ll) * p.step.max_q;
  if (wide && (p.step.n_requests == 1 || shortest * group > FEW)) {
    p.few = 0;                                                 // (all of it, whatever a request brings)
    const int rc = kv8_attention_tcgen05(p, ctx->stream);
    return rc == GB_OK ? 1 : rc;
  }
  if (wide) p.few = FEW;
  // upper bound of the tiles: sum_r ceil(q_len_r * group / rt)
  auto tiles_of = [&](int rt) {
    return p.step.one_each ? (long long)p.step.n_requests * ((group + rt - 1) / rt)
                           : (long long)p.step.n_tokens * group / rt + p.step.n_requests;
  };
  int rt = mma ? 8 : 4;
  long long tiles = tiles_of(rt);
  // Tiles of 16 rows: half as many passes over the keys, once the tiles of 8 are more than the SMs hold at a time.  32 / 8 heads of 128,
  // 4,000 keys, 12 rows a request, us with 8 / 16: 32 requests 98 / 70; 8 requests 37 / 41, 2 requests 22 / 26.  (What stands beside
  // wide portions is single tokens as a rule, in groups of 8 heads at most.)
  const bool rows16 = mma && !wide && (long long)p.step.max_q * group > 8 && tiles * p.kv_heads > 148 * (p.hd == 64 ? 4 : 3);
  if (rows16) tiles = tiles_of(rt = 16);
  if (wide) {                                                  // (the requests that are left have FEW rows at most)
    const long long most = (long long)p.step.n_requests * ((FEW + rt - 1) / rt);
    tiles = tiles < most ? tiles : most;
  }
  if (tiles * p.kv_heads > 0x7fffffff / MAX_PARTS) GB_FAIL(GB_ERR_ARG, "kv8_attention: %lld tiles in one launch", tiles);
  const long long keys = p.window > 0 && p.window + rt < p.step.max_ctx ? p.window + rt : p.step.max_ctx;
  int rc;
  if (mma)
    rc = p.hd == 64 ? launch_mma<64>(p, rows16, tiles, keys, ctx->stream) : launch_mma<128>(p, rows16, tiles, keys, ctx->stream);
  else
    rc = dtype == GB_F32 ? dispatch_any<float>(p, tiles, keys, ctx->stream) : dispatch_any<bf16>(p, tiles, keys, ctx->stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_attention");
  if (!wide) return 1;
  // (The second launch waits for the first, like any kernel for the one in front: what the kernels before them wrote is sure to be seen
  // only behind a launch's own wait.  Portions of 500 and 37 tokens beside three single ones take 60 us so; beside each other, without
  // that wait, the two took 52.)
  rc = kv8_attention_tcgen05(p, ctx->stream);
  return rc == GB_OK ? 2 : rc;
}
