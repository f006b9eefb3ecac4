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
// f0 scale.  The step's requests come from its symbols.
#include "kv8.cuh"
#include "sm100.cuh"

namespace {

using namespace kv8;

struct Attn {
  const void* q; long long ldq;
  void* out; long long ldo;
  const uint8_t* k_pages; const uint8_t* v_pages; const float* k_scales; const float* v_scales;
  int n_pages, page_size, heads, kv_heads, hd, window;
  const int* block_table; int bt_stride;
  Step step;
  int parts;                         // CTAs of a cluster
  float scale_log2;                  // scale * log2(e)
  int* status;
};

constexpr int MAX_PARTS = 8;         // CTAs of a cluster that share a tile's keys

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
  t.r = find_piece(index, p.step.n_requests, true,
                   [&](int i) { return (p.step.q_len[i] * t.group + RT - 1) / RT; }, tile);
  if (t.r < 0) return false;
  const int qlen = p.step.q_len[t.r];
  const int tiles = (qlen * t.group + RT - 1) / RT;
  t.row0 = (tiles - 1 - tile) * RT;                            // the tiles with the most keys first
  t.rows = min(RT, qlen * t.group - t.row0);
  t.qstart = p.step.q_start[t.r];
  t.start = p.step.start_pos[t.r];
  t.hi = t.pos(t.rows - 1) + 1;
  const int first = t.pos(0);
  t.lo = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
  return true;
}

__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(p)), "r"(rank));
  return a;
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
          from_f32<T>(acc / cl[r]);
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
    reinterpret_cast<T*>(p.out)[(size_t)(t.qstart + tok) * p.ldo + (size_t)(kvh * t.group + g) * hd + d] = from_f32<T>(acc / sum);
  }
  sm100::cluster_sync_all();                                   // nobody leaves while another CTA reads its share
}

// ---------------------------------------------------------------- any type, head size and page size
// A warp takes chunks of 32 keys: for the scores a lane has a key, for the output it has pairs of columns.
template <typename T, int NP>
__global__ void __launch_bounds__(128) kv8_attention_any_kernel(const Attn p) {
  constexpr int RT = 4, NW = 4;
  extern __shared__ __align__(16) float sm[];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.hd;
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;
  Tile t;
  if (!find_tile<RT>(p, unit / p.kv_heads, t)) return;          // (the same for every CTA of a cluster)
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

// ---------------------------------------------------------------- bfloat16 on mma.sync
// Tiles of 16 rows.  K and V stay in 8 bits until they are operands: a lane copies the very bytes of its mma fragments from
// the pages into shared memory (cp.async, a ring of STAGES chunks per warp, no barrier but the warp's), and turns them into
// bfloat16 with shifts and masks.  Which entry of a head stands at which place of the contraction is free, as long as q and
// K agree, and which column of the output belongs to which place of the mma, too: so the places are chosen such that
//   - of K, lane (g, t) = (lane / 4, lane % 4) holds hd/4 contiguous bytes of key g of a tile of eight keys, four bytes for
//     each step of 16 entries (bytes 0, 2 in one register, 1, 3 in the other);
//   - of V, it holds hd/8 contiguous bytes (columns g hd/8 ...) of keys 2t, 2t+1, 2t+8, 2t+9 of 16 keys.
// The bits s eeee mmm of a number, moved to s 0000eeee mmm0000 of a bfloat16, stand for number * 2^-120 (subnormal numbers
// included).  The powers of two that are missing go where they are exact and cost nothing: q is multiplied by 2^60 (of q up
// to 2^67, nothing is lost), the scores by 2^60 and the page's scale, the weights by 2^60 and the page's scale, and the
// output by 2^60 at the end.
// The weights are rounded to bfloat16 for the second product (2^-8 of a weight at most, the same as a bfloat16 cache gives);
// their sum is of the 32-bit weights.
// Bound by memory from some 4,000 keys a launch's CTA on, below by the chain of trips (metadata, page ids, keys).
template <int HD> struct Mma {
  static constexpr int RT = 16, NW = 4, STAGES = 4;
  static constexpr int CK = HD <= 64 ? 32 : 16;                // keys of a chunk
  static constexpr int NT = CK / 8;                            // tiles of eight keys in it
  static constexpr int KB = HD / 4, VB = HD / 8;               // bytes of a lane's piece of a key, of a value
  static constexpr int KP = KB % 16 == 0 ? 16 : 8, VP = VB % 16 == 0 ? 16 : VB % 8 == 0 ? 8 : 4;     // bytes of a copy
  static constexpr int K_STAGE = CK * HD, V_STAGE = CK * HD, META = 2 * NT * 4;
  static constexpr int STAGE = K_STAGE + V_STAGE + (META + 15) / 16 * 16;
  static constexpr int JOIN = ((2 * NW + 2) * RT + NW * RT * HD) * 4;
  static constexpr int RING = NW * STAGES * STAGE;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t smem, const void* gmem, bool valid) {
  const int n = valid ? BYTES : 0;                             // 0: the destination is filled with zeros
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem), "l"(gmem), "r"(n), "n"(BYTES) : "memory");
}
template <int WORDS>
__device__ __forceinline__ void ld_words(uint32_t smem, uint32_t* w) {
  if constexpr (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(smem));
  else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(smem));
  else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(smem));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {                // relative error 2^-22; -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Bytes 0 and 2 (1 and 3) of a word as two bfloat16, times 2^-120.
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return ((w << 4) & 0x07f007f0u) | ((w << 8) & 0x80008000u); }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u); }
// 0xff in the bytes that are NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 255u; }

constexpr float TWO_60 = 1152921504606846976.f;

template <int HD>
__global__ void __launch_bounds__(128, 3) kv8_attention_mma_kernel(const Attn p) {
  using C = Mma<HD>;
  constexpr int RT = C::RT, NW = C::NW, NT = C::NT, CK = C::CK, KW = C::KB / 4, VW = C::VB / 4;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;
  Tile t;
  if (!find_tile<RT>(p, unit / p.kv_heads, t)) return;         // (the same for every CTA of a cluster)
  const int c_lo = t.lo / CK, chunks = (t.hi + CK - 1) / CK - c_lo;
  const int parts = max(1, min(p.parts, (chunks + NW - 1) / NW));
  if (part >= parts) return;                                   // (a thread that has left counts as arrived at the cluster's barriers)
  const int* bt = p.block_table + (size_t)t.r * p.bt_stride;
  const int stride = parts * NW, first = part * NW + warp;

  // Lane i looks up the page of tile i of a chunk: id, or -1 where nothing of the tile is visible.
  constexpr int NONE = -1, BAD = -2;
  auto lookup = [&](int c) {
    const int j = (c_lo + c) * CK + lane * 8;
    if (lane >= NT || c >= chunks || j >= t.hi || j + 7 < t.lo) return NONE;
    const int page = bt[j / p.page_size];
    return page >= 0 && page < p.n_pages ? page : BAD;
  };
  const uint32_t ring = sm100::smem_u32(smem) + (uint32_t)(warp * C::STAGES * C::STAGE);
  // Requests chunk c into stage `s`; `page` from lookup(c).  A tile without a page is zeros under a scale of 0, which no
  // page has: none of its keys is visible.
  auto request = [&](int c, int s, int page) {
    const uint32_t k_at = ring + (uint32_t)(s * C::STAGE), v_at = k_at + C::K_STAGE, m_at = v_at + C::V_STAGE;
    const int j = (c_lo + c) * CK + lane * 8;
    long long row = -1;
    if (lane < NT) {
      const bool valid = page >= 0;
      if (page == BAD) atomicExch(p.status, STATUS_BAD_PAGE_READ);
      const size_t ph = valid ? (size_t)page * p.kv_heads + kvh : 0;
      if (valid) row = ((long long)ph * p.page_size + j % p.page_size) * HD;
      cp_async<4>(m_at + lane * 4, p.k_scales + ph, valid);
      cp_async<4>(m_at + (NT + lane) * 4, p.v_scales + ph, valid);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const long long r = __shfl_sync(0xffffffffu, row, i);
      const uint8_t* kp = p.k_pages + (r < 0 ? 0 : r + g * HD + t4 * C::KB);
#pragma unroll
      for (int x = 0; x < C::KB / C::KP; ++x)
        cp_async<C::KP>(k_at + (uint32_t)(((i * (C::KB / C::KP) + x) * 32 + lane) * C::KP), kp + x * C::KP, r >= 0);
      // keys 2t, 2t + 1 of the tile
      const uint8_t* vp = p.v_pages + (r < 0 ? 0 : r + 2 * t4 * HD + g * C::VB);
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int x = 0; x < C::VB / C::VP; ++x)
          cp_async<C::VP>(v_at + (uint32_t)((((2 * i + y) * (C::VB / C::VP) + x) * 32 + lane) * C::VP), vp + (r < 0 ? 0 : y * HD + x * C::VP), r >= 0);
    }
  };
  int pages[C::STAGES];
#pragma unroll
  for (int s = 0; s < C::STAGES; ++s) pages[s] = lookup(first + s * stride);
  pdl_wait();
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) {
    if (first + s * stride < chunks) request(first + s * stride, s, pages[s]);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  int page_next = pages[C::STAGES - 1];

  // q: rows g and g + 8, entries t4 * KB ... + KB, times 2^60
  uint32_t qa[HD / 16][4];
  int rpos[2];
  const bool upper = t.rows > 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = g + 8 * i;
    rpos[i] = -1;                                              // (a row that does not exist sees nothing)
    uint32_t w[HD / 8];
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) w[x] = 0u;
    if (row < t.rows) {
      rpos[i] = t.pos(row);
      const int tok = (t.row0 + row) / t.group, h = (t.row0 + row) - tok * t.group;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.q) + (size_t)(t.qstart + tok) * p.ldq +
                                                        (size_t)(kvh * t.group + h) * HD + t4 * C::KB);
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) {
        const uint4 u = src[x];
        w[4 * x] = u.x; w[4 * x + 1] = u.y; w[4 * x + 2] = u.z; w[4 * x + 3] = u.w;
      }
      const __nv_bfloat162 up = __floats2bfloat162_rn(TWO_60, TWO_60);
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) {
        const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w[x]), up);
        w[x] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      qa[kk][i] = __byte_perm(w[2 * kk], w[2 * kk + 1], 0x5410);       // entries 0, 2 of four
      qa[kk][2 + i] = __byte_perm(w[2 * kk], w[2 * kk + 1], 0x7632);   // entries 1, 3
    }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  const int pos_first = t.pos(0), pos_last = t.pos(t.rows - 1);

  int stage = 0;
  for (int c = first; c < chunks; c += stride) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncwarp();                                              // the chunk has landed, and the stage before is free
    {
      const int ahead = c + (C::STAGES - 1) * stride;
      if (ahead < chunks) request(ahead, stage == 0 ? C::STAGES - 1 : stage - 1, page_next);
      asm volatile("cp.async.commit_group;" ::: "memory");
      page_next = lookup(ahead + stride);
    }
    const uint32_t k_at = ring + (uint32_t)(stage * C::STAGE), v_at = k_at + C::K_STAGE, m_at = v_at + C::V_STAGE;
    stage = stage == C::STAGES - 1 ? 0 : stage + 1;
    float s[NT][4], vs[NT];
    float top[2] = {-INFINITY, -INFINITY};
    bool careful = false;                                      // some page of the chunk has NaN among its values
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float ks;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks) : "r"(m_at + i * 4));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs[i]) : "r"(m_at + (NT + i) * 4));
      careful |= vs[i] < 0.f;
      vs[i] = fabsf(vs[i]) * TWO_60;
      uint32_t w[KW];
#pragma unroll
      for (int x = 0; x < C::KB / C::KP; ++x)
        ld_words<C::KP / 4>(k_at + (uint32_t)(((i * (C::KB / C::KP) + x) * 32 + lane) * C::KP), w + x * (C::KP / 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) mma_bf16(s[i], qa[kk], even_bytes(w[kk]), odd_bytes(w[kk]));
      const float factor = fabsf(ks) * (TWO_60 * p.scale_log2);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] *= factor;
      if (ks < 0.f) {
        // keys with a NaN: lanes 4k .. 4k + 3 hold key k; this lane's columns are keys 2t, 2t + 1
        uint32_t any = 0u;
#pragma unroll
        for (int kk = 0; kk < KW; ++kk) any |= nan_bytes(w[kk]);
        const uint32_t keys = __ballot_sync(0xffffffffu, any != 0u) >> (8 * t4);
        if (keys & 0xfu) s[i][0] = s[i][2] = __int_as_float(0x7fffffff);
        if (keys & 0xf0u) s[i][1] = s[i][3] = __int_as_float(0x7fffffff);
      }
      const int j0 = (c_lo + c) * CK + 8 * i;
      const bool full = ks != 0.f && j0 + 7 <= pos_first && (p.window <= 0 || j0 + p.window > pos_last);
      if (!full) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 2 * t4 + (e & 1), pos = rpos[e >> 1];
          const bool seen = ks != 0.f && j <= pos && (p.window <= 0 || j + p.window > pos);
          s[i][e] = seen ? s[i][e] : -INFINITY;
        }
      }
      top[0] = fmaxf(top[0], fmaxf(s[i][0], s[i][1]));
      if (upper) top[1] = fmaxf(top[1], fmaxf(s[i][2], s[i][3]));
    }
    // The maximum in use follows a row's only when it would fall behind by more than 2^8: weights stay below 256, and most
    // chunks leave the output as it is.
    float corr[2] = {1.f, 1.f}, use[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r == 0 || upper) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        if (top[r] > m[r] + 8.f || (m[r] == -INFINITY && top[r] > -INFINITY)) {
          corr[r] = ex2(m[r] - top[r]);                        // 0 when nothing was seen before
          m[r] = top[r];
          l[r] *= corr[r];
        }
      }
      use[r] = m[r] == -INFINITY ? 0.f : m[r];
    }
    if (corr[0] != 1.f || corr[1] != 1.f) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        o[n][0] *= corr[0]; o[n][1] *= corr[0];
        o[n][2] *= corr[1]; o[n][3] *= corr[1];
      }
    }
#pragma unroll
    for (int x = 0; x < NT / 2; ++x) {                         // 16 keys
      uint32_t a[4], see[4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float* sv = s[2 * x + y];
        const float e0 = ex2(sv[0] - use[0]), e1 = ex2(sv[1] - use[0]);
        l[0] += e0 + e1;
        a[2 * y] = pack_bf16(e0 * vs[2 * x + y], e1 * vs[2 * x + y]);
        a[2 * y + 1] = 0u;
        if (upper) {
          const float e2 = ex2(sv[2] - use[1]), e3 = ex2(sv[3] - use[1]);
          l[1] += e2 + e3;
          a[2 * y + 1] = pack_bf16(e2 * vs[2 * x + y], e3 * vs[2 * x + y]);
        }
      }
      uint32_t v[4][VW];
#pragma unroll
      for (int y = 0; y < 4; ++y)                              // keys 2t, 2t + 1 of the first tile, then of the second
#pragma unroll
        for (int z = 0; z < C::VB / C::VP; ++z)
          ld_words<C::VP / 4>(v_at + (uint32_t)((((4 * x + y) * (C::VB / C::VP) + z) * 32 + lane) * C::VP), v[y] + z * (C::VP / 4));
      if (careful) {
        // A NaN reaches the rows that see its key and no other: the numbers go in as 0, and rows (1: sees) times columns
        // (1: NaN) tell where the output is NaN.
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float* sv = s[2 * x + y];
          see[2 * y] = pack_bf16(sv[0] == -INFINITY ? 0.f : 1.f, sv[1] == -INFINITY ? 0.f : 1.f);
          see[2 * y + 1] = pack_bf16(sv[2] == -INFINITY ? 0.f : 1.f, sv[3] == -INFINITY ? 0.f : 1.f);
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t bad[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            bad[y] = nan_bytes(v[y][w]);
            v[y][w] &= ~bad[y];
          }
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const uint32_t lo = __byte_perm(bad[0], bad[1], z < 2 ? 0x5410 : 0x7632), hi = __byte_perm(bad[2], bad[3], z < 2 ? 0x5410 : 0x7632);
            float n[4] = {0.f, 0.f, 0.f, 0.f};
            mma_bf16(n, see, (z & 1 ? lo : lo << 8) & 0x3f003f00u, (z & 1 ? hi : hi << 8) & 0x3f003f00u);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n[e] > 0.f) o[4 * w + z][e] = __int_as_float(0x7fffffff);
          }
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t l0 = __byte_perm(v[0][w], v[1][w], 0x5410), l1 = __byte_perm(v[0][w], v[1][w], 0x7632);
        const uint32_t h0 = __byte_perm(v[2][w], v[3][w], 0x5410), h1 = __byte_perm(v[2][w], v[3][w], 0x7632);
        mma_bf16(o[4 * w], a, even_bytes(l0), even_bytes(h0));
        mma_bf16(o[4 * w + 1], a, odd_bytes(l0), odd_bytes(h0));
        mma_bf16(o[4 * w + 2], a, even_bytes(l1), even_bytes(h1));
        mma_bf16(o[4 * w + 3], a, odd_bytes(l1), odd_bytes(h1));
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                             // the rings are no longer read
  float* m_s = reinterpret_cast<float*>(smem);                 // [NW + 1][RT], [RT] sums of the CTA
  float* l_s = m_s + (NW + 2) * RT;                            // [NW][RT]
  float* o_s = l_s + NW * RT;                                  // [NW][RT][HD]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = g + 8 * r;
    if (row >= t.rows) continue;
    if (t4 == 0) {
      m_s[warp * RT + row] = m[r];
      l_s[warp * RT + row] = l[r];
    }
    float* at = o_s + ((size_t)warp * RT + row) * HD;
#pragma unroll
    for (int n = 0; n < HD / 8; n += 4)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float4*>(at + (2 * t4 + e) * C::VB + n) =
            make_float4(o[n][2 * r + e] * TWO_60, o[n + 1][2 * r + e] * TWO_60, o[n + 2][2 * r + e] * TWO_60,
                        o[n + 3][2 * r + e] * TWO_60);
  }
  join<bf16, RT, NW>(p, t, kvh, part, parts, m_s, l_s, o_s);
}

// ---------------------------------------------------------------- launches
// Launches `kernel` over the tiles, their kv heads and parts (x in this order, parts fastest: the tiles with the most keys of
// every head start first), a tile's parts as a cluster.
template <typename K>
int launch_parts(K kernel, Attn p, int parts, long long tiles, int threads, size_t smem, cudaStream_t stream) {
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
  GB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return GB_OK;
}

// How many CTAs share a tile's keys: as many as fill `slots` places on the GPU, each with a chunk for every warp.
int key_parts(long long ctas, long long slots, long long chunks, int warps) {
  int parts = 1;
  while (parts < MAX_PARTS && ctas * parts * 2 <= slots && chunks >= (long long)parts * 2 * warps) parts *= 2;
  return parts;
}

template <typename T, int NP>
int launch_any(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  constexpr int RT = 4, NW = 4;
  const size_t smem = (size_t)(RT * p.hd + (2 * NW + 2) * RT + NW * RT * p.hd) * 4 + NW * 32 * (16 + 8);
  return launch_parts(kv8_attention_any_kernel<T, NP>, p, key_parts(tiles * p.kv_heads, 148 * 4, (keys + 31) / 32, NW), tiles, 32 * NW,
                      smem, stream);
}
template <typename T>
int dispatch_any(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  switch ((p.hd + 63) / 64) {
    case 1: return launch_any<T, 1>(p, tiles, keys, stream);
    case 2: return launch_any<T, 2>(p, tiles, keys, stream);
    case 3: return launch_any<T, 3>(p, tiles, keys, stream);
    default: return launch_any<T, 4>(p, tiles, keys, stream);
  }
}

template <int HD>
int launch_mma(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  using C = Mma<HD>;
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_mma_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_set = true;
  }
  return launch_parts(kv8_attention_mma_kernel<HD>, p, key_parts(tiles * p.kv_heads, 148 * 3, (keys + C::CK - 1) / C::CK, C::NW), tiles,
                      32 * C::NW, C::SMEM, stream);
}

}  // namespace

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
  p.window = (int)a[16];
  p.scale_log2 = (float)(f[0] * 1.4426950408889634);
  p.status = ctx->status;
  if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads != 0 || p.hd <= 0 || p.hd % 8 != 0 || p.hd > 256 || p.page_size <= 0)
    GB_FAIL(GB_ERR_ARG, "kv8_attention: %d heads, %d kv heads, head_dim %d, pages of %d: head sizes are multiples of 8 up to 256",
            p.heads, p.kv_heads, p.hd, p.page_size);
  if (dtype != GB_F32 && dtype != GB_BF16) GB_FAIL(GB_ERR_ARG, "kv8_attention: q and out are float32 or bfloat16");
  const int group = p.heads / p.kv_heads;
  const bool mma = dtype == GB_BF16 && (p.hd == 32 || p.hd == 64 || p.hd == 96 || p.hd == 128) && p.page_size % 8 == 0 &&
                   p.ldq % 8 == 0 && ((uintptr_t)p.q & 15) == 0;
  // upper bound of the tiles: sum_r ceil(q_len_r * group / rt)
  const int rt = mma ? 16 : 4;
  const long long tiles = p.step.one_each ? (long long)p.step.n_requests * ((group + rt - 1) / rt)
                                          : (long long)p.step.n_tokens * group / rt + p.step.n_requests;
  if (tiles * p.kv_heads > 0x7fffffff / MAX_PARTS) GB_FAIL(GB_ERR_ARG, "kv8_attention: %lld tiles in one launch", tiles);
  const long long keys = p.window > 0 && p.window + rt < p.step.max_ctx ? p.window + rt : p.step.max_ctx;
  int rc;
  if (mma)
    rc = p.hd == 32 ? launch_mma<32>(p, tiles, keys, ctx->stream) : p.hd == 64 ? launch_mma<64>(p, tiles, keys, ctx->stream)
         : p.hd == 96 ? launch_mma<96>(p, tiles, keys, ctx->stream) : launch_mma<128>(p, tiles, keys, ctx->stream);
  else
    rc = dtype == GB_F32 ? dispatch_any<float>(p, tiles, keys, ctx->stream) : dispatch_any<bf16>(p, tiles, keys, ctx->stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_attention");
  return 1;
}
