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
  // upper bound of the tiles: sum_r ceil(q_len_r * group / RT)
  constexpr int RT = 4;
  const long long tiles = p.step.one_each ? (long long)p.step.n_requests * ((group + RT - 1) / RT)
                                          : (long long)p.step.n_tokens * group / RT + p.step.n_requests;
  if (tiles * p.kv_heads > 0x7fffffff / MAX_PARTS) GB_FAIL(GB_ERR_ARG, "kv8_attention: %lld tiles in one launch", tiles);
  const long long keys = p.window > 0 && p.window + RT < p.step.max_ctx ? p.window + RT : p.step.max_ctx;
  const int rc = dtype == GB_F32 ? dispatch_any<float>(p, tiles, keys, ctx->stream) : dispatch_any<bf16>(p, tiles, keys, ctx->stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_attention");
  return 1;
}
