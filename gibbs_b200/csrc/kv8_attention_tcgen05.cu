// Attention of prompt portions over the 8-bit paged cache (kv8.cuh) on the 5th generation tensor cores, for bfloat16 rows with
// heads of 64 or 128 entries: the formula of kv8_attention.cu, on tcgen05.mma with the accumulators in tensor memory.
//
// A CTA takes 256 consecutive (token, head of a kv head's group) rows of one request, as two tiles of 128, and walks their
// visible keys in tiles of 128:
//
//   warps 8-10   bring K_j and V_j: from the pages by cp.async, some items ahead, then e4m3 to f16, which holds every number exactly,
//                into a ring of swizzled tiles; K_j brings the scales of its pages along
//   warp 11      one thread issues S = Q K_j^T for both row tiles and, when a tile's weights are there, O += P V_j and the next S
//   warps 0-7    a thread has a row: reads S from tensor memory, scales, masks, running maximum and sum in 32 bits, writes the
//                weights in f16 to tensor memory, from where they are the A operand of the second product
//
// The two row tiles take turns: while one is in its softmax the other's products run, and both use the same converted K and V.  (Products
// issued as either tile is ready, without that order: 48 us against 47 at 2,048 tokens, 345 against 327 at 8,192.)
//
// 2,048 tokens, 32 / 8 heads of 64: 45.1 us, 381 TFLOP/s; 8,192 tokens, 16 / 4 heads of 128: 316 us, 870 TFLOP/s.  What bounds it, from
// copies that left work out when it took 47 and 327: heads of 64 take 45 us without the 2^x, 40 without any softmax, 34 without conversion and loads either, so it is
// the hand-overs of a key tile (scores to registers, weights back, product) and a CTA's beginning and end; heads of 128 take 301 us
// without conversion, 296 without softmax and 229 without both.  The special-function unit is at 37 % (a share of the 2^x by a
// polynomial is slower: 49 and 341 us).  Weights go over in halves: whole they take 51 us, in quarters 50.
//
// Scales, as in the kernel for few rows: q's row under the power of two that brings its largest magnitude to 2^14; a score
// times the inverse and the scale of K's page; the scale of V's page in the exponent, x_j = score_j + log2(scale_j), weights
// 2^(x_j - M + 12) in f16 and their sum divided by scale_j, in 32 bits.
//
// Where a launch has few CTAs (a portion of some hundred tokens behind a long context), a cluster shares a tile's keys, and
// joins the shares through distributed shared memory.
#include "kv8_attention.cuh"
#include "sm100.cuh"

namespace {

using namespace kv8;
using namespace sm100;

constexpr int ROWS = 128, KEYS = 128, GROUPS = KEYS / 16;
constexpr int THREADS = 384;                                  // 8 softmax warps, 3 that convert, 1 that issues: 168 registers a thread
constexpr int CONVERTERS = 96;
constexpr int AFTER = 0;
constexpr int META = 4;                                       // tiles whose scales are kept

template <int HD> struct Cfg {
  static constexpr int SUB = HD / 64;                         // 64-column sub-tiles
  // Tensor memory has room for weights of their own beside S and O of two row tiles at head_dim 64: the next S then goes out as soon
  // as S has been read.  At 128 the weights lie over S, and the next S goes out behind the product that reads them.
  static constexpr bool APART = HD == 64;
  static constexpr int RING = APART ? 4 : 3;                  // f16 tiles of K or V
  static constexpr int STAGES = APART ? 4 : 3;                // tiles of K or V as they come
  static constexpr int RAW_TILE = KEYS * HD;
  static constexpr int Q_TILE = ROWS * HD * 2, KV_TILE = KEYS * HD * 2;
  static constexpr int NAN_BYTES = META * KEYS * HD / 8;      // which values of a tile are NaN, a bit each
  static constexpr int SHARE = 2 * ROWS * HD * 4 + 2 * ROWS * 8;
  static constexpr int OPERANDS = 2 * Q_TILE + RING * KV_TILE;
  static constexpr int SMEM = OPERANDS + STAGES * RAW_TILE + NAN_BYTES + 1024;
  static_assert(SHARE <= OPERANDS, "a share of O and its (m, l) fit over the operands");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// A and B in f16, f32 accumulators; B with its N index contiguous for O = P V.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__host__ __device__ constexpr uint32_t idesc_f16_b_mn(int m, int n) { return idesc_f16(m, n) | (1u << 16); }

// D[tmem] (+)= A[tmem] * B[smem]: a lane of tensor memory has a row of A, two entries a column.
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_16_issue(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void cp_async_16(uint32_t smem, const void* gmem, int n) {            // n = 0: filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(n) : "memory");
}
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float2 ld_cluster_f2(const float2* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(const float4* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(p, rank)) : "memory");
  return v;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) kv8_attention_tcgen05_kernel(const Attn p) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full, kv_full[C::RING], kv_empty[C::RING], s_full[2], s_free[2], p_full[2][2], o_done[2];
  __shared__ int marks[META];                                 // whether any page of the tile has NaN among its values
  __shared__ float4 meta[META][GROUPS];                       // of a group of sixteen keys: |scale of K|, log2 and inverse of V's scale,
                                                              // 1 where V's page holds NaN
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = base;                                         // [2][SUB][128 rows][128 B]
  uint8_t* skv = sq + 2 * C::Q_TILE;                          // [RING][SUB][128 keys][128 B]
  uint8_t* sraw = skv + C::RING * C::KV_TILE;                 // [STAGES][128 keys][HD]
  uint32_t* snan = reinterpret_cast<uint32_t*>(sraw + C::STAGES * C::RAW_TILE);          // [META][128 keys][HD / 32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.kv_heads, tpt = ROWS / group;  // tokens of a row tile
  const int part = (int)blockIdx.x % p.parts, unit = (int)blockIdx.x / p.parts, kvh = unit % p.kv_heads;

  int tile = 0;
  const Request q = find_piece(unit / p.kv_heads, p.step, true, [&](int n, int) {
    return n * group > p.few ? (n + 2 * tpt - 1) / (2 * tpt) : 0;
  }, tile);
  if (q.r < 0) return leave();                                 // (the same for every CTA of a cluster)
  const int r = q.r, qlen = q.n, start = q.before, qstart = q.start;
  tile = (qlen + 2 * tpt - 1) / (2 * tpt) - 1 - tile;          // the tiles with the most keys first
  const int tok0 = tile * 2 * tpt, n_tok = min(2 * tpt, qlen - tok0);
  const int hi = start + tok0 + n_tok;                         // keys < hi may be visible
  const int first = start + tok0;
  const int lo = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
  int t_lo = lo / KEYS, t_hi = (hi + KEYS - 1) / KEYS;
  const int parts = max(1, min(p.parts, (t_hi - t_lo) / 2));
  if (part >= parts) return;                                   // (a thread that has left counts as arrived at the cluster's barriers)
  {
    const int whole = t_hi - t_lo, from = t_lo;
    t_lo = from + whole * part / parts;
    t_hi = from + whole * (part + 1) / parts;
  }
  // key tiles of each row tile (the first one may see fewer, the second may have no rows)
  int n_x[2];
  n_x[0] = max(0, min(t_hi, (start + min(tok0 + tpt, tok0 + n_tok) + KEYS - 1) / KEYS) - t_lo);
  n_x[1] = n_tok > tpt ? t_hi - t_lo : 0;
  const int n = max(n_x[0], n_x[1]);

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 8);
    for (int s = 0; s < C::RING; ++s) {
      mbar_init(&kv_full[s], CONVERTERS / 32);
      mbar_init(&kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&s_free[x], 4);
      mbar_init(&p_full[x][0], 4);                             // (a barrier for each half of a tile's weights: a warp may be a half ahead)
      mbar_init(&p_full[x][1], 4);
      mbar_init(&o_done[x], 1);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  // All of tensor memory, but not while waiting for another kernel: a CTA of that one which has started and not taken its columns yet
  // would wait for these.
  pdl_wait();
  if (warp == 11) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t tmem_s[2] = {tmem, tmem + KEYS}, tmem_o[2] = {tmem + 2 * KEYS, tmem + 2 * KEYS + HD};
  const uint32_t tmem_p[2] = {C::APART ? tmem + 2 * KEYS + 2 * HD : tmem, C::APART ? tmem + 2 * KEYS + 2 * HD + KEYS / 2 : tmem + KEYS};

  if (warp >= 8 && warp < 11) {
    // ---- K and V: pages -> f16 tiles ----
    // Item 2 j is K of the CTA's key tile j, item 2 j + 1 its V.  A warp has whole groups of sixteen keys, which lie in one page and
    // there one behind the other: one address for a group, and the rest are constants.  A lane copies the very pieces that it will
    // convert (cp.async, STAGES items ahead), so nothing but its own copies is waited for.  (By TMA, a copy a group, the copies of an
    // item took a warp longer to issue than its conversion.)
    constexpr int PIECES = HD / 16, PER = 16 * PIECES / 32;   // 16-byte pieces of a row; of a group, for a lane
    constexpr int ROWS_STEP = 32 / PIECES;                    // rows from one of a lane's pieces to the next
    constexpr int MINE = (GROUPS + CONVERTERS / 32 - 1) / (CONVERTERS / 32);
    // (The f16 of pieces 4..7 go to the banks of those of pieces 0..3, a sub-tile further: eight lanes that store together have the lower
    // pieces of one row and the upper ones of its neighbour, which the swizzle puts elsewhere.)
    const int w0 = warp - 8, piece = lane % PIECES, row_in = (lane / PIECES) ^ (piece >> 2);     // groups w0, w0 + 3, w0 + 6 < 8
    const int spot = (row_in * PIECES + piece) * 16;          // of this lane among the 512 bytes of a warp's copy
    const int* bt = p.block_table + (size_t)r * p.bt_stride;
    // lane i < 8: page of group i of a tile, -1 where nothing of it is visible (and in the other lanes); as it comes from the table,
    // and looked at only when it is needed, which is after its trip
    auto page_of = [&](int j) {
      const int key = (t_lo + j) * KEYS + lane * 16;
      return (lane >= GROUPS || j >= n || key >= hi || key + 15 < lo) ? -1 : page_id(bt + (key >> p.page_shift));
    };
    auto checked = [&](int page) {
      if (page < p.n_pages) return page;
      if (warp == 8) atomicExch(p.status, STATUS_BAD_PAGE_READ);
      return -1;
    };
    uint8_t* mine = sraw + spot;
    const uint32_t mine_at = smem_u32(mine) + w0 * 16 * HD;
    const size_t head = (size_t)kvh << p.page_shift;
    size_t at[MINE];                                          // where this warp's groups of the last tile asked for lie in the pool
    int rows[MINE];                                            // how many rows from this lane's first on are there
    // Asks for an item, K of a tile and then its V; what is not visible, or behind the context (which holds anything, and 0 * NaN is
    // not 0), comes as zeros.
    auto request = [&](int it, int page) {
      if (it < 2 * n) {
        if (!(it & 1)) {
          const int key0 = (t_lo + (it >> 1)) * KEYS;
#pragma unroll
          for (int y = 0; y < MINE; ++y) {
            const int g = w0 + y * (CONVERTERS / 32), pg = __shfl_sync(0xffffffffu, page, g), key = key0 + 16 * g;
            at[y] = pg < 0 ? 0 : ((((size_t)pg * p.kv_heads) << p.page_shift) + head + (key & (p.page_size - 1))) * HD;
            rows[y] = pg < 0 || g >= GROUPS ? 0 : hi - key - row_in;
          }
        }
        const uint8_t* pool = ((it & 1) ? p.v_pages : p.k_pages) + spot;
        const uint32_t dst = mine_at + (uint32_t)((it % C::STAGES) * C::RAW_TILE);
#pragma unroll
        for (int y = 0; y < MINE; ++y) {
          if (w0 + y * (CONVERTERS / 32) >= GROUPS) continue;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            cp_async_16(dst + (uint32_t)(y * (CONVERTERS / 32) * 16 * HD + i * 512), pool + at[y] + i * 512, rows[y] > i * ROWS_STEP ? 16 : 0);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float ks = 0.f, vs = 0.f, ks_next, vs_next;                // scales of this lane's group, in this tile and in the next
    auto scales = [&](int page, float& k, float& v) {
      k = v = 0.f;
      if (page >= 0) {
        k = p.k_scales[(size_t)page * p.kv_heads + kvh];
        v = p.v_scales[(size_t)page * p.kv_heads + kvh];
      }
    };
    // pages of tile j, j + 1, ... (a request goes out at most STAGES items, two tiles, ahead)
    int pages[4] = {page_of(0), page_of(1), page_of(2), page_of(3)};
#pragma unroll
    for (int i = 0; i < 3; ++i) pages[i] = checked(pages[i]);
#pragma unroll
    for (int it = 0; it < C::STAGES; ++it) request(it, pages[it >> 1]);
    scales(pages[0], ks, vs);
    for (int j = 0; j < n; ++j) {
      scales(pages[1], ks_next, vs_next);                      // asked for a tile ahead
      const uint32_t marked = __ballot_sync(0xffffffffu, lane < GROUPS && vs < 0.f);
      if (warp == 8 && lane == 0) marks[j % META] = marked != 0u;
      if (warp == 8 && lane < GROUPS)
        meta[j % META][lane] = ks == 0.f ? make_float4(0.f, -INFINITY, 0.f, 0.f)
                                         : make_float4(fabsf(ks), log2_of(vs), inverse(vs), vs < 0.f ? 1.f : 0.f);
      if (marked) {
        // Which values of the tile are NaN: rows that see their key have NaN there (the products get 0 instead).  The rows' threads
        // look at it with the scores, which may be ahead of the values: it goes out with the keys.
        asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
        uint16_t* at = reinterpret_cast<uint16_t*>(snan) + (size_t)(j % META) * KEYS * PIECES;
#pragma unroll 1
        for (int g = w0; g < GROUPS; g += CONVERTERS / 32)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(mine + (size_t)((2 * j + 1) % C::STAGES) * C::RAW_TILE + g * 16 * HD + i * 512);
            const uint32_t w[4] = {nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w)};
            uint32_t which = 0u;
#pragma unroll
            for (int x = 0; x < 4; ++x) which |= ((w[x] & 1u) | ((w[x] >> 7) & 2u) | ((w[x] >> 14) & 4u) | ((w[x] >> 21) & 8u)) << (4 * x);
            at[(16 * g + row_in + i * ROWS_STEP) * PIECES + piece] = (uint16_t)which;
          }
      }
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        const int it = 2 * j + kv, s = it % C::RING;
        asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
        uint4 w[MINE][PER];
#pragma unroll
        for (int y = 0; y < MINE; ++y)
#pragma unroll
          for (int i = 0; i < PER; ++i)
            w[y][i] = *reinterpret_cast<const uint4*>(mine + (size_t)(it % C::STAGES) * C::RAW_TILE +
                                                      min(w0 + y * (CONVERTERS / 32), GROUPS - 1) * 16 * HD + i * 512);
        if (!__all_sync(0xffffffffu, mbar_wait(&kv_empty[s], ((it / C::RING) & 1) ^ 1) && !abort_flag)) {
          abort_flag = 1;
          if (lane == 0) atomicExch(p.status, STATUS_TIMEOUT);
          break;
        }
        if (marked && kv == 1) {
#pragma unroll
          for (int y = 0; y < MINE; ++y)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              w[y][i].x &= ~nan_bytes(w[y][i].x);
              w[y][i].y &= ~nan_bytes(w[y][i].y);
              w[y][i].z &= ~nan_bytes(w[y][i].z);
              w[y][i].w &= ~nan_bytes(w[y][i].w);
            }
        }
        // chunks 2 piece, 2 piece + 1 of the row's HD / 8; a sub-tile has 8
        uint8_t* dst = skv + (size_t)s * C::KV_TILE + (size_t)(piece / 4) * KEYS * 128 + row_in * 128;
        constexpr int TURNS = 8 / ROWS_STEP > 1 ? 8 / ROWS_STEP : 1;      // of a lane's rows: different places in the swizzle
        int c0[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; ++i) c0[i] = ((((2 * piece) & 7) ^ ((row_in + i * ROWS_STEP) & 7)) << 4);
#pragma unroll
        for (int y = 0; y < MINE; ++y) {
          const int g = w0 + y * (CONVERTERS / 32);
          if (g >= GROUPS) continue;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            uint4 a, b;
            to_f16(w[y][i].x, a.x, a.y);
            to_f16(w[y][i].y, a.z, a.w);
            to_f16(w[y][i].z, b.x, b.y);
            to_f16(w[y][i].w, b.z, b.w);
            uint8_t* at = dst + g * 16 * 128 + i * ROWS_STEP * 128;
            *reinterpret_cast<uint4*>(at + c0[i % TURNS]) = a;
            *reinterpret_cast<uint4*>(at + (c0[i % TURNS] ^ 16)) = b;
          }
        }
        fence_proxy_async();                                   // read by the tensor core (async proxy)
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[s]);
        request(it + C::STAGES, ((it + C::STAGES) >> 1) == j + 1 ? pages[1] : pages[2]);        // (into the stage that has been read)
      }
      if (abort_flag) break;
      ks = ks_next;
      vs = vs_next;
      pages[0] = pages[1];
      pages[1] = pages[2];
      pages[2] = checked(pages[3]);
      pages[3] = page_of(j + 4);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == 11) {
    // ---- the products ----
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_f16(ROWS, KEYS), idesc_o = idesc_f16_b_mn(ROWS, HD);
      auto issue_s = [&](int x, int j) {
        const uint8_t* kt = skv + (size_t)((2 * j) % C::RING) * C::KV_TILE;
#pragma unroll
        for (int sub = 0; sub < C::SUB; ++sub) {
          const uint64_t da = smem_desc_sw128(sq + (size_t)x * C::Q_TILE + (size_t)sub * ROWS * 128);
          const uint64_t db = smem_desc_sw128(kt + (size_t)sub * KEYS * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem_s[x], da + 2 * k, db + 2 * k, idesc_s, (uint32_t)((sub | k) != 0));
        }
        umma_commit(&s_full[x]);
      };
      auto kv_ready = [&](int it) {
        const bool ok = mbar_wait(&kv_full[it % C::RING], (it / C::RING) & 1);
        tc_fence_after();
        return ok;
      };
      // O += P V_j for a row tile, in two halves of the keys as the weights come; kv_ready(V_j) has been seen
      auto issue_o = [&](int x, int j) {
        const uint8_t* vt = skv + (size_t)((2 * j + 1) % C::RING) * C::KV_TILE;
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k) {
          if (k % (KEYS / 32) == 0) {
            if (!mbar_wait(&p_full[x][k / (KEYS / 32)], j & 1)) return false;
            tc_fence_after();
          }
          // 16 keys = two 8-row groups of 1024 bytes further in V; a second 64-column block of head_dim (128) lies one sub-tile
          // further, which the descriptor's leading offset says
          uint64_t db = smem_desc_sw128(vt + (size_t)k * 16 * 128);
          if (C::SUB > 1) db = (db & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)((KEYS * 128) >> 4) << 16);
          umma_f16_ta(tmem_o[x], tmem_p[x] + 8 * k, db, idesc_o, (uint32_t)((j | k) != 0));
        }
        if (C::APART || j + 1 == n_x[x]) umma_commit(&o_done[x]);
        return true;
      };
      bool ok = mbar_wait(&q_full, 0);
      tc_fence_after();
      if (ok && n > 0) {
        ok = kv_ready(0);
        for (int x = 0; x < 2 && ok; ++x)
          if (n_x[x] > 0) issue_s(x, 0);
        umma_commit(&kv_empty[0]);
      }
      if (C::APART) {
        // The row tiles run half a tile apart, and so do the steps here: S of the first, the product of the second's tile before, ...
        // Step j: S_0(j + 1), O_1(j - 1), S_1(j + 1), O_0(j).  K_{j+1} is done with behind S_1(j + 1), V_{j-1} behind O_1(j - 1).
        for (int j = 0; j <= n && ok && !abort_flag; ++j) {
          const bool more = j + 1 < n;
          if (more) ok = kv_ready(2 * j + 2);
          if (ok && j + 1 < n_x[0]) {
            ok = mbar_wait(&s_free[0], j & 1);
            tc_fence_after();
            if (ok) issue_s(0, j + 1);
          }
          if (ok && j > 0) {
            if (j - 1 < n_x[1]) ok = issue_o(1, j - 1);
            umma_commit(&kv_empty[(2 * j - 1) % C::RING]);
          }
          if (ok && j + 1 < n_x[1]) {
            ok = mbar_wait(&s_free[1], j & 1);
            tc_fence_after();
            if (ok) issue_s(1, j + 1);
          }
          if (ok && more) umma_commit(&kv_empty[(2 * j + 2) % C::RING]);
          if (ok && j < n) ok = kv_ready(2 * j + 1);
          if (ok && j < n_x[0]) ok = issue_o(0, j);
        }
      } else {
        for (int j = 0; j < n && ok && !abort_flag; ++j) {
          ok = kv_ready(2 * j + 1);
          bool next = false;
          for (int x = 0; x < 2 && ok; ++x) {
            if (j >= n_x[x]) continue;
            ok = issue_o(x, j);
            if (ok && j + 1 < n_x[x]) {
              if (!next) ok = kv_ready(2 * j + 2);
              if (!ok) break;
              next = true;
              issue_s(x, j + 1);                               // (behind O_j in the tensor pipe, which reads the weights over S)
            }
          }
          umma_commit(&kv_empty[(2 * j + 1) % C::RING]);
          if (next) umma_commit(&kv_empty[(2 * j + 2) % C::RING]);
        }
      }
      if (!ok) {
        abort_flag = 1;
        atomicExch(p.status, STATUS_TIMEOUT + 1);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = row ----
    const int x = warp >> 2, row = 32 * (warp & 3) + lane;
    const int tl = x * tpt + row / group, h = row % group;     // token within the CTA's 2 tpt, head within the group
    const bool valid = row / group < tpt && tl < n_tok;
    const int pos = first + tl, pos_first = first + x * tpt, pos_last = first + min(n_tok, (x + 1) * tpt) - 1;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    // q under its power of two, in f16, and under the sign of the scale: the factor of the scores is not negative, so the largest
    // score of a group of keys is the largest under its factor too
    float factor;                                              // |scale| * log2(e) / that power
    {
      uint4 w[HD / 8];
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.q) + (size_t)(qstart + tok0 + tl) * p.ldq +
                                                        (size_t)(kvh * group + h) * HD);
      uint32_t top = 0u;                                       // bits of a bfloat16's magnitude compare like the number
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        if (valid) w[i] = src[i];
      }
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
      }
      const int e2 = min(127, max((int)(top >> 7) - 127, -112));
      const float up = copysignf(pow2(min(14 - e2, 126)), p.scale_log2);
      factor = fabsf(p.scale_log2) * pow2(max(e2 - 14, -126));
      uint8_t* dst = sq + (size_t)x * C::Q_TILE + (size_t)row * 128;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[i]);
        uint32_t f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = pack_f16(__uint_as_float(u[e] << 16) * up, __uint_as_float(u[e] & 0xffff0000u) * up);
        *reinterpret_cast<uint4*>(dst + (size_t)(i / 8) * ROWS * 128 + (((i & 7) ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    float m = -INFINITY, l = 0.f;                              // the maximum in use and the sum
    uint32_t poison[HD / 32];                                  // columns that are NaN in this row
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) poison[i] = 0u;
    bool alive = true;
    const uint32_t tmem_x = x ? tmem_s[1] : tmem_s[0], tmem_ox = x ? tmem_o[1] : tmem_o[0], tmem_px = x ? tmem_p[1] : tmem_p[0];
    const int n_mine = x ? n_x[1] : n_x[0];
    for (int j = 0; j < n_mine; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[x], j & 1))) {
        abort_flag = 1;
        if (lane == 0) atomicExch(p.status, STATUS_TIMEOUT + 2);
        alive = false;
        break;
      }
      tc_fence_after();
      const int col0 = (t_lo + j) * KEYS;
      const float4* mt = meta[j % META];
      const bool marked = marks[j % META] != 0;
      const bool full = col0 + KEYS - 1 <= pos_first && (p.window <= 0 || col0 + p.window > pos_last);
      const int hi_c = valid ? pos - col0 : -1, lo_c = (p.window > 0 ? pos - p.window + 1 : 0) - col0;     // columns the row sees
      const bool none = hi_c < lo_c;
      const unsigned span = none ? 0u : (unsigned)(hi_c - lo_c);
      // the whole row of S into registers: the loads on their way together, one wait
      float v[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; c += 32) tmem_ld_32_issue(tmem_x + lane_off + (uint32_t)c, v + c);
      tmem_ld_wait_n<KEYS>(v);
      if (C::APART) {                                          // the next S may come
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[x]);
      }
      if (!full) {
#pragma unroll
        for (int i = 0; i < KEYS; ++i) v[i] = (!none && (unsigned)(i - lo_c) <= span) ? v[i] : -INFINITY;
      }
      // the largest x = score + log2(scale of V) of the row
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const float* u = v + 16 * g;
        float a = max3(u[0], u[1], u[2]), b = max3(u[3], u[4], u[5]);
        a = max3(a, u[6], u[7]);
        b = max3(b, u[8], u[9]);
        a = max3(a, u[10], u[11]);
        b = max3(b, u[12], u[13]);
        a = max3(a, u[14], u[15]);
        const float2 sc = *reinterpret_cast<const float2*>(&mt[g]);
        // (a factor that underflowed would make NaN of a masked column's -inf)
        top = fmaxf(top, fmaf(fmaxf(a, b), fmaxf(factor * sc.x, 1.2e-38f), sc.y));
      }
      // the maximum in use follows only when it would fall behind by more than 2^3: a weight stays below 2^15
      float corr = 1.f;
      if (top > m + 3.f) {                                     // (m -inf: anything seen)
        corr = m == -INFINITY ? 0.f : exp2f(m - top);
        m = top;
        l *= corr;
      }
      const float off = 12.f - (m == -INFINITY ? 0.f : m);
      if (C::APART && j > 0 && !__all_sync(0xffffffffu, mbar_wait(&o_done[x], (j - 1) & 1))) {
        abort_flag = 1;                                        // (P and O of the tile before are read by its product until then)
        if (lane == 0) atomicExch(p.status, STATUS_TIMEOUT + 3);
        alive = false;
        break;
      }
      if (C::APART) tc_fence_after();
      if (j > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
        // (weights over S: S_j was issued behind P V_{j-1}, so O stands still here as well)
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 16) {
          float o[16];
          tmem_ld_16(tmem_ox + lane_off + (uint32_t)c0, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= corr;
          tmem_st_16(tmem_ox + lane_off + (uint32_t)c0, o);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t packed[32];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float* u = v + 64 * half + 16 * g;
          const float4 sc = mt[4 * half + g];
          const float f = fmaxf(factor * sc.x, 1.2e-38f), d = sc.y + off;
          const uint64_t f2 = pk2(f, f), d2 = pk2(d, d);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x0, x1;
            upk2(fma2(pk2(u[i], u[i + 1]), f2, d2), x0, x1);
            const float e0 = ex2(x0), e1 = ex2(x1);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pk2(e0, e1));
            packed[8 * g + i / 2] = pack_f16(e0, e1);
          }
          float a, b;
          upk2(add2(sum[0], sum[1]), a, b);
          l = fmaf(a + b, sc.z, l);
          if (half == 1 && g == AFTER) {                       // (the first half's weights have arrived meanwhile)
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[x][0]);
          }
        }
        tmem_st_16_issue(tmem_px + lane_off + (uint32_t)(32 * half), packed);
        tmem_st_16_issue(tmem_px + lane_off + (uint32_t)(32 * half + 16), packed + 16);
        if (half == 1) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
        }
      }
      if (marked) {
        // values of the tile's pages that are NaN, for the keys that the row sees
        const uint32_t* at = snan + (size_t)(j % META) * KEYS * (HD / 32);
#pragma unroll 1
        for (int i = 0; i < KEYS; ++i) {
          const int key = col0 + i;
          if (mt[i / 16].w != 0.f && valid && key <= pos && (p.window <= 0 || key + p.window > pos)) {
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) poison[w] |= at[i * (HD / 32) + w];
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x][1]);
    }
    if (alive && n_mine > 0 && !__all_sync(0xffffffffu, mbar_wait(&o_done[x], C::APART ? (n_mine - 1) & 1 : 0))) {
      abort_flag = 1;
      if (lane == 0) atomicExch(p.status, STATUS_TIMEOUT + 3);
      alive = false;
    }
    tc_fence_after();
    const float inv = parts > 1 ? 1.f : l != 0.f ? 1.0f / l : 0.f;
    float4* po = reinterpret_cast<float4*>(base) + (size_t)x * (HD / 4) * ROWS;         // [2][HD / 4][128 rows]
    bf16* dst = reinterpret_cast<bf16*>(p.out) + (size_t)(qstart + tok0 + tl) * p.ldo + (size_t)(kvh * group + h) * HD;
    if (parts > 1) asm volatile("bar.sync 2, 256;" ::: "memory");        // (both tiles' products have read the operands)
#pragma unroll 1
    for (int c0 = 0; c0 < HD; c0 += 32) {
      float o[32];
      if (n_mine > 0) tmem_ld_32(tmem_ox + lane_off + (uint32_t)c0, o);
      else
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
      uint32_t bad = 0u;
#pragma unroll
      for (int w = 0; w < HD / 32; ++w) bad = c0 == 32 * w ? poison[w] : bad;
      if (bad) {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = (bad >> i) & 1u ? __int_as_float(0x7fffffff) : o[i];
      }
      if (parts > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          po[(size_t)(c0 / 4 + i) * ROWS + row] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else if (valid) {
#pragma unroll
        for (int c8 = 0; c8 < 4; ++c8) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pk[e] = pack_bf16(o[c8 * 8 + 2 * e] * inv, o[c8 * 8 + 2 * e + 1] * inv);
          *reinterpret_cast<uint4*>(dst + c0 + c8 * 8) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
    }
    if (parts > 1) reinterpret_cast<float2*>(base + 2 * ROWS * HD * 4)[x * ROWS + row] = make_float2(m, l);
  }
  if (parts > 1) {
    cluster_sync_all();                                        // every share lies in its CTA's shared memory
    if (warp < 8) {
      // O = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z, in the keys' order
      const int x = warp >> 2, row = 32 * (warp & 3) + lane;
      const int tl = x * tpt + row / group, h = row % group;
      const bool valid = row / group < tpt && tl < n_tok;
      const float2* ml = reinterpret_cast<const float2*>(base + 2 * ROWS * HD * 4) + x * ROWS + row;
      float top = -INFINITY, sum = 0.f;
      for (int z = 0; z < parts; ++z) top = fmaxf(top, ld_cluster_f2(ml, z).x);
      for (int z = 0; z < parts; ++z) {
        const float2 a = ld_cluster_f2(ml, z);
        sum = fmaf(a.x == -INFINITY ? 0.f : exp2f(a.x - top), a.y, sum);
      }
      const float inv = sum != 0.f ? 1.0f / sum : 0.f;
      bf16* dst = reinterpret_cast<bf16*>(p.out) + (size_t)(qstart + tok0 + tl) * p.ldo + (size_t)(kvh * group + h) * HD;
      const float4* po = reinterpret_cast<const float4*>(base) + (size_t)x * (HD / 4) * ROWS + row;
      // HD / 8 pieces of eight columns; a CTA takes an even share of them
      const int end = HD / 8 * (part + 1) / parts;
      for (int i = HD / 8 * part / parts; i < end; ++i) {
        float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < parts; ++z) {
          const float mz = ld_cluster_f2(ml, z).x, w = mz == -INFINITY ? 0.f : exp2f(mz - top);
          const float4 u = ld_cluster_f4(po + (size_t)(2 * i) * ROWS, z), v = ld_cluster_f4(po + (size_t)(2 * i + 1) * ROWS, z);
          a[0] = fmaf(w, u.x, a[0]); a[1] = fmaf(w, u.y, a[1]); a[2] = fmaf(w, u.z, a[2]); a[3] = fmaf(w, u.w, a[3]);
          a[4] = fmaf(w, v.x, a[4]); a[5] = fmaf(w, v.y, a[5]); a[6] = fmaf(w, v.z, a[6]); a[7] = fmaf(w, v.w, a[7]);
        }
        if (valid) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pk[e] = pack_bf16(a[2 * e] * inv, a[2 * e + 1] * inv);
          *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();                                        // nobody leaves while another CTA reads its share
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == 11) {
    if (abort_flag)
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);        // products still on their way end before their memory is given back
    tmem_dealloc(tmem_slot, 512);
  }
}

constexpr int MAX_SHARES = 8;

template <int HD>
int launch(const Attn& p, long long tiles, long long keys, cudaStream_t stream) {
  static bool attr_set = false;
  if (!attr_set) {
    GB_CUDA(cudaFuncSetAttribute(kv8_attention_tcgen05_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM));
    attr_set = true;
  }
  // CTAs that share a tile's keys: as many as the SMs hold at a time, each with four key tiles at least.  `tiles` is an upper bound that
  // counts one for every request; how many there are is estimated from the longest portion and the mean of the others, which are
  // taken to be as long as their mean, or, where that is few rows, to be single tokens and a portion that has the rest of them.  (Without
  // the others 8 requests of 16 tokens behind 4,000 keys, 32 / 8 heads of 64, take 79 us, by eight CTAs a tile; with them 49, by two.)
  const long long two = 2 * (ROWS / (p.heads / p.kv_heads)), others = p.step.n_requests - 1, rest = p.step.n_tokens - p.step.max_q;
  const bool alike = others > 0 && rest * (p.heads / p.kv_heads) > others * p.few;
  const long long of_others = alike ? others * ((rest / others + two - 1) / two) : (rest + two - 1) / two;
  const long long walks = ((p.step.max_q + two - 1) / two + of_others) * p.kv_heads;
  const long long most = (keys + KEYS - 1) / KEYS / 4;
  int parts = 1;
  for (int x = 2; x <= MAX_SHARES && x <= most; ++x)
    if (walks <= clusters_at_a_time(kv8_attention_tcgen05_kernel<HD>, x, THREADS, Cfg<HD>::SMEM)) parts = x;
  return launch_parts(kv8_attention_tcgen05_kernel<HD>, p, parts, tiles, THREADS, Cfg<HD>::SMEM, stream);
}

}  // namespace

// Requests of more than p.few rows, in one launch; tiles: upper bound of sum_r ceil(q_len_r / (2 * tokens of a row tile)).
int kv8_attention_tcgen05(const kv8::Attn& p, cudaStream_t stream) {
  const int tpt = ROWS / (p.heads / p.kv_heads);
  const long long tiles = p.step.n_requests == 1 ? (p.step.n_tokens + 2 * tpt - 1) / (2 * tpt)
                                                 : (long long)p.step.n_tokens / (2 * tpt) + p.step.n_requests;
  const long long keys = p.window > 0 && p.window + 2 * tpt < p.step.max_ctx ? p.window + 2 * tpt : p.step.max_ctx;
  const int rc = p.hd == 64 ? launch<64>(p, tiles, keys, stream) : launch<128>(p, tiles, keys, stream);
  if (rc != GB_OK) return rc;
  GB_CHECK_LAUNCH("kv8_attention (tcgen05)");
  return GB_OK;
}
