// Copies rows of a cache's tensors: row dst <- row src of every tensor of a group (pages of the tensors that share page ids,
// state slots), for several groups and pairs in one launch.  This is what forking a request costs: the page that both requests
// will write on, its scales, and the state slot.
//
// The tensors' rows are cut into pieces of at most 4 KB once, when the cache is made; a warp moves one piece of one pair, in
// one trip (eight 16-byte loads a lane in flight).  The pairs travel in the launch's arguments: no copy to the device goes in
// front.  Bound by memory: every byte is read once and written once; 1,000 pages of twelve tensors, 197 MB in and out, 36.6 us, 5.4
// TB/s.  One page and a state slot: 2.7 us a launch in a chain of them.
#include <exception>
#include <vector>

#include "common.cuh"

namespace {

constexpr int MAX_GROUPS = 16, MAX_PAIRS = 440;

struct Piece {
  char* base; long long stride; long long bytes;              // piece of row i at base + i * stride
};
struct Copies {
  const Piece* pieces;
  int n_groups, last;                                         // last: of the call's launches
  int first_piece[MAX_GROUPS + 1], first_pair[MAX_GROUPS + 1];
  unsigned first_unit[MAX_GROUPS + 1];                        // a unit: a pair and a piece
  int2 pairs[MAX_PAIRS];                                      // (src, dst)
};
static_assert(sizeof(Copies) <= 4096, "the arguments of a launch");

// Only another launch of the same call may start early: kernels read what earlier steps left in pages and slots ahead of their wait, and
// the rows that are written here are such.
__global__ void __launch_bounds__(256) row_copies_kernel(const __grid_constant__ Copies c) {
  if (!c.last) pdl_trigger();
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= c.first_unit[c.n_groups]) return;
  int g = 0;
  while (unit >= c.first_unit[g + 1]) ++g;
  const unsigned n = (unsigned)(c.first_piece[g + 1] - c.first_piece[g]), at = unit - c.first_unit[g];
  const int2 pair = c.pairs[c.first_pair[g] + (int)(at / n)];
  const Piece p = c.pieces[c.first_piece[g] + (int)(at % n)];
  const char* src = p.base + (long long)pair.x * p.stride;
  char* dst = p.base + (long long)pair.y * p.stride;
  pdl_wait();
  if ((((uintptr_t)src | (uintptr_t)dst | (uintptr_t)p.bytes) & 15) == 0) {
    float4 v[8];
    const int vecs = (int)(p.bytes >> 4);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < vecs) v[i] = reinterpret_cast<const float4*>(src)[lane + 32 * i];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < vecs) reinterpret_cast<float4*>(dst)[lane + 32 * i] = v[i];
  } else if ((((uintptr_t)src | (uintptr_t)dst | (uintptr_t)p.bytes) & 3) == 0) {
    for (int i = lane; i < (int)(p.bytes >> 2); i += 32) reinterpret_cast<int*>(dst)[i] = reinterpret_cast<const int*>(src)[i];
  } else {
    for (int i = lane; i < (int)p.bytes; i += 32) dst[i] = src[i];
  }
  if (c.last) __threadfence();                                 // (in place for the whole GPU before this block ends)
}

// Ids within the group, no destination twice, none that is a source too.
int check_pairs(int g, const int* pairs, int n, int rows) {
  for (int i = 0; i < n; ++i)
    for (int k = 0; k < 2; ++k)
      if (pairs[2 * i + k] < 0 || pairs[2 * i + k] >= rows)
        GB_FAIL(GB_ERR_ARG, "row copies: pair %d of group %d: row %d of %d", i, g, pairs[2 * i + k], rows);
  if (n == 1) {
    if (pairs[0] == pairs[1]) GB_FAIL(GB_ERR_ARG, "row copies: row %d of group %d onto itself", pairs[0], g);
    return GB_OK;
  }
  try {
    static thread_local std::vector<unsigned char> to;         // 1: a destination (all 0 between calls)
    if (to.size() < (size_t)rows) to.resize((size_t)rows, 0);
    int bad = -1, twice = 0;
    for (int i = 0; i < n && bad < 0; ++i) {
      if (to[pairs[2 * i + 1]]) bad = i, twice = 1;
      to[pairs[2 * i + 1]] = 1;
    }
    for (int i = 0; i < n && bad < 0; ++i)
      if (to[pairs[2 * i]]) bad = i;
    for (int i = 0; i < n; ++i) to[pairs[2 * i + 1]] = 0;
    if (bad >= 0)
      GB_FAIL(GB_ERR_ARG, "row copies: row %d of group %d is a destination %s", pairs[2 * bad + (twice ? 1 : 0)], g,
              twice ? "twice" : "and a source");
  } catch (const std::exception& e) {
    GB_FAIL(GB_ERR_ARG, "row copies: %s", e.what());
  }
  return GB_OK;
}

}  // namespace

GB_API int gb_row_copies_piece_bytes() { return 4096; }

// What a call needs in one array of 64-bit words: w0 the pieces (device memory, one record of three words each: address in row
// 0, bytes between rows, bytes; group after group), w1 stream, w2 groups, then for each group its pairs (host memory, (src, dst)
// as 32-bit integers) and their number, then for each group its pieces and rows.
// Every source is read as it was before the call: a row that is a destination twice, or a destination and a source, is
// refused, as is a row outside the group.  Returns the number of kernels launched, or a negative error code.
GB_API int gb_row_copies(const long long* w) {
  const void* pieces = reinterpret_cast<const void*>(w[0]);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(w[1]);
  const int n_groups = (int)w[2];
  if (n_groups < 0 || n_groups > MAX_GROUPS) GB_FAIL(GB_ERR_ARG, "row copies: %d groups, %d at most", n_groups, MAX_GROUPS);
  const int* pairs[MAX_GROUPS];
  int n_pairs[MAX_GROUPS], n_pieces[MAX_GROUPS];
  for (int g = 0; g < n_groups; ++g) {
    pairs[g] = reinterpret_cast<const int*>(w[3 + 2 * g]);
    n_pairs[g] = (int)w[4 + 2 * g];
    n_pieces[g] = (int)w[3 + 2 * n_groups + 2 * g];
    const int rc = check_pairs(g, pairs[g], n_pairs[g], (int)w[4 + 2 * n_groups + 2 * g]);
    if (rc != GB_OK) return rc;
  }
  int launched = 0;
  long long to_copy = 0;                                       // pairs (of groups that have pieces) that no launch has yet
  for (int g = 0; g < n_groups; ++g) to_copy += n_pieces[g] > 0 ? n_pairs[g] : 0;
  int g0 = 0, done = 0;                                        // group and pair of it that come next
  while (g0 < n_groups) {
    // as many pairs as the arguments hold, group after group
    Copies c;
    c.pieces = reinterpret_cast<const Piece*>(pieces);
    c.n_groups = n_groups;
    int used = 0;
    long long units = 0, piece = 0;
    for (int g = 0; g < n_groups; ++g) {
      c.first_piece[g] = (int)piece;
      c.first_pair[g] = used;
      c.first_unit[g] = (unsigned)units;
      piece += n_pieces[g];
      if (g != g0 || used == MAX_PAIRS) continue;
      const int left = n_pairs[g] - done, take = left < MAX_PAIRS - used ? left : MAX_PAIRS - used;
      for (int i = 0; i < take; ++i) c.pairs[used + i] = make_int2(pairs[g][2 * (done + i)], pairs[g][2 * (done + i) + 1]);
      used += take;
      done += take;
      units += (long long)take * n_pieces[g];
      to_copy -= n_pieces[g] > 0 ? take : 0;
      if (done == n_pairs[g]) {
        ++g0;
        done = 0;
      }
    }
    c.first_piece[n_groups] = (int)piece;
    c.first_pair[n_groups] = used;
    c.first_unit[n_groups] = (unsigned)units;
    if (units > 0x7fffffffll) GB_FAIL(GB_ERR_ARG, "gb_row_copies: %lld pieces in one launch", units);
    if (units == 0) continue;
    c.last = to_copy == 0;
    gb_launch(row_copies_kernel, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, stream, c);
    GB_CHECK_LAUNCH("gb_row_copies");
    ++launched;
  }
  return launched;
}
