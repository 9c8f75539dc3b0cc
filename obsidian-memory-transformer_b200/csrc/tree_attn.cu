// tree_attn.cu -- attention of T drafted tokens per sequence (T = 1: a plain
// decode step) over a KV cache in 16 bits or in int8 codes with a scale per
// row.
//
//   o_t = sum_j p_tj v_j ,  p_t = softmax_j(q_t . k_j / sqrt(D))
//
// over the cached context j in [0, len_b) and, at positions len_b .. len_b + T,
// the token itself and its ancestors (parents).  G = heads / kv_heads query
// heads share a cached head.
//
// The keys of a (sequence, head) -- context, then draft -- are cut into tiles of
// 128 to 240 positions.  The tiles of the whole batch, whatever the lengths, form one
// list that the persistent CTAs (one per SM) share out evenly; a CTA that ends or
// starts inside a head leaves a partial (max, sum, output) there, and
// tree_combine_kernel merges them, one warp per query row.  Every cached byte is
// read once for a block of rows (up to 128 rows, 64 over int8 caches; more rows are more
// blocks, and each goes through the cache again); that read is the bound.  Only tiles that
// reach past the context look at the mask: a 64-bit ancestor set per token, found by
// pointer doubling.
//
// Two kernels contract the tiles, by the rows G * T that share a cached head:
//
// * tree_mma_kernel, up to 16 rows: warp 0 streams K and V
//   tiles by TMA into a ring of swizzled slots; the consumer warps contract them on
//   mma.sync m16n8k16 with the keys as M (a decode step's few rows are the 8 or 16
//   columns; a 128-row tcgen05 tile would idle).  A warp takes 16 keys at a time
//   through S^T = K Q^T, softmax and O^T += V^T P^T on its own; P^T is S^T's
//   accumulator transposed in registers.  Nothing is exchanged until the segment's
//   end, where the warps' (max, sum, output) are merged in shared memory.  int8 codes
//   become f16 in registers (exact), with the row's scale applied to the fp32 score (K)
//   and to the probability (V); those conversions are most of its instructions, so
//   int8 caches run 15 consumer warps up to 8 rows (16 warps with the producer: 128
//   registers a thread) and 11 beyond (168), 16-bit ones 8.  A tile is 16 keys for every warp:
//   each warp waits for every load in turn (a warp that skipped tiles could take a
//   barrier's phase for the one before).
// * tree_tc_kernel, more rows: tcgen05, keys as the 128 lanes:
//   S^T [128 keys x N rows] = K Q^T and O^T [D x N] += V^T P, N = 32, 64 or (16-bit
//   caches) 128 rows.  K and V tiles are used as they lie (K-major and M-major
//   operands), the softmax work grows with the rows, and a thread owns a key: its mask
//   test, its scales and the clean-up of rows past the end are its own.  int8 codes
//   become f16 tiles in shared memory first.
//
// Measured (bf16 queries, calls back to back; the second of two figures once the clock has
// dropped under load).  Read-bound: one row per head of 128 dims over a 16-bit cache, 16 x
// 32 heads x 8192 to 16384 positions, 0.47 ms for 3.2 GB (6.9 TB/s); int8, 64 x 32 heads x 4096
// to 8192, 0.52 to 0.61 ms for 3.3 GB (5.5 to 6.4 TB/s).  9 to 16 int8 rows of 128 dims: 8 x 32
// heads x 16384 positions 0.25 to 0.29 ms, where DRAM (45%) and issue slots (51%) both
// wait for the chain of a warp's tile: conversions, products, exponentials.
// Time of a 128-position tile, CTA by CTA, over 8 x 32 heads x 16384 positions in us (to read:
// 0.74 for 64 dims, 1.48 for 128; int8 0.39 and 0.76):
//   rows            16    32    64   128
//   64 dims       0.77  1.00  1.33  1.90   up to 16 rows read-bound, then by the softmax's
//   128 dims      1.38  1.46  1.64   2.7   latencies (exponentials, votes, barriers)
//   64 dims int8  0.80  1.28  1.82   3.6   (two blocks of 64 rows) latencies and, with
//   128 dims int8 1.23  1.54  2.53   5.0   64 rows of 128 dims, three slots of f16 tiles
// A segment's start and end cost 7 to 9 us (half of it queries, masks and the
// tail's clean-up; 13 before those were overlapped and rid of divisions).
//
// In both, a row's reference maximum is only raised when a score exceeds it by more
// than 2^8.  Weights that go to the tensor core as f16 are held 2^7 higher (Raise), so that
// the many small ones of a long context stay above its smallest numbers.  A non-finite
// value of a drafted token must not reach the tokens that do not see it (0 * inf): it is
// taken out of the tile, and the combine kernel adds it to the rows that do; over int8
// caches, whose non-finite rows have the scale NaN, their weights become NaN instead.
//
// The reference has no counterpart: its cache manager is a stub
// (python_bindings/src/main.cpp:101-135).
#include <type_traits>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kTcTile = 128;      // cache positions per tile of the tcgen05 kernel
constexpr int kTBatch = 512;      // sequences per launch
constexpr int kScanWords = 3 * (kTBatch + 2);  // what tree_scan leaves
constexpr int kTMaxGrid = 256;    // CTAs that share the tiles, whatever the device
constexpr int kTMaxTokens = 64;   // drafted tokens (one 64-bit ancestor mask)
// A row's reference in log2 units: `lower` below its maximum when it is set, raised when a
// score passes it by `at`.  Weights that stay in fp32 or become bf16 are at most 2^8.  f16
// ends at 2^16, and below 2^-14 its steps are 2^-24 whatever the weight: with the largest
// between 2^7 and 2^15, half such a step is at most 2^-32 of it (2^-25 with a reference at
// the maximum: 65536 keys of 2^-26 each then vanished).
template <bool F16>
struct Raise {
  static constexpr float lower = F16 ? 7.0f : 0.0f;
  static constexpr float at = 8.0f + lower;
  static constexpr float most = F16 ? 32768.0f : 256.0f;  // 2^at
};

struct TreeParams {
  const void* q;
  int64_t qb, qt, qh;  // element strides of q: batch, token, head
  void* o;
  int64_t ob, ot, oh;
  const void* kc;
  const void* vc;
  const float* ks;
  const float* vs;
  const int* lens;
  const int* ntok;
  const int* parents;
  int B, T, G, kvh, nrb, rb;  // nrb: row blocks per cached head, of rb rows
  int tile;                   // positions per tile
  float inv_g;                // 1 / G
  int64_t P;
  float sl2;
  float* part;
  int grid;  // CTAs that share the tiles
  int* err;
};

template <int D>
constexpr int part_stride() { return D + 4; }  // output, max, sum, "values were taken out"

// Context length and tokens (0: nothing to do) of sequence b.
__device__ __forceinline__ bool tree_seq(const TreeParams& p, int b, int& len, int& n) {
  len = p.lens[b];
  n = p.ntok ? p.ntok[b] : p.T;
  const bool ok = len >= 0 && n >= 0 && n <= p.T && static_cast<int64_t>(len) + n <= p.P;
  if (!ok) len = n = 0;
  return ok;
}

// TILE, RB: p.tile and p.rb where the kernel knows them (integer divisions by a variable
// are most of what finding a tile costs), else 0.
template <int TILE>
__device__ __forceinline__ int tiles_of(const TreeParams& p, int len, int n) {
  return n > 0 ? (len + n - 1) / (TILE ? TILE : p.tile) + 1 : 0;
}
template <int RB>
__device__ __forceinline__ int row_blocks(const TreeParams& p, int n) {
  const int rb = RB ? RB : p.rb;
  return (p.G * n + rb - 1) / rb;
}
// x / G for 0 <= x < 2^13 (G <= 64: (x + 1/2) / G is 2^-7 away from every integer)
__device__ __forceinline__ int over_g(const TreeParams& p, int x) {
  return static_cast<int>((static_cast<float>(x) + 0.5f) * p.inv_g);
}

// First tile of every sequence in the batch's list, and the sequences' lengths and
// token counts after it ([kTBatch + 2] words each), by one warp.
template <int TILE, int RB>
__device__ __forceinline__ void tree_scan(const TreeParams& p, uint32_t* base, int lane) {
  uint32_t carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    uint32_t w = 0;
    if (b < p.B) {
      int len, n;
      tree_seq(p, b, len, n);
      w = static_cast<uint32_t>(p.kvh) * row_blocks<RB>(p, n) * tiles_of<TILE>(p, len, n);
      base[kTBatch + 2 + b] = static_cast<uint32_t>(len);
      base[2 * (kTBatch + 2) + b] = static_cast<uint32_t>(n);
    }
    uint32_t s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (b < p.B) base[b] = carry + s - w;
    carry += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) base[p.B] = carry;
}

// The list is shared by min(grid, total) CTAs, so that no share is empty: the
// partials of a head are those of consecutive CTAs.
// The first total % shares of them take a tile more than the others.
struct Shares {
  uint32_t each, more;
  __device__ __forceinline__ Shares(uint32_t total, uint32_t shares)
      : each(shares ? total / shares : 0u), more(total - each * shares) {}
  __device__ __forceinline__ uint32_t start(uint32_t c) const { return c * each + min(c, more); }
  __device__ __forceinline__ uint32_t of(uint32_t tile) const {
    const uint32_t head = more * (each + 1);
    return tile < head ? tile / (each + 1) : more + (tile - head) / each;
  }
};

// Where tile w of the list lies.
struct TreeSpan {
  int b, h, rb, len, n, rows, tile, tiles;  // tile: index within the head's keys
};
template <int TILE, int RB>
__device__ __forceinline__ TreeSpan tree_find(const TreeParams& p, const uint32_t* base, uint32_t w) {
  int lo = 0, hi = p.B;  // base[lo] <= w < base[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (base[mid] <= w) lo = mid;
    else hi = mid;
  }
  TreeSpan s;
  s.b = lo;
  s.len = static_cast<int>(base[kTBatch + 2 + lo]);
  s.n = static_cast<int>(base[2 * (kTBatch + 2) + lo]);
  s.tiles = tiles_of<TILE>(p, s.len, s.n);
  const int nrb = row_blocks<RB>(p, s.n);
  const uint32_t at = w - base[lo];
  const uint32_t item = at / s.tiles;
  s.tile = static_cast<int>(at - item * s.tiles);
  s.h = static_cast<int>(nrb == 1 ? item : item / nrb);
  s.rb = static_cast<int>(item - s.h * nrb);
  s.rows = min(RB, p.G * s.n - s.rb * RB);
  return s;
}

// Ancestor sets (the token itself included) of the drafted tokens that the rows
// row0 .. row0 + rows (at most 64) of a sequence belong to, into mask[0 .. rows), by
// one warp: log2(n) rounds of pointer doubling over the n tokens.  A parent that
// does not come before its token counts as none and sets the device error word.
__device__ __forceinline__ void tree_masks(const TreeParams& p, int b, int n, int row0, int rows,
                                           unsigned long long* mask, int lane) {
  unsigned long long m[2];
  int up[2];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = lane + 32 * i;
    m[i] = (2ull << t) - 1;  // a chain
    up[i] = -1;
    if (p.parents != nullptr) {
      m[i] = 1ull << t;
      up[i] = t < n ? p.parents[static_cast<int64_t>(b) * p.T + t] : -1;
      if (up[i] >= t || up[i] < -1) {
        bad = true;
        up[i] = -1;
      }
    }
  }
  if (bad) atomicExch(p.err, kErrBadParent);
#pragma unroll 1
  for (int reach = 1; reach < n && p.parents != nullptr; reach *= 2) {
    unsigned long long a[2];
    int nx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // set and parent of this token's farthest known ancestor
      const int from = up[i] & 31;
      const unsigned long long m0 = __shfl_sync(0xffffffffu, m[0], from);
      const unsigned long long m1 = __shfl_sync(0xffffffffu, m[1], from);
      const int u0 = __shfl_sync(0xffffffffu, up[0], from);
      const int u1 = __shfl_sync(0xffffffffu, up[1], from);
      a[i] = up[i] < 0 ? 0ull : up[i] < 32 ? m0 : m1;
      nx[i] = up[i] < 0 ? -1 : up[i] < 32 ? u0 : u1;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] |= a[i];
      up[i] = nx[i];
    }
  }
  __syncwarp();  // the sets of the segment before have been read
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = lane + 32 * i, tok = over_g(p, row0 + r);
    const unsigned long long m0 = __shfl_sync(0xffffffffu, m[0], tok & 31);
    const unsigned long long m1 = __shfl_sync(0xffffffffu, m[1], tok & 31);
    if (r < rows) mask[r] = tok >= n ? 0ull : tok < 32 ? m0 : m1;
  }
  __syncwarp();
}

// Bit 15 of each half of a word whose 16-bit value is not finite (its exponent bits are
// all ones).
template <class T>
__device__ __forceinline__ uint32_t non_finite_halves(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((w & kExp) + kOne) & 0x80008000u;
}
template <class T>
__device__ __forceinline__ uint32_t non_finite_in(const uint4& x) {
  return non_finite_halves<T>(x.x) | non_finite_halves<T>(x.y) | non_finite_halves<T>(x.z) |
         non_finite_halves<T>(x.w);
}
template <class T>
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
  return w & ~((non_finite_halves<T>(w) >> 15) * 0xffffu);
}
// One 16-byte unit of a tile's V row: zeroed (`drop`: nothing is there), or
// without its non-finite values (a drafted token); returns whether any was found.
template <class T>
__device__ __forceinline__ bool clean_unit(uint8_t* at, bool drop) {
  const uint4 x = *reinterpret_cast<const uint4*>(at);
  if (!drop && non_finite_in<T>(x) == 0u) return false;
  *reinterpret_cast<uint4*>(at) =
      drop ? make_uint4(0u, 0u, 0u, 0u)
           : make_uint4(finite_of<T>(x.x), finite_of<T>(x.y), finite_of<T>(x.z), finite_of<T>(x.w));
  return !drop;
}

// -------------------------------------------------------------- mma helpers --
template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(addr)
               : "memory");
  return r;
}
// Two of a word's four codes (biased by 128) as an f16 pair: 0x6400 | u is
// 1024 + u, and 1024 + u - 1152 = u - 128 is exact.
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t sel) {
  const uint32_t x = __byte_perm(biased, 0x64646464u, sel);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  return r;
}
// Power of two that brings the largest magnitude `am` of a query row to
// [2^14, 2^15) (1 where it is 0 or not finite).
__device__ __forceinline__ float query_scale(float am) {
  int ex = static_cast<int>(__float_as_uint(am) >> 23);  // 2^(ex-127) <= am
  if (ex == 0 || ex == 255) ex = 141;
  return __uint_as_float(static_cast<uint32_t>(min(268 - ex, 254)) << 23);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}
template <int THREADS>
__device__ __forceinline__ void cons_sync() {
  asm volatile("barrier.cta.sync 1, %0;" ::"n"(THREADS) : "memory");
}
// 8 x 8 16-bit transpose over the warp (a row of two values per lane).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ----------------------------------------------------------- mma.sync kernel --
constexpr int kMRows = 16;  // most rows of a block

template <int D, bool Q8, int NR>  // NR: 8-row columns of a block
struct MmaSmem {
  static constexpr int kWarps = !Q8 ? 8 : NR == 1 ? 15 : 11;  // consumers
  static constexpr int kKeys = 16 * kWarps;                // positions per tile
  static constexpr int kRows = 8 * NR;
  static constexpr int kRow = D * (Q8 ? 1 : 2);            // bytes per cached row
  static constexpr int kBox = kRow > 128 ? 128 : kRow;     // bytes per row of a TMA box
  static constexpr int kBoxes = kRow / kBox;
  static constexpr int kTile = kKeys * kRow;               // K or V tile
  static constexpr int kMergeRow = D + 4;                  // output, max, sum
  static constexpr int kMerge = kWarps * kRows * kMergeRow * 4;
  static constexpr int kFit = (212 * 1024 - kMerge) / kTile;
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static_assert(kTile % 1024 == 0 && kSlots >= 4, "swizzle atoms; K and V of two tiles");
  static constexpr int kOffMerge = kSlots * kTile;         // [warps][rows]
  static constexpr int kOffMask = kOffMerge + kMerge;  // [warps][rows]
  static constexpr int kOffBase = kOffMask + kWarps * kRows * 8;
  static constexpr int kOffBar = kOffBase + kScanWords * 4;
  static constexpr int kOffFlag = kOffBar + 2 * kSlots * 8;
  static constexpr int kBytes = kOffFlag + 128 + 1024;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

// Shared-memory offset of 16-byte unit c of row r of a tile (the TMA swizzle).
template <class S>
__device__ __forceinline__ uint32_t tile_unit(int r, int c) {
  if constexpr (S::kBox == 128)
    return static_cast<uint32_t>((c >> 3) * (S::kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  else  // 64-byte rows, 64-byte swizzle
    return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <class T, int D, bool Q8, int NR>
__global__ void __launch_bounds__(32 * (MmaSmem<D, Q8, NR>::kWarps + 1), 1)
    tree_mma_kernel(const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const TreeParams p) {
  using S = MmaSmem<D, Q8, NR>;
  constexpr int NS = S::kSlots, KS = D / 16, NU = D / 16, NW = S::kWarps;
  constexpr int ROWS = S::kRows;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value && !Q8;  // type of the products
  using RaiseS = Raise<!Q8 && !BF>;  // of the scores (int8: the sums' weights, in fp32)
  using RaiseP = Raise<!BF>;         // of what goes to the tensor core
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* merge = reinterpret_cast<float*>(smem + S::kOffMerge);
  uint32_t* base = reinterpret_cast<uint32_t*>(smem + S::kOffBase);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
  uint64_t* empty = full + NS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffFlag);
  int* wait_ok = reinterpret_cast<int*>(smem + S::kOffFlag) + 1;  // [NW]
  int* taken = wait_ok + NW;  // [2], by segment parity
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, NW);
    }
    *abort_flag = 0;
    taken[0] = taken[1] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  grid_wait();
  if (warp == 0) tree_scan<S::kKeys, ROWS>(p, base, lane);
  __syncthreads();
  grid_release();
  const uint32_t total = base[p.B];
  const uint32_t shares = min(total, gridDim.x);
  if (blockIdx.x >= shares) return;
  const Shares share(total, shares);
  const uint32_t w0 = share.start(blockIdx.x), w1 = share.start(blockIdx.x + 1);

  if (warp == 0) {
    // ---- producer: K(0), V(0), K(1), ... into the ring
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (uint32_t w = w0; ok && w < w1;) {
        const TreeSpan s = tree_find<S::kKeys, ROWS>(p, base, w);
        const int nt = min(static_cast<int>(w1 - w), s.tiles - s.tile);
        const int row = static_cast<int>((static_cast<int64_t>(s.b) * p.kvh + s.h) * p.P) +
                        s.tile * S::kKeys;
        for (int t = 0; t < 2 * nt; ++t) {
          const int st = it % NS;
          if (!mbar_wait_bounded(empty + st, ((it / NS) & 1) ^ 1, abort_flag, p.err,
                                 kErrWaitEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full + st, S::kTile);
          uint8_t* dst = smem + st * S::kTile;
#pragma unroll
          for (int x = 0; x < S::kBoxes; ++x)
            tma_load_2d(dst + x * S::kKeys * 128, (t & 1) ? &tmV : &tmK, full + st, x * 64,
                        row + (t >> 1) * S::kKeys);
          ++it;
        }
        w += nt;
      }
      if (!ok) {  // let the copies in flight land before the CTA exits
        volatile int never = 0;
        for (int j = (it > NS ? it - NS : 0); j < it; ++j)
          mbar_wait_bounded(full + j % NS, (j / NS) & 1, &never, p.err, kErrWaitOther);
      }
    }
    return;
  }

  // ---- consumers: keys wk .. wk + 15 of every tile
  const int cw = warp - 1, g = lane >> 2, c = lane & 3, i8 = lane >> 3, r8 = lane & 7;
  const int wk = cw * 16, ct = threadIdx.x - 32;
  unsigned long long* mask = reinterpret_cast<unsigned long long*>(smem + S::kOffMask) + cw * ROWS;
  int it = 0, seg = 0;  // the CTA's tiles so far; parity of its segments
  for (uint32_t w = w0; w < w1; seg ^= 1) {
    const TreeSpan sp = tree_find<S::kKeys, ROWS>(p, base, w);
    const int nt = min(static_cast<int>(w1 - w), sp.tiles - sp.tile);
    const int64_t head = static_cast<int64_t>(sp.b) * p.kvh + sp.h;
    const int keys = sp.len + sp.n;
    // the scales of this warp's 16 keys (K in lanes 0-15, V in lanes 16-31), loaded
    // kAhead tiles before their use: a tile's time is less than a load takes
    constexpr int kAhead = 2;
    float sc_next[kAhead];
    auto load_scale = [&](int t) -> float {
      const int key = (sp.tile + t) * S::kKeys + wk + (lane & 15);
      return key < keys ? (lane < 16 ? p.ks : p.vs)[head * p.P + key] : 0.0f;
    };
    if constexpr (Q8)
#pragma unroll
      for (int i = 0; i < kAhead; ++i) sc_next[i] = load_scale(i);
    // Q as B fragments (row g of each 8-row column).  int8 codes: lane c of a quad
    // holds dims c * D/4 .. (the codes' own order, any order of the dims gives the
    // same products) in f16, each row scaled by a power of two so that its largest value
    // is below 2^15 (bf16 values reach beyond f16; the scale is undone in fp32).
    uint32_t bq[NR][KS][2];
    float qinv[NR][2];  // of rows 2c, 2c + 1
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int r = nr * 8 + g, rr = sp.rb * ROWS + r;
      const int t = over_g(p, rr), gg = rr - t * p.G;
      const T* qp = static_cast<const T*>(p.q) + sp.b * p.qb + t * p.qt +
                    (static_cast<int64_t>(sp.h) * p.G + gg) * p.qh;
      const bool live = r < sp.rows;
      if constexpr (!Q8) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bq[nr][s][0] = live ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + 2 * c) : 0u;
          bq[nr][s][1] = live ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + 8 + 2 * c) : 0u;
        }
        qinv[nr][0] = qinv[nr][1] = p.sl2;
      } else {
        uint4 raw[KS / 2];
        float am = 0.0f;
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          raw[s] = live ? *reinterpret_cast<const uint4*>(qp + c * (D / 4) + 8 * s)
                        : make_uint4(0u, 0u, 0u, 0u);
          const T* e = reinterpret_cast<const T*>(&raw[s]);
#pragma unroll
          for (int i = 0; i < 8; ++i) am = fmaxf(am, fabsf(to_f32(e[i])));
        }
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
        const float qs = query_scale(am), inv = p.sl2 / qs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const T* e = reinterpret_cast<const T*>(&raw[s / 2]) + (s & 1) * 4;
          bq[nr][s][0] = pack16<false>(to_f32(e[0]) * qs, to_f32(e[1]) * qs);
          bq[nr][s][1] = pack16<false>(to_f32(e[2]) * qs, to_f32(e[3]) * qs);
        }
        qinv[nr][0] = __shfl_sync(0xffffffffu, inv, 8 * c);
        qinv[nr][1] = __shfl_sync(0xffffffffu, inv, 8 * c + 4);
      }
    }
    if ((sp.tile + nt) * S::kKeys > sp.len)
      tree_masks(p, sp.b, sp.n, sp.rb * ROWS, ROWS, mask, lane);
    // o[nr][u]: dims of 16-byte-pair u (rows of the A tile) x rows 2c, 2c + 1
    float o[NR][NU][4], l[NR][2], mref[NR][2], eref[NR][2], frow[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nr][u][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nr][j] = frow[nr][j] = 0.0f;
        mref[nr][j] = eref[nr][j] = -INFINITY;
      }
    }

    bool ok = true;
    for (int t = 0; t < nt; ++t) {
      const int sk = 2 * (it + t), sv = sk + 1;
      const int key0 = (sp.tile + t) * S::kKeys + wk;
      float ks[2] = {1.0f, 1.0f}, vsc[2], lvs[2];
      if constexpr (Q8) {
        const float sc = sc_next[0];
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) sc_next[i] = sc_next[i + 1];
        sc_next[kAhead - 1] = load_scale(t + kAhead);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // keys g, g + 8
          ks[h] = __shfl_sync(0xffffffffu, sc, g + 8 * h);
          vsc[h] = __shfl_sync(0xffffffffu, sc, 16 + g + 8 * h);
          asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lvs[h]) : "f"(vsc[h]));
        }
      }
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(full + sk % NS, (sk / NS) & 1, abort_flag,
                                                     p.err, kErrWaitFull));
      if (!ok) break;
      const uint32_t ak = smem_u32(smem + (sk % NS) * S::kTile);
      const bool tail = key0 + 16 > sp.len;

      // ---- S^T: keys g, g + 8 x rows 2c, 2c + 1
      float acc[NR][4];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nr][i] = 0.0f;
      if constexpr (!Q8) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t ka[4];
          ldsm4(ak + tile_unit<S>(wk + (i8 & 1) * 8 + r8, 2 * s + (i8 >> 1)), ka);
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) mma16816<BF>(acc[nr], ka, bq[nr][s][0], bq[nr][s][1]);
        }
      } else {
        constexpr int NL = D / 64;  // 16-byte units per lane and key
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          const uint4 lo = lds128(ak + tile_unit<S>(wk + g, NL * c + u));
          const uint4 hi = lds128(ak + tile_unit<S>(wk + 8 + g, NL * c + u));
          const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = a[i] ^ 0x80808080u, y = b[i] ^ 0x80808080u;
            const uint32_t ka[4] = {codes_f16(x, 0x4140), codes_f16(y, 0x4140),
                                    codes_f16(x, 0x4342), codes_f16(y, 0x4342)};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
              mma16816<false>(acc[nr], ka, bq[nr][4 * u + i][0], bq[nr][4 * u + i][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + sk % NS);
      // ---- log2 scores; does any pass its row's reference by more than the margin?
      bool need = false;
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float s = acc[nr][2 * h + j] * qinv[nr][j];
            if constexpr (Q8) s *= ks[h];
            if (tail) {
              const int at = key0 + g + 8 * h - sp.len;  // place in the draft
              if (at >= 0 && !(at < sp.n && (mask[nr * 8 + 2 * c + j] >> at & 1ull)))
                s = -INFINITY;
            }
            acc[nr][2 * h + j] = s;
          }
          need |= fmaxf(acc[nr][j], acc[nr][2 + j]) > mref[nr][j] + RaiseS::at;
          if constexpr (Q8)
            need |= fmaxf(acc[nr][j] + lvs[0], acc[nr][2 + j] + lvs[1]) > eref[nr][j] + RaiseP::at;
        }
      if (__any_sync(0xffffffffu, need)) {
        // raise the references to the maxima (and rescale what is summed)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float a = fmaxf(mref[nr][j], fmaxf(acc[nr][j], acc[nr][2 + j]) - RaiseS::lower);
            float e = eref[nr][j];
            if constexpr (Q8)
              e = fmaxf(e, fmaxf(acc[nr][j] + lvs[0], acc[nr][2 + j] + lvs[1]) - RaiseP::lower);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
              if constexpr (Q8) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, x));
            }
            const float fl = mref[nr][j] == -INFINITY ? 0.0f : ex2_approx(mref[nr][j] - a);
            float fo = fl;
            if constexpr (Q8)
              fo = eref[nr][j] == -INFINITY ? 0.0f : ex2_approx(eref[nr][j] - e);
            l[nr][j] *= fl;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              o[nr][u][j] *= fo;
              o[nr][u][2 + j] *= fo;
            }
            mref[nr][j] = a;
            eref[nr][j] = e;
            // capped: p, at most 2^8, times it stays finite (times a scale of 0 it would else
            // be a NaN where the largest scores are those of keys with nearly no V scale)
            if constexpr (Q8) frow[nr][j] = e == -INFINITY ? 0.0f : ex2_approx(fminf(a - e, 119.0f));
          }
      }
      // ---- probabilities, transposed to the B fragment of the value product
      uint32_t bp[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float pr[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float s = acc[nr][2 * h + j];
            pr[j] = ex2_approx(s - (mref[nr][j] == -INFINITY ? 0.0f : mref[nr][j]));
            l[nr][j] += pr[j];
            if constexpr (Q8) {
              // p * v's scale, against its own reference: at most 2^15.  A scale NaN makes
              // a NaN of it, whatever p; a row that does not see the key takes nothing of it.
              pr[j] = pr[j] * frow[nr][j] * vsc[h];
              if (tail && s == -INFINITY) pr[j] = 0.0f;
            }
          }
          bp[nr][h] = transpose8x8(pack16<BF>(pr[0], pr[1]));
        }
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(full + sv % NS, (sv / NS) & 1, abort_flag,
                                                     p.err, kErrWaitFull));
      if (!ok) break;
      uint8_t* tv = smem + (sv % NS) * S::kTile;
      const uint32_t av = smem_u32(tv);
      if constexpr (!Q8) {
        if (tail) {  // rows past the end may hold anything, and drafted ones infinities
          for (int u = lane; u < 16 * (S::kRow / 16); u += 32) {
            const int r = u / (S::kRow / 16);
            if (key0 + r >= sp.len &&
                clean_unit<T>(tv + tile_unit<S>(wk + r, u % (S::kRow / 16)), key0 + r >= keys))
              taken[seg] = 1;
          }
          __syncwarp();
        }
      }
      // ---- O^T += V^T P^T, 16 dims at a time
      if constexpr (!Q8) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          uint32_t va[4];
          ldsm4_t(av + tile_unit<S>(wk + (i8 >> 1) * 8 + r8, 2 * u + (i8 & 1)), va);
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) mma16816<BF>(o[nr][u], va, bp[nr][0], bp[nr][1]);
        }
      } else {
        // a 16-byte unit holds 16 dims; the transposed 16-bit element is a pair of
        // neighbouring dims: the even ones become rows 0-7 of the A tile, the odd ones 8-15
#pragma unroll
        for (int u = 0; u < NU; u += 2) {
          uint32_t vb[4];
          ldsm4_t(av + tile_unit<S>(wk + (i8 & 1) * 8 + r8, u + (i8 >> 1)), vb);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t y0 = vb[2 * x] ^ 0x80808080u, y1 = vb[2 * x + 1] ^ 0x80808080u;
            const uint32_t va[4] = {codes_f16(y0, 0x4240), codes_f16(y0, 0x4341),
                                    codes_f16(y1, 0x4240), codes_f16(y1, 0x4341)};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
              mma16816<false>(o[nr][u + x], va, bp[nr][0], bp[nr][1]);
          }
        }
      }
      if constexpr (!Q8) {
        if (tail) fence_proxy_async_smem();  // the clean-up above, before the next TMA write
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + sv % NS);
    }
    it += nt;

    // ---- the segment's partial: the warps' (max, sum, output) merged
    float* mine = merge + cw * ROWS * S::kMergeRow;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          l[nr][j] += __shfl_xor_sync(0xffffffffu, l[nr][j], x);
        const int r = nr * 8 + 2 * c + j;
        if (r < sp.rows) {
          float* row = mine + r * S::kMergeRow;
          if constexpr (Q8) {
            // back to the scores' own reference
            const float f = eref[nr][j] == -INFINITY ? 0.0f : ex2_approx(eref[nr][j] - mref[nr][j]);
#pragma unroll
            for (int u = 0; u < NU; ++u)
              *reinterpret_cast<float2*>(row + u * 16 + 2 * g) =
                  make_float2(o[nr][u][j] * f, o[nr][u][2 + j] * f);
          } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              row[u * 16 + g] = o[nr][u][j];
              row[u * 16 + 8 + g] = o[nr][u][2 + j];
            }
          }
          if (g == 0) {
            row[D] = mref[nr][j];
            row[D + 1] = l[nr][j];
          }
        }
      }
    if (lane == 0) wait_ok[cw] = ok;
    cons_sync<NW * 32>();
    bool all_ok = true;
#pragma unroll
    for (int k = 0; k < NW; ++k) all_ok &= wait_ok[k] != 0;
    if (!all_ok) return;  // a wait ran out: every consumer leaves here
    const int64_t item = head * p.nrb + sp.rb;
    float* pp = p.part + (static_cast<int64_t>(blockIdx.x) + item) * ROWS * part_stride<D>();
    for (int i = ct; i < sp.rows * (D / 4); i += NW * 32) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      const float* in = merge + r * S::kMergeRow;
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < NW; ++k) m = fmaxf(m, in[k * ROWS * S::kMergeRow + D]);
      const float ref = m == -INFINITY ? 0.0f : m;
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float* x = in + k * ROWS * S::kMergeRow;
        const float f = ex2_approx(x[D] - ref);
        const float4 y = *reinterpret_cast<const float4*>(x + d);
        a.x = fmaf(y.x, f, a.x);
        a.y = fmaf(y.y, f, a.y);
        a.z = fmaf(y.z, f, a.z);
        a.w = fmaf(y.w, f, a.w);
        sum = fmaf(x[D + 1], f, sum);
      }
      float* row = pp + r * part_stride<D>();
      *reinterpret_cast<float4*>(row + d) = a;
      if (d == 0)
        *reinterpret_cast<float4*>(row + D) =
            make_float4(m, sum, Q8 ? 0.0f : static_cast<float>(taken[seg]), 0.0f);
    }
    cons_sync<NW * 32>();  // the merge rows are free
    if (ct == 0) taken[seg] = 0;  // set again two segments on, past another barrier
    w += nt;
  }
}

// ------------------------------------------------------------ tcgen05 kernel --
// Shared memory: Q [N rows x D] (K-major), P [128 keys x N] (N contiguous; twice up to 64
// rows, so that P(j + 1) is written while P(j) is contracted), a ring
// of 128-position K and V tiles, all in 128-byte-swizzled chunks of 64 columns.  int8
// caches: two or four warps fill that ring from a ring of code tiles.

template <int D, int N, bool Q8>
struct TcSmem {
  static constexpr int kTile = kTcTile * D * 2;        // K or V tile
  static constexpr int kQChunk = N * 128;             // N rows x 64 dims
  static constexpr int kQ = (D / 64) * kQChunk;
  static constexpr int kPChunk = kTcTile * 128;        // 128 keys x 64 rows
  static constexpr int kPOne = ((N + 63) / 64) * kPChunk;
  // int8, 32 rows of 128 dims: a fourth slot of f16 tiles instead of the second P (1.80 ->
  // 1.53 us a tile; 64 rows lose 2% by it)
  static constexpr bool kFour = Q8 && D == 128 && N == 32;
  static constexpr int kPs = N <= 64 && !kFour ? 2 : 1;  // P buffers
  static constexpr int kP = kPs * kPOne;
  static constexpr int kOffP = kQ;
  static constexpr int kOffRing = kOffP + kP;
  // 128 rows: the sums by the tensor core, behind the ring 16 keys x 64 ones
  static constexpr bool kSum = N == 128 && !Q8;
  static constexpr int kOnes = kSum ? 2048 : 0;
  static constexpr int kLeft = 212 * 1024 - kOffRing;
  static constexpr int kFit = kLeft / kTile;
  static constexpr int kSlots = Q8 ? (D == 64 ? 6 : kFour ? 4 : 3) : kFit > 8 ? 8 : kFit;
  static constexpr int kCodes = Q8 ? kTcTile * D : 0;        // K or V tile of codes
  static constexpr int kSlots8 = !Q8 ? 0 : D == 64 ? 8 : kFour ? 3 : 4;
  static constexpr int kOffCodes = kOffRing + kSlots * kTile;
  static_assert(kSlots * kTile + kSlots8 * kCodes <= kLeft, "the rings fit");
  // the softmax warps wait for V tiles in a sequence's last tiles only (see there)
  static_assert(kSlots >= 3, "the load before a tile's V load in its slot has completed by then");
  static constexpr int kOffOnes = kOffCodes + kSlots8 * kCodes;
  static constexpr int kOffMax = kOffOnes + kOnes;  // [2][4][N] maxima / sums
  static constexpr int kOffRef = kOffMax + 8 * N * 4;        // [6][N] per row, see the kernel
  static constexpr int kOffMask = kOffRef + 6 * N * 4;       // [softmax warps][rows] ancestor sets
  static constexpr int kOffBase = kOffMask + 4 * N * 8;
  static constexpr int kOffBar = (kOffBase + kScanWords * 4 + 7) / 8 * 8;
  static constexpr int kBars = 2 * kSlots + 2 * kSlots8 + 10;
  static constexpr int kOffFlag = kOffBar + kBars * 8;
  static constexpr int kRows = 32, kGroups = N / kRows;  // softmax: groups of four warps
  // int8: warps 2, 3 convert, and two more, but not with 64 rows of 64 dims: the 13th warp
  // costs the softmax registers (168 -> 128; 2.26 us a tile against 1.66), which 128 dims,
  // bound by the conversion, are worth (2.44 us against 2.84)
  static constexpr int kConv = N == 64 && D == 64 ? 2 : 4;
  static constexpr int kThreads = 128 + 128 * kGroups + (Q8 ? 32 * (kConv - 2) : 0);
  static constexpr int kBytes = kOffFlag + 80 + 1024;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

// Maxima (or sums) over the warp's 32 lanes of v[0 .. 31]; lane i gets that of v[i].
template <bool SUM>
__device__ __forceinline__ float across_lanes(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool up = lane & o;
      const float give = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      const float got = __shfl_xor_sync(0xffffffffu, give, o);
      v[i] = SUM ? keep + got : fmaxf(keep, got);
    }
  return v[0];
}

// Barrier of the softmax warps (THREADS of them); true where any predicate holds.
template <int THREADS>
__device__ __forceinline__ bool soft_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "n"(THREADS)
      : "memory");
  return r != 0;
}
template <int THREADS>
__device__ __forceinline__ void soft_sync() {
  asm volatile("barrier.cta.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// warp 0: TMA producer (K(0), V(0), K(1), ... into the ring); warp 1: TMEM and
// the MMAs, in the order S(0), S(1), O(0), S(2), O(1), ... within a head's
// segment; from warp 4 on, four warps for every 32 rows: softmax, thread = key = TMEM
// lane, a tile's 32 exponentials in registers.  TMEM: S^T twice, O^T.  With 128 rows that
// leaves a thread 96 registers, too few for its 32 sums as well: they are those of P's
// 16-bit values, contracted with ones (rows 64-127 of O^T for 64 dims, an accumulator of
// their own for 128), which saves reading S twice: 27 tokens of 4 heads a cached head,
// 55 -> 50 us.  (Up to 64 rows the sums stay in fp32 registers: contracting them cost 5%.)
// int8 caches: warps 2, 3 (and the last two) turn the codes into f16 tiles (exact); a thread's
// key has its K scale on the scores and its V scale on the probabilities, as in
// tree_mma_kernel.
template <class T, int D, int N, bool Q8>
__global__ void __launch_bounds__(TcSmem<D, N, Q8>::kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const TreeParams p) {
  using S = TcSmem<D, N, Q8>;
  constexpr int NS = S::kSlots, N8 = S::kSlots8;
  constexpr int RW = S::kRows, kSoft = 128 * S::kGroups, PB = S::kPs;
  constexpr bool SUM = S::kSum;
  using RaiseS = Raise<!Q8 && std::is_same<T, __half>::value>;
  using RaiseP = Raise<Q8 || std::is_same<T, __half>::value>;
  constexpr uint32_t kCols = 4 * N;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* smax = reinterpret_cast<float*>(smem + S::kOffMax);
  // per row: -reference (0: none yet), the rescaling of the sums; int8: the scores'
  // factor, the reference with the V scale, the rescaling of O, 2^(reference - that one)
  float* nref = reinterpret_cast<float*>(smem + S::kOffRef);
  float* fact = nref + N;
  float* srow = fact + N;
  float* eref = srow + N;
  float* facto = eref + N;
  float* frow = facto + N;
  uint32_t* base = reinterpret_cast<uint32_t*>(smem + S::kOffBase);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
  uint64_t* empty = full + NS;
  uint64_t* q_full = empty + NS;  // an arrival per softmax warp: q_full, s_free, p_full
  uint64_t* s_full = q_full + 1;  // [2]
  uint64_t* s_free = s_full + 2;  // [2]
  uint64_t* p_full = s_free + 2;  // [2], as is pv_done: by P buffer
  uint64_t* pv_done = p_full + 2;
  uint64_t* drained = pv_done + 2;
  uint64_t* full8 = drained + 1;  // the ring of code tiles
  uint64_t* empty8 = full8 + N8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffFlag);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + S::kOffFlag) + 1;
  int* wait_ok = reinterpret_cast<int*>(tslot) + 1;  // [softmax warps]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    for (int i = 0; i < S::kBars; ++i) {
      const bool per_warp = full + i == q_full || full + i == s_free || full + i == s_free + 1 ||
                            full + i == p_full || full + i == p_full + 1;
      const bool conv = Q8 && (i < NS || (full + i >= empty8 && full + i < empty8 + N8));
      mbar_init(full + i, per_warp ? kSoft / 32 : conv ? S::kConv : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(tslot, kCols);
  }
  if constexpr (SUM) {
    if (warp >= 2 && warp < 4) {
      constexpr uint32_t k1 = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
      for (int i = threadIdx.x - 64; i < S::kOnes / 16; i += 64)
        reinterpret_cast<uint4*>(smem + S::kOffOnes)[i] = make_uint4(k1, k1, k1, k1);
      fence_proxy_async_smem();
    }
  }
  grid_wait();
  if (warp == 0) tree_scan<kTcTile, N>(p, base, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_release();
  const uint32_t tmem = *tslot, tO = tmem + 2 * N, tL = tO + N;
  const uint32_t total = base[p.B];
  const uint32_t shares = min(total, gridDim.x);
  uint32_t w0 = 0, w1 = 0;  // no tiles: every role falls through to the end
  if (blockIdx.x < shares) {
    const Shares share(total, shares);
    w0 = share.start(blockIdx.x);
    w1 = share.start(blockIdx.x + 1);
  }

  if (warp == 0) {
    if (lane == 0) {
      // into the ring of tiles, or of code tiles
      constexpr int NP = Q8 ? N8 : NS, kBytes = Q8 ? S::kCodes : S::kTile;
      constexpr int kBoxes = Q8 ? 1 : D / 64;
      uint64_t* pfull = Q8 ? full8 : full;
      uint64_t* pempty = Q8 ? empty8 : empty;
      int it = 0;  // ring slots used
      bool ok = true;
      for (uint32_t w = w0; ok && w < w1;) {
        const TreeSpan s = tree_find<kTcTile, N>(p, base, w);
        const int nt = min(static_cast<int>(w1 - w), s.tiles - s.tile);
        const int row = static_cast<int>((static_cast<int64_t>(s.b) * p.kvh + s.h) * p.P) +
                        s.tile * kTcTile;
        for (int t = 0; ok && t < 2 * nt; ++t) {
          const int st = it % NP;
          if (!mbar_wait_bounded(pempty + st, ((it / NP) & 1) ^ 1, abort_flag, p.err,
                                 kErrWaitEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(pfull + st, kBytes);
          uint8_t* dst = smem + (Q8 ? S::kOffCodes : S::kOffRing) + st * kBytes;
#pragma unroll
          for (int x = 0; x < kBoxes; ++x)
            tma_load_2d(dst + x * kTcTile * 128, (t & 1) ? &tmV : &tmK, pfull + st, x * 64,
                        row + (t >> 1) * kTcTile);
          ++it;
        }
        w += nt;
      }
      if (!ok) {  // let the copies in flight land before the CTA exits
        volatile int never = 0;
        for (int j = (it > NP ? it - NP : 0); j < it; ++j)
          mbar_wait_bounded(pfull + j % NP, (j / NP) & 1, &never, p.err, kErrWaitOther);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr bool kBF = std::is_same<T, __nv_bfloat16>::value && !Q8;
      constexpr uint32_t idS = idesc_f16(128, N, kBF);
      // A = V^T: M (dims) contiguous; B = P: N (rows) contiguous
      constexpr uint32_t idO = idesc_f16(128, N, kBF, true) | (1u << 15);
      const uint32_t ones = smem_u32(smem + S::kOffOnes);
      const uint32_t aQ = smem_u32(smem), aP = smem_u32(smem + S::kOffP);
      const uint32_t ring = smem_u32(smem + S::kOffRing);
      int it = 0, seg = 0;  // tiles, segments so far
      bool ok = true;
      auto slot_wait = [&](int slot) {
        return mbar_wait_bounded(full + slot % NS, (slot / NS) & 1, abort_flag, p.err, kErrWaitFull);
      };
      auto issue_s = [&](int j) -> bool {  // tile j of the CTA into S buffer j % 2
        if (!slot_wait(2 * j)) return false;
        if (j >= 2 && !mbar_wait_bounded(s_free + (j & 1), ((j >> 1) - 1) & 1, abort_flag, p.err,
                                         kErrWaitOther))
          return false;
        tc_fence_after();
        const uint32_t aK = ring + (2 * j % NS) * S::kTile;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma_f16(tmem + (j & 1) * N,
                     make_desc_kmajor_sw128(aK + (k >> 2) * kTcTile * 128 + (k & 3) * 32),
                     make_desc_kmajor_sw128(aQ + (k >> 2) * S::kQChunk + (k & 3) * 32), idS, k != 0);
        tc_commit(s_full + (j & 1));
        tc_commit(empty + 2 * j % NS);
        return true;
      };
      auto issue_o = [&](int j, bool first) -> bool {
        const int pb = j % PB;
        if (!mbar_wait_bounded(p_full + pb, (j / PB) & 1, abort_flag, p.err, kErrWaitFull))
          return false;
        if (!slot_wait(2 * j + 1)) return false;
        tc_fence_after();
        const uint32_t aV = ring + ((2 * j + 1) % NS) * S::kTile;
#pragma unroll
        for (int k = 0; k < kTcTile / 16; ++k) {
          // D = 64: the upper 64 lanes are the ones' (or repeat the lower ones)
          const uint32_t av = aV + k * 2048;
          const uint32_t chunk = D == 128 ? kTcTile * 128 : SUM ? ones - av : 0u;
          const uint64_t bP = make_desc_mnmajor_sw128(aP + pb * S::kPOne + k * 2048, S::kPChunk);
          tc_mma_f16(tO, make_desc_mnmajor_sw128(av, chunk), bP, idO, !first || k != 0);
          if constexpr (D == 128 && SUM)
            tc_mma_f16(tL, make_desc_mnmajor_sw128(ones, 0), bP, idO, !first || k != 0);
        }
        tc_commit(pv_done + pb);
        tc_commit(empty + (2 * j + 1) % NS);
        return true;
      };
      for (uint32_t w = w0; ok && w < w1; ++seg) {
        const TreeSpan s = tree_find<kTcTile, N>(p, base, w);
        const int nt = min(static_cast<int>(w1 - w), s.tiles - s.tile);
        ok = mbar_wait_bounded(q_full, seg & 1, abort_flag, p.err, kErrWaitFull);
        if (ok) ok = issue_s(it);
        for (int t = 0; ok && t < nt; ++t) {
          if (t + 1 < nt) ok = issue_s(it + t + 1);
          if (ok) ok = issue_o(it + t, t == 0);
        }
        it += nt;
        w += nt;
      }
      if (!ok) {  // what was issued completes before TMEM and shared memory go
        volatile int never = 0;
        tc_commit(drained);
        mbar_wait_bounded(drained, 0, &never, p.err, kErrWaitOther);
      }
    }
  } else if (warp >= 4 && warp < 4 + kSoft / 32) {
    // ---- softmax: key `kt` of every tile, rows r0 .. r0 + RW
    const int sw = warp - 4, q4 = warp & 3, kt = q4 * 32 + lane, tid = threadIdx.x - 128;
    const int r0 = (sw >> 2) * RW;
    const uint32_t lane_off = static_cast<uint32_t>(q4 * 32) << 16;
    unsigned long long* mask =
        reinterpret_cast<unsigned long long*>(smem + S::kOffMask) + sw * RW;
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) -> bool {
      const bool r = mbar_wait_bounded(bar, parity, abort_flag, p.err, kErrWaitAccum);
      return __all_sync(0xffffffffu, r);
    };
    auto wait_pv = [&](int j) -> bool {  // tile j's value product is in O
      return wait_warp(pv_done + j % PB, (j / PB) & 1);
    };
    int it = 0;
    bool ok = true;
    for (uint32_t w = w0; ok && w < w1;) {
      const TreeSpan sp = tree_find<kTcTile, N>(p, base, w);
      const int nt = min(static_cast<int>(w1 - w), sp.tiles - sp.tile);
      const int64_t head = static_cast<int64_t>(sp.b) * p.kvh + sp.h;
      bool taken = false;
      // Q into its swizzled chunks (the last scores of the segment before have been
      // read, so its MMAs are done), all loads in flight together and with the masks; rows
      // past the block are zeros
      {
        constexpr int U = D / 8, NQ = N * U / kSoft;  // 16-byte units per row / thread
        uint4 v[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          const int r = (tid + i * kSoft) / U, x = (tid + i * kSoft) % U;
          const int rr = sp.rb * N + r, t = over_g(p, rr);
          const T* qp = static_cast<const T*>(p.q) + sp.b * p.qb + t * p.qt +
                        (static_cast<int64_t>(sp.h) * p.G + (rr - t * p.G)) * p.qh;
          v[i] = r < sp.rows ? reinterpret_cast<const uint4*>(qp)[x]
                             : make_uint4(0, 0, 0, 0);
        }
        if ((sp.tile + nt) * kTcTile > sp.len)
          tree_masks(p, sp.b, sp.n, sp.rb * N + r0, RW, mask, lane);
        if constexpr (Q8) {
          // f16, each row scaled by a power of two (undone by srow); the row's U units
          // lie in U neighbouring lanes
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            const T* e = reinterpret_cast<const T*>(&v[i]);
            float am = 0.0f;
#pragma unroll
            for (int y = 0; y < 8; ++y) am = fmaxf(am, fabsf(to_f32(e[y])));
#pragma unroll
            for (int o = 1; o < U; o <<= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
            const float qs = query_scale(am);
            uint32_t f[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              f[y] = pack16<false>(to_f32(e[2 * y]) * qs, to_f32(e[2 * y + 1]) * qs);
            v[i] = make_uint4(f[0], f[1], f[2], f[3]);
            if ((tid + i * kSoft) % U == 0) srow[(tid + i * kSoft) / U] = p.sl2 / qs;
          }
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          const int r = (tid + i * kSoft) / U, x = (tid + i * kSoft) % U;
          *reinterpret_cast<uint4*>(smem + (x >> 3) * S::kQChunk + r * 128 +
                                    (((x & 7) ^ (r & 7)) << 4)) = v[i];
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      float l[SUM ? 1 : RW];
#pragma unroll
      for (int i = 0; i < (SUM ? 1 : RW); ++i) l[i] = 0.0f;
      // the scales of this thread's key, loaded two tiles ahead
      float ks_next[2], vs_next[2];
      auto load_scales = [&](int t, int slot) {
        const int key = (sp.tile + t) * kTcTile + kt;
        const bool in = key < sp.len + sp.n;
        ks_next[slot] = in ? p.ks[head * p.P + key] : 0.0f;
        vs_next[slot] = in ? p.vs[head * p.P + key] : 0.0f;
      };
      if constexpr (Q8) {
        load_scales(0, 0);
        load_scales(1, 1);
      }

      for (int t = 0; t < nt; ++t, ++it) {
        const int at = (sp.tile + t) * kTcTile + kt - sp.len;  // this key's place in the draft
        const bool tail = (sp.tile + t + 1) * kTcTile > sp.len, first = t == 0;
        // the rows that see this key, as bits: all of a context key, of a drafted one those
        // whose token's set holds it
        uint32_t seen = ~0u;
        if (tail && at >= 0) {
          seen = 0u;
          if (at < sp.n)
#pragma unroll 8
            for (int i = 0; i < RW; ++i) seen |= static_cast<uint32_t>(mask[i] >> at & 1ull) << i;
        }
        float ksc = 1.0f, vsc = 1.0f, lvs = 0.0f;
        bool no_scale = false;  // V's scale is a NaN
        if constexpr (Q8) {
          ksc = ks_next[0];
          asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lvs) : "f"(vs_next[0]));
          no_scale = vs_next[0] != vs_next[0];
          vsc = fminf(vs_next[0], 3.0e38f);
          ks_next[0] = ks_next[1];
          vs_next[0] = vs_next[1];
          load_scales(t + 2, 1);
        }
        bool got = wait_warp(s_full + (it & 1), (it >> 1) & 1);
        tc_fence_after();
        auto scores = [&](uint32_t (&s)[32]) {
          tmem_ld_32x32b_x32(tmem + (it & 1) * N + lane_off + r0, s);
          tmem_wait_ld_tie(s);
          if constexpr (Q8) {  // the row's factor, then the key's (last where nothing is masked)
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 y = *reinterpret_cast<const float4*>(srow + r0 + i);
              const float y4[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                s[i + x] = __float_as_uint(__uint_as_float(s[i + x]) * y4[x]);
                if (tail) s[i + x] = __float_as_uint(__uint_as_float(s[i + x]) * ksc);
              }
            }
          }
          if (tail) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen >> i & 1u)) s[i] = __float_as_uint(-INFINITY);
          }
        };
        if (!Q8 && tail && got && sw < 4) {  // this thread's V row, once it has landed
          // A wait tells a phase from the next only: this one, of load 2 it + 1, is right if load
          // 2 it + 1 - NS of the same slot has completed.  S(it) has been waited for; it was
          // issued after S(it - 1) and O(it - 2), which waited for the loads up to 2 it except V's
          // of tile it - 1, 2 it - 1: any but NS = 2.
          const int slot = 2 * it + 1;
          got = wait_warp(full + slot % NS, (slot / NS) & 1);
          if (got && at >= 0) {
            uint8_t* tv = smem + S::kOffRing + (slot % NS) * S::kTile;
            auto unit = [&](int u) {
              return tv + (u >> 3) * kTcTile * 128 + kt * 128 + (((u & 7) ^ (kt & 7)) << 4);
            };
            if (at >= sp.n) {
#pragma unroll
              for (int u = 0; u < D / 8; ++u)
                *reinterpret_cast<uint4*>(unit(u)) = make_uint4(0u, 0u, 0u, 0u);
            } else {
              uint32_t any = 0u;
#pragma unroll
              for (int u = 0; u < D / 8; ++u)
                any |= non_finite_in<T>(*reinterpret_cast<const uint4*>(unit(u)));
              if (any != 0u)
#pragma unroll 1
                for (int u = 0; u < D / 8; ++u) taken |= clean_unit<T>(unit(u), false);
            }
          }
        }
        // ---- does a score pass its row's reference by more than the margin?  The
        // exponentials are taken at once and looked at afterwards
        const float unit = !Q8 ? p.sl2 : tail ? 1.0f : ksc;  // scores to log2 units
        auto expo = [&](uint32_t (&x)[32]) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 nr = *reinterpret_cast<const float4*>(nref + r0 + i);
            const float n4[4] = {nr.x, nr.y, nr.z, nr.w};
#pragma unroll
            for (int y = 0; y < 4; ++y)
              x[i + y] = __float_as_uint(ex2_approx(fmaf(__uint_as_float(x[i + y]), unit, n4[y])));
          }
        };
        // int8: p * v's scale goes into P, against its own reference: at most 2^15 (a scale
        // NaN counts as 3e38 until P is stored)
        uint32_t pk[16];
        auto weigh = [&](const uint32_t (&x)[32]) -> float {
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 y = *reinterpret_cast<const float4*>(frow + r0 + i);
            const float y4[4] = {y.x, y.y, y.z, y.w};
            float z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              z[j] = __uint_as_float(x[i + j]) * y4[j] * vsc;
              top = fmaxf(top, z[j]);
            }
            pk[i / 2] = pack16<false>(z[0], z[1]);
            pk[i / 2 + 1] = pack16<false>(z[2], z[3]);
          }
          return top;
        };
        uint32_t e[32];
        // int8: always where drafted keys are, so that no row's result hangs on the scales of
        // keys that it does not see
        bool need = first || !got || (Q8 && tail);
        if (!need) {
          float top = -INFINITY;
          scores(e);
          expo(e);
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(e[i]));
          need = top > RaiseS::most;
          if constexpr (Q8) need |= weigh(e) > RaiseP::most;
        }
        if (soft_any<kSoft>(need)) {
          if (got) {
            uint32_t s[32];
            scores(s);
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(s[i]) * unit;
            if constexpr (Q8) {
              float x[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = v[i] + lvs;
              smax[(4 + q4) * N + r0 + lane] = across_lanes<false>(x, lane);
            }
            smax[q4 * N + r0 + lane] = across_lanes<false>(v, lane);
          }
          if (lane == 0) wait_ok[sw] = got;
          soft_sync<kSoft>();
          bool all_ok = true;
#pragma unroll
          for (int k = 0; k < kSoft / 32; ++k) all_ok &= wait_ok[k] != 0;
          if (!all_ok) {  // a wait ran out: the softmax warps leave together
            ok = false;
            break;
          }
          if (tid < N) {
            const float top = fmaxf(fmaxf(smax[tid], smax[N + tid]),
                                    fmaxf(smax[2 * N + tid], smax[3 * N + tid]));
            const float old = first ? -INFINITY : -nref[tid];
            const float now = fmaxf(old, top - RaiseS::lower);
            // a row without a score above -inf keeps 0: its probabilities are 0 (or NaN)
            nref[tid] = now == -INFINITY ? 0.0f : -now;
            fact[tid] = first ? 0.0f : ex2_approx(old - now);
            if constexpr (Q8) {
              const float* m = smax + 4 * N + tid;
              const float old_e = first ? -INFINITY : eref[tid];
              const float now_e = fmaxf(old_e, fmaxf(fmaxf(m[0], m[N]), fmaxf(m[2 * N], m[3 * N])) -
                                                   RaiseP::lower);
              eref[tid] = now_e;
              facto[tid] = old_e == -INFINITY ? 0.0f : ex2_approx(old_e - now_e);
              // capped: p, at most 2^8, times it stays finite
              frow[tid] = now_e == -INFINITY ? 0.0f : ex2_approx(fminf(now - now_e, 119.0f));
            }
          }
          soft_sync<kSoft>();
          // O is final up to the tile before; rescale it and the sums (where the wait
          // runs out, the next vote ends the segment)
          if (!first && wait_pv(it - 1)) {
            tc_fence_after();
            auto rescale = [&](uint32_t at, const float* by) {
              uint32_t ov[32];
              tmem_ld_32x32b_x32(at + lane_off + r0, ov);
              tmem_wait_ld_tie(ov);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                ov[i] = __float_as_uint(__uint_as_float(ov[i]) * by[r0 + i]);
              tmem_st_32x32b_x32(at + lane_off + r0, ov);
            };
            rescale(tO, Q8 ? facto : fact);
            if constexpr (!SUM) {
#pragma unroll
              for (int i = 0; i < RW; ++i) l[i] *= fact[r0 + i];
            } else if (D == 128 && q4 == 0) {
              rescale(tL, fact);
            }
            tmem_wait_st();
          }
          scores(e);
          expo(e);
          if constexpr (Q8) weigh(e);
        }
        // ---- P: 16 bits, this key's row
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free + (it & 1));  // S may be overwritten
        if constexpr (!SUM) {
#pragma unroll
          for (int i = 0; i < 32; ++i) l[i] += __uint_as_float(e[i]);
        }
        if constexpr (!Q8) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            pk[i / 2] = pack16<std::is_same<T, __nv_bfloat16>::value>(__uint_as_float(e[i]),
                                                                      __uint_as_float(e[i + 1]));
        }
        if (Q8 && no_scale) {  // NaN for every row that sees the key, whatever its weight
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            pk[i / 2] |= (seen >> i & 1u) * 0x7fffu | (seen >> (i + 1) & 1u) * 0x7fff0000u;
        }
        // this P buffer is free once the tile that was in it has been contracted
        if (it >= PB) wait_pv(it - PB);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int u = r0 / 8 + x;
          *reinterpret_cast<uint4*>(smem + S::kOffP + (it % PB) * S::kPOne + (u >> 3) * S::kPChunk +
                                    kt * 128 + (((u & 7) ^ (kt & 7)) << 4)) =
              make_uint4(pk[4 * x], pk[4 * x + 1], pk[4 * x + 2], pk[4 * x + 3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + it % PB);
      }
      if (!ok) break;
      // ---- the segment's partial
      if constexpr (!SUM) smax[q4 * N + r0 + lane] = across_lanes<true>(l, lane);
      if constexpr (Q8) {  // O back to the scores' own reference
        if (tid < N) smax[4 * N + tid] = eref[tid] == -INFINITY ? 0.0f : ex2_approx(eref[tid] + nref[tid]);
      }
      ok = wait_pv(it - 1);
      if constexpr (SUM) {  // the ones' rows, alike in every lane
        if (ok && q4 == (D == 128 ? 0 : 2)) {
          tc_fence_after();
          uint32_t lv[32];
          tmem_ld_32x32b_x32((D == 128 ? tL : tO) + lane_off + r0, lv);
          tmem_wait_ld_tie(lv);
          float x = __uint_as_float(lv[0]);
#pragma unroll
          for (int i = 1; i < 32; ++i) x = lane == i ? __uint_as_float(lv[i]) : x;
          smax[r0 + lane] = x;
        }
      }
      const bool any_taken = soft_any<kSoft>(taken);
      if (ok) {
        tc_fence_after();
        const int64_t item = head * p.nrb + sp.rb;
        float* pp = p.part + (static_cast<int64_t>(blockIdx.x) + item) * N * part_stride<D>();
        if (tid < sp.rows) {
          float* row = pp + tid * part_stride<D>();
          const float sum = SUM ? smax[tid]
                                : (smax[tid] + smax[N + tid]) + (smax[2 * N + tid] + smax[3 * N + tid]);
          row[D] = sum == 0.0f ? -INFINITY : -nref[tid];  // a row that sees nothing here
          row[D + 1] = sum;
          row[D + 2] = any_taken ? 1.0f : 0.0f;
        }
        if (D == 128 || q4 < 2) {  // thread = output dim
          uint32_t ov[32];
          tmem_ld_32x32b_x32(tO + lane_off + r0, ov);
          tmem_wait_ld_tie(ov);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (r0 + i < sp.rows)
              pp[(r0 + i) * part_stride<D>() + kt] =
                  __uint_as_float(ov[i]) * (Q8 ? smax[4 * N + r0 + i] : 1.0f);
        }
        tc_fence_before();
      }
      // nref, smax and O are used again by the next segment only after this
      if (soft_any<kSoft>(!ok)) ok = false;
      w += nt;
    }
  } else if constexpr (Q8) {
    // ---- codes to f16 tiles
    const int ct = (warp < 4 ? warp - 2 : warp - 2 - kSoft / 32) * 32 + lane;
    constexpr int U = D / 16, NU = kTcTile * U / (32 * S::kConv);  // 16-code units per row / thread
    const int nloads = 2 * static_cast<int>(w1 - w0);
    auto wait_conv = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu,
                        mbar_wait_bounded(bar, parity, abort_flag, p.err, kErrWaitOther));
    };
    for (int it = 0; it < nloads; ++it) {
      const int s8 = it % N8, st = it % NS;
      if (!wait_conv(full8 + s8, (it / N8) & 1)) break;
      const uint8_t* src = smem + S::kOffCodes + s8 * S::kCodes;
      uint4 x[NU];
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int u = ct + i * 32 * S::kConv, key = u / U, c = u % U;
        const int at = D == 128 ? key * 128 + ((c ^ (key & 7)) << 4)
                                : key * 64 + ((c ^ ((key >> 1) & 3)) << 4);
        x[i] = *reinterpret_cast<const uint4*>(src + at);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty8 + s8);
      if (!wait_conv(empty + st, ((it / NS) & 1) ^ 1)) break;
      uint8_t* dst = smem + S::kOffRing + st * S::kTile;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int u = ct + i * 32 * S::kConv, key = u / U, c = u % U;
        const uint32_t wd[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t f[8];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t z = wd[y] ^ 0x80808080u;
          f[2 * y] = codes_f16(z, 0x4140);
          f[2 * y + 1] = codes_f16(z, 0x4342);
        }
        // the upper chunk's units in the other order: no bank conflicts between the chunks
        const bool swap = (c >> 2) & 1;
        uint8_t* row = dst + (c >> 2) * kTcTile * 128 + key * 128;
        const int w0u = ((c & 3) * 2 + swap) ^ (key & 7), w1u = ((c & 3) * 2 + !swap) ^ (key & 7);
        const uint4 lo = make_uint4(f[0], f[1], f[2], f[3]), hi = make_uint4(f[4], f[5], f[6], f[7]);
        *reinterpret_cast<uint4*>(row + (w0u << 4)) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(row + (w1u << 4)) = swap ? lo : hi;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + st);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

// ----------------------------------------------------------------- combine --
constexpr int kCWarps = 8;  // query rows per CTA

// One warp per query row: its block's partials are those of consecutive shares.
template <class T, int D>
__global__ void __launch_bounds__(32 * kCWarps) tree_combine_kernel(const TreeParams p) {
  constexpr int DL = D / 32;
  __shared__ uint32_t base[kScanWords];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_release();
  if (warp == 0) tree_scan<0, 0>(p, base, lane);
  __syncthreads();
  const uint32_t total = base[p.B];
  const uint32_t shares = min(total, static_cast<uint32_t>(p.grid));
  const int R = p.G * p.T;
  const int row = blockIdx.x * kCWarps + warp;
  if (row >= p.B * p.kvh * R) {
    grid_wait();
    return;
  }
  const int bh = row / R, r = row - bh * R;
  const int b = bh / p.kvh, h = bh - b * p.kvh;
  const int t = r / p.G, head = h * p.G + (r - t * p.G);
  const int len = static_cast<int>(base[kTBatch + 2 + b]);
  const int n = static_cast<int>(base[2 * (kTBatch + 2) + b]);
  if (h == 0 && r == 0 && lane == 0) {
    int x, y;
    if (!tree_seq(p, b, x, y)) atomicExch(p.err, kErrBadCacheLen);
  }
  float acc[DL], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < DL; ++i) acc[i] = 0.0f;
  grid_wait();  // the partials are complete
  if (t < n) {
    const int rb = r / p.rb, tiles = tiles_of<0>(p, len, n), nrb = row_blocks<0>(p, n);
    const uint32_t t0 = base[b] + (static_cast<uint32_t>(h) * nrb + rb) * tiles;
    const Shares share(total, shares);
    const uint32_t c0 = share.of(t0), c1 = share.of(t0 + tiles - 1);
    const int64_t item = static_cast<int64_t>(bh) * p.nrb + rb;
    const float* pr = p.part + ((c0 + item) * p.rb + (r - rb * p.rb)) * part_stride<D>();
    bool taken = false;
    for (uint32_t c = c0; c <= c1; ++c, pr += static_cast<int64_t>(p.rb) * part_stride<D>()) {
      const float4 st = *reinterpret_cast<const float4*>(pr + D);  // max, sum, taken
      float x[DL];
#pragma unroll
      for (int i = 0; i < DL; ++i) x[i] = pr[lane * DL + i];
      const float mn = fmaxf(m, st.x);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      const float fa = exp2f(m - ref), fb = exp2f(st.x - ref);
      l = l * fa + st.y * fb;
#pragma unroll
      for (int i = 0; i < DL; ++i) acc[i] = acc[i] * fa + x[i] * fb;
      m = mn;
      taken |= st.z != 0.0f;
    }
    if (taken) {
      // infinities and NaN of the drafted values that this token sees
      const T* v = static_cast<const T*>(p.vc) + (static_cast<int64_t>(bh) * p.P + len) * D + lane * DL;
      for (int a = t, steps = 0; a >= 0 && steps < kTMaxTokens; ++steps) {
#pragma unroll
        for (int i = 0; i < DL; ++i) {
          const float x = to_f32(v[static_cast<int64_t>(a) * D + i]);
          if (!(fabsf(x) <= 3.402823466e38f)) acc[i] += x;
        }
        const int up = p.parents ? p.parents[static_cast<int64_t>(b) * p.T + a] : a - 1;
        a = up < a ? up : -1;
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a NaN sum stays one
  T* og = static_cast<T*>(p.o) + b * p.ob + t * p.ot + head * p.oh + lane * DL;
  T y[DL];
#pragma unroll
  for (int i = 0; i < DL; ++i) y[i] = from_f32<T>(acc[i] * inv);
  if constexpr (DL == 4) *reinterpret_cast<uint2*>(og) = *reinterpret_cast<const uint2*>(y);
  else *reinterpret_cast<uint32_t*>(og) = *reinterpret_cast<const uint32_t*>(y);
}

// ---------------------------------------------------------------- launchers --
// Rows of a block.  Up to 16 rows go to mma.sync; more to tcgen05, in the smallest block
// that holds them, of at most 128 rows (64 for int8 caches).  17 int8 rows of 128 dims, 8 x
// 32 heads x 16384 positions: 0.34 ms in one block, about 0.52 in two of mma.sync; 12 rows
// 0.26 ms on mma.sync.
int block_rows(int rows, bool q8) {
  if (rows <= 8) return 8;
  if (rows <= kMRows) return kMRows;
  if (rows <= 32) return 32;
  return rows <= 64 || q8 ? 64 : 128;
}

size_t tree_slots(int B, int T, int G, int kvh, int grid, int rb, int& nrb) {
  nrb = (G * T + rb - 1) / rb;
  return static_cast<size_t>(B) * kvh * nrb + grid;
}

// Tile length, and the CTAs that share the tiles (at most kTMaxGrid).
void set_tiles(TreeParams& p, int tile) {
  const int64_t most = static_cast<int64_t>(p.B) * p.kvh * p.nrb * ((p.P + tile - 1) / tile);
  LTM_REQUIRE(most < (1ll << 31), "too many tiles");
  const int sms = device_sm_count() < kTMaxGrid ? device_sm_count() : kTMaxGrid;
  p.tile = tile;
  p.grid = static_cast<int>(most < sms ? most : sms);
}

template <class T, int D>
void launch_combine(const TreeParams& p, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.kvh * p.G * p.T;
  // launched while the tiles are still contracted; it waits for them on the device
  launch_dependent(tree_combine_kernel<T, D>,
                   dim3(static_cast<unsigned>((rows + kCWarps - 1) / kCWarps)), 32 * kCWarps, 0, st,
                   p);
  check_launch("tree_combine_kernel", st);
}

template <class T, int D, bool Q8, int NR>
void launch_mma(TreeParams p, cudaStream_t st) {
  using S = MmaSmem<D, Q8, NR>;
  set_tiles(p, S::kKeys);
  const CUtensorMapDataType dt = Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tma_dtype_of<T>();
  const uint64_t rows = static_cast<uint64_t>(p.B) * p.kvh * p.P;
  const CUtensorMapSwizzle sw =
      S::kBox == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap tk, tv;
  make_tma_2d(&tk, p.kc, dt, Q8 ? 1 : 2, rows, D, D, S::kBox / (Q8 ? 1 : 2), S::kKeys, sw);
  make_tma_2d(&tv, p.vc, dt, Q8 ? 1 : 2, rows, D, D, S::kBox / (Q8 ? 1 : 2), S::kKeys, sw);
  auto kern = tree_mma_kernel<T, D, Q8, NR>;
  allow_smem(kern, S::kBytes);
  launch_dependent(kern, dim3(static_cast<unsigned>(p.grid)), 32 * (S::kWarps + 1), S::kBytes, st,
                   tk, tv, p);
  check_launch("tree_mma_kernel", st);
  launch_combine<T, D>(p, st);
}

template <class T, int D, int N, bool Q8>
void launch_tc(TreeParams p, cudaStream_t st) {
  using S = TcSmem<D, N, Q8>;
  set_tiles(p, kTcTile);
  const uint64_t rows = static_cast<uint64_t>(p.B) * p.kvh * p.P;
  CUtensorMap tk, tv;
  const CUtensorMapDataType dt = Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tma_dtype_of<T>();
  const CUtensorMapSwizzle sw =
      Q8 && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  make_tma_2d(&tk, p.kc, dt, Q8 ? 1 : 2, rows, D, D, Q8 ? D : 64, kTcTile, sw);
  make_tma_2d(&tv, p.vc, dt, Q8 ? 1 : 2, rows, D, D, Q8 ? D : 64, kTcTile, sw);
  auto kern = tree_tc_kernel<T, D, N, Q8>;
  allow_smem(kern, S::kBytes);
  launch_dependent(kern, dim3(static_cast<unsigned>(p.grid)), S::kThreads, S::kBytes, st, tk, tv,
                   p);
  check_launch("tree_tc_kernel", st);
  launch_combine<T, D>(p, st);
}

}  // namespace
}  // namespace ltm_b200

using namespace ltm_b200;

namespace {
void check_tree(int B, int T, int heads, int kv_heads, int head_dim, int64_t P) {
  LTM_REQUIRE(B >= 0 && T >= 0 && heads >= 1 && kv_heads >= 1 && P >= 1, "bad size");
  if (head_dim != 64 && head_dim != 128) LTM_UNSUPPORTED("head_dim must be 64 or 128");
  LTM_REQUIRE(heads % kv_heads == 0, "num_heads must be a multiple of kv_heads");
  if (T > kTMaxTokens) LTM_UNSUPPORTED("more than 64 drafted tokens");
  if (heads / kv_heads > 64) LTM_UNSUPPORTED("more than 64 query heads per cached head");
  LTM_REQUIRE(P < (1ll << 31), "max_positions exceeds int32");
}
}  // namespace

extern "C" ltm_status ltm_tree_attention_workspace(int B, int T, int num_heads, int kv_heads,
                                                   int head_dim, size_t* bytes) {
  return guarded([&] {
    LTM_REQUIRE(bytes != nullptr, "NULL pointer");
    check_tree(B, T, num_heads, kv_heads, head_dim, 1);
    const int G = num_heads / kv_heads;
    int nrb = 0;
    size_t most = 0;
    for (int q8 = 0; q8 < 2; ++q8) {
      const int rb = block_rows(G * T, q8 != 0);
      const size_t n = tree_slots(B < kTBatch ? B : kTBatch, T, G, kv_heads, kTMaxGrid, rb, nrb) * rb;
      if (n > most) most = n;
    }
    *bytes = most * (head_dim + 4) * sizeof(float);
  });
}

extern "C" ltm_status ltm_tree_attention(
    const void* q, const int64_t* q_strides, const void* k_cache, const void* v_cache,
    const float* k_scale, const float* v_scale, int64_t max_positions, const int32_t* cache_lens,
    const int32_t* num_tokens, const int32_t* parents, void* o, const int64_t* o_strides, int B,
    int T, int num_heads, int kv_heads, int head_dim, ltm_dtype dtype, void* workspace,
    size_t workspace_bytes, void* stream) {
  return guarded([&] {
    check_tree(B, T, num_heads, kv_heads, head_dim, max_positions);
    if (dtype != LTM_DTYPE_F16 && dtype != LTM_DTYPE_BF16)
      LTM_UNSUPPORTED("tree attention needs f16 or bf16 activations");
    if (B == 0 || T == 0) return;
    LTM_REQUIRE(q && q_strides && k_cache && v_cache && cache_lens && o && o_strides && workspace,
                "NULL pointer");
    LTM_REQUIRE((k_scale == nullptr) == (v_scale == nullptr), "give both scales or neither");
    const uintptr_t mis = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) |
                          reinterpret_cast<uintptr_t>(k_cache) |
                          reinterpret_cast<uintptr_t>(v_cache) |
                          reinterpret_cast<uintptr_t>(workspace);
    LTM_REQUIRE((mis & 15) == 0, "q, the output, the caches and the workspace must be 16-byte aligned");
    for (int i = 0; i < 3; ++i)
      LTM_REQUIRE(q_strides[i] % 8 == 0 && o_strides[i] % 8 == 0,
                  "q and output strides must be multiples of 8 elements");
    const int G = num_heads / kv_heads;
    const bool q8 = k_scale != nullptr;
    const int rb = block_rows(G * T, q8);
    TreeParams p{};
    p.qt = q_strides[1];
    p.qh = q_strides[2];
    p.qb = q_strides[0];
    p.ob = o_strides[0];
    p.ot = o_strides[1];
    p.oh = o_strides[2];
    p.T = T;
    p.G = G;
    p.inv_g = 1.0f / static_cast<float>(G);
    p.kvh = kv_heads;
    p.P = max_positions;
    p.sl2 = 1.4426950408889634f / sqrtf(static_cast<float>(head_dim));
    p.part = static_cast<float*>(workspace);
    p.err = device_error_ptr();
    const cudaStream_t st = as_stream(stream);
    const size_t row = static_cast<size_t>(head_dim) * (q8 ? 1 : 2);
    for (int b0 = 0; b0 < B; b0 += kTBatch) {
      p.B = B - b0 < kTBatch ? B - b0 : kTBatch;
      const int64_t heads0 = static_cast<int64_t>(b0) * kv_heads;
      LTM_REQUIRE(static_cast<int64_t>(p.B) * kv_heads * max_positions < (1ll << 31),
                  "cache rows exceed int32");
      LTM_REQUIRE(static_cast<int64_t>(p.B) * num_heads * T < (1ll << 31) - kCWarps,
                  "query rows exceed int32");
      p.rb = rb;
      const size_t slots = tree_slots(p.B, T, G, kv_heads, kTMaxGrid, rb, p.nrb);
      LTM_REQUIRE(workspace_bytes >= slots * rb * (head_dim + 4) * sizeof(float),
                  "workspace too small");
      p.q = static_cast<const uint8_t*>(q) + 2 * b0 * p.qb;
      p.o = static_cast<uint8_t*>(o) + 2 * b0 * p.ob;
      p.kc = static_cast<const uint8_t*>(k_cache) + heads0 * max_positions * row;
      p.vc = static_cast<const uint8_t*>(v_cache) + heads0 * max_positions * row;
      p.ks = q8 ? k_scale + heads0 * max_positions : nullptr;
      p.vs = q8 ? v_scale + heads0 * max_positions : nullptr;
      p.lens = cache_lens + b0;
      p.ntok = num_tokens ? num_tokens + b0 : nullptr;
      p.parents = parents ? parents + static_cast<int64_t>(b0) * T : nullptr;
      auto go = [&](auto t_c, auto d_c, auto q_c) {
        using E = decltype(t_c);
        constexpr int D = decltype(d_c)::value;
        constexpr bool Q = decltype(q_c)::value;
        if (rb == 8) {
          launch_mma<E, D, Q, 1>(p, st);
        } else if (rb == kMRows) {
          launch_mma<E, D, Q, 2>(p, st);
        } else if (rb == 32) {
          launch_tc<E, D, 32, Q>(p, st);
        } else if (rb == 64) {
          launch_tc<E, D, 64, Q>(p, st);
        } else if constexpr (!Q) {
          launch_tc<E, D, 128, false>(p, st);
        }
      };
      auto by_q = [&](auto t_c, auto d_c) {
        if (q8) go(t_c, d_c, std::true_type{});
        else go(t_c, d_c, std::false_type{});
      };
      auto by_d = [&](auto t_c) {
        if (head_dim == 64) by_q(t_c, std::integral_constant<int, 64>{});
        else by_q(t_c, std::integral_constant<int, 128>{});
      };
      if (dtype == LTM_DTYPE_BF16) by_d(__nv_bfloat16{});
      else by_d(__half{});
    }
  });
}
