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
// The mask only concerns the T newest positions, so the work is split there:
//
// * tree_context_kernel: all G * T rows of a (sequence, head) against the
//   context.  No mask but the context's end.  Every cached byte is read once;
//   that read is the bound.  The tiles (128 positions of one head) of the whole
//   batch, whatever the lengths, form one list that the persistent CTAs (one
//   per SM) share out evenly; a CTA that ends or starts inside a head leaves a
//   partial (max, sum, output) there.
//   Warp 0 streams K and V tiles by TMA into a ring of swizzled stages; eight
//   consumer warps contract them on mma.sync m16n8k16 (the rows of a decode
//   step fill a fraction of a 128-row tcgen05 tile): each warp scores 16 of the
//   tile's keys, writes its probabilities to shared memory, and accumulates
//   its D / 8 output dims over all 128 keys.  The rows' reference maximum is
//   shared and only raised when a score exceeds it by more than 2^8.
//   int8 codes become f16 in registers (exact), with the row's scale applied
//   to the fp32 score (K) and to the probability (V).
// * tree_combine_kernel: one warp per query row walks the row's ancestors in
//   fp32 (a few rows of shared memory, no mask arithmetic, so a non-finite
//   value of one branch cannot reach another), merges the context's partials
//   and writes the output.
//
// The reference has no counterpart: its cache manager is a stub
// (python_bindings/src/main.cpp:101-135).
#include <type_traits>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kTTile = 128;       // cache positions per tile
constexpr int kTCons = 8;         // consumer warps
constexpr int kTBatch = 512;      // sequences per launch
constexpr int kTMaxTokens = 64;   // drafted tokens (one 64-bit ancestor mask)
constexpr float kTRaise = 8.0f;   // log2 of the largest probability before the reference is raised

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
  int B, T, G, kvh, nrb;  // nrb: row blocks per cached head
  int64_t P;
  float sl2;
  float* part;
  int grid;  // CTAs of the context kernel
  int* err;
};

template <int D>
constexpr int part_stride() { return D + 4; }  // output, max, sum (16-byte rows)

// Context length (0: nothing to do) and tokens of sequence b.
__device__ __forceinline__ bool tree_seq(const TreeParams& p, int b, int& len, int& n) {
  len = p.lens[b];
  n = p.ntok ? p.ntok[b] : p.T;
  const bool ok = len >= 0 && n >= 0 && n <= p.T && static_cast<int64_t>(len) + n <= p.P;
  if (!ok) len = n = 0;
  return ok;
}

__device__ __forceinline__ int tiles_of(int len) { return (len + kTTile - 1) / kTTile; }
template <int RB>
__device__ __forceinline__ int row_blocks(const TreeParams& p, int n) {
  return (p.G * n + RB - 1) / RB;
}

// First tile of every sequence in the batch's list (one warp).
template <int RB>
__device__ __forceinline__ void tree_scan(const TreeParams& p, uint32_t* base, int lane) {
  uint32_t carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    uint32_t w = 0;
    if (b < p.B) {
      int len, n;
      tree_seq(p, b, len, n);
      w = static_cast<uint32_t>(p.kvh) * row_blocks<RB>(p, n) * tiles_of(len);
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
__device__ __forceinline__ uint32_t share_start(uint32_t c, uint32_t total, uint32_t grid) {
  return static_cast<uint32_t>(static_cast<uint64_t>(c) * total / grid);
}
__device__ __forceinline__ uint32_t share_of(uint32_t tile, uint32_t total, uint32_t grid) {
  return static_cast<uint32_t>((static_cast<uint64_t>(tile + 1) * grid - 1) / total);
}

// Where tile w of the list lies.
struct TreeSpan {
  int b, h, rb, len, rows, tile, tiles;  // tile: index within the head's context
};
template <int RB>
__device__ __forceinline__ TreeSpan tree_find(const TreeParams& p, const uint32_t* base, uint32_t w) {
  int lo = 0, hi = p.B;  // base[lo] <= w < base[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (base[mid] <= w) lo = mid;
    else hi = mid;
  }
  TreeSpan s;
  s.b = lo;
  int n;
  tree_seq(p, lo, s.len, n);
  s.tiles = tiles_of(s.len);
  const int nrb = row_blocks<RB>(p, n);
  const uint32_t at = w - base[lo];
  const uint32_t item = at / s.tiles;
  s.tile = static_cast<int>(at - item * s.tiles);
  s.h = static_cast<int>(item / nrb);
  s.rb = static_cast<int>(item - s.h * nrb);
  s.rows = min(RB, p.G * n - s.rb * RB);
  return s;
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
// Barrier of the consumer warps; true where any thread's predicate holds.
__device__ __forceinline__ bool cons_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "n"(kTCons * 32)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void cons_sync() {
  asm volatile("barrier.cta.sync 1, %0;" ::"n"(kTCons * 32) : "memory");
}

// ------------------------------------------------------------ shared memory --
template <int D, bool Q8, int MT>
struct TreeSmem {
  static constexpr int kRow = D * (Q8 ? 1 : 2);                 // bytes per cached row
  static constexpr int kBox = kRow > 128 ? 128 : kRow;          // bytes per row of a TMA box
  static constexpr int kBoxes = kRow / kBox;
  static constexpr int kTile = kTTile * kRow;                   // K or V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = 196608 / kStage > 8 ? 8 : 196608 / kStage;
  static constexpr int RB = 16 * MT;
  static constexpr int kOffP = kStages * kStage;                // probabilities [RB][128] 16-bit
  static constexpr int kOffMax = kOffP + RB * kTTile * 2;       // [8][RB] x 2 row maxima, sums
  static constexpr int kOffBase = kOffMax + 2 * kTCons * RB * 4;
  static constexpr int kOffBar = kOffBase + (kTBatch + 2) * 4;
  static constexpr int kOffFlag = kOffBar + 2 * kStages * 8;
  static constexpr int kBytes = kOffFlag + 64 + 1024;
};

// Shared-memory offset of 16-byte unit c of row r of a tile (the TMA swizzle).
template <class S>
__device__ __forceinline__ uint32_t tile_unit(int r, int c) {
  if constexpr (S::kBox == 128)
    return static_cast<uint32_t>((c >> 3) * (kTTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  else  // 64-byte rows, 64-byte swizzle
    return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <class T, int D, bool Q8, int MT>
__global__ void __launch_bounds__(32 * (kTCons + 1), 1)
    tree_context_kernel(const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const TreeParams p) {
  using S = TreeSmem<D, Q8, MT>;
  constexpr int NS = S::kStages, KS = D / 16, RB = S::RB;
  constexpr int NO = D / 64;  // 8-dim output blocks per warp
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value && !Q8;  // type of the products
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* smax = reinterpret_cast<float*>(smem + S::kOffMax);  // [kTCons][RB]
  float* sevm = smax + kTCons * RB;                           // [kTCons][RB]
  uint32_t* base = reinterpret_cast<uint32_t*>(smem + S::kOffBase);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
  uint64_t* empty = full + NS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffFlag);
  int* wait_ok = reinterpret_cast<int*>(smem + S::kOffFlag) + 1;  // [kTCons]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, kTCons);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 0) tree_scan<RB>(p, base, lane);
  __syncthreads();
  const uint32_t total = base[p.B];
  if (total == 0) return;
  const uint32_t shares = min(total, gridDim.x);
  if (blockIdx.x >= shares) return;
  const uint32_t w0 = share_start(blockIdx.x, total, shares);
  const uint32_t w1 = share_start(blockIdx.x + 1, total, shares);

  if (warp == 0) {
    // ---- producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (uint32_t w = w0; ok && w < w1;) {
        const TreeSpan s = tree_find<RB>(p, base, w);
        const int nt = min(static_cast<int>(w1 - w), s.tiles - s.tile);
        const int row = static_cast<int>((static_cast<int64_t>(s.b) * p.kvh + s.h) * p.P) +
                        s.tile * kTTile;
        for (int t = 0; t < nt; ++t, ++it) {
          const int st = it % NS;
          if (!mbar_wait_bounded(empty + st, ((it / NS) & 1) ^ 1, abort_flag, p.err,
                                 kErrWaitEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full + st, S::kStage);
          uint8_t* dst = smem + st * S::kStage;
#pragma unroll
          for (int x = 0; x < S::kBoxes; ++x) {
            tma_load_2d(dst + x * kTTile * 128, &tmK, full + st, x * 64, row + t * kTTile);
            tma_load_2d(dst + S::kTile + x * kTTile * 128, &tmV, full + st, x * 64,
                        row + t * kTTile);
          }
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

  // ---- consumers: this warp's keys of a tile are cw * 16 .. + 15
  const int cw = warp - 1, g = lane >> 2, c = lane & 3;
  const uint32_t sP = smem_u32(smem + S::kOffP);
  int it = 0;
  for (uint32_t w = w0; w < w1;) {
    const TreeSpan sp = tree_find<RB>(p, base, w);
    const int nt = min(static_cast<int>(w1 - w), sp.tiles - sp.tile);
    const int64_t head = static_cast<int64_t>(sp.b) * p.kvh + sp.h;
    // Q as A fragments.  int8 codes: lane c of a quad holds dims c * D/4 ..
    // (the codes' own order, any order of the dims gives the same products) in
    // f16, each row scaled by a power of two so that its largest value is
    // below 2^15 (bf16 values reach beyond f16; the scale is undone in fp32).
    uint32_t aq[MT][KS][4];
    float qinv[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + g;
        const int rr = sp.rb * RB + r;
        const int t = rr / p.G, gg = rr - t * p.G;
        const T* qp = static_cast<const T*>(p.q) + sp.b * p.qb + t * p.qt +
                      (static_cast<int64_t>(sp.h) * p.G + gg) * p.qh;
        const bool live = r < sp.rows;
        if constexpr (!Q8) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            aq[mt][s][hf] = live ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + 2 * c) : 0u;
            aq[mt][s][hf + 2] =
                live ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + 8 + 2 * c) : 0u;
          }
          qinv[mt][hf] = p.sl2;
        } else {
          uint2 raw[KS];
          float am = 0.0f;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            raw[s] = live ? *reinterpret_cast<const uint2*>(qp + c * (D / 4) + 4 * s)
                          : make_uint2(0u, 0u);
            const T* e = reinterpret_cast<const T*>(&raw[s]);
#pragma unroll
            for (int i = 0; i < 4; ++i) am = fmaxf(am, fabsf(to_f32(e[i])));
          }
          am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
          am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
          int ex = static_cast<int>(__float_as_uint(am) >> 23);  // 2^(ex-127) <= am
          if (ex == 0 || ex == 255) ex = 141;                     // 0 or infinite: as it is
          const float qs = __uint_as_float(static_cast<uint32_t>(min(268 - ex, 254)) << 23);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const T* e = reinterpret_cast<const T*>(&raw[s]);
            aq[mt][s][hf] = pack16<false>(to_f32(e[0]) * qs, to_f32(e[1]) * qs);
            aq[mt][s][hf + 2] = pack16<false>(to_f32(e[2]) * qs, to_f32(e[3]) * qs);
          }
          qinv[mt][hf] = p.sl2 / qs;
        }
      }
    float o[MT][NO][4], l[MT][2], mref[MT][2], eref[MT][2], frow[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < NO; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.0f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        l[mt][hf] = 0.0f;
        mref[mt][hf] = eref[mt][hf] = -INFINITY;
        frow[mt][hf] = 0.0f;
      }
    }
    // the scales of this warp's 16 keys: K in lanes 0-15, V in lanes 16-31
    const float* scp = nullptr;
    float sc_next = 0.0f;
    if constexpr (Q8) {
      scp = (lane < 16 ? p.ks : p.vs) + head * p.P + cw * 16 + (lane & 15);
      const int key = sp.tile * kTTile + cw * 16 + (lane & 15);
      sc_next = key < sp.len ? __ldg(scp + sp.tile * kTTile) : 0.0f;
    }

    for (int t = 0; t < nt; ++t, ++it) {
      const int st = it % NS;
      const int key0 = (sp.tile + t) * kTTile;
      const float sc = sc_next;
      if constexpr (Q8) {
        if (t + 1 < nt)
          sc_next = key0 + kTTile + cw * 16 + (lane & 15) < sp.len ? __ldg(scp + key0 + kTTile)
                                                                   : 0.0f;
      }
      const bool got = __all_sync(
          0xffffffffu,
          mbar_wait_bounded(full + st, (it / NS) & 1, abort_flag, p.err, kErrWaitFull));
      uint8_t* tk = smem + st * S::kStage;
      uint8_t* tv = tk + S::kTile;
      const uint32_t ak = smem_u32(tk), av = smem_u32(tv);
      const bool tail = key0 + kTTile > sp.len;

      // ---- scores of this warp's 16 keys
      float acc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[mt][n][i] = 0.0f;
      if constexpr (!Q8) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t kb[4];
          const int i = lane >> 3;
          ldsm4(ak + tile_unit<S>(cw * 16 + (i >> 1) * 8 + (lane & 7), 2 * s + (i & 1)), kb);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16816<BF>(acc[mt][0], aq[mt][s], kb[0], kb[1]);
            mma16816<BF>(acc[mt][1], aq[mt][s], kb[2], kb[3]);
          }
        }
      } else {
        constexpr int NU = D / 64;  // 16-byte units per lane and key
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            const uint4 raw = lds128(ak + tile_unit<S>(cw * 16 + n * 8 + g, NU * c + u));
            const uint32_t wd[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = wd[i] ^ 0x80808080u;
              const uint32_t b0 = codes_f16(x, 0x4140), b1 = codes_f16(x, 0x4342);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                mma16816<false>(acc[mt][n], aq[mt][4 * u + i], b0, b1);
            }
          }
      }
      // ---- log2 scores; does any pass the reference by more than the margin?
      float ksc[2][2], vsc[2][2], lvs[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (Q8) {
            ksc[n][i] = __shfl_sync(0xffffffffu, sc, n * 8 + 2 * c + i);
            vsc[n][i] = __shfl_sync(0xffffffffu, sc, 16 + n * 8 + 2 * c + i);
            lvs[n][i] = __log2f(vsc[n][i]);
          } else {
            ksc[n][i] = vsc[n][i] = 1.0f;
            lvs[n][i] = 0.0f;
          }
        }
      bool need = !got;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float s = acc[mt][n][i] * qinv[mt][i >> 1];
            if constexpr (Q8) s *= ksc[n][i & 1];
            if (tail && key0 + cw * 16 + n * 8 + 2 * c + (i & 1) >= sp.len) s = -INFINITY;
            acc[mt][n][i] = s;
            need |= s > mref[mt][i >> 1] + kTRaise;
            if constexpr (Q8) need |= s + lvs[n][i & 1] > eref[mt][i >> 1] + kTRaise;
          }
      if constexpr (!Q8) {
        // rows past the context may hold anything: 0 * NaN must not reach the sums
        if (tail) {
          for (int u = lane; u < 16 * (S::kRow / 16); u += 32) {
            const int r = cw * 16 + u / (S::kRow / 16);
            if (key0 + r >= sp.len)
              *reinterpret_cast<uint4*>(tv + tile_unit<S>(r, u % (S::kRow / 16))) =
                  make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (cons_any(need)) {
        // raise the references to the tile's maxima (and rescale what is summed)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float a = -INFINITY, e = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                a = fmaxf(a, acc[mt][n][2 * hf + i]);
                if constexpr (Q8) e = fmaxf(e, acc[mt][n][2 * hf + i] + lvs[n][i]);
              }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
              a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
              if constexpr (Q8) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, x));
            }
            if (c == 0) {
              smax[cw * RB + mt * 16 + hf * 8 + g] = a;
              if constexpr (Q8) sevm[cw * RB + mt * 16 + hf * 8 + g] = e;
            }
          }
        if (lane == 0) wait_ok[cw] = got;
        cons_sync();
        bool all_ok = true;
#pragma unroll
        for (int k = 0; k < kTCons; ++k) all_ok &= wait_ok[k] != 0;
        if (!all_ok) return;  // a wait ran out: every consumer leaves here
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int r = mt * 16 + hf * 8 + g;
            float a = mref[mt][hf], e = eref[mt][hf];
#pragma unroll
            for (int k = 0; k < kTCons; ++k) {
              a = fmaxf(a, smax[k * RB + r]);
              if constexpr (Q8) e = fmaxf(e, sevm[k * RB + r]);
            }
            const float fl = mref[mt][hf] == -INFINITY ? 0.0f : ex2_approx(mref[mt][hf] - a);
            float fo = fl;
            if constexpr (Q8)
              fo = eref[mt][hf] == -INFINITY ? 0.0f : ex2_approx(eref[mt][hf] - e);
            l[mt][hf] *= fl;
#pragma unroll
            for (int n = 0; n < NO; ++n) {
              o[mt][n][2 * hf] *= fo;
              o[mt][n][2 * hf + 1] *= fo;
            }
            mref[mt][hf] = a;
            eref[mt][hf] = e;
            if constexpr (Q8) frow[mt][hf] = e == -INFINITY ? 0.0f : ex2_approx(a - e);
          }
      }
      // ---- probabilities into shared memory
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r = mt * 16 + hf * 8 + g;
          const float mu = mref[mt][hf] == -INFINITY ? 0.0f : mref[mt][hf];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            float x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              x[i] = ex2_approx(acc[mt][n][2 * hf + i] - mu);
              l[mt][hf] += x[i];
              if constexpr (Q8) {
                // p * v's scale, against its own reference: at most 2^8.  The
                // factor only overflows where p is 0.
                float f = vsc[n][i] * frow[mt][hf];
                f = f > 3.0e38f ? 3.0e38f : f;
                x[i] *= f;
              }
            }
            const uint32_t at = sP + r * 256 + (((2 * cw + n) ^ (r & 7)) << 4) + 4 * c;
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(pack16<BF>(x[0], x[1]))
                         : "memory");
          }
        }
      cons_sync();
      // ---- output dims of this warp over the tile's 128 keys
      const int i8 = lane >> 3, r8 = lane & 7;
#pragma unroll
      for (int s2 = 0; s2 < kTTile / 32; ++s2) {
        uint32_t vb[2][NO][2];  // [16-key step][output block][k half]
        if constexpr (!Q8 && D == 128) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[4];
            ldsm4_t(av + tile_unit<S>(32 * s2 + 16 * h + (i8 & 1) * 8 + r8, 2 * cw + (i8 >> 1)), r);
            vb[h][0][0] = r[0];
            vb[h][0][1] = r[1];
            vb[h][NO - 1][0] = r[2];
            vb[h][NO - 1][1] = r[3];
          }
        } else {
          // int8: 16-byte units hold 16 dims; the transposed 16-bit element is
          // a pair of neighbouring dims, split into an even and an odd block
          uint32_t r[4];
          const int unit = Q8 ? (D == 128 ? cw : cw >> 1) : cw;
          ldsm4_t(av + tile_unit<S>(32 * s2 + i8 * 8 + r8, unit), r);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
              if constexpr (!Q8) {
                vb[h][0][kh] = r[2 * h + kh];
              } else {
                const uint32_t x = r[2 * h + kh] ^ 0x80808080u;
                if constexpr (D == 128) {
                  vb[h][0][kh] = codes_f16(x, 0x4240);
                  vb[h][NO - 1][kh] = codes_f16(x, 0x4341);
                } else {
                  vb[h][0][kh] = codes_f16(x, (cw & 1) ? 0x4341 : 0x4240);
                }
              }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t ap[4];
            const int r = mt * 16 + (i8 & 1) * 8 + r8;
            const int unit = 4 * s2 + 2 * h + (i8 >> 1);
            ldsm4(sP + r * 256 + ((unit ^ (r & 7)) << 4), ap);
#pragma unroll
            for (int n = 0; n < NO; ++n) mma16816<BF>(o[mt][n], ap, vb[h][n][0], vb[h][n][1]);
          }
      }
      if constexpr (!Q8) {
        if (tail) fence_proxy_async_smem();  // the zeros above, before the next TMA write
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
    }

    // ---- the segment's partial: row sums over the warps, output to the true reference
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float a = l[mt][hf];
        a += __shfl_xor_sync(0xffffffffu, a, 1);
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        if (c == 0) smax[cw * RB + mt * 16 + hf * 8 + g] = a;
      }
    cons_sync();
    const int64_t item = head * p.nrb + sp.rb;
    float* pp = p.part + (static_cast<int64_t>(blockIdx.x) + item) * RB * part_stride<D>();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + g;
        if (r < sp.rows) {
          float* row = pp + r * part_stride<D>();
          float f = 1.0f;
          if constexpr (Q8)
            f = eref[mt][hf] == -INFINITY ? 0.0f : ex2_approx(eref[mt][hf] - mref[mt][hf]);
          const float* a = o[mt][0];
          const float* b = o[mt][NO - 1];
          if constexpr (Q8 && D == 128) {
            *reinterpret_cast<float4*>(row + cw * 16 + 4 * c) =
                make_float4(a[2 * hf] * f, b[2 * hf] * f, a[2 * hf + 1] * f, b[2 * hf + 1] * f);
          } else if constexpr (Q8) {
            row[(cw >> 1) * 16 + 4 * c + (cw & 1)] = a[2 * hf] * f;
            row[(cw >> 1) * 16 + 4 * c + 2 + (cw & 1)] = a[2 * hf + 1] * f;
          } else {
#pragma unroll
            for (int n = 0; n < NO; ++n)
              *reinterpret_cast<float2*>(row + cw * (D / 8) + n * 8 + 2 * c) =
                  make_float2(o[mt][n][2 * hf], o[mt][n][2 * hf + 1]);
          }
          if (cw == 0 && c == 0) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kTCons; ++k) sum += smax[k * RB + r];
            row[D] = mref[mt][hf];
            row[D + 1] = sum;
          }
        }
      }
    w += nt;
  }
}

// ----------------------------------------------------------------- combine --
constexpr int kCRows = 32;  // query rows per CTA of the combine kernel

// D / 32 values of a lane from a row in shared memory.
template <class T, bool Q8, int DL>
__device__ __forceinline__ void draft_part(const uint8_t* row, int lane, float scale,
                                           float (&x)[DL]) {
  if constexpr (Q8) {
    const int8_t* e = reinterpret_cast<const int8_t*>(row) + lane * DL;
#pragma unroll
    for (int i = 0; i < DL; ++i) x[i] = static_cast<float>(e[i]) * scale;
  } else {
    const T* e = reinterpret_cast<const T*>(row) + lane * DL;
#pragma unroll
    for (int i = 0; i < DL; ++i) x[i] = to_f32(e[i]);
  }
}

template <class T, int D, bool Q8, int RB>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeParams p) {
  constexpr int DL = D / 32;
  constexpr int kRow = D * (Q8 ? 1 : 2), kUnits = kRow / 16;
  extern __shared__ __align__(16) uint8_t draft[];  // K rows, V rows of the drafted tokens
  __shared__ uint32_t base[kTBatch + 2];
  __shared__ float scales[2][kTMaxTokens];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int bh = blockIdx.x, b = bh / p.kvh, h = bh % p.kvh;
  int len, n;
  const bool valid = tree_seq(p, b, len, n);
  if (!valid && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicExch(p.err, kErrBadCacheLen);
  if (warp == 0) tree_scan<RB>(p, base, lane);
  const int64_t row0 = static_cast<int64_t>(bh) * p.P + len;
  uint8_t* sk = draft;
  uint8_t* sv = draft + p.T * kRow;
  for (int i = threadIdx.x; i < 2 * n * kUnits; i += blockDim.x) {
    const int u = i < n * kUnits ? i : i - n * kUnits;
    const uint8_t* src = static_cast<const uint8_t*>(i < n * kUnits ? p.kc : p.vc) + row0 * kRow;
    reinterpret_cast<uint4*>(i < n * kUnits ? sk : sv)[u] =
        __ldg(reinterpret_cast<const uint4*>(src) + u);
  }
  if constexpr (Q8) {
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x)
      scales[i >= n][i >= n ? i - n : i] = __ldg((i >= n ? p.vs : p.ks) + row0 + (i >= n ? i - n : i));
  }
  __syncthreads();
  const uint32_t total = base[p.B];
  const uint32_t shares = min(total, static_cast<uint32_t>(p.grid));
  const int tiles = tiles_of(len), nrb = row_blocks<RB>(p, n);
  const int r1 = min(p.G * p.T, (static_cast<int>(blockIdx.y) + 1) * kCRows);
  for (int r = blockIdx.y * kCRows + warp; r < r1; r += blockDim.x >> 5) {
    const int t = r / p.G, gg = r - t * p.G;
    const int head = h * p.G + gg;
    T* og = static_cast<T*>(p.o) + b * p.ob + t * p.ot + head * p.oh + lane * DL;
    float acc[DL], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] = 0.0f;
    if (t < n) {
      const T* qp = static_cast<const T*>(p.q) + b * p.qb + t * p.qt + head * p.qh + lane * DL;
      float q[DL];
#pragma unroll
      for (int i = 0; i < DL; ++i) q[i] = to_f32(qp[i]);
      // ancestors of token t (itself included) as a 64-bit mask
      unsigned long long mask = 0ull;
      if (p.parents == nullptr) {
        mask = t == 63 ? ~0ull : (1ull << (t + 1)) - 1ull;
      } else {
        const int* par = p.parents + static_cast<int64_t>(b) * p.T;
        const int p_lo = lane < n ? par[lane] : -1, p_hi = lane + 32 < n ? par[lane + 32] : -1;
        for (int a = t; a >= 0;) {
          mask |= 1ull << a;
          const int lo = __shfl_sync(0xffffffffu, p_lo, a & 31);
          const int hi = __shfl_sync(0xffffffffu, p_hi, a & 31);
          int up = a < 32 ? lo : hi;
          if (up >= a || up < -1) {  // not a tree: the token counts as a root
            if (lane == 0) atomicExch(p.err, kErrBadParent);
            up = -1;
          }
          a = up;
        }
      }
      // scores of the ancestors: lane a & 31 keeps that of token a
      float s_lo = -INFINITY, s_hi = -INFINITY;
      for (unsigned long long left = mask; left != 0ull;) {
        int a[4];
        float d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          a[k] = left != 0ull ? __ffsll(left) - 1 : -1;
          left &= left - 1ull;  // 0 stays 0
          float x[DL];
          const int at = a[k] < 0 ? t : a[k];
          draft_part<T, Q8, DL>(sk + at * kRow, lane, Q8 ? scales[0][at] : 1.0f, x);
          d[k] = 0.0f;
#pragma unroll
          for (int i = 0; i < DL; ++i) d[k] = fmaf(q[i], x[i], d[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int k = 0; k < 4; ++k) d[k] += __shfl_xor_sync(0xffffffffu, d[k], o);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (a[k] >= 0 && (a[k] & 31) == lane) (a[k] < 32 ? s_lo : s_hi) = d[k] * p.sl2;
      }
      m = fmaxf(s_lo, s_hi);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float mu = m == -INFINITY ? 0.0f : m;
      // a NaN score must stay one: lanes without an ancestor add 0
      const bool has_lo = (mask >> lane) & 1ull, has_hi = (mask >> (lane + 32)) & 1ull;
      const float e_lo = has_lo ? exp2f(s_lo - mu) : 0.0f, e_hi = has_hi ? exp2f(s_hi - mu) : 0.0f;
      l = e_lo + e_hi;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      for (unsigned long long left = mask; left != 0ull; left &= left - 1ull) {
        const int a = __ffsll(left) - 1;
        const float lo = __shfl_sync(0xffffffffu, e_lo, a & 31);
        const float hi = __shfl_sync(0xffffffffu, e_hi, a & 31);
        const float e = a < 32 ? lo : hi;
        float x[DL];
        draft_part<T, Q8, DL>(sv + a * kRow, lane, Q8 ? scales[1][a] : 1.0f, x);
#pragma unroll
        for (int i = 0; i < DL; ++i) acc[i] = fmaf(e, x[i], acc[i]);
      }
      // the context's partials of this row's block
      if (tiles > 0) {
        const int rb = r / RB;
        const uint32_t t0 = base[b] + (static_cast<uint32_t>(h) * nrb + rb) * tiles;
        const uint32_t c0 = share_of(t0, total, shares);
        const uint32_t c1 = share_of(t0 + tiles - 1, total, shares);
        const int64_t item = static_cast<int64_t>(bh) * p.nrb + rb;
        const float* pr = p.part + ((c0 + item) * RB + (r - rb * RB)) * part_stride<D>();
        for (uint32_t cc = c0; cc <= c1; ++cc, pr += RB * part_stride<D>()) {
          const float pm = pr[D], pl = pr[D + 1];
          float x[DL];
#pragma unroll
          for (int i = 0; i < DL; ++i) x[i] = pr[lane * DL + i];
          const float mn = fmaxf(m, pm);
          const float ref = mn == -INFINITY ? 0.0f : mn;
          const float fa = exp2f(m - ref), fb = exp2f(pm - ref);
          l = l * fa + pl * fb;
#pragma unroll
          for (int i = 0; i < DL; ++i) acc[i] = acc[i] * fa + x[i] * fb;
          m = mn;
        }
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a NaN sum stays one
#pragma unroll
    for (int i = 0; i < DL; ++i) og[i] = from_f32<T>(acc[i] * inv);
  }
}

// ---------------------------------------------------------------- launchers --
int row_tiles(int G, int T) { return G * T <= 16 ? 1 : 2; }  // 16-row tiles per block

size_t tree_slots(int B, int T, int G, int kvh, int grid, int& nrb) {
  const int RB = 16 * row_tiles(G, T);
  nrb = (G * T + RB - 1) / RB;
  return static_cast<size_t>(B) * kvh * nrb + grid;
}

template <class T, int D, bool Q8, int MT>
void launch_tree(const TreeParams& p, cudaStream_t st) {
  using S = TreeSmem<D, Q8, MT>;
  const CUtensorMapDataType dt = Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : std::is_same<T, __nv_bfloat16>::value
                                     ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t rows = static_cast<uint64_t>(p.B) * p.kvh * p.P;
  const CUtensorMapSwizzle sw =
      S::kBox == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap tk, tv;
  make_tma_2d(&tk, p.kc, dt, Q8 ? 1 : 2, rows, D, D, S::kBox / (Q8 ? 1 : 2), kTTile, sw);
  make_tma_2d(&tv, p.vc, dt, Q8 ? 1 : 2, rows, D, D, S::kBox / (Q8 ? 1 : 2), kTTile, sw);
  auto kern = tree_context_kernel<T, D, Q8, MT>;
  LTM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
  kern<<<p.grid, 32 * (kTCons + 1), S::kBytes, st>>>(tk, tv, p);
  check_launch("tree_context_kernel", st);
  auto comb = tree_combine_kernel<T, D, Q8, 16 * MT>;
  const int R = p.G * p.T;
  const int warps = R < 8 ? R : 8;
  const dim3 grid(static_cast<unsigned>(p.B) * p.kvh, (R + kCRows - 1) / kCRows);
  comb<<<grid, 32 * warps, 2 * p.T * S::kRow, st>>>(p);
  check_launch("tree_combine_kernel", st);
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
    // a context kernel never has more CTAs than this device-independent cap
    const size_t slots = tree_slots(B < kTBatch ? B : kTBatch, T, G, kv_heads, 256, nrb);
    *bytes = slots * 16 * row_tiles(G, T) * (head_dim + 4) * sizeof(float);
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
    const int mt = row_tiles(G, T);
    const bool q8 = k_scale != nullptr;
    TreeParams p{};
    p.qt = q_strides[1];
    p.qh = q_strides[2];
    p.qb = q_strides[0];
    p.ob = o_strides[0];
    p.ot = o_strides[1];
    p.oh = o_strides[2];
    p.T = T;
    p.G = G;
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
      const int64_t most = static_cast<int64_t>(p.B) * kv_heads *
                           ((G * T + 16 * mt - 1) / (16 * mt)) *
                           ((max_positions + kTTile - 1) / kTTile);
      LTM_REQUIRE(most < (1ll << 31), "too many tiles");
      const int sms = device_sm_count() < 256 ? device_sm_count() : 256;
      p.grid = static_cast<int>(most < sms ? most : sms);
      const size_t slots = tree_slots(p.B, T, G, kv_heads, p.grid, p.nrb);
      LTM_REQUIRE(workspace_bytes >= slots * 16 * mt * (head_dim + 4) * sizeof(float),
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
        if (mt == 1) launch_tree<E, D, Q, 1>(p, st);
        else launch_tree<E, D, Q, 2>(p, st);
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
