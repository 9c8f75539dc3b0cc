// kvcache.cu -- the KV cache as a store of its own: writing new keys / values
// (int8 codes with one scale per token and head, or the activation type),
// reading rows back, and moving whole beams' caches after a beam selection.
//
// Cache layout (that of decode.cu): [B, kv_heads, max_positions, head_dim],
// head-major, contiguous; the scales of an int8 cache are fp32
// [B, kv_heads, max_positions].
//
//   write:  s = max_d |x_d| / 127 ;  q_d = clamp(round_half_away(x_d / s), -127, 127)
//           (s == 0 -> q = 0); a row that holds an infinity or a NaN gets the
//           scale NaN and zero codes, so every later read of it gives NaN.
//   read:   y_d = q_d * s, one fp32 product rounded to the output type.
//
// The reference declares the cache manager as stubs only
// (python_bindings/src/main.cpp:101-135); the quantizer's formula is that of
// src/core/quantization/quantizer.cu:94-142 with a row per token and head.
//
// Rows are handled by groups of lanes that hold 16 bytes each, several rows per lane in
// flight.  Measured (inputs larger than L2): the int8 write of 4 x 8192 tokens, 32 heads of
// 128 dims, from bf16 142 to 147 us for 0.81 GB (5.7 TB/s; arithmetic: 11 instructions a value),
// from f16 134 us (6.1 TB/s), from fp32 232 us for 1.35 GB (5.8 TB/s); into a 16-bit cache 162 us
// for 1.07 GB (6.6 TB/s, the copy bandwidth); reading the int8 cache back 64 us for 0.41 GB
// (6.3 TB/s); the reorder of 32 beams' caches 473 us, at the copy bandwidth.
#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kWarps = 8;    // warps per CTA of the write and read kernels
constexpr int kVals = 16;    // values of a row per lane
constexpr int kRowsFly = 4;  // rows in flight per lane group (write)
constexpr int kReadFly = 8;  // rows in flight per lane group (read)

struct RowStrides {
  int64_t b, t, h;  // elements between batches, tokens, heads
};

// Sequence b takes part iff its positions [len, len + n) lie in the cache.
// n is num_tokens[b] (or T); returns false, and flags the device error word,
// where a length or a count is out of range.
__device__ __forceinline__ bool seq_span(const int* lens, const int* num_tokens, int b, int T,
                                         int64_t P, int& len, int& n, int* err) {
  len = lens[b];
  n = num_tokens ? num_tokens[b] : T;
  const bool ok = len >= 0 && n >= 0 && n <= T && static_cast<int64_t>(len) + n <= P;
  if (!ok && err != nullptr) atomicExch(err, kErrBadCacheLen);
  return ok;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// prmt with its sign modes: selector nibble 8 | i gives byte i's sign, eight times.
__device__ __forceinline__ uint32_t signs_of(uint32_t lo, uint32_t hi, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(lo), "r"(hi), "r"(sel));
  return r;
}

// Scale of a row from its largest |x|: the IEEE quotient amax / 127, by Markstein's
// correction of the product with the rounded reciprocal (q = a y, q + (a - 127 q) y with
// fused multiply-adds; compared with the division for every mantissa on the CPU); small
// amax, where the correction could underflow, is divided.
constexpr float kTiny = 8.0779357e-28f;  // 2^-90
__device__ __forceinline__ float row_scale(float amax) {
  constexpr float kY = 1.0f / 127.0f;
  float s = amax * kY;
  s = fmaf(fmaf(-s, 127.0f, amax), kY, s);
  if (amax < kTiny) s = __fdiv_rn(amax, 127.0f);
  return s;
}

// What the codes of a row take from it.
struct RowQuant {
  uint64_t inv, ms;  // 1 / s (approximate) and -s, twice
  float up;          // 2^50 / s
  uint32_t keep;     // all ones, or 0: zero codes
};

// Sum rounded down, two at a time.
__device__ __forceinline__ uint64_t f2_add_down(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Codes of four values of a row, in magnitudes (a) and signs (a byte of ones for each
// negative value): the IEEE quotient q = RN(a / s) rounded half up, without a division.
//
// 16-bit values: the product with the reciprocal, corrected once by its remainder, is the
// quotient up to 2^-45, and floor((q - 1/2) + 1) the code (q - 1/2 is exact from 1/4 on;
// below, the code is 0).  Compared on the CPU with the division for every mantissa of the
// row's largest value, every smaller value down to 2^-8 of it, and reciprocals up to 2 units
// in the last place off: all codes alike.
//
// fp32 values can come closer to a tie than that.  n = floor(a / s) or, just above an
// integer, one less, from the reciprocal (off by at most 2e-5); then the code is n + 1
// where q >= c = n + 1/2, else n.  RN ties to even and c is even, so q >= c iff
// a / s >= (c + c') / 2, c' the float below c:
//   w = (a - c s) + (a - c' s) >= 0 .
// Near the threshold both differences are exact as fused multiply-adds for s >= 2^-97: a
// and c s are multiples of 2^(e-24) (s in [2^e, 2^(e+1))) that differ by less than
// 2^-14 s, and a - c' s, a multiple of 2^(e+k-46) for c in [2^k, 2^(k+1)), is there about
// s 2^(k-24); so w, where it is negative, is at most -2^(e-47), and 1 + 2^50 w / s,
// clamped to [0, 1], is the step.  Farther away the signs are certain.  c' is RN(c -
// 2^-24 c): c is a power of two only as 1/2, otherwise 2^-24 c lies between half a unit
// and one.
//
// (Dividing where the estimate is near a tie cost 250 us for a prompt of 4 x 8192 tokens,
// 32 heads of 128: most warps of 16-bit rows hold a tie.)
template <class T>
__device__ __forceinline__ uint32_t quant4(const float (&a)[4], uint32_t neg, const RowQuant& r) {
  constexpr float kShift = 12582912.0f;  // 1.5 * 2^23: the sum's low byte is the integer
  constexpr float kBelow = 1.0f - 5.9604644775390625e-8f;  // 1 - 2^-24
  const uint64_t mhalf2 = f2_pack(-0.5f, -0.5f);
  float big[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint64_t a2 = f2_pack(a[i], a[i + 1]);
    if constexpr (sizeof(T) == 2) {
      const uint64_t q0 = f2_mul(a2, r.inv);
      const uint64_t q = f2_fma(f2_fma(q0, r.ms, a2), r.inv, q0);
      f2_unpack(f2_add_down(f2_add(q, mhalf2), f2_pack(kShift + 1.0f, kShift + 1.0f)), big[i],
                big[i + 1]);
    } else {
      const uint64_t shift2 = f2_pack(kShift, kShift);
      const uint64_t b = f2_add(f2_fma(a2, r.inv, mhalf2), shift2);
      const uint64_t c = f2_add(f2_sub(b, shift2), f2_pack(0.5f, 0.5f));
      const uint64_t below = f2_mul(c, f2_pack(kBelow, kBelow));
      float w0, w1, s0, s1;
      f2_unpack(f2_add(f2_fma(c, r.ms, a2), f2_fma(below, r.ms, a2)), w0, w1);
      asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(s0) : "f"(w0), "f"(r.up), "f"(1.0f));
      asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(s1) : "f"(w1), "f"(r.up), "f"(1.0f));
      f2_unpack(f2_add(b, f2_pack(s0, s1)), big[i], big[i + 1]);
    }
  }
  const uint32_t m =  // magnitudes, at most 127 each
      __byte_perm(__byte_perm(__float_as_uint(big[0]), __float_as_uint(big[1]), 0x0040),
                  __byte_perm(__float_as_uint(big[2]), __float_as_uint(big[3]), 0x0040), 0x5410);
  // byte-wise (m ^ neg) - neg without carries between bytes
  return (((m ^ neg) & (r.keep & 0x7f7f7f7fu)) + (neg & (r.keep & 0x01010101u))) ^
         (neg & (r.keep & 0x80808080u));
}

// Bits of the largest |x| of a 16-byte vector.
template <class T>
__device__ __forceinline__ uint32_t abs_max_bits(const uint4& raw) {
  if constexpr (sizeof(T) == 4) {
    return max(max(raw.x & 0x7fffffffu, raw.y & 0x7fffffffu),
               max(raw.z & 0x7fffffffu, raw.w & 0x7fffffffu));
  } else {  // two 16-bit patterns a word: without the sign they compare as integers
    return __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu),
                         __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
  }
}
// The larger half of a pair, as the bits of its fp32 value.
template <class T>
__device__ __forceinline__ uint32_t widen_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    const uint32_t h = max(m & 0xffffu, m >> 16);
    const uint16_t u = static_cast<uint16_t>(h);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&u)));
  }
}

// |x| and signs (a byte of ones where negative) of values 4g .. 4g + 3 of a lane.
template <class T, int NP>
__device__ __forceinline__ void magnitudes(const uint4 (&raw)[NP], int g, float (&a)[4],
                                           uint32_t& neg) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t x[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = fabsf(__uint_as_float(x[i]));
    neg = __byte_perm(signs_of(x[0], x[1], 0x00fb), signs_of(x[2], x[3], 0x00fb), 0x5410);
  } else {
    const uint4& r = raw[g / 2];
    const uint32_t x[2] = {g % 2 ? r.z : r.x, g % 2 ? r.w : r.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = x[i] & 0x7fff7fffu;
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
        a[2 * i] = f.x;
        a[2 * i + 1] = f.y;
      } else {
        a[2 * i] = __uint_as_float(y << 16);
        a[2 * i + 1] = __uint_as_float(y & 0xffff0000u);
      }
    }
    neg = signs_of(x[0], x[1], 0xfdb9);
  }
}

// New tokens into the caches: input read once, codes and scales written once.  The int8
// write is bound by its arithmetic (67% of the issue slots, 62% of the integer pipe, 50% of
// the DRAM; 4 rows in flight, because a warp's fixed part is 125 instructions: 2 rows cost
// 16 us more), the 16-bit one by memory.  A lane holds 16 values of a row (two or four 16-byte pieces a
// group's width apart, so that loads and stores are contiguous over the group),
// a group of D / 16 lanes a row; a warp takes kRowsFly * 32 / group
// consecutive tokens of one head, K or V, so that its int8 rows are one
// contiguous block and its scales whole 32-byte sectors; neighbouring warps take
// neighbouring heads of the same tokens: the reads cover whole projection rows.
template <class T, int D, bool Q8>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 2 ? 4 : 2)
    cache_append_kernel(const T* k, RowStrides sk, const T* v, RowStrides sv,
                        void* __restrict__ kc, void* __restrict__ vc, float* __restrict__ ks,
                        float* __restrict__ vs, int64_t P, const int* lens, const int* num_tokens,
                        int Tn, int heads, int tgroups, int* err) {
  constexpr int N = 16 / sizeof(T);   // values per piece
  constexpr int NP = kVals / N;       // pieces per lane
  constexpr int G = D / kVals;        // lanes per row
  constexpr int RP = 32 / G;          // rows per warp and step
  constexpr int TOK = RP * kRowsFly;  // tokens per warp
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const int hv = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);  // K heads, then V heads
  if (hv >= 2 * heads) return;
  const bool is_v = hv >= heads;
  const int h = is_v ? hv - heads : hv;
  const int b = blockIdx.x / tgroups, tg = blockIdx.x - b * tgroups;
  int len, n;
  const bool ok = seq_span(lens, num_tokens, b, Tn, P, len, n,
                           (tg == 0 && hv == 0 && lane == 0) ? err : nullptr);
  if (!ok) return;
  const T* src = (is_v ? v + b * sv.b + h * sv.h : k + b * sk.b + h * sk.h);
  const int64_t st = is_v ? sv.t : sk.t;
  const int sub = lane / G, gl = lane % G;
  uint4 raw[kRowsFly][NP];
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int t = tg * TOK + j * RP + sub;
    const uint4* at = reinterpret_cast<const uint4*>(src + t * st) + gl;
#pragma unroll
    for (int q = 0; q < NP; ++q)
      raw[j][q] = t < n ? at[q * G] : make_uint4(0, 0, 0, 0);
  }
  const int64_t row0 = (static_cast<int64_t>(b) * heads + h) * P + len;
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int t = tg * TOK + j * RP + sub;
    if (tg * TOK + j * RP >= n) break;  // uniform over the warp
    if constexpr (Q8) {
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const uint32_t a = abs_max_bits<T>(raw[j][q]);
        if constexpr (sizeof(T) == 4) m = max(m, a);
        else m = __vmaxu2(m, a);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        const uint32_t a = __shfl_xor_sync(0xffffffffu, m, o);
        if constexpr (sizeof(T) == 4) m = max(m, a);
        else m = __vmaxu2(m, a);
      }
      const uint32_t abs_bits = widen_bits<T>(m);
      const bool bad = abs_bits >= 0x7f800000u;  // an infinity or a NaN
      const float amax = __uint_as_float(abs_bits);
      const bool tiny = amax < kTiny;
      float s = row_scale(amax);
      const float inv = rcp_approx(s);
      const RowQuant rq{f2_pack(inv, inv), f2_pack(-s, -s), inv * 1.125899906842624e15f,
                        bad || tiny ? 0u : ~0u};
      uint32_t code[kVals / 4];
#pragma unroll
      for (int g = 0; g < kVals / 4; ++g) {
        float a[4];
        uint32_t neg;
        magnitudes<T>(raw[j], g, a, neg);
        code[g] = quant4<T>(a, neg, rq);
      }
      if (tiny && s > 0.0f) {  // divided
#pragma unroll
        for (int g = 0; g < kVals / 4; ++g) {
          float a[4];
          uint32_t neg;
          magnitudes<T>(raw[j], g, a, neg);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = static_cast<int>(fminf(roundf(__fdiv_rn(a[i], s)), 127.0f));
            code[g] |= static_cast<uint32_t>((neg >> (8 * i) & 1u ? -c : c) & 0xff) << (8 * i);
          }
        }
      }
      if (bad) s = __int_as_float(0x7fc00000);
      if (t < n) {
        int8_t* dst = static_cast<int8_t*>(is_v ? vc : kc) + (row0 + t) * D + gl * N;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          if constexpr (N == 8)
            *reinterpret_cast<uint2*>(dst + q * G * N) = make_uint2(code[2 * q], code[2 * q + 1]);
          else
            *reinterpret_cast<uint32_t*>(dst + q * G * N) = code[q];
        }
        if (gl == 0) (is_v ? vs : ks)[row0 + t] = s;
      }
    } else {
      if (t < n) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(is_v ? vc : kc) + (row0 + t) * D) + gl;
#pragma unroll
        for (int q = 0; q < NP; ++q) dst[q * G] = raw[j][q];
      }
    }
  }
}

// Rows [first_b, first_b + n) of every head back as O values; positions
// outside [0, min(P, len_b)) give zeros.  Bound by memory.  A lane writes 16 bytes
// (so that a warp's stores are contiguous) of the 4 or 8 codes, or the 8 values of a
// 16-bit cache, that it holds of a row.
template <class O, int D, bool Q8>
__global__ void __launch_bounds__(kWarps * 32)
    cache_read_kernel(const void* cache, const float* scale, int64_t P, const int* first,
                      const int* lens, int heads, int n, int start, O* __restrict__ out) {
  constexpr int V = 16 / sizeof(O);
  using Raw = std::conditional_t<!Q8, uint4, std::conditional_t<V == 8, uint2, uint32_t>>;
  constexpr int G = D / V;
  constexpr int RP = 32 / G;
  constexpr int ROWS = RP * kReadFly;
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31;
  const int bh = blockIdx.x;
  const int64_t i0 = start + static_cast<int64_t>(blockIdx.y * kWarps + (threadIdx.x >> 5)) * ROWS;
  if (i0 >= n) return;
  const int b = bh / heads;
  const int64_t p0 = first ? first[b] : 0;
  const int64_t end = lens ? min(P, static_cast<int64_t>(lens[b])) : P;
  const int sub = lane / G, gl = lane % G;
  Raw raw[kReadFly];
  float s[kReadFly];
#pragma unroll
  for (int j = 0; j < kReadFly; ++j) {
    const int64_t i = i0 + j * RP + sub;
    const int64_t p = p0 + i;
    const bool live = i < n && p >= 0 && p < end;
    const int64_t row = bh * P + p;
    raw[j] = live ? reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(cache) +
                                                 row * D * (Q8 ? 1 : 2))[gl]
                  : Raw{};
    s[j] = Q8 && live ? scale[row] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < kReadFly; ++j) {
    const int64_t i = i0 + j * RP + sub;
    if (i >= n) continue;
    O* dst = out + (static_cast<int64_t>(bh) * n + i) * D + gl * V;
    if constexpr (Q8) {
      const int8_t* q = reinterpret_cast<const int8_t*>(&raw[j]);
      O y[V];
#pragma unroll
      for (int u = 0; u < V; ++u) y[u] = from_f32<O>(static_cast<float>(q[u]) * s[j]);
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
    } else {
      *reinterpret_cast<uint4*>(dst) = raw[j];
    }
  }
}

// ------------------------------------------------------------------- reorder --
constexpr int kMaxReorder = 64;  // caches per launch (the kernel's parameter block)
constexpr int kMaxBeams = 32;

struct ReorderParams {
  void* cache[kMaxReorder];
  int row_bytes[kMaxReorder];
};

// One 16-byte (or 4-byte) column of all W beams of one group belongs to one
// thread: it loads what the moved beams take (their sources), then stores it.
// No other thread touches those bytes, so any map -- swaps, cycles, copies -- is
// done in place without a second cache; beams that keep their slot cost nothing.
template <class V, int WMAX>
__device__ __forceinline__ void reorder_columns(uint8_t* base, int64_t beam_bytes, int64_t lo,
                                                int64_t hi, const int* src, int W, int part,
                                                int parts) {
  const int64_t n = (hi - lo) / static_cast<int64_t>(sizeof(V));
  const int64_t step = static_cast<int64_t>(parts) * blockDim.x;
  for (int64_t c = static_cast<int64_t>(part) * blockDim.x + threadIdx.x; c < n; c += step) {
    uint8_t* at = base + lo + c * sizeof(V);
    V r[WMAX];
#pragma unroll
    for (int i = 0; i < WMAX; ++i)
      if (i < W && src[i] != i) r[i] = *reinterpret_cast<const V*>(at + src[i] * beam_bytes);
#pragma unroll
    for (int i = 0; i < WMAX; ++i)
      if (i < W && src[i] != i) *reinterpret_cast<V*>(at + i * beam_bytes) = r[i];
  }
}

template <int WMAX>
__global__ void __launch_bounds__(256)
    cache_reorder_kernel(const __grid_constant__ ReorderParams p, const int* beams,
                         const int* first, const int* lens, int W,
                         int heads, int64_t P, int parts, int* err) {
  __shared__ int src[WMAX];
  grid_wait();
  grid_release();
  const int bh = blockIdx.x / parts, part = blockIdx.x % parts;
  const int b = bh / heads, h = bh % heads;
  int mine = threadIdx.x;
  bool ok = true, moved = false;
  if (threadIdx.x < W) {
    mine = beams[b * W + threadIdx.x];
    ok = mine >= 0 && mine < W;
    moved = mine != static_cast<int>(threadIdx.x);
    src[threadIdx.x] = mine;
  }
  const int64_t lo = first ? first[b] : 0, hi = lens ? lens[b] : P;
  if (lo < 0 || hi > P || lo > hi) ok = false;
  const bool all_ok = __syncthreads_and(ok);
  const bool any = __syncthreads_or(moved);
  if (!all_ok) {
    if (threadIdx.x == 0 && part == 0 && h == 0 && blockIdx.y == 0) atomicExch(err, kErrBadBeam);
    return;
  }
  if (!any) return;
  const int rb = p.row_bytes[blockIdx.y];
  const int64_t head_bytes = P * rb, beam_bytes = head_bytes * heads;
  uint8_t* base = static_cast<uint8_t*>(p.cache[blockIdx.y]) +
                  static_cast<int64_t>(b) * W * beam_bytes + h * head_bytes;
  if (rb % 16 == 0)
    reorder_columns<uint4, WMAX>(base, beam_bytes, lo * rb, hi * rb, src, W, part, parts);
  else
    reorder_columns<uint32_t, WMAX>(base, beam_bytes, lo * rb, hi * rb, src, W, part, parts);
}

// ---------------------------------------------------------------- launchers --
void check_rows(const void* p, const int64_t* strides, size_t esize, const char* what) {
  const int64_t per = static_cast<int64_t>(16 / esize);
  LTM_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0,
              std::string(what) + " must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    LTM_REQUIRE(strides[i] % per == 0, std::string(what) + ": strides must be multiples of 16 bytes");
}

void check_dims(int B, int heads, int head_dim, int64_t P) {
  LTM_REQUIRE(B >= 0 && heads >= 1 && P >= 1, "bad size");
  if (head_dim != 64 && head_dim != 128) LTM_UNSUPPORTED("head_dim must be 64 or 128");
  LTM_REQUIRE(P < (1ll << 31), "max_positions exceeds int32");
}

bool overlap(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + bytes && y < x + bytes;
}

template <class F>
void by_head_dim(int D, F&& f) {
  if (D == 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace ltm_b200

using namespace ltm_b200;

extern "C" ltm_status ltm_kv_cache_append(const void* k, const int64_t* k_strides, const void* v,
                                          const int64_t* v_strides, ltm_dtype dtype, void* k_cache,
                                          void* v_cache, float* k_scale, float* v_scale,
                                          int64_t max_positions, const int32_t* cache_lens,
                                          const int32_t* num_tokens, int B, int T, int kv_heads,
                                          int head_dim, void* stream) {
  return guarded([&] {
    check_dims(B, kv_heads, head_dim, max_positions);
    LTM_REQUIRE(T >= 0, "bad size");
    LTM_REQUIRE(dtype == LTM_DTYPE_F32 || dtype == LTM_DTYPE_F16 || dtype == LTM_DTYPE_BF16,
                "unknown dtype");
    if (B == 0 || T == 0) return;
    LTM_REQUIRE(k && v && k_strides && v_strides && k_cache && v_cache && cache_lens,
                "NULL pointer");
    LTM_REQUIRE((k_scale == nullptr) == (v_scale == nullptr), "give both scales or neither");
    const bool q8 = k_scale != nullptr;
    if (!q8 && dtype == LTM_DTYPE_F32) LTM_UNSUPPORTED("fp32 caches (int8, f16 or bf16)");
    check_rows(k, k_strides, dtype_size(dtype), "k");
    check_rows(v, v_strides, dtype_size(dtype), "v");
    LTM_REQUIRE(((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) &
                 15) == 0, "the caches must be 16-byte aligned");
    const size_t rows = static_cast<size_t>(B) * kv_heads * max_positions;
    LTM_REQUIRE(!overlap(k_cache, v_cache, rows * head_dim * (q8 ? 1 : dtype_size(dtype))) &&
                    !(q8 && overlap(k_scale, v_scale, rows * 4)),
                "the K and V caches overlap");
    const RowStrides sk{k_strides[0], k_strides[1], k_strides[2]};
    const RowStrides sv{v_strides[0], v_strides[1], v_strides[2]};
    const int tok = 32 / (head_dim / kVals) * kRowsFly;
    const int tgroups = (T + tok - 1) / tok;
    LTM_REQUIRE(static_cast<int64_t>(B) * tgroups < (1ll << 31), "too many tokens");
    const int warps = 2 * kv_heads < kWarps ? 2 * kv_heads : kWarps;
    const int gy = (2 * kv_heads + warps - 1) / warps;
    LTM_REQUIRE(gy < (1 << 16), "too many heads");
    const dim3 grid(static_cast<unsigned>(B) * tgroups, static_cast<unsigned>(gy));
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(dtype, [&](auto tag) {
      using E = decltype(tag);
      by_head_dim(head_dim, [&](auto d_c) {
        constexpr int D = decltype(d_c)::value;
        auto go = [&](auto q_c) {
          launch_dependent(cache_append_kernel<E, D, decltype(q_c)::value>, grid, warps * 32, 0, st,
                           static_cast<const E*>(k), sk, static_cast<const E*>(v), sv, k_cache,
                           v_cache, k_scale, v_scale, max_positions, cache_lens, num_tokens, T,
                           kv_heads, tgroups, device_error_ptr());
        };
        if constexpr (std::is_same<E, float>::value) {
          go(std::true_type{});
        } else {
          if (q8) go(std::true_type{});
          else go(std::false_type{});
        }
      });
    });
    check_launch("cache_append_kernel", st);
  });
}

extern "C" ltm_status ltm_kv_cache_read(const void* cache, const float* scale, ltm_dtype out_dtype,
                                        int64_t max_positions, const int32_t* first,
                                        const int32_t* cache_lens, int B, int kv_heads,
                                        int head_dim, int n, void* out, void* stream) {
  return guarded([&] {
    check_dims(B, kv_heads, head_dim, max_positions);
    LTM_REQUIRE(n >= 0, "bad size");
    LTM_REQUIRE(out_dtype == LTM_DTYPE_F32 || out_dtype == LTM_DTYPE_F16 ||
                    out_dtype == LTM_DTYPE_BF16, "unknown dtype");
    if (B == 0 || n == 0) return;
    LTM_REQUIRE(cache && out, "NULL pointer");
    if (!scale && out_dtype == LTM_DTYPE_F32) LTM_UNSUPPORTED("fp32 caches (int8, f16 or bf16)");
    LTM_REQUIRE(((reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                "the cache and the output must be 16-byte aligned");
    const int rows = 32 / (head_dim * static_cast<int>(dtype_size(out_dtype)) / 16) * kReadFly * kWarps;  // per CTA
    LTM_REQUIRE(static_cast<int64_t>(B) * kv_heads < (1ll << 31), "too many rows");
    constexpr int64_t kMostBlocks = 65535;  // of a launch, in y
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(out_dtype, [&](auto tag) {
      using O = decltype(tag);
      by_head_dim(head_dim, [&](auto d_c) {
        constexpr int D = decltype(d_c)::value;
        auto go = [&](auto q_c) {
          for (int64_t start = 0; start < n; start += kMostBlocks * rows) {
            const int64_t gy = std::min<int64_t>((n - start + rows - 1) / rows, kMostBlocks);
            launch_dependent(cache_read_kernel<O, D, decltype(q_c)::value>,
                             dim3(static_cast<unsigned>(B) * kv_heads, static_cast<unsigned>(gy)),
                             kWarps * 32, 0, st, cache, scale, max_positions, first, cache_lens,
                             kv_heads, n, static_cast<int>(start), static_cast<O*>(out));
            check_launch("cache_read_kernel", st);
          }
        };
        if constexpr (std::is_same<O, float>::value) {
          go(std::true_type{});
        } else {
          if (scale) go(std::true_type{});
          else go(std::false_type{});
        }
      });
    });
  });
}

extern "C" ltm_status ltm_kv_cache_reorder(void* const* caches, const int64_t* row_bytes,
                                           int n_caches, const int32_t* beams,
                                           const int32_t* first, const int32_t* cache_lens, int B,
                                           int W, int kv_heads, int64_t max_positions,
                                           void* stream) {
  return guarded([&] {
    LTM_REQUIRE(n_caches >= 0 && B >= 0 && W >= 1 && kv_heads >= 1 && max_positions >= 1,
                "bad size");
    LTM_REQUIRE(max_positions < (1ll << 31), "max_positions exceeds int32");
    if (W > kMaxBeams) LTM_UNSUPPORTED("more than 32 beams");
    if (n_caches == 0 || B == 0) return;
    LTM_REQUIRE(caches && row_bytes && beams, "NULL pointer");
    int64_t widest = 0;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans(n_caches);
    for (int i = 0; i < n_caches; ++i) {
      LTM_REQUIRE(caches[i] != nullptr, "NULL pointer");
      LTM_REQUIRE(row_bytes[i] > 0 && row_bytes[i] % 4 == 0 && row_bytes[i] <= 4096,
                  "row bytes must be a multiple of 4, at most 4096");
      const uintptr_t a = reinterpret_cast<uintptr_t>(caches[i]);
      LTM_REQUIRE(a % (row_bytes[i] % 16 == 0 ? 16 : 4) == 0, "a cache is not aligned to its rows");
      spans[i] = {a, a + static_cast<uintptr_t>(B) * W * kv_heads * max_positions * row_bytes[i]};
      if (row_bytes[i] > widest) widest = row_bytes[i];
    }
    std::sort(spans.begin(), spans.end());
    for (int i = 1; i < n_caches; ++i)
      LTM_REQUIRE(spans[i].first >= spans[i - 1].second,
                  "caches overlap (each may be listed once)");
    const cudaStream_t st = as_stream(stream);
    for (int i0 = 0; i0 < n_caches; i0 += kMaxReorder) {
      const int n = n_caches - i0 < kMaxReorder ? n_caches - i0 : kMaxReorder;
      ReorderParams p{};
      for (int i = 0; i < n; ++i) {
        p.cache[i] = caches[i0 + i];
        p.row_bytes[i] = static_cast<int>(row_bytes[i0 + i]);
      }
      // enough CTAs to fill the device several times, at most one column per thread
      const int64_t columns = (max_positions * widest / 16 + 255) / 256;
      const int64_t others = static_cast<int64_t>(B) * kv_heads * n;
      int64_t nx = (static_cast<int64_t>(device_sm_count()) * 64 + others - 1) / others;
      if (nx > columns) nx = columns;
      if (nx < 1) nx = 1;
      const int64_t gx = nx * B * kv_heads;
      LTM_REQUIRE(gx < (1ll << 31), "too many heads");
      const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(n));
      auto go = [&](auto w_c) {
        launch_dependent(cache_reorder_kernel<decltype(w_c)::value>, grid, 256, 0, st, p, beams,
                         first, cache_lens, W, kv_heads, max_positions, static_cast<int>(nx),
                         device_error_ptr());
      };
      if (W <= 4) go(std::integral_constant<int, 4>{});
      else if (W <= 8) go(std::integral_constant<int, 8>{});
      else if (W <= 16) go(std::integral_constant<int, 16>{});
      else go(std::integral_constant<int, 32>{});
      check_launch("cache_reorder_kernel", st);
    }
  });
}
