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
// All three kernels are bound by memory.  Rows are handled by groups of lanes
// that hold 16 bytes each, several rows per lane in flight.
#include <type_traits>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kWarps = 8;   // warps per CTA of the write and read kernels
constexpr int kRowsFly = 4;  // rows in flight per lane group

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

// One row of a lane group: codes and scale of V values per lane.  All 32 lanes
// call it (lanes without a row pass zeros).  abs_bits: the largest |x| of the
// row as bits, where an infinity or a NaN compares above every finite value.
template <int V>
__device__ __forceinline__ float quant_row(const float (&v)[V], uint32_t abs_bits,
                                           int8_t (&out)[V]) {
  const bool bad = abs_bits >= 0x7f800000u;
  const float amax = bad ? 0.0f : __uint_as_float(abs_bits);
  const float s = __fdiv_rn(amax, 127.0f);
  // a reciprocal of a scale this small overflows: such rows take the division
  const bool tiny = s < 1e-37f;
  float w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = (bad || tiny) ? 0.0f : v[i];
  quant_i8_exact_warp<V>(w, tiny ? 0.0f : s, tiny ? 0.0f : recip_or_zero(s), out);
  if (tiny && s > 0.0f && !bad) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float r = roundf(__fdiv_rn(v[i], s));
      out[i] = static_cast<int8_t>(static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f)));
    }
  }
  return bad ? __int_as_float(0x7fc00000) : s;
}

// New tokens into the caches.  A warp takes kRowsFly * (32 / group) consecutive
// tokens of one head, K or V: its int8 rows are then one contiguous block and
// its scales whole 32-byte sectors; neighbouring warps take neighbouring heads
// of the same tokens, so that the reads cover whole projection rows.
template <class T, int D, bool Q8>
__global__ void __launch_bounds__(kWarps * 32)
    cache_append_kernel(const T* __restrict__ k, RowStrides sk, const T* __restrict__ v,
                        RowStrides sv, void* __restrict__ kc, void* __restrict__ vc,
                        float* __restrict__ ks, float* __restrict__ vs, int64_t P,
                        const int* __restrict__ lens, const int* __restrict__ num_tokens, int B,
                        int Tn, int heads, int tgroups, int64_t tasks, int* err) {
  constexpr int V = 16 / sizeof(T);   // values per lane and row
  constexpr int G = D / V;            // lanes per row
  constexpr int RP = 32 / G;          // rows per warp and step
  constexpr int TOK = RP * kRowsFly;  // tokens per warp task
  const int lane = threadIdx.x & 31;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const int h = static_cast<int>(task % heads);
  int64_t rest = task / heads;
  const bool is_v = rest & 1;
  rest >>= 1;
  const int tg = static_cast<int>(rest % tgroups), b = static_cast<int>(rest / tgroups);
  int len, n;
  const bool ok = seq_span(lens, num_tokens, b, Tn, P, len, n,
                           (tg == 0 && h == 0 && !is_v && lane == 0) ? err : nullptr);
  if (!ok) return;
  const T* src = (is_v ? v + b * sv.b + h * sv.h : k + b * sk.b + h * sk.h);
  const int64_t st = is_v ? sv.t : sk.t;
  const int sub = lane / G, gl = lane % G;
  uint4 raw[kRowsFly];
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int t = tg * TOK + j * RP + sub;
    raw[j] = make_uint4(0, 0, 0, 0);
    if (t < n) raw[j] = __ldg(reinterpret_cast<const uint4*>(src + t * st) + gl);
  }
  const int64_t row0 = (static_cast<int64_t>(b) * heads + h) * P + len;
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int t = tg * TOK + j * RP + sub;
    if (tg * TOK + j * RP >= n) break;  // uniform over the warp
    if constexpr (Q8) {
      const T* e = reinterpret_cast<const T*>(&raw[j]);
      float x[V];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = to_f32(e[i]);
        m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      int8_t out[V];
      const float s = quant_row<V>(x, m, out);
      if (t < n) {
        int8_t* dst = static_cast<int8_t*>(is_v ? vc : kc) + (row0 + t) * D + gl * V;
        if constexpr (V == 8)
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(out);
        else
          *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(out);
        if (gl == 0) (is_v ? vs : ks)[row0 + t] = s;
      }
    } else {
      if (t < n)
        reinterpret_cast<uint4*>(static_cast<T*>(is_v ? vc : kc) + (row0 + t) * D)[gl] = raw[j];
    }
  }
}

// Rows [first_b, first_b + n) of every head back as O values; positions
// outside [0, min(P, len_b)) give zeros.  A lane holds 16 codes (or 8 values of
// a 16-bit cache, copied).
template <class O, int D, bool Q8>
__global__ void __launch_bounds__(kWarps * 32)
    cache_read_kernel(const void* __restrict__ cache, const float* __restrict__ scale, int64_t P,
                      const int* __restrict__ first, const int* __restrict__ lens, int heads,
                      int n, int groups, int64_t tasks, O* __restrict__ out) {
  constexpr int V = Q8 ? 16 : 8;
  constexpr int G = D / V;
  constexpr int RP = 32 / G;
  constexpr int ROWS = RP * kRowsFly;
  const int lane = threadIdx.x & 31;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const int g = static_cast<int>(task % groups);
  const int64_t bh = task / groups;
  const int b = static_cast<int>(bh / heads);
  const int64_t p0 = first ? first[b] : 0;
  const int64_t end = lens ? min(P, static_cast<int64_t>(lens[b])) : P;
  const int sub = lane / G, gl = lane % G;
  uint4 raw[kRowsFly];
  float s[kRowsFly];
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int i = g * ROWS + j * RP + sub;
    const int64_t p = p0 + i;
    raw[j] = make_uint4(0, 0, 0, 0);
    s[j] = 0.0f;
    if (i < n && p >= 0 && p < end) {
      const int64_t row = bh * P + p;
      raw[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(cache) +
                                                    row * D * (Q8 ? 1 : 2)) +
                     gl);
      if constexpr (Q8) s[j] = __ldg(scale + row);
    }
  }
#pragma unroll
  for (int j = 0; j < kRowsFly; ++j) {
    const int i = g * ROWS + j * RP + sub;
    if (i >= n) continue;
    O* dst = out + (bh * n + i) * D + gl * V;
    if constexpr (Q8) {
      const int8_t* q = reinterpret_cast<const int8_t*>(&raw[j]);
      constexpr int W = 16 / sizeof(O);  // values per 16-byte store
#pragma unroll
      for (int c = 0; c < V / W; ++c) {
        O y[W];
#pragma unroll
        for (int u = 0; u < W; ++u) y[u] = from_f32<O>(static_cast<float>(q[c * W + u]) * s[j]);
        reinterpret_cast<uint4*>(dst)[c] = *reinterpret_cast<const uint4*>(y);
      }
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
    cache_reorder_kernel(const __grid_constant__ ReorderParams p, const int* __restrict__ beams,
                         const int* __restrict__ first, const int* __restrict__ lens, int W,
                         int heads, int64_t P, int parts, int* err) {
  __shared__ int src[WMAX];
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

unsigned grid_of(int64_t tasks) {
  const int64_t g = (tasks + kWarps - 1) / kWarps;
  LTM_REQUIRE(g < (1ll << 31), "too many rows");
  return static_cast<unsigned>(g);
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
    const RowStrides sk{k_strides[0], k_strides[1], k_strides[2]};
    const RowStrides sv{v_strides[0], v_strides[1], v_strides[2]};
    const int per = static_cast<int>(16 / dtype_size(dtype));
    const int tok = 32 / (head_dim / per) * kRowsFly;
    const int tgroups = (T + tok - 1) / tok;
    const int64_t tasks = static_cast<int64_t>(B) * tgroups * 2 * kv_heads;
    const unsigned grid = grid_of(tasks);
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(dtype, [&](auto tag) {
      using E = decltype(tag);
      by_head_dim(head_dim, [&](auto d_c) {
        constexpr int D = decltype(d_c)::value;
        auto go = [&](auto q_c) {
          cache_append_kernel<E, D, decltype(q_c)::value><<<grid, kWarps * 32, 0, st>>>(
              static_cast<const E*>(k), sk, static_cast<const E*>(v), sv, k_cache, v_cache,
              k_scale, v_scale, max_positions, cache_lens, num_tokens, B, T, kv_heads, tgroups,
              tasks, device_error_ptr());
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
    const int rows = 32 / (head_dim / (scale ? 16 : 8)) * kRowsFly;
    const int groups = (n + rows - 1) / rows;
    const int64_t tasks = static_cast<int64_t>(B) * kv_heads * groups;
    const unsigned grid = grid_of(tasks);
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(out_dtype, [&](auto tag) {
      using O = decltype(tag);
      by_head_dim(head_dim, [&](auto d_c) {
        constexpr int D = decltype(d_c)::value;
        auto go = [&](auto q_c) {
          cache_read_kernel<O, D, decltype(q_c)::value><<<grid, kWarps * 32, 0, st>>>(
              cache, scale, max_positions, first, cache_lens, kv_heads, n, groups, tasks,
              static_cast<O*>(out));
        };
        if constexpr (std::is_same<O, float>::value) {
          go(std::true_type{});
        } else {
          if (scale) go(std::true_type{});
          else go(std::false_type{});
        }
      });
    });
    check_launch("cache_read_kernel", st);
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
    for (int i = 0; i < n_caches; ++i) {
      LTM_REQUIRE(caches[i] != nullptr, "NULL pointer");
      LTM_REQUIRE(row_bytes[i] > 0 && row_bytes[i] % 4 == 0 && row_bytes[i] <= 4096,
                  "row bytes must be a multiple of 4, at most 4096");
      const uintptr_t a = reinterpret_cast<uintptr_t>(caches[i]);
      LTM_REQUIRE(a % (row_bytes[i] % 16 == 0 ? 16 : 4) == 0, "a cache is not aligned to its rows");
      for (int j = 0; j < i; ++j)
        LTM_REQUIRE(caches[j] != caches[i], "the same cache is listed twice");
      if (row_bytes[i] > widest) widest = row_bytes[i];
    }
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
        cache_reorder_kernel<decltype(w_c)::value><<<grid, 256, 0, st>>>(
            p, beams, first, cache_lens, W, kv_heads, max_positions, static_cast<int>(nx),
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
