// beam.cu -- one selection step of a beam search: the K best continuations of
// every request over its W beams x V tokens.
//
//   total[w, x] = score_w + logit[w, x] - log(sum_y exp(logit[w, y]))
//   K largest totals, descending; equal totals: the lowest w * V + x first.
//   A finished beam (done) continues as itself only: its end token keeps
//   score_w, every other token has -inf.
// A logit NaN counts as -inf and +inf as its type's largest value; a score that
// is NaN counts as -inf.
//
// Every logit is read once (the bound): beam_chunk_kernel gives each CTA up to
// 8192 or 16384 logits of one row, held in shared memory.  It takes the chunk's maximum, the
// sum of exponentials, and its K best by filtering: the smallest of n >= K group
// maxima is a value that at least K logits reach, and usually few more do (about
// n (1 + 1/2 + ... + 1/n) for n groups, 22 for 8), so only those are compacted and ranked.
// Where too many pass (long runs of equal or masked logits) the K best are
// taken one by one instead.  beam_merge_kernel (one CTA per request) evaluates the
// totals of the chunks' sorted lists in 64 bits (the fp32 logarithm of the row's sum
// aside), because nearly equal totals of different beams decide the order, and filters
// and ranks them the same way; within a row the order is that of the logits.
//
// Measured: 64 requests x 8 beams x 32000 bf16 logits, K = 16, 22.5 us (chunks 18, merge 8
// partly under them): the 33 MB take 5 us to read, the chunks are bound by their
// instructions (65% of the issue slots; 20 a logit, half of them a chunk's fixed part:
// maxima of groups, candidates, ranks) and their barriers.  With the logits in registers,
// three CTAs per SM, it took 26.5 us.  One request of 4 beams: 8.9 us, of which the host
// needs most to queue two kernels (6.8 us in a captured graph).
//
// The reference's generation loop samples on the host
// (python_bindings/ltm/inference.py:131-260).
#include <type_traits>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kBThreads = 256;
constexpr int kPer = 32, kPerMany = 64;      // logits per thread
constexpr int kMaxCand = 1024;               // candidates ranked in shared memory
constexpr int kMaxK = 64;
constexpr int kMaxW = 32;
constexpr uint32_t kNegInf = 0x007fffffu;    // ordered(-inf)

// Order-preserving bits of a float: larger float <=> larger integer.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 -> +0: equal values have equal keys
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
// NaN -> -inf (fmaxf gives the other operand for a NaN), +inf -> the type's largest value.
template <class T>
__device__ __forceinline__ float logit_value(float x) {
  constexpr float kMost = std::is_same<T, float>::value    ? 3.402823466e38f
                          : std::is_same<T, __half>::value ? 65504.0f
                                                           : 3.389531390e38f;
  return fminf(fmaxf(x, -INFINITY), kMost);
}
__device__ __forceinline__ uint64_t list_key(float x, int token) {
  return (static_cast<uint64_t>(ordered(x)) << 32) | ~static_cast<uint32_t>(token);
}

// Larger of two 16-byte vectors' elements (a NaN gives way), element by element.
template <class T>
__device__ __forceinline__ uint4 vec_max(const uint4& a, const uint4& b) {
  uint4 r;
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  uint32_t z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      z[i] = __float_as_uint(fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&x[i]),
                                *reinterpret_cast<const __half2*>(&y[i]));
      z[i] = *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]),
                                       *reinterpret_cast<const __nv_bfloat162*>(&y[i]));
      z[i] = *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  r.x = z[0];
  r.y = z[1];
  r.z = z[2];
  r.w = z[3];
  return r;
}

template <class T>
__device__ __forceinline__ uint4 vec_none() {  // -inf everywhere
  constexpr uint32_t k = std::is_same<T, float>::value    ? 0xff800000u
                         : std::is_same<T, __half>::value ? 0xfc00fc00u
                                                          : 0xff80ff80u;
  return make_uint4(k, k, k, k);
}

// A 16-byte vector of shared memory with -inf at the elements whose token, t0 for the
// first, lies outside [c0, c1).
template <class T>
__device__ __noinline__ void cut_vector(uint4* v, int t0, int c0, int c1) {
  constexpr int N = 16 / sizeof(T);
  T* e = reinterpret_cast<T*>(v);
#pragma unroll 1
  for (int j = 0; j < N; ++j)
    if (t0 + j < c0 || t0 + j >= c1) e[j] = from_f32<T>(-INFINITY);
}

__device__ __forceinline__ void copy_vector(uint4* dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}

// Ranks of n values by counting those before each, by the whole CTA; up to 32 lanes share
// one value's comparisons (the comparisons of one thread after the other would be most of
// a short list's time).
template <class Get, class Before, class Put>
__device__ __forceinline__ void rank_in_place(int n, Get&& get, Before&& before, Put&& put) {
  int g = 1;
  while (g < 32 && 2 * g * n <= kBThreads) g *= 2;
  const int tid = threadIdx.x, sub = tid & (g - 1), own = tid / g;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kBThreads / g) {
    const int i = i0 + own;
    const auto x = get(i < n ? i : n - 1);
    int rank = 0;
#pragma unroll 4
    for (int j = sub; j < n; j += g) rank += before(get(j), x);
#pragma unroll 1
    for (int o = g / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (sub == 0 && i < n) put(rank, x);
  }
}

constexpr float kLog2e = 1.4426950408889634f;

struct BeamPartial {
  float m, sum;  // maximum logit of the chunk and sum of exp(logit - m)
};

// Workspace: [rows, nchunk] BeamPartial, then [rows, nchunk, K] sorted keys
// (ordered logit << 32 | ~token; 0 = none).
//
// The chunk stays in shared memory (16-byte vectors of the row's aligned span; a thread
// copies and works through its own, tid + i * 256), so that a thread needs few registers
// and five CTAs share an SM: their loads, exponentials and filters overlap.
template <class T, int PER>
__global__ void __launch_bounds__(kBThreads, 5)
    beam_chunk_kernel(const T* logits, int64_t ldb, int64_t ldw, const float* scores,
                      const uint8_t* done, int end, int W, int V, int K, int nchunk, int groups,
                      BeamPartial* __restrict__ stats, uint64_t* __restrict__ lists) {
  constexpr int N = 16 / sizeof(T);  // logits per vector
  constexpr int NV = PER / N;        // vectors per thread
  constexpr int kChunk = kBThreads * PER, kVecs = kBThreads * NV;
  __shared__ uint4 s_x[kVecs + 1];  // a misaligned chunk takes one vector more: thread 0's
  __shared__ float s_group[kBThreads];
  __shared__ float s_sum[kBThreads / 32];
  __shared__ uint64_t s_cand[kMaxCand];
  __shared__ uint64_t s_best[kBThreads / 32];
  __shared__ int s_owner[kBThreads];
  __shared__ int s_count, s_slots;
  grid_wait();
  grid_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / nchunk, chunk = blockIdx.x - row * nchunk;
  const int b = row / W, w = row - b * W;
  const int c0 = chunk * kChunk, c1 = min(V, c0 + kChunk);
  const int64_t item = blockIdx.x;
  uint64_t* list = lists + item * K;

  // ---- load: whole vectors, in the first and last also what lies beside the chunk (it is
  // in the same 16 bytes as logits of it), which is cut away afterwards
  const uintptr_t at = reinterpret_cast<uintptr_t>(logits + b * ldb + w * ldw + c0);
  const uint8_t* src = reinterpret_cast<const uint8_t*>(at & ~static_cast<uintptr_t>(15));
  const int shift = static_cast<int>((at & 15) / sizeof(T));
  const int t0 = c0 - shift;  // token of element 0
  const int nvec = (c1 - t0 + N - 1) / N;
  const bool more = tid == 0 && nvec > kVecs;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tid + i * kBThreads;
    if (v < nvec) copy_vector(s_x + v, src + v * 16);
    else s_x[v] = vec_none<T>();
  }
  if (more) copy_vector(s_x + kVecs, src + kVecs * 16);
  asm volatile("cp.async.commit_group;" ::: "memory");
  const float score = scores[row];
  const bool is_done = done != nullptr && done[row] != 0;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (is_done || !(score > -INFINITY)) {
    // no logit matters: the end token (if this chunk has it), then the lowest tokens
    const bool has = is_done && score > -INFINITY && end >= c0 && end < c1;
    if (tid < K) {
      int x = c0 + tid;
      float y = -INFINITY;
      if (has) {
        if (tid == 0) {
          x = end;
          y = 0.0f;
        } else if (x - 1 < end) {
          x -= 1;
        }
      }
      list[tid] = x < c1 ? list_key(y, x) : 0ull;
    }
    if (tid == 0) stats[item] = BeamPartial{0.0f, 1.0f};
    return;
  }
  if (tid == 0) s_count = s_slots = 0;
  if (tid == 0 && shift > 0) cut_vector<T>(s_x, t0, c0, c1);
  if (more) cut_vector<T>(s_x + kVecs, t0 + kVecs * N, c0, c1);
  else if ((nvec - 1) % kBThreads == tid && nvec <= kVecs)
    cut_vector<T>(s_x + nvec - 1, t0 + (nvec - 1) * N, c0, c1);

  // Maximum, bound and sum.  The first pass takes the logits as they are; a NaN
  // or +inf among them makes the sum a NaN, and they are replaced before a second.
  float m, tau, tm;
  while (true) {
    uint4 vm = s_x[tid];
#pragma unroll
    for (int i = 1; i < NV; ++i) vm = vec_max<T>(vm, s_x[tid + i * kBThreads]);
    if (more) vm = vec_max<T>(vm, s_x[kVecs]);
    tm = -INFINITY;
    {
      const T* e = reinterpret_cast<const T*>(&vm);
#pragma unroll
      for (int j = 0; j < N; ++j) tm = fmaxf(tm, to_f32(e[j]));
    }
    // maxima of the groups of equal tid % groups (so that a short chunk fills them all)
    float gm = tm;
    for (int o = 16; o >= groups; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    s_group[tid] = gm;
    __syncthreads();
    float g0 = -INFINITY, g1 = -INFINITY;  // groups lane and lane + 32 (mod groups)
#pragma unroll
    for (int i = 0; i < kBThreads / 32; i += 2) {
      g0 = fmaxf(g0, s_group[i * 32 + lane]);
      g1 = fmaxf(g1, s_group[i * 32 + 32 + lane]);
    }
    if (groups <= 32) g0 = g1 = fmaxf(g0, g1);
    m = unordered(__reduce_max_sync(0xffffffffu, ordered(fmaxf(g0, g1))));
    tau = unordered(__reduce_min_sync(0xffffffffu, ordered(fminf(g0, g1))));
    const float ref = m == -INFINITY ? 0.0f : m;
    const uint64_t ref2 = f2_pack(ref, ref), log2e2 = f2_pack(kLog2e, kLog2e);
    uint64_t sum2 = 0ull;  // two sums
    auto add = [&](const uint4& v) {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float x0, x1;
        f2_unpack(f2_mul(f2_sub(f2_pack(to_f32(e[j]), to_f32(e[j + 1])), ref2), log2e2), x0, x1);
        sum2 = f2_add(sum2, f2_pack(ex2_approx(x0), ex2_approx(x1)));
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) add(s_x[tid + i * kBThreads]);
    if (more) add(s_x[kVecs]);
    float sum, odd;
    f2_unpack(sum2, sum, odd);
    sum += odd;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    if (!__syncthreads_or(sum != sum)) break;
    auto replace = [&](uint4* v) {
      T* e = reinterpret_cast<T*>(v);
#pragma unroll 1
      for (int j = 0; j < N; ++j) e[j] = from_f32<T>(logit_value<T>(to_f32(e[j])));
    };
#pragma unroll 1
    for (int i = 0; i < NV; ++i) replace(s_x + tid + i * kBThreads);
    if (more) replace(s_x + kVecs);
  }
  // ---- the threads that hold a value at the bound: their vectors, by the whole CTA
  auto offer = [&](float y, int x) {
    if (y >= tau && x >= c0 && x < c1) {
      const int i = atomicAdd(&s_count, 1);
      if (i < kMaxCand) s_cand[i] = list_key(y, x);
    }
  };
  auto offer_vector = [&](int v) {
    const uint4 x = s_x[v];
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int j = 0; j < N; ++j) offer(to_f32(e[j]), t0 + v * N + j);
  };
  if (tm >= tau) {
    s_owner[atomicAdd(&s_slots, 1)] = tid;
    if (more) offer_vector(kVecs);
  }
  if (tid == 0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kBThreads / 32; ++i) t += s_sum[i];
    stats[item] = BeamPartial{m, t};
  }
  __syncthreads();
  const int nown = s_slots * NV;
#pragma unroll 1
  for (int i = tid; i < nown; i += kBThreads)
    offer_vector(s_owner[i / NV] + (i % NV) * kBThreads);
  __syncthreads();
  const int n = s_count;
  if (n <= kMaxCand) {
    rank_in_place(
        n, [&](int i) { return s_cand[i]; }, [](uint64_t x, uint64_t y) { return x > y; },
        [&](int rank, uint64_t x) {
          if (rank < K) list[rank] = x;
        });
    for (int i = n + tid; i < K; i += kBThreads) list[i] = 0ull;
    return;
  }
  // too many: the K best one after the other (each below the last one taken)
  uint64_t last = ~0ull;
#pragma unroll 1
  for (int kk = 0; kk < K; ++kk) {
    uint64_t best = 0ull;
    auto look = [&](int v) {
      const uint4 q = s_x[v];
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int x = t0 + v * N + j;
        const uint64_t full = list_key(to_f32(e[j]), x);
        if (x >= c0 && x < c1 && full < last && full > best) best = full;
      }
    };
#pragma unroll 1
    for (int i = 0; i < NV; ++i) look(tid + i * kBThreads);
    if (more) look(kVecs);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBThreads / 32; ++i) best = max(best, s_best[i]);
    if (tid == 0) list[kk] = best;
    last = best;
  }
}

// Order-preserving bits of a double.
__device__ __forceinline__ uint64_t ordered64(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t u) {
  return __longlong_as_double(
      static_cast<long long>((u >> 63) ? (u & 0x7fffffffffffffffull) : ~u));
}

// A continuation: larger total first, then the lower flat index.
struct __align__(16) Total {
  uint64_t t;  // ordered bits of the total; 0 = none
  uint32_t f;  // beam * V + token (below 2^29)
  uint32_t pad;
};
__device__ __forceinline__ bool before(const Total& a, const Total& b) {
  return a.t > b.t || (a.t == b.t && a.f < b.f);
}

constexpr int kMergeCand = 512;   // continuations ranked in shared memory
constexpr int kMergeKeys = 8192;  // entries whose keys fit in shared memory
constexpr int kMergeAll = 128;    // entries that are ranked without a bound
constexpr int kMergeSlack = 24;   // continuations past K that are ranked rather than sorted out

// What the merge knows of a request's rows.
struct Rows {
  double score[kMaxW], lse[kMaxW];  // score, log(sum of exp(logit - max))
  float max[kMaxW];
  uint8_t done[kMaxW];
};

// Total of a logit (ordered bits) of row w.
__device__ __forceinline__ uint64_t total_bits(const Rows& r, int w, uint32_t u) {
  double t = -INFINITY;
  if (u > kNegInf && r.score[w] > -INFINITY)
    t = r.done[w] ? r.score[w]
                  : r.score[w] + ((static_cast<double>(unordered(u)) - r.max[w]) - r.lse[w]);
  return ordered64(t);
}

struct Outputs {  // [B, K]
  float* scores;
  int *beams, *tokens;
  uint8_t* done;
};
// Output k: continuation f = beam * V + token of total t (ordered bits).
__device__ __forceinline__ void write_out(const Outputs& o, const Rows& r, int64_t k, uint64_t t,
                                          uint32_t f, int V, int end) {
  const int w = static_cast<int>(f / static_cast<uint32_t>(V));
  const int tok = static_cast<int>(f) - w * V;
  o.scores[k] = static_cast<float>(unordered64(t));
  o.beams[k] = w;
  o.tokens[k] = tok;
  if (o.done) o.done[k] = r.done[w] || tok == end;
}

constexpr float kFar = 16777216.0f;  // 2^24: steps of 2^-28
__device__ __forceinline__ bool far_out(const Rows& r, int w) {
  const float x = fmaxf(fabsf(r.max[w]), fabsf(static_cast<float>(r.score[w])));
  return x >= kFar && x < INFINITY && !r.done[w];
}

// For a request with a row so far out that 64 bits may give different logits one total (a
// score of fp32's lowest value, say, or a logit of +inf): a chunk's list, ordered by the
// logits, then may lack continuations of a total that it holds.  Only those equal to the
// K-th total matter (of greater ones there are fewer than K, so they are all in the lists),
// and of those the lowest indices are the request's: the outputs from k0 + c on, c the number
// of greater totals, are written anew from the logits, beam after beam.  By the whole CTA.
template <class T>
__device__ void ties_by_index(const T* logits, int64_t ldw, const Rows& r, const Outputs& o,
                              int64_t k0, int W, int V, int K, int end) {
  __shared__ int s_found[kBThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto total = [&](int w, int x) {  // (a finished beam's end token whatever its logit)
    if (r.done[w]) return total_bits(r, w, x == end ? ordered(0.0f) : kNegInf);
    return total_bits(r, w, ordered(logit_value<T>(to_f32(logits[w * ldw + x]))));
  };
  __syncthreads();  // the outputs are written
  const uint64_t tk = total(o.beams[k0 + K - 1], o.tokens[k0 + K - 1]);
  if (tk == ordered64(-INFINITY)) return;  // equal logits (-inf) only
  // no row far out that reaches the K-th total: as with beams that have lost already
  if (!__syncthreads_or(tid < W && far_out(r, tid) &&
                        total_bits(r, tid, ordered(r.max[tid])) >= tk))
    return;
  int at = __syncthreads_count(tid < K && total(o.beams[k0 + tid], o.tokens[k0 + tid]) > tk);
#pragma unroll 1
  for (int w = 0; w < W && at < K; ++w) {
    if (!(r.score[w] > -INFINITY)) continue;
    if (!r.done[w] && (r.max[w] == -INFINITY || total_bits(r, w, ordered(r.max[w])) < tk)) continue;
    const int n = r.done[w] ? end + 1 : V;
#pragma unroll 1
    for (int i0 = r.done[w] ? end : 0; i0 < n && at < K; i0 += kBThreads) {
      // most of a row holds none: 16 tokens a thread until there is one
      while (!r.done[w] && i0 + 16 * kBThreads <= n) {
        T y[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) y[x] = logits[w * ldw + i0 + x * kBThreads + tid];
        bool any = false;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          any |= total_bits(r, w, ordered(logit_value<T>(to_f32(y[x])))) == tk;
        if (__syncthreads_or(any)) break;
        i0 += 16 * kBThreads;
      }
      const int i = i0 + tid;
      const bool hit = i < n && total(w, i) == tk;
      const uint32_t hits = __ballot_sync(0xffffffffu, hit);
      if (lane == 0) s_found[warp] = __popc(hits);
      __syncthreads();
      int mine = at + __popc(hits & ((1u << lane) - 1u));
#pragma unroll 1
      for (int x = 0; x < kBThreads / 32; ++x) {
        if (x < warp) mine += s_found[x];
        at += s_found[x];
      }
      if (hit && mine < K) write_out(o, r, k0 + mine, tk, static_cast<uint32_t>(w) * V + i, V, end);
      __syncthreads();
    }
  }
}
__device__ __noinline__ void order_ties(const void* logits, ltm_dtype dtype, int64_t ldb,
                                        int64_t ldw, const Rows& r, const Outputs& o, int W, int V,
                                        int K, int end) {
  const int64_t b = blockIdx.x, at = b * ldb;
  if (dtype == LTM_DTYPE_F32)
    ties_by_index(static_cast<const float*>(logits) + at, ldw, r, o, b * K, W, V, K, end);
  else if (dtype == LTM_DTYPE_F16)
    ties_by_index(static_cast<const __half*>(logits) + at, ldw, r, o, b * K, W, V, K, end);
  else
    ties_by_index(static_cast<const __nv_bfloat16*>(logits) + at, ldw, r, o, b * K, W, V, K, end);
}

// One CTA per request.  Its W * nchunk lists are sorted, so the best
// d = ceil(K / lists) entries of every list hold K continuations, and the least of
// those d-th entries is a total that at least K reach.  From there a bisection on
// the upper 32 bits of the totals (one count per step) raises the bound until
// few more than K are left, whatever the beams' scores; those are ranked.  Where
// shared memory does not take them (equal totals), the K best are taken one by
// one.  Loops stay rolled: for one request the code's own fetch is most of the time.
__global__ void __launch_bounds__(kBThreads)
    beam_merge_kernel(const void* logits, ltm_dtype dtype, int64_t ldb, int64_t ldw,
                      const float* scores, const uint8_t* done, int end, int W, int V, int K,
                      int nchunk, const BeamPartial* stats, const uint64_t* lists,
                      const __grid_constant__ Outputs out) {
  __shared__ Rows rows;
  __shared__ int s_far;  // a row is far out
  __shared__ Total s_cand[kMergeCand];
  __shared__ Total s_best[kBThreads / 32];
  __shared__ uint32_t s_key[kMergeKeys];
  __shared__ uint32_t s_lim[2 * kBThreads / 32];
  __shared__ int s_count[2];
  grid_release();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nlists = W * nchunk, entries = nlists * K;
  const uint64_t* mine = lists + static_cast<int64_t>(b) * entries;
  for (int w = tid; w < W; w += kBThreads) {
    const float sc = scores[b * W + w];
    rows.score[w] = sc == sc ? sc : -INFINITY;
    rows.done[w] = done != nullptr && done[b * W + w] != 0;
  }
  if (tid == 0) s_far = 0;
  grid_wait();  // the chunks' kernel has completed
  const bool all = entries <= kMergeAll;  // few enough to rank as they are
  const uint64_t own = all && tid < entries ? mine[tid] : 0ull;  // in flight with the sums
  __syncthreads();
  // a row's maximum and sum over its chunks: one warp per row
#pragma unroll 1
  for (int w = warp; w < W; w += kBThreads / 32) {
    const int row = b * W + w;
    float m = -INFINITY, sum = 0.0f;
#pragma unroll 1
    for (int c0 = 0; c0 < nchunk; c0 += 32) {
      BeamPartial st{-INFINITY, 0.0f};
      if (c0 + lane < nchunk) st = stats[static_cast<int64_t>(row) * nchunk + c0 + lane];
      const float mm =
          fmaxf(m, unordered(__reduce_max_sync(0xffffffffu, ordered(st.m))));
      float part = st.m == -INFINITY ? 0.0f : st.sum * expf(st.m - mm);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      sum = (m == -INFINITY ? 0.0f : sum * expf(m - mm)) + part;
      m = mm;
    }
    if (lane == 0) {
      rows.max[w] = m;
      rows.lse[w] = static_cast<double>(logf(sum));
      if (far_out(rows, w)) s_far = 1;
    }
  }
  __syncthreads();
  auto total = [&](int l, uint64_t key) -> Total {  // of a key of list l
    if (key == 0ull) return Total{0ull, ~0u, 0u};
    const int w = l / nchunk;
    return Total{total_bits(rows, w, static_cast<uint32_t>(key >> 32)),
                 static_cast<uint32_t>(w) * V + ~static_cast<uint32_t>(key), 0u};
  };
  auto entry = [&](int l, int i) { return total(l, mine[i]); };  // entry i of all
  auto put = [&](int k, const Total& x) {
    write_out(out, rows, static_cast<int64_t>(b) * K + k, x.t, x.f, V, end);
  };
  auto finish = [&] {
    if (s_far) order_ties(logits, dtype, ldb, ldw, rows, out, W, V, K, end);
  };
  auto rank_all = [&](int n) {
    rank_in_place(
        n, [&](int i) { return s_cand[i]; },
        [](const Total& a, const Total& b) { return before(a, b); },
        [&](int rank, const Total& x) {
          if (rank < K) put(rank, x);
        });
  };
  if (all) {
    if (tid < entries) s_cand[tid] = total(tid / K, own);
    __syncthreads();
    rank_all(entries);
    finish();
    return;
  }
  // ---- the bound: `low` is reached by at least K continuations
  const bool staged = entries <= kMergeKeys;
  auto key_of = [&](int i) -> uint32_t {
    return staged ? s_key[i] : static_cast<uint32_t>(entry(i / K, i).t >> 32);
  };
  if (staged)
#pragma unroll 1
    for (int i = tid; i < entries; i += kBThreads)
      s_key[i] = static_cast<uint32_t>(entry(i / K, i).t >> 32);
  __syncthreads();
  const int d = min(K, (K + nlists - 1) / nlists) - 1;
  uint32_t low = ~0u, high = 0u;
#pragma unroll 1
  for (int l = tid; l < nlists; l += kBThreads) {
    low = min(low, key_of(l * K + d));
    high = max(high, key_of(l * K));
  }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) {
    s_lim[warp] = low;
    s_lim[8 + warp] = high;
  }
  __syncthreads();
  for (int i = 0; i < kBThreads / 32; ++i) {
    low = min(low, s_lim[i]);
    high = max(high, s_lim[8 + i]);
  }
  low = max(low, 1u);  // a list without that many entries bounds nothing
  if (tid < 2) s_count[tid] = 0;
  __syncthreads();
  // how many reach x; the two counters take turns
  int turn = 0;
  auto reach = [&](uint32_t x) -> int {
    int c = 0;
#pragma unroll 1
    for (int i = tid; i < entries; i += kBThreads) c += key_of(i) >= x;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0 && c) atomicAdd(&s_count[turn], c);
    __syncthreads();
    c = s_count[turn];
    turn ^= 1;
    __syncthreads();
    if (tid == 0) s_count[turn ^ 1] = 0;
    return c;
  };
  int n = reach(low);
  while (n > K + kMergeSlack && low < high) {
    const uint32_t mid = low + (high - low + 1) / 2;
    const int c = reach(mid);
    if (c >= K) {
      low = mid;
      n = c;
    } else {
      high = mid - 1;
    }
  }
  __syncthreads();
  if (n <= kMergeCand) {
    if (tid == 0) s_count[0] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < entries; i += kBThreads)
      if (key_of(i) >= low) s_cand[atomicAdd(&s_count[0], 1)] = entry(i / K, i);
    __syncthreads();
    rank_all(n);
    finish();
    return;
  }
  Total last{~0ull, 0u, 0u};
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    Total best{0ull, ~0u, 0u};
#pragma unroll 1
    for (int i = tid; i < entries; i += kBThreads) {
      const Total x = entry(i / K, i);
      if (before(last, x) && before(x, best)) best = x;
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
      const Total y{__shfl_xor_sync(0xffffffffu, best.t, o), __shfl_xor_sync(0xffffffffu, best.f, o), 0u};
      if (before(y, best)) best = y;
    }
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < kBThreads / 32; ++i)
      if (before(s_best[i], best)) best = s_best[i];
    if (tid == 0) put(k, best);
    last = best;
  }
  finish();
}

int chunks_of(int V, int per) { return (V + kBThreads * per - 1) / (kBThreads * per); }

// Logits per thread: 32, or 64 of 16 bits where the chunks of 8192 would be more than
// the device holds at a time: half as many chunks share each one's fixed part (the
// filter and its barriers).  64 x 8 rows of 32000 bf16 logits, 64 against 32 a thread: K = 4
// 16.7 / 25.0 us, 16 22.5 / 27.8, 17 35.9 / 45.0, 64 86 / 120; of 128 x 8 rows of 16384 24.0 /
// 27.1 (K = 16), of 64 x 4 of 128256 34.2 / 46.9.
int logits_per_thread(int64_t rows, int V, ltm_dtype dt) {
  const bool many = rows * chunks_of(V, kPer) > 4 * device_sm_count();
  return many && dt != LTM_DTYPE_F32 && V > kBThreads * kPer ? kPerMany : kPer;
}

}  // namespace
}  // namespace ltm_b200

using namespace ltm_b200;

extern "C" ltm_status ltm_beam_select_workspace(int B, int W, int V, int K, size_t* bytes) {
  return guarded([&] {
    LTM_REQUIRE(bytes != nullptr, "NULL pointer");
    LTM_REQUIRE(B >= 0 && W >= 1 && V >= 1 && K >= 1, "bad size");
    const int64_t items = static_cast<int64_t>(B) * W * chunks_of(V, kPer);
    *bytes = static_cast<size_t>(items) * (sizeof(BeamPartial) + static_cast<size_t>(K) * 8);
  });
}

extern "C" ltm_status ltm_beam_select(const void* logits, ltm_dtype dtype, int64_t batch_stride,
                                      int64_t beam_stride, const float* scores,
                                      const uint8_t* done, int end_token, int B, int W, int V,
                                      int K, float* out_scores, int32_t* out_beams,
                                      int32_t* out_tokens, uint8_t* out_done, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  return guarded([&] {
    LTM_REQUIRE(B >= 0 && W >= 1 && V >= 1 && K >= 1, "bad size");
    if (W > kMaxW) LTM_UNSUPPORTED("more than 32 beams");
    if (K > kMaxK) LTM_UNSUPPORTED("more than 64 continuations");
    LTM_REQUIRE(static_cast<int64_t>(W) * V >= K, "fewer tokens than continuations");
    LTM_REQUIRE(V <= (1 << 24), "vocabulary too large");
    LTM_REQUIRE(dtype == LTM_DTYPE_F32 || dtype == LTM_DTYPE_F16 || dtype == LTM_DTYPE_BF16,
                "unknown dtype");
    LTM_REQUIRE((done == nullptr) == (out_done == nullptr), "give done and out_done or neither");
    LTM_REQUIRE(done == nullptr || (end_token >= 0 && end_token < V),
                "finished beams need an end token inside the vocabulary");
    if (B == 0) return;
    LTM_REQUIRE(logits && scores && out_scores && out_beams && out_tokens && workspace,
                "NULL pointer");
    LTM_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0,
                "logits are not aligned to their type");
    LTM_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
    const int64_t rows = static_cast<int64_t>(B) * W, most = rows * chunks_of(V, kPer);
    LTM_REQUIRE(most < (1ll << 31), "too many beams");
    LTM_REQUIRE(workspace_bytes >= most * (sizeof(BeamPartial) + static_cast<size_t>(K) * 8),
                "workspace too small");
    const int per = logits_per_thread(rows, V, dtype), nchunk = chunks_of(V, per);
    const int64_t items = rows * nchunk;
    BeamPartial* stats = static_cast<BeamPartial*>(workspace);
    uint64_t* lists = reinterpret_cast<uint64_t*>(stats + items);
    int groups = 8;
    while (groups < K) groups *= 2;
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      auto go = [&](auto per_c) {
        launch_dependent(beam_chunk_kernel<T, decltype(per_c)::value>,
                         dim3(static_cast<unsigned>(items)), kBThreads, 0, st,
                         static_cast<const T*>(logits), batch_stride, beam_stride, scores, done,
                         end_token, W, V, K, nchunk, groups, stats, lists);
      };
      if constexpr (sizeof(T) == 2) {
        if (per == kPerMany) return go(std::integral_constant<int, kPerMany>{});
      }
      go(std::integral_constant<int, kPer>{});
    });
    check_launch("beam_chunk_kernel", st);
    // launched while the chunks still run; it waits for their completion on the device
    launch_dependent(beam_merge_kernel, dim3(static_cast<unsigned>(B)), kBThreads, 0, st, logits,
                     dtype, batch_stride, beam_stride, scores, done, end_token, W, V, K, nchunk,
                     static_cast<const BeamPartial*>(stats), static_cast<const uint64_t*>(lists),
                     Outputs{out_scores, out_beams, out_tokens, out_done});
    check_launch("beam_merge_kernel", st);
  });
}
