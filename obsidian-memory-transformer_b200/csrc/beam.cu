// beam.cu -- one selection step of a beam search: the K best continuations of
// every request over its W beams x V tokens.
//
//   total[w, x] = score_w + logit[w, x] - log(sum_y exp(logit[w, y]))
//   K largest totals, descending; equal totals: the lowest w * V + x first.
//   A finished beam (done) continues as itself only: its end token keeps
//   score_w, every other token has -inf.
// A logit NaN counts as -inf and +inf as the largest finite float; a score that
// is NaN counts as -inf.
//
// Every logit is read once (the bound): beam_chunk_kernel gives each CTA up to
// 8192 logits of one row, held in registers.  It takes the chunk's maximum, the
// sum of exponentials, and its K best by filtering: the smallest of n >= K group
// maxima is a value that at least K logits reach, and usually few more do (about
// n * H_n for n groups, 22 for 8 beams), so only those are compacted and ranked.
// Where too many pass (long runs of equal or masked logits) the K best are
// taken one by one instead.  beam_merge_kernel (one CTA per request) evaluates the
// totals of the chunks' sorted lists in 64 bits, because nearly equal totals of
// different beams decide the order, and filters and ranks them the same way;
// within a row the order is that of the logits.
//
// The reference's generation loop samples on the host
// (python_bindings/ltm/inference.py:131-260).
#include <type_traits>

#include "block.cuh"

namespace ltm_b200 {
namespace {

constexpr int kBThreads = 256;
constexpr int kPer = 32;                     // logits per thread
constexpr int kChunk = kBThreads * kPer;     // logits per CTA
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
// fmaxf gives the other operand for a NaN.
__device__ __forceinline__ float logit_value(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);
}
__device__ __forceinline__ uint64_t list_key(float x, int token) {
  return (static_cast<uint64_t>(ordered(x)) << 32) | ~static_cast<uint32_t>(token);
}

struct BeamPartial {
  float m, sum;  // maximum logit of the chunk and sum of exp(logit - m)
};

// Workspace: [rows, nchunk] BeamPartial, then [rows, nchunk, K] sorted keys
// (ordered logit << 32 | ~token; 0 = none).
template <class T>
__global__ void __launch_bounds__(kBThreads, 3)
    beam_chunk_kernel(const T* __restrict__ logits, int64_t ldb, int64_t ldw,
                      const float* __restrict__ scores, const uint8_t* __restrict__ done, int end,
                      int W, int V, int K, int nchunk, int groups, BeamPartial* __restrict__ stats,
                      uint64_t* __restrict__ lists) {
  __shared__ float s_group[kBThreads];
  __shared__ float s_sum[kBThreads / 32];
  __shared__ uint64_t s_cand[kMaxCand];
  __shared__ uint64_t s_best[kBThreads / 32];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / nchunk, chunk = blockIdx.x - row * nchunk;
  const int b = row / W, w = row - b * W;
  const int c0 = chunk * kChunk, c1 = min(V, c0 + kChunk);
  const int64_t item = blockIdx.x;
  uint64_t* list = lists + item * K;

  // ---- load: 16-byte vectors of the row's aligned span, all in flight at once; then the
  // vectors that the chunk's ends cut, element by element
  constexpr int N = 16 / sizeof(T);  // logits per vector
  constexpr int NV = kPer / N;       // vectors per thread
  const T* r = logits + b * ldb + w * ldw;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
  // token of element j of vector i: t0 + i * 256 * N + j
  const int t0 = c0 - shift + tid * N;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int x = t0 + i * kBThreads * N;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (x >= c0 && x + N <= c1) raw[i] = __ldg(reinterpret_cast<const uint4*>(r + x));
  }
  const float score = scores[row];
  const bool is_done = done != nullptr && done[row] != 0;
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
  if (tid == 0) s_count = 0;
  // elements that are not there are -inf here and left out by their index below
  float v[kPer];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) v[i * N + j] = logit_value(to_f32(e[j]));
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int x = t0 + i * kBThreads * N;
    if (!(x >= c0 && x + N <= c1)) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[i * N + j] = (x + j >= c0 && x + j < c1) ? logit_value(to_f32(r[x + j])) : -INFINITY;
    }
  }
  // a misaligned row's last `shift` logits lie past the vectors: one per thread
  const int xe = c0 - shift + kChunk + tid;
  const bool has_extra = tid < shift && xe < c1;
  const float extra = has_extra ? logit_value(to_f32(r[xe])) : -INFINITY;

  float vm[NV];  // maximum of each vector
  float tm = extra;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vm[i] = v[i * N];
#pragma unroll
    for (int j = 1; j < N; ++j) vm[i] = fmaxf(vm[i], v[i * N + j]);
    tm = fmaxf(tm, vm[i]);
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
  const float m = unordered(__reduce_max_sync(0xffffffffu, ordered(fmaxf(g0, g1))));
  const float tau = unordered(__reduce_min_sync(0xffffffffu, ordered(fminf(g0, g1))));
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = __expf(extra - ref);
  auto offer = [&](float y, int x) {
    if (y >= tau && x >= c0 && x < c1) {
      const int at = atomicAdd(&s_count, 1);
      if (at < kMaxCand) s_cand[at] = list_key(y, x);
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < N; ++j) sum += __expf(v[i * N + j] - ref);
    if (vm[i] >= tau) {
#pragma unroll
      for (int j = 0; j < N; ++j) offer(v[i * N + j], t0 + i * kBThreads * N + j);
    }
  }
  if (has_extra) offer(extra, xe);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kBThreads / 32; ++i) t += s_sum[i];
    stats[item] = BeamPartial{m, t};
  }
  const int n = s_count;
  if (n <= kMaxCand) {
    for (int i = tid; i < n; i += kBThreads) {
      const uint64_t mine = s_cand[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += s_cand[j] > mine;
      if (rank < K) list[rank] = mine;
    }
    for (int i = n + tid; i < K; i += kBThreads) list[i] = 0ull;
    return;
  }
  // too many: the K best one after the other (each below the last one taken)
  uint64_t last = ~0ull;
  for (int kk = 0; kk < K; ++kk) {
    uint64_t best = 0ull;
    auto look = [&](float y, int x) {
      const uint64_t full = list_key(y, x);
      if (x >= c0 && x < c1 && full < last && full > best) best = full;
    };
#pragma unroll
    for (int i = 0; i < kPer; ++i) look(v[i], t0 + (i / N) * kBThreads * N + i % N);
    if (has_extra) look(extra, xe);
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
struct Total {
  uint64_t t;  // ordered bits of the total; 0 = none
  uint64_t f;  // beam * V + token
};
__device__ __forceinline__ bool before(const Total& a, const Total& b) {
  return a.t > b.t || (a.t == b.t && a.f < b.f);
}

constexpr int kMergeCand = 512;  // continuations ranked in shared memory

// One CTA per request.  Its W * nchunk lists are sorted, so the best d entries
// of every list, d = ceil(K / lists), hold K continuations: the least of those
// d-th entries bounds the K-th best from below, more sharply by the K-th of
// the lists' heads where there are K of them.  What reaches the bound is ranked;
// where that is more than shared memory takes, the K best are taken one by one.
__global__ void __launch_bounds__(kBThreads)
    beam_merge_kernel(const float* __restrict__ scores, const uint8_t* __restrict__ done, int end,
                      int W, int V, int K, int nchunk, const BeamPartial* __restrict__ stats,
                      const uint64_t* __restrict__ lists, float* __restrict__ out_scores,
                      int* __restrict__ out_beams, int* __restrict__ out_tokens,
                      uint8_t* __restrict__ out_done) {
  __shared__ double s_m[kMaxW], s_ls[kMaxW], s_score[kMaxW];
  __shared__ uint8_t s_done[kMaxW];
  __shared__ Total s_cand[kMergeCand];
  __shared__ Total s_best[kBThreads / 32];
  __shared__ uint64_t s_low[kBThreads / 32];
  __shared__ int s_count;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nlists = W * nchunk;
  const uint64_t* mine = lists + static_cast<int64_t>(b) * nlists * K;
  if (tid == 0) s_count = 0;
  // a row's maximum and sum over its chunks: one warp per row
  for (int w = warp; w < W; w += kBThreads / 32) {
    const int row = b * W + w;
    const float sc = scores[row];
    float m = -INFINITY;
    double sum = 0.0;
    for (int c0 = 0; c0 < nchunk; c0 += 32) {
      BeamPartial st{-INFINITY, 0.0f};
      if (c0 + lane < nchunk) st = stats[static_cast<int64_t>(row) * nchunk + c0 + lane];
      float mm = st.m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
      mm = fmaxf(mm, m);
      double part = st.m == -INFINITY ? 0.0 : static_cast<double>(st.sum * expf(st.m - mm));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      sum = (m == -INFINITY ? 0.0 : sum * static_cast<double>(expf(m - mm))) + part;
      m = mm;
    }
    if (lane == 0) {
      s_m[w] = m;
      s_ls[w] = log(sum);
      s_score[w] = sc == sc ? sc : -INFINITY;
      s_done[w] = done != nullptr && done[row] != 0;
    }
  }
  __syncthreads();
  auto entry = [&](int l, int pos) -> Total {
    const uint64_t key = mine[static_cast<int64_t>(l) * K + pos];
    if (key == 0ull) return Total{0ull, ~0ull};
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    const int w = l / nchunk;
    double t = -INFINITY;
    if (u > kNegInf && s_score[w] > -INFINITY)
      t = s_done[w] ? s_score[w]
                    : s_score[w] + ((static_cast<double>(unordered(u)) - s_m[w]) - s_ls[w]);
    return Total{ordered64(t), static_cast<uint64_t>(w) * V + ~static_cast<uint32_t>(key)};
  };
  auto put = [&](int k, const Total& x) {
    const int w = static_cast<int>(x.f / V), tok = static_cast<int>(x.f - static_cast<uint64_t>(w) * V);
    const int64_t o = static_cast<int64_t>(b) * K + k;
    out_scores[o] = static_cast<float>(unordered64(x.t));
    out_beams[o] = w;
    out_tokens[o] = tok;
    if (out_done) out_done[o] = s_done[w] || tok == end;
  };
  // ---- the bound (ordered bits of a total that at least K continuations reach)
  uint64_t low = ~0ull;
  if (nlists >= K && nlists <= kMergeCand) {
    for (int l = tid; l < nlists; l += kBThreads) s_cand[l] = entry(l, 0);
    __syncthreads();
    for (int l = tid; l < nlists; l += kBThreads) {
      const Total x = s_cand[l];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < nlists; ++j) rank += before(s_cand[j], x);
      if (rank == K - 1) s_low[0] = x.t;
    }
    __syncthreads();
    low = s_low[0];
    __syncthreads();  // s_cand is written again below
  } else {
    const int d = min(K, (K + nlists - 1) / nlists) - 1;
    for (int l = tid; l < nlists; l += kBThreads) low = min(low, entry(l, d).t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
    if (lane == 0) s_low[warp] = low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBThreads / 32; ++i) low = min(low, s_low[i]);
  }
  low = max(low, static_cast<uint64_t>(1));  // a list without that many entries bounds nothing
  const int entries = nlists * K;
  for (int i = tid; i < entries; i += kBThreads) {
    const Total x = entry(i / K, i % K);
    if (x.t >= low) {
      const int at = atomicAdd(&s_count, 1);
      if (at < kMergeCand) s_cand[at] = x;
    }
  }
  __syncthreads();
  const int n = s_count;
  if (n <= kMergeCand) {
    for (int i = tid; i < n; i += kBThreads) {
      const Total x = s_cand[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += before(s_cand[j], x);
      if (rank < K) put(rank, x);
    }
    return;
  }
  Total last{~0ull, 0ull};
  for (int k = 0; k < K; ++k) {
    Total best{0ull, ~0ull};
    for (int i = tid; i < entries; i += kBThreads) {
      const Total x = entry(i / K, i % K);
      if (before(last, x) && before(x, best)) best = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Total y{__shfl_xor_sync(0xffffffffu, best.t, o), __shfl_xor_sync(0xffffffffu, best.f, o)};
      if (before(y, best)) best = y;
    }
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBThreads / 32; ++i)
      if (before(s_best[i], best)) best = s_best[i];
    if (tid == 0) put(k, best);
    last = best;
  }
}

int chunks_of(int V) { return (V + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace ltm_b200

using namespace ltm_b200;

extern "C" ltm_status ltm_beam_select_workspace(int B, int W, int V, int K, size_t* bytes) {
  return guarded([&] {
    LTM_REQUIRE(bytes != nullptr, "NULL pointer");
    LTM_REQUIRE(B >= 0 && W >= 1 && V >= 1 && K >= 1, "bad size");
    const int64_t items = static_cast<int64_t>(B) * W * chunks_of(V);
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
    const int nchunk = chunks_of(V);
    const int64_t items = static_cast<int64_t>(B) * W * nchunk;
    LTM_REQUIRE(items < (1ll << 31), "too many beams");
    LTM_REQUIRE(workspace_bytes >= items * (sizeof(BeamPartial) + static_cast<size_t>(K) * 8),
                "workspace too small");
    BeamPartial* stats = static_cast<BeamPartial*>(workspace);
    uint64_t* lists = reinterpret_cast<uint64_t*>(stats + items);
    int groups = 8;
    while (groups < K) groups *= 2;
    const cudaStream_t st = as_stream(stream);
    dispatch_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      beam_chunk_kernel<T><<<static_cast<unsigned>(items), kBThreads, 0, st>>>(
          static_cast<const T*>(logits), batch_stride, beam_stride, scores, done, end_token, W, V,
          K, nchunk, groups, stats, lists);
    });
    check_launch("beam_chunk_kernel", st);
    beam_merge_kernel<<<B, kBThreads, 0, st>>>(
        scores, done, end_token, W, V, K, nchunk, stats, lists, out_scores, out_beams, out_tokens,
        out_done);
    check_launch("beam_merge_kernel", st);
  });
}
