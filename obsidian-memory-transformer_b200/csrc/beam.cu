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
// 8192 logits of one row, held in registers as order-preserving integers.  It
// takes the chunk's maximum, the sum of exponentials, and its K best by
// filtering: the smallest of n >= K group maxima is a value that at least K
// logits reach, and usually few more do (about n * H_n for n groups, 22 for 8
// beams), so only those are compacted and ranked.  Where too many pass (long
// runs of equal or masked logits) the K best are taken one by one instead.
// beam_merge_kernel (one warp per request) merges the chunks' sorted lists by
// their totals, evaluated in 64 bits because nearly equal totals of different
// beams decide the order; within a row the order is that of the logits.
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
constexpr uint32_t kNone = 0u;               // not a logit (past the row's end)
constexpr uint32_t kNegInf = 0x007fffffu;    // ordered(-inf)

// Order-preserving bits of a float: larger float <=> larger integer.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (!(x == x)) return kNegInf;
  x = fminf(x, 3.402823466e38f) + 0.0f;  // -0 -> +0: equal values have equal keys
  return ordered(x);
}

struct BeamPartial {
  float m, sum;  // maximum logit of the chunk and sum of exp(logit - m)
};

// Workspace: [rows, nchunk] BeamPartial, then [rows, nchunk, K] sorted keys
// (ordered logit << 32 | ~token; 0 = none).
template <class T>
__global__ void __launch_bounds__(kBThreads)
    beam_chunk_kernel(const T* __restrict__ logits, int64_t ldb, int64_t ldw,
                      const float* __restrict__ scores, const uint8_t* __restrict__ done, int end,
                      int W, int V, int K, int nchunk, int groups, BeamPartial* __restrict__ stats,
                      uint64_t* __restrict__ lists) {
  __shared__ uint32_t s_group[kMaxK];
  __shared__ float s_sum[kBThreads / 32];
  __shared__ uint64_t s_cand[kMaxCand];
  __shared__ uint64_t s_best[kBThreads / 32];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / nchunk, chunk = blockIdx.x % nchunk;
  const int b = row / W, w = row % W;
  const int c0 = chunk * kChunk, c1 = min(V, c0 + kChunk);
  const int64_t item = blockIdx.x;
  uint64_t* list = lists + item * K;
  const bool is_done = done != nullptr && done[row] != 0;
  const float score = scores[row];

  if (is_done || !(score > -INFINITY)) {
    // no logit matters: the end token (if this chunk has it), then the lowest tokens
    const bool has = is_done && score > -INFINITY && end >= c0 && end < c1;
    if (tid < K) {
      int x = tid;
      uint32_t u = kNegInf;
      if (has) {
        if (tid == 0) {
          x = end - c0;
          u = ordered(0.0f);
        } else {
          x = tid - 1 < end - c0 ? tid - 1 : tid;
        }
      }
      list[tid] = c0 + x < c1
                      ? (static_cast<uint64_t>(u) << 32) | ~static_cast<uint32_t>(c0 + x)
                      : 0ull;
    }
    if (tid == 0) stats[item] = BeamPartial{0.0f, 1.0f};
    return;
  }

  // ---- load: 16-byte vectors of the row's aligned span, the ragged ends one by one
  constexpr int N = 16 / sizeof(T);       // logits per vector
  constexpr int NV = kPer / N;            // vectors per thread
  const T* r = logits + b * ldb + w * ldw;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
  uint32_t u[kPer];
  // token of element j of vector i: c0 - shift + (i * 256 + tid) * N + j
  const int t0 = c0 - shift + tid * N;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int x = t0 + i * kBThreads * N;
    if (x >= c0 && x + N <= c1) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(r + x));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < N; ++j) u[i * N + j] = logit_key(to_f32(e[j]));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        u[i * N + j] = (x + j >= c0 && x + j < c1) ? logit_key(to_f32(r[x + j])) : kNone;
    }
  }
  // a misaligned row's last `shift` logits lie past the vectors: one per thread
  uint32_t extra = kNone;
  const int xe = c0 - shift + kChunk + tid;
  if (tid < shift && xe < c1) extra = logit_key(to_f32(r[xe]));

  uint32_t um = extra;
#pragma unroll
  for (int i = 0; i < kPer; ++i) um = max(um, u[i]);
  // maxima of `groups` groups of consecutive lanes (8 warps down to 4 lanes each)
  const int gl = kBThreads / groups;
  for (int o = gl >> 1; o > 0; o >>= 1) um = max(um, __shfl_xor_sync(0xffffffffu, um, o));
  if (tid % gl == 0) s_group[tid / gl] = um;
  if (tid == 0) s_count = 0;
  __syncthreads();
  uint32_t hi = kNone, tau = 0xffffffffu;
  for (int i = 0; i < groups; ++i) {
    const uint32_t g = s_group[i];
    hi = max(hi, g);
    tau = min(tau, g);
  }
  if (tau == kNone) tau = 1u;
  const float m = unordered(hi);
  const float ref = hi <= kNegInf ? 0.0f : m;
  float sum = 0.0f;
  auto visit = [&](uint32_t key, int x) {
    if (key > kNegInf) sum += __expf(unordered(key) - ref);
    if (key >= tau) {
      const int at = atomicAdd(&s_count, 1);
      if (at < kMaxCand) s_cand[at] = (static_cast<uint64_t>(key) << 32) | ~static_cast<uint32_t>(x);
    }
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) visit(u[i], t0 + (i / N) * kBThreads * N + i % N);
  visit(extra, xe);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    float t = 0.0f;
    for (int i = 0; i < kBThreads / 32; ++i) t += s_sum[i];
    stats[item] = BeamPartial{m, t};
  }
  const int n = s_count;
  if (n <= kMaxCand) {
    for (int i = tid; i < n; i += kBThreads) {
      const uint64_t mine = s_cand[i];
      int rank = 0;
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
    auto look = [&](uint32_t key, int x) {
      const uint64_t full = (static_cast<uint64_t>(key) << 32) | ~static_cast<uint32_t>(x);
      if (key != kNone && full < last && full > best) best = full;
    };
#pragma unroll
    for (int i = 0; i < kPer; ++i) look(u[i], t0 + (i / N) * kBThreads * N + i % N);
    look(extra, xe);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
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

__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v >> 32));
  const uint32_t lo = __reduce_max_sync(
      0xffffffffu, static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// One warp per request: lane l owns the lists l, l + 32, ... (row-major over
// beams and chunks) and keeps the best head among them.
__global__ void __launch_bounds__(32)
    beam_merge_kernel(const float* __restrict__ scores, const uint8_t* __restrict__ done, int end,
                      int W, int V, int K, int nchunk, const BeamPartial* __restrict__ stats,
                      const uint64_t* __restrict__ lists, float* __restrict__ out_scores,
                      int* __restrict__ out_beams, int* __restrict__ out_tokens,
                      uint8_t* __restrict__ out_done) {
  extern __shared__ int s_pos[];  // next entry of every list
  __shared__ double s_m[kMaxW], s_ls[kMaxW], s_score[kMaxW];
  __shared__ uint8_t s_done[kMaxW];
  const int b = blockIdx.x, lane = threadIdx.x;
  const int nlists = W * nchunk;
  for (int i = lane; i < nlists; i += 32) s_pos[i] = 0;
  // a row's maximum and sum over its chunks
  if (lane < W) {
    const int row = b * W + lane;
    const BeamPartial* st = stats + static_cast<int64_t>(row) * nchunk;
    float m = -INFINITY;
    for (int c = 0; c < nchunk; ++c) m = fmaxf(m, st[c].m);
    double sum = 0.0;
    for (int c = 0; c < nchunk; ++c)
      if (st[c].m > -INFINITY)
        sum += static_cast<double>(st[c].sum) * exp(static_cast<double>(st[c].m) - m);
    const float sc = scores[row];
    s_m[lane] = m;
    s_ls[lane] = log(sum);
    s_score[lane] = sc == sc ? sc : -INFINITY;
    s_done[lane] = done != nullptr && done[row] != 0;
  }
  __syncwarp();
  const uint64_t* mine = lists + static_cast<int64_t>(b) * nlists * K;
  // total of a list's entry as ordered bits; 0 = the list is used up
  auto total_of = [&](int l, int pos) -> uint64_t {
    if (pos >= K) return 0ull;
    const uint64_t key = mine[static_cast<int64_t>(l) * K + pos];
    if (key == 0ull) return 0ull;
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    const int w = l / nchunk;
    double t = -INFINITY;
    if (u > kNegInf && s_score[w] > -INFINITY)
      t = s_done[w] ? s_score[w]
                    : s_score[w] + ((static_cast<double>(unordered(u)) - s_m[w]) - s_ls[w]);
    return ordered64(t);
  };
  auto flat_of = [&](int l, int pos) -> uint64_t {
    const uint64_t key = mine[static_cast<int64_t>(l) * K + pos];
    return static_cast<uint64_t>(l / nchunk) * V + static_cast<uint32_t>(~static_cast<uint32_t>(key));
  };
  uint64_t best = 0ull, flat = ~0ull;
  int from = -1;
  auto rescan = [&] {
    best = 0ull;
    flat = ~0ull;
    from = -1;
    for (int l = lane; l < nlists; l += 32) {
      const uint64_t t = total_of(l, s_pos[l]);
      if (t == 0ull) continue;
      const uint64_t f = flat_of(l, s_pos[l]);
      if (t > best || (t == best && f < flat)) {
        best = t;
        flat = f;
        from = l;
      }
    }
  };
  rescan();
  for (int k = 0; k < K; ++k) {
    const uint64_t top = warp_max64(best);
    // of the lanes that hold it, the lowest flat index
    const uint64_t inv = (best == top && from >= 0) ? ~flat : 0ull;
    const uint64_t win = warp_max64(inv);
    if (inv == win && win != 0ull) {
      const int w = static_cast<int>(flat / V), x = static_cast<int>(flat - static_cast<uint64_t>(w) * V);
      const int64_t o = static_cast<int64_t>(b) * K + k;
      out_scores[o] = static_cast<float>(unordered64(best));
      out_beams[o] = w;
      out_tokens[o] = x;
      if (out_done) out_done[o] = s_done[w] || x == end;
      s_pos[from] += 1;
      rescan();
    }
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
    beam_merge_kernel<<<B, 32, static_cast<size_t>(W) * nchunk * sizeof(int), st>>>(
        scores, done, end_token, W, V, K, nchunk, stats, lists, out_scores, out_beams, out_tokens,
        out_done);
    check_launch("beam_merge_kernel", st);
  });
}
