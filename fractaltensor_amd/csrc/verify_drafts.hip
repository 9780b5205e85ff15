// Verification of drafted tokens: which of them a target model accepts, and the token that follows the accepted ones.
//
// Token d_i, drafted with probability q_i(d_i), is accepted while u_i q_i(d_i) < p_i(d_i) for a uniform u_i of [0, 1); at the first
// that is not, the next token is drawn from max(p_i - q_i, 0), and behind K accepted ones from p_K.  Tokens that leave
// this way are distributed as the target's own.
//
// Exactness: probabilities of 16 or 32 bits and their products of two are exact in 64 bits, so acceptance does not depend on
// the arithmetic; sums are in 64 bits, and a drawn token could differ from another order of summation only where u * total lies
// within some 2^-50 of a border.  Every sum has a fixed order: the same call gives the same tokens.
//
// Of the K + 1 rows of a sequence at most one of the target's and one of the draft's is read: the rows are known once the K
// single probabilities are.  The first launch sums the weights of kSegment tokens a workgroup, the second finds the segment and
// in it the token.
#include <algorithm>

#include "kv_common.h"

namespace ftk {

constexpr int kSegment = 2048, kVerifyThreads = 256, kVerifyMost = 64;   // tokens of a segment; drafted tokens of a sequence
constexpr int kSegmentsMost = 1024;

struct VerifyArgs {
  const void *target, *draft;      // [B, K + 1, V], [B, K, V] or NULL
  const void* drafts;              // [B, K]
  const float *accept, *sample;    // [B, K], [B]
  const int* counts;               // [B] or NULL
  void* tokens;                    // [B, K + 1]
  int* accepted;                   // [B]
  double* sums;                    // [B][segments][2]: of the weights, of the target's row
  int K, V, wide_ids, segments, segment;
};

template <typename P>
__device__ __forceinline__ double probability(const void* p, long long i) {
  return (double)(float)((const P*)p)[i];
}
__device__ __forceinline__ long long drafted(const VerifyArgs& a, long long i) {
  return a.wide_ids ? ((const long long*)a.drafts)[i] : (long long)((const int*)a.drafts)[i];
}

// How many drafted tokens of sequence b are accepted, and whether one is rejected behind them; a lane a token.
template <typename P>
__device__ __forceinline__ int accepted_of(const VerifyArgs& a, int b, bool* rejected) {
  const int lane = threadIdx.x & 63;
  const int count = a.counts ? min(max(a.counts[b], 0), a.K) : a.K;
  bool take = false;
  if (lane < count) {
    const long long at = (long long)b * a.K + lane, id = drafted(a, at);
    if (id >= 0 && id < a.V) {
      const double p = probability<P>(a.target, ((long long)b * (a.K + 1) + lane) * a.V + id);
      const double q = a.draft ? probability<P>(a.draft, at * a.V + id) : 1.0;
      take = (double)a.accept[at] * q < p;
    }
  }
  const unsigned long long refused = __builtin_amdgcn_ballot_w64(!take);
  const int n = min(refused ? (int)__builtin_ctzll(refused) : 64, count);
  *rejected = n < count;
  return n;
}

// The weights that the next token is drawn from.
template <typename P>
struct Weights {
  const P *p, *q;        // rows; q NULL: the target's alone
  long long without;     // a token of weight zero, or -1
  __device__ __forceinline__ Weights(const VerifyArgs& a, int b, int n, bool rejected) {
    p = (const P*)a.target + ((long long)b * (a.K + 1) + n) * a.V;
    q = rejected && a.draft ? (const P*)a.draft + ((long long)b * a.K + n) * a.V : nullptr;
    without = rejected && !a.draft ? drafted(a, (long long)b * a.K + n) : -1;
  }
  static __device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }   // (NaN: 0)
  __device__ __forceinline__ double all(double pv) const { return positive(pv); }
  __device__ __forceinline__ double rest(double pv, double qv, int i) const { return i == without ? 0.0 : positive(pv - qv); }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// VEC: rows lie at 16-byte boundaries.
template <typename P, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyArgs a) {
  const int b = blockIdx.x / a.segments, s = blockIdx.x - b * a.segments;
  bool rejected;
  const int n = accepted_of<P>(a, b, &rejected);
  const Weights<P> w(a, b, n, rejected);
  const int from = s * a.segment, to = min(a.V, from + a.segment);
  double rest = 0.0, all = 0.0;
  if constexpr (VEC) {
    constexpr int E = 16 / sizeof(P);
    struct alignas(16) Piece {
      P x[E];
    };
    for (int i = from + (int)threadIdx.x * E; i < to; i += kVerifyThreads * E) {
      const Piece p = *reinterpret_cast<const Piece*>(w.p + i);
      Piece q{};
      if (w.q) q = *reinterpret_cast<const Piece*>(w.q + i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        all += w.all((double)(float)p.x[e]);
        rest += w.rest((double)(float)p.x[e], w.q ? (double)(float)q.x[e] : 0.0, i + e);
      }
    }
  } else {
    for (int i = from + (int)threadIdx.x; i < to; i += kVerifyThreads) {
      const double p = (double)(float)w.p[i];
      all += w.all(p);
      rest += w.rest(p, w.q ? (double)(float)w.q[i] : 0.0, i);
    }
  }
  __shared__ double part[2][kVerifyThreads / 64];
  rest = wave_sum(rest);
  all = wave_sum(all);
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = rest;
    part[1][threadIdx.x >> 6] = all;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double x = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyThreads / 64; ++i) x += part[threadIdx.x][i];
    a.sums[2LL * blockIdx.x + threadIdx.x] = x;
  }
}

// The sum of the values of the threads before this one, and that of all.
__device__ __forceinline__ double sum_before(double x, double* waves, double* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = y;
  __syncthreads();
  double before = 0.0, sum = 0.0;
#pragma unroll
  for (int i = 0; i < kVerifyThreads / 64; ++i) {
    if (i < wave) before += waves[i];
    sum += waves[i];
  }
  *all = sum;
  return before + (y - x);
}

template <typename P>
__global__ __launch_bounds__(kVerifyThreads) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x;
  bool rejected;
  const int n = accepted_of<P>(a, b, &rejected);
  const Weights<P> w(a, b, n, rejected);
  __shared__ double waves[kVerifyThreads / 64];
  __shared__ int found, last;
  __shared__ double begin;
  if (tid == 0) {
    found = INT_MAX;
    last = -1;
    begin = 0.0;
  }
  // the segment: kSegmentsMost / threads segments a thread
  constexpr int PER = kSegmentsMost / kVerifyThreads;
  double own[2][PER], sum[2] = {0.0, 0.0}, total[2], before[2];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = tid * PER + i;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      own[k][i] = s < a.segments ? a.sums[2 * ((long long)b * a.segments + s) + k] : 0.0;
      sum[k] += own[k][i];
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) before[k] = sum_before(sum[k], waves, &total[k]);
  const int k = rejected && total[0] > 0.0 ? 0 : 1;            // nothing is left of the target's row: the row itself
  const double aim = (double)a.sample[b] * total[k];
  {
    double at = before[k];
    int mine = INT_MAX, positive = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      at += own[k][i];
      if (own[k][i] > 0.0) {
        positive = tid * PER + i;
        if (at > aim && mine == INT_MAX) mine = positive;
      }
    }
    __syncthreads();
    if (mine != INT_MAX) atomicMin(&found, mine);
    if (positive >= 0) atomicMax(&last, positive);
    __syncthreads();
  }
  const int segment = found != INT_MAX ? found : last;         // (u so near 1 that rounding leaves none above)
  if (segment >= tid * PER && segment < (tid + 1) * PER) {
    double at = before[k];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (tid * PER + i < segment) at += own[k][i];
    begin = at;
  }
  __syncthreads();
  double at = begin;
  __syncthreads();
  if (tid == 0) {
    found = INT_MAX;
    last = -1;
  }
  __syncthreads();
  // the token: eight neighbours a thread, kSegment tokens at a time
  constexpr int E = kSegment / kVerifyThreads;
  const int from = segment * a.segment, to = segment < 0 ? from : min(a.V, from + a.segment);
  for (int i0 = from; i0 < to; i0 += kSegment) {
    double x[E], mine = 0.0, whole;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + tid * E + e;
      x[e] = 0.0;
      if (i < to) {
        const double p = (double)(float)w.p[i];
        x[e] = k == 0 ? w.rest(p, w.q ? (double)(float)w.q[i] : 0.0, i) : w.all(p);
      }
      mine += x[e];
    }
    double here = at + sum_before(mine, waves, &whole);
    int first = INT_MAX, positive = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      here += x[e];
      if (x[e] > 0.0) {
        positive = i0 + tid * E + e;
        if (here > aim && first == INT_MAX) first = positive;
      }
    }
    if (first != INT_MAX) atomicMin(&found, first);
    if (positive >= 0) atomicMax(&last, positive);
    at += whole;
    __syncthreads();
  }
  if (tid <= a.K) {
    const int next = found != INT_MAX ? found : last;
    const long long id = tid < n ? drafted(a, (long long)b * a.K + tid) : tid == n ? (long long)next : -1;
    const long long to_at = (long long)b * (a.K + 1) + tid;
    if (a.wide_ids) ((long long*)a.tokens)[to_at] = id;
    else ((int*)a.tokens)[to_at] = (int)id;
    if (tid == 0) a.accepted[b] = n;
  }
}

static int segment_of(int V) { return kSegment * ((V + kSegment * kSegmentsMost - 1) / (kSegment * kSegmentsMost)); }

}  // namespace ftk

extern "C" {

size_t ftk_verify_drafts_workspace_bytes(int sequences, int vocabulary) {
  if (sequences <= 0 || vocabulary <= 0 || vocabulary > (1 << 30)) return 0;
  const int segment = ftk::segment_of(vocabulary);
  return (size_t)sequences * ((vocabulary + segment - 1) / segment) * 2 * sizeof(double);
}

int ftk_verify_drafts(const void* target, const void* draft, int type, const void* drafts, int drafts_are_64bit, const float* accept_uniforms,
                      const float* sample_uniforms, const int* draft_lens, void* tokens, int* accepted, int sequences, int drafted, int vocabulary,
                      void* workspace, size_t workspace_bytes, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_verify_drafts";
  if (sequences < 0 || vocabulary <= 0 || drafted < 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the vocabulary must be positive, the other sizes not negative", who);
  if (drafted > kVerifyMost - 1 || vocabulary > (1 << 30)) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: at most %d drafted tokens and a vocabulary of 2^30", who, kVerifyMost - 1);
  if (type != FTK_F16 && type != FTK_BF16 && type != FTK_F32) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: probabilities are fp16, bf16 or fp32", who);
  if (sequences == 0) return FTK_OK;
  if (!target || !sample_uniforms || !tokens || !accepted || (drafted > 0 && (!drafts || !accept_uniforms)))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: operands must be non-NULL", who);
  const int size = type == FTK_F32 ? 4 : 2, id_size = drafts_are_64bit ? 8 : 4;
  if ((uintptr_t)target % size || (uintptr_t)draft % size || (uintptr_t)drafts % id_size || (uintptr_t)tokens % id_size ||
      (((uintptr_t)accept_uniforms | (uintptr_t)sample_uniforms | (uintptr_t)draft_lens | (uintptr_t)accepted) & 3))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their elements", who);
  const size_t need = ftk_verify_drafts_workspace_bytes(sequences, vocabulary);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7)) return fail(FTK_ERR_WORKSPACE, "%s: needs an 8-byte aligned workspace of %zu bytes", who, need);
  VerifyArgs a{target, drafted ? draft : nullptr, drafts, accept_uniforms, sample_uniforms, draft_lens, tokens, accepted, (double*)workspace, drafted, vocabulary,
               drafts_are_64bit != 0, 0, segment_of(vocabulary)};
  a.segments = (vocabulary + a.segment - 1) / a.segment;
  const long long blocks = (long long)sequences * a.segments;
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
  const bool vec = aligned16(target) && aligned16(draft) && (long long)vocabulary * size % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  auto with = [&](auto p) -> int {
    using P = decltype(p);
    if (vec) hipLaunchKernelGGL((verify_sums_kernel<P, true>), dim3((unsigned)blocks), dim3(kVerifyThreads), 0, s, a);
    else hipLaunchKernelGGL((verify_sums_kernel<P, false>), dim3((unsigned)blocks), dim3(kVerifyThreads), 0, s, a);
    if (int rc = check_launch("verify_sums_kernel")) return rc;
    hipLaunchKernelGGL((verify_pick_kernel<P>), dim3(sequences), dim3(kVerifyThreads), 0, s, a);
    return check_launch("verify_pick_kernel");
  };
  return type == FTK_F32 ? with(0.0f) : type == FTK_F16 ? with(_Float16{}) : with(__bf16{});
}

}  // extern "C"
