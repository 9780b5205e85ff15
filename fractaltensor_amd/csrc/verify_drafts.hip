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
// single probabilities are.
//
// Vocabularies up to 65536: one launch, a workgroup of 1024 threads to a sequence.  A thread sums four neighbouring weights at a time
// and leaves the sums in LDS; what is left is to find one among these, and to look at four weights again.  Bound by a chain of some six
// memory latencies and by what one compute unit reads: 10 us for 4 sequences of 32000 and 4 drafted tokens in fp32 (two launches 13.5).
//
// Larger ones: the first launch sums the weights of kSegment tokens a workgroup, the second finds the segment and in it the token.
// Bound by reading the two rows: 12 + 9 us for 64 sequences of 131072 in fp32 (a workgroup to a sequence 28).
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
  if (s == 0 && threadIdx.x == 0) a.accepted[b] = n;
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

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ double wave_scan(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// The first lane of a wave whose positive weights (`sum` of them, `end` with all before it) pass the aim; else the last that has any; else -1.
__device__ __forceinline__ int pick_lane(double sum, double end, double aim) {
  const unsigned long long some = __builtin_amdgcn_ballot_w64(sum > 0.0), past = __builtin_amdgcn_ballot_w64(sum > 0.0 && end > aim);
  return past ? (int)__builtin_ctzll(past) : some ? 63 - (int)__builtin_clzll(some) : -1;
}

// Tokens of a sequence: the accepted drafts, the next one, then -1.
__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int n, int next) {
  const int i = threadIdx.x;
  if (i > a.K) return;
  const long long id = i < n ? drafted(a, (long long)b * a.K + i) : i == n ? (long long)next : -1;
  const long long at = (long long)b * (a.K + 1) + i;
  if (a.wide_ids) ((long long*)a.tokens)[at] = id;
  else ((int*)a.tokens)[at] = (int)id;
  if (i == 0) a.accepted[b] = n;
}

template <typename P, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // a lane of the first wave has the sums of up to kSegmentsMost / 64 neighbouring segments; they are asked for before anything is waited for
  constexpr int PER = kSegmentsMost / 64;
  const int per = (a.segments + 63) / 64;
  double own[2][PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = lane * per + i;
    const bool in = wave == 0 && i < per && s < a.segments;
    const double2 x = in ? *reinterpret_cast<const double2*>(a.sums + 2 * ((long long)b * a.segments + s)) : double2{0.0, 0.0};
    own[0][i] = x.x;
    own[1][i] = x.y;
  }
  const double u = (double)a.sample[b];
  const int n = a.accepted[b];                                 // by the first launch
  const bool rejected = n < (a.counts ? min(max(a.counts[b], 0), a.K) : a.K);
  const Weights<P> w(a, b, n, rejected);
  __shared__ double waves[kVerifyThreads / 64], begin, goal;
  __shared__ int chosen, source, found, last;
  if (wave == 0) {
    double sum[2] = {0.0, 0.0}, end[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < PER; ++i) sum[k] += own[k][i];
      end[k] = wave_scan(sum[k]);
    }
    const double rest = __shfl(end[0], 63), all = __shfl(end[1], 63);
    const int k = rejected && rest > 0.0 ? 0 : 1;              // nothing is left of the target's row: the row itself
    const double aim = u * (k ? all : rest);
    const int at = pick_lane(k ? sum[1] : sum[0], k ? end[1] : end[0], aim);
    if (lane == 0) {
      chosen = -1;
      found = INT_MAX;
      last = -1;
      source = k;
      goal = aim;
    }
    if (lane == at) {
      double here = (k ? end[1] : end[0]) - (k ? sum[1] : sum[0]);
      int s = -1;
      double before = here;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const double x = k ? own[1][i] : own[0][i];
        if (x > 0.0 && (s < 0 || before <= aim)) {             // `before`: with the segment that is held
          begin = here;
          s = lane * per + i;
          before = here + x;
        }
        here += x;
      }
      chosen = s;
    }
  }
  __syncthreads();
  // the token: eight neighbours a thread, kSegment tokens at a time
  constexpr int E = kSegment / kVerifyThreads;
  const int k = source, segment = chosen, from = segment * a.segment, to = segment < 0 ? from : min(a.V, from + a.segment);
  const double aim = goal;
  double at = begin;
  for (int i0 = from; i0 < to; i0 += kSegment) {
    const int first_i = i0 + tid * E;
    P p[E] = {}, q[E] = {};
    if constexpr (VEC) {
      constexpr int W = 16 / sizeof(P);
      struct alignas(16) Piece {
        P x[W];
      };
#pragma unroll
      for (int j = 0; j < E; j += W)
        if (first_i + j < to) {
          const Piece a16 = *reinterpret_cast<const Piece*>(w.p + first_i + j);
          Piece b16{};
          if (k == 0 && w.q) b16 = *reinterpret_cast<const Piece*>(w.q + first_i + j);
#pragma unroll
          for (int e = 0; e < W; ++e) {
            p[j + e] = a16.x[e];
            q[j + e] = b16.x[e];
          }
        }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (first_i + e < to) {
          p[e] = w.p[first_i + e];
          if (k == 0 && w.q) q[e] = w.q[first_i + e];
        }
    }
    double x[E], mine = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = k == 0 ? w.rest((double)(float)p[e], (double)(float)q[e], first_i + e) : w.all((double)(float)p[e]);
      mine += x[e];
    }
    const double end = wave_scan(mine);
    if (lane == 63) waves[wave] = end;
    __syncthreads();
    double here = at + (end - mine);
#pragma unroll
    for (int i = 0; i < kVerifyThreads / 64; ++i) {
      if (i < wave) here += waves[i];
      at += waves[i];
    }
    int first = INT_MAX, positive = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      here += x[e];
      if (x[e] > 0.0) {
        positive = first_i + e;
        if (here > aim && first == INT_MAX) first = positive;
      }
    }
    if (first != INT_MAX) atomicMin(&found, first);
    if (positive >= 0) atomicMax(&last, positive);
    __syncthreads();
  }
  write_tokens(a, b, n, found != INT_MAX ? found : last);
}

// One launch: chunks of four weights to each of 1024 threads, at most kChunks of them.
constexpr int kRowThreads = 1024, kChunk = 4 * kRowThreads, kChunks = 16;

template <typename P, bool VEC>
__global__ __launch_bounds__(kRowThreads) void verify_row_kernel(VerifyArgs a) {
  extern __shared__ double part[];                             // [chunks][threads]
  __shared__ double totals[kChunks];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  bool rejected;
  const int n = accepted_of<P>(a, b, &rejected);
  const double u = (double)a.sample[b];
  const Weights<P> w(a, b, n, rejected);
  const int chunks = (a.V + kChunk - 1) / kChunk;
  struct alignas(4 * sizeof(P)) Piece {
    P x[4];
  };
  auto four = [&](int i, bool rest, double (&x)[4]) __attribute__((always_inline)) {
    Piece p{}, q{};
    if constexpr (VEC) {
      if (i < a.V) {
        p = *reinterpret_cast<const Piece*>(w.p + i);
        if (rest && w.q) q = *reinterpret_cast<const Piece*>(w.q + i);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < a.V) {
          p.x[e] = w.p[i + e];
          if (rest && w.q) q.x[e] = w.q[i + e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = rest ? w.rest((double)(float)p.x[e], (double)(float)q.x[e], i + e) : w.all((double)(float)p.x[e]);
  };
  bool rest = rejected;
  double total;
  for (;;) {
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
      double x[4];
      four(c * kChunk + 4 * tid, rest, x);
      part[c * kRowThreads + tid] = (x[0] + x[1]) + (x[2] + x[3]);
    }
    __syncthreads();
    if (wave < chunks) {                                       // a wave a chunk, the lanes' sums of every 64th in order
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < kRowThreads / 64; ++i) sum += part[wave * kRowThreads + 64 * i + lane];
      sum = wave_sum(sum);
      if (lane == 0) totals[wave] = sum;
    }
    __syncthreads();
    total = 0.0;
    for (int c = 0; c < chunks; ++c) total += totals[c];
    if (!rest || total > 0.0) break;
    rest = false;                                              // nothing is left of the target's row: the row itself
    __syncthreads();
  }
  const double aim = u * total;
  if (wave != 0) return;
  // the chunk, the 64 sums in it, the four weights
  int next = -1;
  {
    const double own = lane < chunks ? totals[lane] : 0.0, end = wave_scan(own);
    const int c = pick_lane(own, end, aim);
    if (c >= 0) {
      double before = __shfl(end - own, c);
      constexpr int ROUNDS = kRowThreads / 64;
      double sums[ROUNDS], group = 0.0;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        sums[i] = wave_sum(part[c * kRowThreads + 64 * i + lane]);   // (in every lane)
        if (lane == i) group = sums[i];
      }
      const double group_end = wave_scan(group);
      const int g = pick_lane(group, before + group_end, aim);
      if (g >= 0) {
        before += __shfl(group_end - group, g);
        const double mine = part[c * kRowThreads + 64 * g + lane], mine_end = wave_scan(mine);
        const int t = pick_lane(mine, before + mine_end, aim);
        if (t >= 0) {
          double here = before + __shfl(mine_end - mine, t);
          double x[4];
          const int i = c * kChunk + 4 * (64 * g + t);
          four(i, rest, x);
          bool past = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            here += x[e];
            if (x[e] > 0.0 && !past) {
              next = i + e;
              past = here > aim;
            }
          }
        }
      }
    }
  }
  write_tokens(a, b, n, next);
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
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return fail(FTK_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes", who, need);
  VerifyArgs a{target, drafted ? draft : nullptr, drafts, accept_uniforms, sample_uniforms, draft_lens, tokens, accepted, (double*)workspace, drafted, vocabulary,
               drafts_are_64bit != 0, 0, segment_of(vocabulary)};
  a.segments = (vocabulary + a.segment - 1) / a.segment;
  const long long blocks = (long long)sequences * a.segments;
  if (blocks > INT_MAX) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: grid too large", who);
  const bool vec = aligned16(target) && aligned16(draft) && (long long)vocabulary * size % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  auto with = [&](auto p) -> int {
    using P = decltype(p);
    const bool quads = (uintptr_t)target % (4 * size) == 0 && (uintptr_t)draft % (4 * size) == 0 && vocabulary % 4 == 0;
    auto row = [&](auto vec_c) -> int {
      constexpr bool VEC = decltype(vec_c)::value;
      const int lds = (vocabulary + kChunk - 1) / kChunk * kRowThreads * (int)sizeof(double);
      static DeviceOnce once;
      unsigned bit;
      if (once.pending(&bit)) {
        FTK_HIP(hipFuncSetAttribute((const void*)verify_row_kernel<P, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, kChunks * kRowThreads * (int)sizeof(double)));
        once.done(bit);
      }
      hipLaunchKernelGGL((verify_row_kernel<P, VEC>), dim3(sequences), dim3(kRowThreads), lds, s, a);
      return check_launch("verify_row_kernel");
    };
    if (vocabulary <= kChunk * kChunks) return quads ? row(std::true_type{}) : row(std::false_type{});
    if (vec) hipLaunchKernelGGL((verify_sums_kernel<P, true>), dim3((unsigned)blocks), dim3(kVerifyThreads), 0, s, a);
    else hipLaunchKernelGGL((verify_sums_kernel<P, false>), dim3((unsigned)blocks), dim3(kVerifyThreads), 0, s, a);
    if (int rc = check_launch("verify_sums_kernel")) return rc;
    if (vec) hipLaunchKernelGGL((verify_pick_kernel<P, true>), dim3(sequences), dim3(kVerifyThreads), 0, s, a);
    else hipLaunchKernelGGL((verify_pick_kernel<P, false>), dim3(sequences), dim3(kVerifyThreads), 0, s, a);
    return check_launch("verify_pick_kernel");
  };
  return type == FTK_F32 ? with(0.0f) : type == FTK_F16 ? with(_Float16{}) : with(__bf16{});
}

}  // extern "C"
