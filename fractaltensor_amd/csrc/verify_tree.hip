// Verification of a tree of drafted tokens: from the root on, the target model's own next token is drawn at each node, and where the draft has a child with that
// token, the way goes on there; else the token is the one that follows.  Tokens that leave this way are drawn from the target whatever the drafts are, so that no
// probabilities of the draft are needed.
//
// A workgroup of 1024 threads to a sequence, which reads the rows of the nodes on its way and no others.  A wave has a sixteenth of a row: the
// sums of the sixteenths name the one that holds the token, whose weights are then read once more, by all threads, a few neighbours each.  Bound by a chain
// of latencies for each node (its row, the sixteenth, the children) and by what one compute unit reads.
//
// Sums are in 64 bits in a fixed order; a drawn token could differ from another order of summation only where u * total lies within some 2^-50 of a border.
#include <algorithm>

#include "kv_common.h"

namespace ftk {

constexpr int kTreeThreads = 1024, kTreeWaves = kTreeThreads / 64, kWayMost = 64;

struct TreeArgs {
  const void* target;            // [tokens, V]
  const void* ids;               // [tokens]
  const int *parents, *starts;   // [tokens], [sequences + 1]
  const float* uniforms;         // [sequences, most]
  void* next;                    // [sequences, most]
  int *path, *accepted;          // [sequences, most], [sequences]
  int tokens, V, most, wide_ids;
  int part;                      // of a row, a wave: a multiple of 64 * E
};

__device__ __forceinline__ double positive(double x) { return x > 0.0 ? x : 0.0; }   // (NaN: 0)

__device__ __forceinline__ double tree_wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double tree_wave_scan(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// VEC: rows lie at 16-byte boundaries.
template <typename P, bool VEC>
__global__ __launch_bounds__(kTreeThreads) void verify_tree_kernel(TreeArgs a) {
  constexpr int E = 16 / sizeof(P);
  struct alignas(16) Piece {
    P x[E];
  };
  __shared__ double sums[kTreeWaves], waves[kTreeWaves];
  __shared__ int found, last, child;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int start = min(max(load_uniform(a.starts, b), 0), a.tokens), n = min(max(load_uniform(a.starts, b + 1), start), a.tokens) - start;
  const auto four = [&](const P* row, int i, int to) __attribute__((always_inline)) {
    Piece p{};
    if constexpr (VEC) {
      if (i < to) p = *reinterpret_cast<const Piece*>(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < to) p.x[e] = row[i + e];
    }
    return p;
  };
  int node = n > 0 ? 0 : -1, steps = 0;
  for (; steps < a.most && node >= 0; ++steps) {
    const P* const row = (const P*)a.target + (long long)(start + node) * a.V;
    const double u = (double)a.uniforms[(long long)b * a.most + steps];
    // ---- the sixteenth
    {
      const int from = wave * a.part, to = min(a.V, from + a.part);
      double sum = 0.0;
#pragma unroll 8
      for (int i = from + lane * E; i < to; i += 64 * E) {
        const Piece p = four(row, i, to);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += positive((double)(float)p.x[e]);
        sum += s;
      }
      sum = tree_wave_sum(sum);
      if (lane == 0) sums[wave] = sum;
      if (tid == 0) {
        found = INT_MAX;
        last = -1;
        child = INT_MAX;
      }
    }
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < kTreeWaves; ++i) total += sums[i];
    const double aim = u * total;
    int part = -1;
    double at = 0.0, before = 0.0;                               // in front of the part
#pragma unroll
    for (int i = 0; i < kTreeWaves; ++i) {
      if (sums[i] > 0.0 && (part < 0 || before + sums[part] <= aim)) {
        part = i;
        before = at;
      }
      at += sums[i];
    }
    // ---- the token: E neighbours a thread, 1024 E at a time
    if (part >= 0) {
      const int from = part * a.part, to = min(a.V, from + a.part);
      double base = before;
      for (int i0 = from; i0 < to; i0 += kTreeThreads * E) {
        const int i = i0 + tid * E;
        const Piece p = four(row, i, to);
        double x[E], mine = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[e] = positive((double)(float)p.x[e]);
          mine += x[e];
        }
        const double end = tree_wave_scan(mine);
        if (lane == 63) waves[wave] = end;
        __syncthreads();
        double here = base + (end - mine);
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
          if (w < wave) here += waves[w];
          base += waves[w];
        }
        int first = INT_MAX, some = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          here += x[e];
          if (x[e] > 0.0) {
            some = i + e;
            if (here > aim && first == INT_MAX) first = some;
          }
        }
        if (first != INT_MAX) atomicMin(&found, first);
        if (some >= 0) atomicMax(&last, some);
        __syncthreads();
      }
    }
    const int token = found != INT_MAX ? found : last;
    // ---- the child that has it
    if (token >= 0)
      for (int i = node + 1 + tid; i < n; i += kTreeThreads) {
        const long long id = a.wide_ids ? ((const long long*)a.ids)[start + i] : (long long)((const int*)a.ids)[start + i];
        if (a.parents[start + i] == node && id == token) atomicMin(&child, i);
      }
    if (tid == 0) {
      const long long to = (long long)b * a.most + steps;
      if (a.wide_ids) ((long long*)a.next)[to] = token;
      else ((int*)a.next)[to] = token;
      a.path[to] = node;
    }
    __syncthreads();
    node = child != INT_MAX ? child : -1;
    __syncthreads();                                             // (found, last and child begin again)
  }
  for (int i = steps + tid; i < a.most; i += kTreeThreads) {
    const long long to = (long long)b * a.most + i;
    if (a.wide_ids) ((long long*)a.next)[to] = -1;
    else ((int*)a.next)[to] = -1;
    a.path[to] = -1;
  }
  if (tid == 0) a.accepted[b] = max(steps - 1, 0);
}

}  // namespace ftk

extern "C" {

int ftk_verify_tree(const void* target, int type, const void* ids, int ids_are_64bit, const int* parents, const int* starts, const float* uniforms, void* next, int* path,
                    int* accepted, int sequences, int tokens, int most, int vocabulary, ftk_stream_t stream) {
  using namespace ftk;
  const char* who = "ftk_verify_tree";
  if (sequences < 0 || tokens < 0 || vocabulary <= 0 || most <= 0) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the vocabulary and the way must be positive, the other sizes not negative", who);
  if (most > kWayMost || vocabulary > (1 << 30)) return fail(FTK_ERR_UNSUPPORTED_SHAPE, "%s: at most %d tokens of a sequence and a vocabulary of 2^30", who, kWayMost);
  if (type != FTK_F16 && type != FTK_BF16 && type != FTK_F32) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: probabilities are fp16, bf16 or fp32", who);
  if (sequences == 0) return FTK_OK;
  if (!starts || !uniforms || !next || !path || !accepted || (tokens > 0 && (!target || !ids || !parents)))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: operands must be non-NULL", who);
  const int size = type == FTK_F32 ? 4 : 2, id_size = ids_are_64bit ? 8 : 4;
  if ((uintptr_t)target % size || (uintptr_t)ids % id_size || (uintptr_t)next % id_size ||
      (((uintptr_t)parents | (uintptr_t)starts | (uintptr_t)uniforms | (uintptr_t)path | (uintptr_t)accepted) & 3))
    return fail(FTK_ERR_INVALID_ARGUMENT, "%s: operands must be aligned to their elements", who);
  const int unit = 64 * (16 / size);
  TreeArgs a{target, ids, parents, starts, uniforms, next, path, accepted, tokens, vocabulary, most, ids_are_64bit != 0, 0};
  a.part = (int)(((long long)vocabulary + (long long)unit * kTreeWaves - 1) / ((long long)unit * kTreeWaves) * unit);
  const bool vec = aligned16(target) && (long long)vocabulary * size % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  auto with = [&](auto p) -> int {
    using P = decltype(p);
    if (vec) hipLaunchKernelGGL((verify_tree_kernel<P, true>), dim3(sequences), dim3(kTreeThreads), 0, s, a);
    else hipLaunchKernelGGL((verify_tree_kernel<P, false>), dim3(sequences), dim3(kTreeThreads), 0, s, a);
    return check_launch("verify_tree_kernel");
  };
  return type == FTK_F32 ? with(0.0f) : type == FTK_F16 ? with(_Float16{}) : with(__bf16{});
}

}  // extern "C"
