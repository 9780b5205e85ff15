// Verification of a tree of drafted tokens: from the root on, the target model's own next token is drawn at each node, and where the draft has a child with that
// token, the way goes on there; else the token is the one that follows.  Tokens that leave this way are drawn from the target whatever the drafts are, so that no
// probabilities of the draft are needed.
//
// A draw takes a workgroup of 1024 threads: a wave has a sixteenth of the row, in registers where they hold it, its lanes' sums of pieces of 16 bytes
// are kept, the sums of the sixteenths name the wave that has the token, and that wave finds the piece and in it the token.  Bound by a chain of latencies (the row,
// the sums, the scan) and by what one compute unit reads.  The draws of a sequence do not depend on one another, only which of them count does.  So there are two ways:
//
//   one behind the other   a workgroup to a sequence draws at the nodes on its way, and reads no other rows
//   all at once            a workgroup to each node, then a small launch that walks
//
// by what is less: all rows at HBM's rate, or a chain of draws.
//
// Sums are in 64 bits in a fixed order, the same on both ways; a drawn token could differ from another order of summation only where u * total lies within some 2^-50 of a border.
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
  int* drawn;                    // [tokens], all at once
  int sequences, tokens, V, most, wide_ids;
  int part;                      // of a row, a wave: a multiple of 64 pieces
};

// x plus that of the lane that CONTROL names, in the rows of 16 lanes that ROWS names; nothing where there is none.
template <int CONTROL, int ROWS>
__device__ __forceinline__ double plus_lane(double x) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)bits, CONTROL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(bits >> 32), CONTROL, ROWS, 0xf, false);
  return x + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// Inclusive sum over the lanes of a wave, or of each 16: lanes 1, 2, 4 and 8 in front within 16, then the last of the 16 and of the 32 in front.  (Register to register: exchanges
// through LDS take five times as long, and a draw is a chain of such sums.)
__device__ __forceinline__ double scan16(double x) { return plus_lane<0x118, 0xf>(plus_lane<0x114, 0xf>(plus_lane<0x112, 0xf>(plus_lane<0x111, 0xf>(x)))); }
__device__ __forceinline__ double scan64(double x) { return plus_lane<0x143, 0xc>(plus_lane<0x142, 0xa>(scan16(x))); }
__device__ __forceinline__ double of_lane(double x, int lane) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)bits, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(bits >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// The first lane of a wave whose positive weights (`sum` of them, `end` with all before it) pass the aim; else the last that has any; else -1.
__device__ __forceinline__ int tree_pick(double sum, double end, double aim) {
  const unsigned long long some = __builtin_amdgcn_ballot_w64(sum > 0.0), past = __builtin_amdgcn_ballot_w64(sum > 0.0 && end > aim);
  return past ? (int)__builtin_ctzll(past) : some ? 63 - (int)__builtin_clzll(some) : -1;
}

struct TreeShared {
  v4u pieces[kTreeThreads];
  double sums[kTreeWaves], waves[kTreeWaves];
  int found, last;
};

// The token that u draws from a row, -1 if it has no positive weight; all threads of the workgroup call it, and may call it again.  A wave has pieces from its part of the row
// on, 64 neighbouring ones at a time, the first HELD of a lane's in registers.  VEC: rows lie at 16-byte boundaries.
template <typename P, bool VEC, int HELD>
__device__ __forceinline__ int draw(const TreeArgs& a, const P* row, double u, TreeShared& shared) {
  constexpr int E = 16 / sizeof(P);
  static_assert(HELD <= kTreeWaves);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = (a.part + 64 * E - 1) / (64 * E);
  // piece `lane` of the c-th 64 of part w
  const auto place = [&](int w, int c) __attribute__((always_inline)) { return w * a.part + (64 * c + lane) * E; };
  const auto read = [&](int w, int c) __attribute__((always_inline)) {
    const int i = place(w, c), to = c < count ? min(a.V, (w + 1) * a.part) : 0;
    v4u p = {0, 0, 0, 0};
    if constexpr (VEC) {
      if (i < to) p = *reinterpret_cast<const v4u*>(row + i);
    } else {
      P x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i + e < to ? row[i + e] : P(0.0f);
      p = __builtin_bit_cast(v4u, x);
    }
    return p;
  };
  const auto weight = [&](v4u p, int e) __attribute__((always_inline)) {
    float x;
    if constexpr (sizeof(P) == 4) x = __uint_as_float(p[e]);
    else if constexpr (std::is_same<P, _Float16>::value) x = e & 1 ? Half::high(p[e / 2]) : Half::low(p[e / 2]);
    else x = e & 1 ? Brain::high(p[e / 2]) : Brain::low(p[e / 2]);
    return (double)__builtin_amdgcn_fmed3f(x, 0.0f, INFINITY);   // (NaN: 0)
  };
  const auto sum_of = [&](v4u p) __attribute__((always_inline)) {
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) s += weight(p, e);
    return s;
  };
  v4u held[HELD];
#pragma unroll
  for (int c = 0; c < HELD; ++c) held[c] = read(wave, c);
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < HELD; ++c) sum += sum_of(held[c]);
#pragma unroll 8
  for (int c = HELD; c < count; ++c) sum += sum_of(read(wave, c));
  sum = of_lane(scan64(sum), 63);
  if (lane == 0) shared.sums[wave] = sum;
  if (tid == 0) {
    shared.found = INT_MAX;
    shared.last = -1;
  }
  __syncthreads();
  // the wave that has the token
  const double own = shared.sums[lane & (kTreeWaves - 1)], end = scan16(own);
  const double aim = u * of_lane(end, kTreeWaves - 1);
  const int part = tree_pick(lane < kTreeWaves ? own : 0.0, end, aim);
  if (part < 0) {
    __syncthreads();
    return -1;
  }
  // Its pieces go to all threads, 1024 at a time, one each.
  double base = of_lane(end - own, part);
  if (wave == part) {
#pragma unroll
    for (int c = 0; c < HELD; ++c) shared.pieces[64 * c + lane] = held[c];
  }
  __syncthreads();
  for (int c0 = 0; c0 < count; c0 += kTreeWaves) {
    const v4u p = c0 == 0 && wave < HELD ? shared.pieces[tid] : read(part, c0 + wave);
    const double s = sum_of(p), s_end = scan64(s);
    if (lane == 63) shared.waves[wave] = s_end;
    __syncthreads();
    const double w = shared.waves[lane & (kTreeWaves - 1)], w_end = scan16(w);
    double here = base + of_lane(w_end - w, wave) + (s_end - s);
    base += of_lane(w_end, kTreeWaves - 1);
    int first = INT_MAX, some = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double x = weight(p, e);
      here += x;
      if (x > 0.0) {
        some = place(part, c0 + wave) + e;
        if (here > aim && first == INT_MAX) first = some;
      }
    }
    // lanes are in the order of the row
    const unsigned long long past = __builtin_amdgcn_ballot_w64(first != INT_MAX), any = __builtin_amdgcn_ballot_w64(some >= 0);
    if (past) {
      if (lane == (int)__builtin_ctzll(past)) atomicMin(&shared.found, first);
    } else if (any) {
      if (lane == 63 - (int)__builtin_clzll(any)) atomicMax(&shared.last, some);
    }
    __syncthreads();
    if (shared.found != INT_MAX) break;
  }
  const int token = shared.found != INT_MAX ? shared.found : shared.last;
  __syncthreads();                                               // (found and last begin again)
  return token;
}

__device__ __forceinline__ long long id_of(const TreeArgs& a, int i) { return a.wide_ids ? ((const long long*)a.ids)[i] : (long long)((const int*)a.ids)[i]; }
__device__ __forceinline__ void put(const TreeArgs& a, int b, int step, long long token, int node) {
  const long long at = (long long)b * a.most + step;
  if (a.wide_ids) ((long long*)a.next)[at] = token;
  else ((int*)a.next)[at] = (int)token;
  a.path[at] = node;
}
struct TreeRows {
  int start, n;
};
__device__ __forceinline__ TreeRows rows_of(const TreeArgs& a, int b) {
  const int start = min(max(load_uniform(a.starts, b), 0), a.tokens);
  return {start, min(max(load_uniform(a.starts, b + 1), start), a.tokens) - start};
}

constexpr int kNodes = 512;      // of a sequence whose ids and parents are kept at hand

// One behind the other.
template <typename P, bool VEC, int HELD>
__global__ __launch_bounds__(kTreeThreads) void verify_tree_kernel(TreeArgs a) {
  __shared__ TreeShared shared;
  __shared__ long long ids[kNodes];
  __shared__ int parents[kNodes], child[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const TreeRows r = rows_of(a, b);
  for (int i = tid; i < min(r.n, kNodes); i += kTreeThreads) {
    ids[i] = id_of(a, r.start + i);
    parents[i] = a.parents[r.start + i];
  }
  if (tid == 0) child[0] = child[1] = INT_MAX;
  int node = r.n > 0 ? 0 : -1, steps = 0;
  for (; steps < a.most && node >= 0; ++steps) {
    // (its barriers also end the step before)
    const int token = draw<P, VEC, HELD>(a, (const P*)a.target + (long long)(r.start + node) * a.V, (double)a.uniforms[(long long)b * a.most + steps], shared);
    int* const found = &child[steps & 1];
    if (token >= 0)
      for (int i = node + 1 + tid; i < r.n; i += kTreeThreads) {
        const bool near = i < kNodes;
        if ((near ? parents[i] : a.parents[r.start + i]) == node && (near ? ids[i] : id_of(a, r.start + i)) == token) atomicMin(found, i);
      }
    if (tid == 0) {
      put(a, b, steps, token, node);
      child[~steps & 1] = INT_MAX;                               // the next step's
    }
    __syncthreads();
    node = *found != INT_MAX ? *found : -1;
  }
  for (int i = steps + tid; i < a.most; i += kTreeThreads) put(a, b, i, -1, -1);
  if (tid == 0) a.accepted[b] = max(steps - 1, 0);
}

// All at once: what each node draws, with the uniform number of its depth.
template <typename P, bool VEC, int HELD>
__global__ __launch_bounds__(kTreeThreads) void verify_nodes_kernel(TreeArgs a) {
  __shared__ TreeShared shared;
  const int row = blockIdx.x;
  const int b = count_at_most(a.sequences, row, [&](int i) { return a.starts[i + 1]; });
  if (b >= a.sequences) return;
  const TreeRows r = rows_of(a, b);
  if (row < r.start || row >= r.start + r.n) return;
  int depth = 0;
  for (int at = row - r.start; depth < a.most && at > 0; ++depth) {   // (at falls with every step)
    const int up = load_uniform(a.parents, r.start + at);
    if (up < 0 || up >= at) return;                              // no way leads there from the root
    at = up;
  }
  if (depth >= a.most) return;
  const int token = draw<P, VEC, HELD>(a, (const P*)a.target + (long long)row * a.V, (double)a.uniforms[(long long)b * a.most + depth], shared);
  if (threadIdx.x == 0) a.drawn[row] = token;
}

// The way through what has been drawn: a wave to a sequence.
__global__ __launch_bounds__(64) void verify_walk_kernel(TreeArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const TreeRows r = rows_of(a, b);
  int token[4], parent[4];                                       // of the first 256 nodes, a lane four
  long long id[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = 64 * k + lane;
    const bool in = i < r.n;
    token[k] = in ? a.drawn[r.start + i] : -1;
    parent[k] = in ? a.parents[r.start + i] : -1;
    id[k] = in ? id_of(a, r.start + i) : -1;
  }
  int node = r.n > 0 ? 0 : -1, steps = 0;
  for (; steps < a.most && node >= 0; ++steps) {
    int t = -1;
    if (node < 256) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = __builtin_amdgcn_readlane(token[k], node & 63);
        if (node >> 6 == k) t = x;
      }
    } else {
      t = load_uniform(a.drawn, r.start + node);
    }
    if (lane == 0) put(a, b, steps, t, node);
    int next = -1;
    if (t >= 0) {
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        const unsigned long long m = __builtin_amdgcn_ballot_w64(64 * k + lane > node && parent[k] == node && id[k] == t);
        if (m) next = 64 * k + (int)__builtin_ctzll(m);
      }
      for (int i0 = 256; next < 0 && i0 < r.n; i0 += 64) {
        const int i = i0 + lane;
        const unsigned long long m = __builtin_amdgcn_ballot_w64(i < r.n && i > node && a.parents[r.start + i] == node && id_of(a, r.start + i) == t);
        if (m) next = i0 + (int)__builtin_ctzll(m);
      }
    }
    node = next;
  }
  for (int i = steps + lane; i < a.most; i += 64) put(a, b, i, -1, -1);
  if (lane == 0) a.accepted[b] = max(steps - 1, 0);
}

// Whether all rows are read.  A draw takes 2 us and 6.5 for every 100000 tokens of the vocabulary; a way has some five of them, if there are as many tokens.  All at once, a draw, 5 us
// more and the bytes at 5.5 TB/s.  (Eight draws of a chain, one behind the other and all at once: 35 and 12 us for 16 sequences of 32000 in fp32, 85 and 21 of 131072; trees of up to 31 tokens of
// 64 sequences, 131072 in bf16: 46 us, where all the rows are 250 MB.)
static bool all_at_once(int sequences, int tokens, int most, int V, double row_bytes) {
  const double draw = 2.0 + 6.5e-5 * V, way = std::min({(double)most, 5.0, 1.0 + (double)tokens / sequences});
  return 5.0 + draw + tokens * row_bytes / 5.5e6 < way * draw;
}

}  // namespace ftk

extern "C" {

size_t ftk_verify_tree_workspace_bytes(int tokens) { return tokens > 0 ? (size_t)tokens * sizeof(int) : 0; }

int ftk_verify_tree(const void* target, int type, const void* ids, int ids_are_64bit, const int* parents, const int* starts, const float* uniforms, void* next, int* path,
                    int* accepted, int sequences, int tokens, int most, int vocabulary, void* workspace, size_t workspace_bytes, ftk_stream_t stream) {
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
  if (workspace && ((uintptr_t)workspace & 15)) return fail(FTK_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
  TreeArgs a{target, ids, parents, starts, uniforms, next, path, accepted, (int*)workspace, sequences, tokens, vocabulary, most, ids_are_64bit != 0, 0};
  a.part = (int)(((long long)vocabulary + (long long)unit * kTreeWaves - 1) / ((long long)unit * kTreeWaves) * unit);
  const bool vec = aligned16(target) && (long long)vocabulary * size % 16 == 0;
  const bool all = workspace && workspace_bytes >= ftk_verify_tree_workspace_bytes(tokens) && tokens > 0 && all_at_once(sequences, tokens, most, vocabulary, (double)vocabulary * size);
  const hipStream_t s = (hipStream_t)stream;
  auto with = [&](auto p) -> int {
    using P = decltype(p);
    auto launch = [&](auto vec_c, auto held_c) -> int {
      constexpr bool VEC = decltype(vec_c)::value;
      constexpr int HELD = decltype(held_c)::value;
      if (!all) {
        hipLaunchKernelGGL((verify_tree_kernel<P, VEC, HELD>), dim3(sequences), dim3(kTreeThreads), 0, s, a);
        return check_launch("verify_tree_kernel");
      }
      hipLaunchKernelGGL((verify_nodes_kernel<P, VEC, HELD>), dim3(tokens), dim3(kTreeThreads), 0, s, a);
      if (int rc = check_launch("verify_nodes_kernel")) return rc;
      hipLaunchKernelGGL(verify_walk_kernel, dim3(sequences), dim3(64), 0, s, a);
      return check_launch("verify_walk_kernel");
    };
    // up to eight pieces a thread in registers, or sixteen
    auto with_held = [&](auto vec_c) { return a.part <= 8 * unit ? launch(vec_c, std::integral_constant<int, 8>{}) : launch(vec_c, std::integral_constant<int, 16>{}); };
    return vec ? with_held(std::true_type{}) : with_held(std::false_type{});
  };
  return type == FTK_F32 ? with(0.0f) : type == FTK_F16 ? with(_Float16{}) : with(__bf16{});
}

}  // extern "C"
