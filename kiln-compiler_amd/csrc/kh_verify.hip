// kh_verify.hip - which drafted tokens the target model keeps (kh_verify_op), and
// the token after them.
//
// A sequence's walk down its tree needs single probabilities until a token is
// refused (or the path ends): then one row of V probabilities is summed, and a
// second look into it finds where the running sum passes a random part of the
// whole. Sums and what they are sums of are 64-bit numbers: with V tokens of
// 1 / V each a running sum that is off by 2^-24 names another token now and
// then. They are kept by stretches of 1024 tokens, so that the second look reads
// one stretch.
//
// verify_kernel does all that with a workgroup per sequence. Where the
// sequences alone do not fill the chip, sums_kernel does the first sum of every
// sequence with a wave per stretch beforehand: 64 chains over 128000 tokens of
// fp32 14.6 us (the target's and the draft's row, 4.5 TB/s of the 5.2 that a copy
// reaches) and 7.8 us for the walk, two dependent looks into the sums and one
// stretch. One chain of 5 over 50257: 10.8 us, one workgroup reading 400 KB; 32
// trees without the draft's probabilities, 2.3 rows a path one after the other:
// 13 us. The sums of 64 bits cost what the loads wait for anyway; sums between
// lanes by permutes through the LDS took 3 to 5 us more.
#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <string>
#include <vector>

#include "kh_common.hpp"
#include "kh_internal.hpp"

namespace kh {

int abi_fail(int code, const std::string &msg);   // kh_plan.hip: sets kh_last_error

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxTokens = 256;     // drafted tokens of a sequence, as tree_attention's
constexpr int kStretch = 1024;      // tokens of a sum that is kept
constexpr int kMaxStretches = 1024; // ... of a row: longer rows have longer stretches
constexpr int kThreads = 1024;
constexpr int kSumThreads = 256;

struct VerifyWork {
  kh_verify_op p;
  int stretch;      // tokens of a stretch: a multiple of kStretch
  int stretches;
  double *sums;     // [sequence][stretch] of the first row summed, or null
};

// -- a row's weights: the target's probabilities less what refusals took ---------

template <int PT>
struct Probs;
template <>
struct Probs<KH_TYPE_F32> {
  typedef float T;
  static constexpr int N = 4;
};
template <>
struct Probs<KH_TYPE_BF16> {
  typedef __bf16 T;
  static constexpr int N = 8;
};
template <>
struct Probs<KH_TYPE_F16> {
  typedef _Float16 T;
  static constexpr int N = 8;
};

// N adjacent probabilities from x on, those at or past `end` 0. (A row starts at
// any multiple of its elements' size.)
template <int PT>
__device__ __forceinline__ void load_probs(const void *row, int x, int end, float (&y)[Probs<PT>::N]) {
  typedef typename Probs<PT>::T T;
  constexpr int N = Probs<PT>::N;
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
  const T *at = static_cast<const T *>(row) + x;
  if (x + N <= end) {
    const vec v = *reinterpret_cast<const loose *>(at);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = x + e < end ? (float)at[e] : 0.0f;
  }
}

// What is left of weight v after the refusals took their part of q (not below 0): 0
// where that is not above it (or is no number).
__device__ __forceinline__ double left_of(double v, double q, const double *took, int refusals) {
  for (int j = 0; j < refusals; ++j) {
    const double r = v - took[j] * q;
    v = r > 0.0 ? r : 0.0;
  }
  return v;
}

// Probabilities as they count: of the target 0 where they are not above it (or no
// number), of the draft 0 where they are below it; a NaN of the draft's stays, for
// which its token is refused and nothing of it is left.
__host__ __device__ inline float target_counted(float x) { return x > 0.0f ? x : 0.0f; }
__host__ __device__ inline float draft_counted(float x) { return __builtin_elementwise_maximum(x, 0.0f); }   // (one instruction, which keeps a NaN)

// The weights that are left of probabilities p: a refusal at a time for all, so that
// what it took is read once.
template <int STEPS, int N>
__device__ __forceinline__ void weigh(const float (&p)[STEPS][N], const float (&q)[STEPS][N], const double *took, int refusals, double (&v)[STEPS][N]) {
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) v[i][e] = target_counted(p[i][e]);
  for (int j = 0; j < refusals; ++j) {
    const double r = took[j];
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double left = v[i][e] - r * draft_counted(q[i][e]);
        v[i][e] = left > 0.0 ? left : 0.0;
      }
  }
}

// v moved between lanes by a DPP control, 0 where nothing comes (DPP moves take a
// few cycles where a permute through the LDS takes a hundred).
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A running sum over the lanes, own part included.
__device__ __forceinline__ double scan_lanes(double v) {
  v += moved<0x111, 0xF>(v);   // row_shr:1, 2, 4, 8
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);   // row_bcast:15 to rows 1 and 3
  v += moved<0x143, 0xC>(v);   // row_bcast:31 to rows 2 and 3
  return v;
}

__device__ __forceinline__ double lane_of(double v, int lane) {   // (a uniform lane: a scalar)
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double add_lanes(double v) { return lane_of(scan_lanes(v), 63); }

// The sum of a stretch's weights, by one wave; the same in every lane.
template <int PT, bool Q>
__device__ __forceinline__ double stretch_sum(const VerifyWork &w, const void *target, const void *draft, int x0, const double *took, int refusals) {
  constexpr int N = Probs<PT>::N, STEPS = kStretch / (64 * N);
  const int lane = threadIdx.x & 63, end = min(w.p.vocab, x0 + w.stretch);
  double sum = 0.0;
  for (int x1 = x0; x1 < end; x1 += kStretch) {
    float p[STEPS][N], q[STEPS][N];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int x = min(x1 + (64 * i + lane) * N, end);
      load_probs<PT>(target, x, end, p[i]);
      if (Q && refusals) load_probs<PT>(draft, x, end, q[i]);
    }
    double v[STEPS][N];
    weigh(p, q, took, Q ? refusals : 0, v);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += v[i][e];
  }
  return add_lanes(sum);
}

// The first token whose running sum passes `part` of the whole (the last with a
// weight where rounding leaves none), -1 where there is no weight at all; by one
// wave. sums: the stretches'.
template <int PT, bool Q>
__device__ int find_token(const VerifyWork &w, const void *target, const void *draft, const double *sums, double part, const double *took, int refusals) {
  constexpr int N = Probs<PT>::N;
  const int lane = threadIdx.x & 63;
  // the stretch
  double before = 0.0, base = 0.0;
  int found = -1, last = -1;
  double last_before = 0.0;
  for (int c0 = 0; c0 < w.stretches && found < 0; c0 += 64) {
    const double mine = c0 + lane < w.stretches ? sums[c0 + lane] : 0.0;
    const double run = scan_lanes(mine);
    const uint64_t past = __ballot(mine > 0.0 && before + run > part), some = __ballot(mine > 0.0);
    if (some) {   // (ballots are scalars)
      const int at = 63 - __builtin_clzll(some);
      last = c0 + at;
      last_before = before + lane_of(run, at) - lane_of(mine, at);
    }
    if (past) {
      const int at = __builtin_ctzll(past);
      found = c0 + at;
      base = before + lane_of(run, at) - lane_of(mine, at);
    }
    before += lane_of(run, 63);
  }
  if (found < 0) {
    if (last < 0) return -1;
    found = last;
    base = last_before;
  }
  // the token: a lane looks at 16 that lie together
  constexpr int STEPS = kStretch / (64 * N);
  const int x0 = found * w.stretch, end = min(w.p.vocab, x0 + w.stretch);
  int answer = -1, fallback = -1;
  for (int x1 = x0; x1 < end && answer < 0; x1 += kStretch) {
    const int x = min(x1 + lane * (kStretch / 64), end);
    float p[STEPS][N], q[STEPS][N];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      load_probs<PT>(target, min(x + i * N, end), end, p[i]);
      if (Q && refusals) load_probs<PT>(draft, min(x + i * N, end), end, q[i]);
    }
    double v[STEPS][N], mine = 0.0;
    weigh(p, q, took, Q ? refusals : 0, v);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) mine += v[i][e];
    const double run = scan_lanes(mine);
    double at = base + (run - mine);
    int first = -1, any = -1;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        at += v[i][e];
        if (v[i][e] > 0.0) {
          any = x + i * N + e;
          if (first < 0 && at > part) first = any;
        }
      }
    const uint64_t past = __ballot(first >= 0), some = __ballot(any >= 0);
    if (past) answer = __builtin_amdgcn_readlane(first, __builtin_ctzll(past));
    if (some) fallback = __builtin_amdgcn_readlane(any, 63 - __builtin_clzll(some));
    base += lane_of(run, 63);
  }
  return answer >= 0 ? answer : fallback;
}

// -- the walk ------------------------------------------------------------------

struct Walk {   // in the LDS
  int token[kMaxTokens], parent[kMaxTokens], path[kMaxTokens];
  double u[kMaxTokens], p[kMaxTokens], q[kMaxTokens];
  double took[kMaxTokens];
};

__device__ __forceinline__ double uniform_of(const VerifyWork &w, int s, int i) {
  const int64_t at = s * w.p.uniforms_s + i;
  const double u = w.p.uniforms_wide ? static_cast<const double *>(w.p.uniforms)[at] : (double)static_cast<const float *>(w.p.uniforms)[at];
  return u;
}

template <int PT>
__device__ __forceinline__ const void *row_of(const void *probs, int64_t at) {
  return static_cast<const typename Probs<PT>::T *>(probs) + at;
}

// Tokens, what they follow (-2: nothing) and, with the draft's probabilities,
// both models' of each.
template <int PT, bool Q>
__device__ __forceinline__ void load_walk(const VerifyWork &w, int s, Walk &t) {
  typedef typename Probs<PT>::T T;
  for (int i = threadIdx.x; i < w.p.draft; i += blockDim.x) {
    const int64_t token = w.p.tokens_wide ? static_cast<const int64_t *>(w.p.tokens)[s * w.p.tokens_s + i]
                                          : (int64_t)static_cast<const int32_t *>(w.p.tokens)[s * w.p.tokens_s + i];
    int up = w.p.parents ? w.p.parents[s * w.p.parents_s + i] : i - 1;
    t.u[i] = uniform_of(w, s, i);
    const bool in = token >= 0 && token < w.p.vocab;
    if (i > 0 && (up < 0 || up >= i || !in)) up = -2;
    t.token[i] = in ? (int)token : -1;
    t.parent[i] = up;
    if (Q && i > 0 && up >= 0) {
      t.p[i] = target_counted((float)static_cast<const T *>(w.p.target)[s * w.p.target_s + up * w.p.target_n + token]);
      t.q[i] = draft_counted((float)static_cast<const T *>(w.p.drafted)[s * w.p.drafted_s + up * w.p.drafted_n + token]);
    }
  }
  __syncthreads();
}

// What every lane knows alike, as a scalar: a branch on it takes the whole wave,
// which the ballots behind it need.
__device__ __forceinline__ bool all_know(bool x) { return __builtin_amdgcn_readfirstlane((int)x) != 0; }
__device__ __forceinline__ int all_know(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The next token after `i` that follows `now` (and is `token`, unless that is
// -1), `draft` where there is none; every wave alike.
__device__ __forceinline__ int next_child(const VerifyWork &w, const Walk &t, int i, int now, int token) {
  const int lane = threadIdx.x & 63;
  for (int i0 = (i + 1) & ~63; i0 < w.p.draft; i0 += 64) {
    const int j = i0 + lane;
    const bool is = j > i && j < w.p.draft && t.parent[j] == now && (token < 0 || t.token[j] == token);
    const uint64_t found = __ballot(is);
    if (found) return all_know(i0 + (int)__builtin_ctzll(found));
  }
  return w.p.draft;
}

// Down the tree while single probabilities decide: stops at the first refusal
// (its token is `at`), or with at = draft behind the last token.
struct Place {
  int now, at, count;   // the current token, the child asked last, tokens kept
};
template <bool Q>
__device__ __forceinline__ void descend(const VerifyWork &w, Walk &t, Place &r) {
  if (!Q) return;   // (every step draws)
  for (;;) {
    r.at = next_child(w, t, r.at, r.now, -1);
    if (r.at >= w.p.draft) return;
    if (!all_know(t.u[r.at] * t.q[r.at] < t.p[r.at])) return;
    r.now = r.at;
    t.path[r.count++] = r.now;   // (every thread the same)
  }
}

// The sums of the first row that a sequence needs: a wave per stretch.
template <int PT, bool Q>
__global__ __launch_bounds__(kSumThreads) void sums_kernel(const VerifyWork w) {
  __shared__ Walk t;
  const int s = blockIdx.y, c = blockIdx.x * (kSumThreads / 64) + (threadIdx.x >> 6);
  Place r = {0, 0, 1};
  int refusals = 0;
  if (Q) {
    load_walk<PT, Q>(w, s, t);
    descend<Q>(w, t, r);
    refusals = r.at < w.p.draft ? 1 : 0;
    t.took[0] = 1.0;
    __syncthreads();
  }
  if (c >= w.stretches) return;
  const double sum = stretch_sum<PT, Q>(w, row_of<PT>(w.p.target, s * w.p.target_s + r.now * w.p.target_n),
                                        row_of<PT>(w.p.drafted, s * w.p.drafted_s + r.now * w.p.drafted_n), c * w.stretch, t.took, refusals);
  if ((threadIdx.x & 63) == 0) w.sums[(int64_t)s * w.stretches + c] = sum;
}

// A workgroup per sequence: the whole walk; the first sums from sums_kernel where
// that ran.
template <int PT, bool Q>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyWork w) {
  __shared__ Walk t;
  __shared__ double sums[kMaxStretches];
  __shared__ int drawn;
  const int s = blockIdx.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (w.sums)
    for (int c = threadIdx.x; c < w.stretches; c += blockDim.x) sums[c] = w.sums[(int64_t)s * w.stretches + c];
  load_walk<PT, Q>(w, s, t);
  const bool used = all_know(t.parent[0] == -1);
  Place r = {0, 0, used ? 1 : 0};
  t.path[0] = 0;
  int token = -1;

  bool first = w.sums != nullptr;
  // the stretches' sums of the current row, and their whole
  auto add = [&](int refusals) {
    __syncthreads();   // (took, and nobody reads the old sums)
    if (!first) {
      const void *target = row_of<PT>(w.p.target, s * w.p.target_s + r.now * w.p.target_n);
      const void *draft = row_of<PT>(w.p.drafted, s * w.p.drafted_s + r.now * w.p.drafted_n);
      for (int c = wave; c < w.stretches; c += waves) {
        const double sum = stretch_sum<PT, Q>(w, target, draft, c * w.stretch, t.took, refusals);
        if ((threadIdx.x & 63) == 0) sums[c] = sum;
      }
    }
    first = false;
    __syncthreads();
    double whole = 0.0;   // (every wave in the same order)
    for (int c = threadIdx.x & 63; c < w.stretches; c += 64) whole += sums[c];
    return add_lanes(whole);
  };
  auto draw = [&](double u, double whole, int refusals) {
    if (wave == 0) {
      const double part = (u > 0.0 ? u : 0.0) * whole;
      const int x = whole < INFINITY
                        ? find_token<PT, Q>(w, row_of<PT>(w.p.target, s * w.p.target_s + r.now * w.p.target_n),
                                            row_of<PT>(w.p.drafted, s * w.p.drafted_s + r.now * w.p.drafted_n), sums, part, t.took, refusals)
                        : -1;
      if (threadIdx.x == 0) drawn = x;
    }
    __syncthreads();
    return all_know(drawn);
  };

  if (used) {
    if (Q) {
      double whole = 0.0;
      int refusals = 0;
      bool summed = false;
      descend<Q>(w, t, r);
      while (r.at < w.p.draft) {   // token r.at is refused
        t.took[refusals] = refusals ? whole : 1.0;
        whole = add(++refusals);
        summed = true;
        r.at = next_child(w, t, r.at, r.now, -1);
        if (r.at >= w.p.draft) break;
        if (all_know(t.u[r.at] * whole * t.q[r.at] < left_of(t.p[r.at], t.q[r.at], t.took, refusals))) {
          r.now = r.at;
          t.path[r.count++] = r.now;
          __syncthreads();   // (took is read)
          refusals = 0;
          summed = false;
          descend<Q>(w, t, r);
        }
      }
      if (!summed) whole = add(0);
      if (refusals && all_know(!(whole > 0.0))) whole = add(refusals = 0);   // nothing is left: the target's own
      token = draw(t.u[0], whole, refusals);
    } else {
      for (;;) {
        token = draw(t.u[r.now], add(0), 0);
        r.at = token < 0 ? w.p.draft : next_child(w, t, r.now, r.now, token);
        if (r.at >= w.p.draft) break;
        r.now = r.at;
        t.path[r.count++] = r.now;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < w.p.draft; i += blockDim.x) w.p.rows[(int64_t)s * w.p.draft + i] = i < r.count ? t.path[i] : -1;
  if (threadIdx.x == 0) {
    w.p.counts[s] = r.count;
    w.p.next[s] = token;
  }
}

VerifyWork work_of(const kh_verify_op &p) {
  VerifyWork w;
  w.p = p;
  w.stretch = kStretch * (int)((p.vocab + (int64_t)kStretch * kMaxStretches - 1) / ((int64_t)kStretch * kMaxStretches));
  w.stretches = (p.vocab + w.stretch - 1) / w.stretch;
  w.sums = nullptr;
  return w;
}

// Sequences that leave compute units without work have the first sums of all
// made beforehand, where that is more than four stretches a wave: a row of 50257 fp32
// probabilities (and the draft's) takes one workgroup 10.8 us in all, 4.6 and 5.1
// in two launches; 64 rows of 128000 23.0, and 14.3 and 7.9 us.
bool ahead(const kh_verify_op &p) { return p.batch < current_device().cus && work_of(p).stretches > 4 * (kThreads / 64); }

template <int PT, bool Q>
void launch_of(const VerifyWork &w, hipStream_t stream) {
  if (w.sums) {
    const dim3 grid((unsigned)((w.stretches + kSumThreads / 64 - 1) / (kSumThreads / 64)), (unsigned)w.p.batch);
    sums_kernel<PT, Q><<<grid, kSumThreads, 0, stream>>>(w);
  }
  verify_kernel<PT, Q><<<(unsigned)w.p.batch, kThreads, 0, stream>>>(w);
}

hipError_t launch(const kh_verify_op &p, void *workspace, hipStream_t stream) {
  if (p.batch == 0) return hipSuccess;
  VerifyWork w = work_of(p);
  if (ahead(p)) w.sums = static_cast<double *>(workspace);
  switch (p.type) {
    case KH_TYPE_F32: p.drafted ? launch_of<KH_TYPE_F32, true>(w, stream) : launch_of<KH_TYPE_F32, false>(w, stream); break;
    case KH_TYPE_BF16: p.drafted ? launch_of<KH_TYPE_BF16, true>(w, stream) : launch_of<KH_TYPE_BF16, false>(w, stream); break;
    default: p.drafted ? launch_of<KH_TYPE_F16, true>(w, stream) : launch_of<KH_TYPE_F16, false>(w, stream);
  }
  return hipGetLastError();
}

size_t workspace_bytes(const kh_verify_op &p) { return ahead(p) ? (size_t)p.batch * work_of(p).stretches * sizeof(double) : 0; }

// -- the meaning on the CPU ----------------------------------------------------------

float prob(const void *p, int64_t i, int type) {
  if (type == KH_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == KH_TYPE_BF16) return (float)static_cast<const __bf16 *>(p)[i];
  return (float)static_cast<const _Float16 *>(p)[i];
}

void host_verify(const kh_verify_op &p) {
  std::vector<double> left((size_t)p.vocab);
  for (int s = 0; s < p.batch; ++s) {
    int now = 0, token = -1;
    std::vector<int> path;
    auto follows = [&](int i) { return p.parents ? p.parents[s * p.parents_s + i] : i - 1; };
    auto token_of = [&](int i) {
      return p.tokens_wide ? static_cast<const int64_t *>(p.tokens)[s * p.tokens_s + i] : (int64_t)static_cast<const int32_t *>(p.tokens)[s * p.tokens_s + i];
    };
    auto uniform = [&](int i) {
      const int64_t at = s * p.uniforms_s + i;
      return p.uniforms_wide ? static_cast<const double *>(p.uniforms)[at] : (double)static_cast<const float *>(p.uniforms)[at];
    };
    auto fresh = [&] {
      double whole = 0.0;
      for (int x = 0; x < p.vocab; ++x) {
        left[(size_t)x] = target_counted(prob(p.target, s * p.target_s + now * p.target_n + x, p.type));
        whole += left[(size_t)x];
      }
      return whole;
    };
    auto draw = [&](double u) {
      double whole = 0.0, run = 0.0;
      int last = -1;
      for (double v : left) whole += v;
      if (!(whole < INFINITY)) return -1;
      const double part = (u > 0.0 ? u : 0.0) * whole;
      for (int x = 0; x < p.vocab; ++x) {
        if (!(left[(size_t)x] > 0.0)) continue;
        run += left[(size_t)x];
        last = x;
        if (run > part) return x;
      }
      return last;
    };
    if (follows(0) == -1) {
      path.push_back(0);
      fresh();
      double whole = 1.0;
      if (!p.drafted) token = draw(uniform(0));
      for (int i = 1; i < p.draft; ++i) {
        const int64_t c = token_of(i);
        if (follows(i) != now || c < 0 || c >= p.vocab) continue;
        if (!p.drafted) {
          if (c != token) continue;
        } else {
          const int64_t row = s * p.drafted_s + now * p.drafted_n;
          if (!(uniform(i) * whole * draft_counted(prob(p.drafted, row + c, p.type)) < left[(size_t)c])) {
            double rest = 0.0;
            for (int x = 0; x < p.vocab; ++x) {
              const double v = left[(size_t)x] - whole * draft_counted(prob(p.drafted, row + x, p.type));
              left[(size_t)x] = v > 0.0 ? v : 0.0;
              rest += left[(size_t)x];
            }
            whole = rest;
            continue;
          }
        }
        now = i;
        path.push_back(i);
        fresh();
        whole = 1.0;
        if (!p.drafted) token = draw(uniform(now));
      }
      if (p.drafted) {
        if (!(whole > 0.0)) fresh();
        token = draw(uniform(0));
      }
    }
    for (int i = 0; i < p.draft; ++i) p.rows[(int64_t)s * p.draft + i] = i < (int)path.size() ? path[(size_t)i] : -1;
    p.counts[s] = (int)path.size();
    p.next[s] = token;
  }
}

int check(const kh_verify_op *p, bool pointers) {
  if (!p) return abi_fail(KH_ERR_INVALID, "null argument");
  if (p->batch < 0 || p->draft < 1 || p->vocab < 1 || p->type < KH_TYPE_F32 || p->type > KH_TYPE_F16)
    return abi_fail(KH_ERR_INVALID, "bad sizes or types");
  if (p->draft > kMaxTokens)
    return abi_fail(KH_ERR_UNSUPPORTED, std::to_string(p->draft) + " drafted tokens of a sequence (at most " + std::to_string(kMaxTokens) + ")");
  if (p->batch > 65535) return abi_fail(KH_ERR_UNSUPPORTED, std::to_string(p->batch) + " sequences (at most 65535)");
  if (p->vocab > 1 << 24) return abi_fail(KH_ERR_UNSUPPORTED, "a vocabulary of " + std::to_string(p->vocab) + " tokens (at most 2^24)");
  if (!pointers || p->batch == 0) return KH_OK;
  auto odd = [](const void *x, int n) { return x == nullptr || (uintptr_t)x % n; };
  const int size = p->type == KH_TYPE_F32 ? 4 : 2;
  if (odd(p->tokens, p->tokens_wide ? 8 : 4) || odd(p->target, size) || odd(p->uniforms, p->uniforms_wide ? 8 : 4) ||
      (p->parents && odd(p->parents, 4)) || (p->drafted && odd(p->drafted, size)) || odd(p->rows, 4) || odd(p->counts, 4) || odd(p->next, 4))
    return abi_fail(KH_ERR_INVALID, "a null or unaligned pointer");
  return KH_OK;
}

// No C++ exception leaves a C entry.
template <class F>
int guarded(F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return abi_fail(KH_ERR_CAPACITY, "out of host memory");
  } catch (const std::exception &e) {
    return abi_fail(KH_ERR_INVALID, e.what());
  }
}

}  // namespace
}  // namespace kh

extern "C" {

int kh_verify_workspace_bytes(const kh_verify_op *op, size_t *bytes) {
  return kh::guarded([&] {
    if (!bytes) return kh::abi_fail(KH_ERR_INVALID, "null argument");
    const int rc = kh::check(op, false);
    if (rc == KH_OK) *bytes = kh::workspace_bytes(*op);
    return rc;
  });
}

int kh_verify_run(const kh_verify_op *op, void *workspace, size_t bytes, void *stream) {
  return kh::guarded([&] {
    const int rc = kh::check(op, true);
    if (rc != KH_OK) return rc;
    const size_t need = kh::workspace_bytes(*op);
    if (bytes < need || (need && !workspace))
      return kh::abi_fail(KH_ERR_CAPACITY, "workspace of " + std::to_string(bytes) + " bytes, the operator needs " + std::to_string(need));
    if ((uintptr_t)workspace % 16) return kh::abi_fail(KH_ERR_INVALID, "workspace: not 16-byte aligned");
    const hipError_t e = kh::launch(*op, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? (int)KH_OK : kh::abi_fail(KH_ERR_HIP, std::string("kh_verify_run: ") + hipGetErrorString(e));
  });
}

int kh_verify_host(const kh_verify_op *op) {
  return kh::guarded([&] {
    const int rc = kh::check(op, true);
    if (rc == KH_OK) kh::host_verify(*op);
    return rc;
  });
}

}  // extern "C"
