// paged_verify.hip -- sampled verification of drafted rows (exl3p_verify in
// include/exl3_paged.h) for MI355X (gfx950, wave64): the rows' softmax
// statistics, the walk down each sequence's tree, and the token sampled where it
// ends.
#include "paged_common.h"

namespace {

struct F32 {
  typedef float T;
  static constexpr uint32_t EXP = 0x7F800000u;
};

// Elements of 16 bytes of a row as floats.
template <typename E>
struct Vec {
  static constexpr int N = 16 / sizeof(typename E::T);
  static __device__ __forceinline__ void unpack(u32x4 raw, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(typename E::T) == 4) {
        const uint32_t v = raw[i];  // (a bit cast of an element itself takes the first)
        x[i] = __builtin_bit_cast(float, v);
      } else {
        x[2 * i] = to_f32<E>(raw[i] & 0xFFFFu);
        x[2 * i + 1] = to_f32<E>(raw[i] >> 16);
      }
    }
  }
};
// Elements e .. of a row as they are, -inf in place of those outside it.
template <typename E>
__device__ __forceinline__ u32x4 block_of(const char *row, int e, int vocab) {
  constexpr int N = Vec<E>::N, S = sizeof(typename E::T);
  if (e >= 0 && e + N <= vocab) return *reinterpret_cast<const u32x4 *>(row + (int64_t)e * S);
  constexpr uint32_t LOW = S == 4 ? 0xFF800000u : E::EXP | 0x8000u;
  u32x4 raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = 0;
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const int x = e + i * (N / 4) + k;
      uint32_t one = LOW;
      if (x >= 0 && x < vocab) {
        if constexpr (S == 4)
          one = reinterpret_cast<const uint32_t *>(row)[x];
        else
          one = reinterpret_cast<const uint16_t *>(row)[x];
      }
      v |= one << (16 * k);
    }
    raw[i] = v;
  }
  return raw;
}
// Drafts' probabilities of tokens e .., 0 outside the vocabulary; of any alignment.
template <typename Q, int N>
__device__ __forceinline__ void drafts_of(const typename Q::T *q, int e, int vocab, float (&y)[N]) {
  if (e >= 0 && e + N <= vocab) {
    typename Q::T t[N];
    __builtin_memcpy(t, q + e, sizeof(t));
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = (float)t[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = e + k >= 0 && e + k < vocab ? (float)q[e + k] : 0.0f;
  }
}
template <typename E>
__device__ __forceinline__ float one_of(const void *p, size_t i) {
  return (float)static_cast<const typename E::T *>(p)[i];
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr int ST = 256;       // threads of most workgroups,
constexpr int PIECE = 8192;   // elements of a row that one takes,
constexpr int DRAW = 4096;    // and of a row that is sampled
constexpr int ALONE = 1024;   // threads of a workgroup that walks alone
constexpr int SHORT = 32;     // rows of a sequence that the sampling walks by itself
constexpr int MIDDLE = 128;   // rows of a sequence whose walk takes little LDS

// A piece's largest logit, the first place of it, and the sum of its weights
// 2^((logit - top) log2(e) / T).
struct Part {
  float top;
  int32_t best;
  double mass;
};

// What a walk waits for: nothing, it has ended; what p~ has left after a refusal; a
// row's statistics; whether a refusal has left anything (within a launch alone).
enum Need : int32_t { END, REST, STATS, DOUBT };

// A walk: the row that it is at (among its sequence's), the last child looked at, and
// of p~ and q~ there: what p~ has left, what is left of q (siblings drawn without
// replacement), the share of q that p has lost and what the last refusal adds to it once that
// is known to leave something; the row's statistics.  (64 bytes: a larger one is not kept in
// registers, and verify_tree_64 takes 92 us, not 59.)
struct State {
  int32_t at, seen, need, best;
  double left, drawn, share, step;
  double mass;  // -1: the row has no distribution
  float top;
  int32_t spare;  // what follows where the refusals leave nothing: a child, or
};
static_assert(sizeof(State) == 64, "");
constexpr int AS_BEFORE = -1, NO_MATTER = -2;
constexpr double SCANT = 0x1p-16;  // what p~ has left is nothing, perhaps: 32-bit sums are off by less
__device__ __forceinline__ State begun() {
  return State{0, 0, STATS, 0, 1.0, 1.0, 0.0, 0.0, -1.0, 0.0f, NO_MATTER};
}

// Where a sequence's walk ended: what the sampling needs.
struct Tip {
  int32_t row;   // of the step's tensors, -1: nothing to sample
  int32_t at;    // among the sequence's
  float top, heat;
  double share;  // of q that p has lost, times the row's mass
  double u;
};

struct VerifyArgs {
  const void *logits;
  int64_t ls;
  const void *draft;
  int64_t ds;
  Step st;
  int vocab, pieces, draws;
  const int32_t *parent, *ids;
  const float *temperature;
  const double *u;
  int32_t *target;
  int distinct;
  int lazy;       // rows' statistics are formed when a walk gets there
  Part *part;     // [rows][pieces]
  State *state;   // [2][seqs]: a round reads one and leaves the other
  double *rest;   // [2][seqs][pieces]: what p~ has left, likewise
  Tip *tip;       // [seqs]
  double *sums;   // [seqs][draws][2]: of what p has left, of p
  int *arrived;   // [seqs]: sampling workgroups that are done
};

// A temperature's factor of the logits, in powers of two, f32's largest at most.
__device__ __forceinline__ float rate_of(float heat) {
  return fminf(LOG2E / heat, 3.0e38f);
}

// v of lane (this lane ^ m) without the LDS crossbar (exl3::xor_lanes).  For m below 16 a row
// of 16 lanes may take part alone.
template <typename T>
__device__ __forceinline__ T across(T v, int m) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, exl3::xor_lanes(__builtin_bit_cast(float, v), m));
  } else {
    const u32x2 x = __builtin_bit_cast(u32x2, v);
    const uint32_t lo = x[0], hi = x[1];
    return __builtin_bit_cast(T, u32x2{across(lo, m), across(hi, m)});
  }
}
// Sum over the lanes up to and with this one, as scan's.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const u32x2 x = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[0], CTRL, ROWS, 0xF, false),
                                          (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[1], CTRL, ROWS, 0xF, false)});
}
__device__ __forceinline__ double scan(double v) {
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);
  v += moved<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += across(v, m);
  return v;
}
__device__ __forceinline__ float larger(float a, float b) {  // NaN if either is
  return __builtin_elementwise_maximum(a, b);
}

// A sequence's rows and temperature.
struct Seq {
  int begin, n;
  float heat, rate;
  double inv;
  bool fit, greedy;
};
__device__ __forceinline__ Seq seq_of(const VerifyArgs &a, int s) {
  Seq q;
  q.begin = min(max(a.st.cu[s], 0), a.st.rows);
  q.n = min(min(max(a.st.cu[s + 1], q.begin), a.st.rows) - q.begin, min(a.st.max_rows, EXL3P_TREE_MAX));
  q.heat = a.temperature ? a.temperature[s] : 1.0f;
  q.rate = rate_of(q.heat);
  q.inv = 1.0 / (double)q.heat;
  q.fit = q.heat >= 0.0f && q.heat < INFINITY;
  q.greedy = q.heat == 0.0f;
  return q;
}

// ------------------------------------------------------------ rows' statistics

// A row's first element of a piece: the piece's blocks of 16 bytes lie on their
// boundaries, the row may not.
template <typename E>
__device__ __forceinline__ const char *row_of(const VerifyArgs &a, int t) {
  return static_cast<const char *>(a.logits) + (int64_t)t * a.ls * (int)sizeof(typename E::T);
}
template <typename E>
__device__ __forceinline__ int first_of(const char *row, int piece, int size) {
  return piece * size - (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
}

// A workgroup takes PIECE logits of a row into registers: the largest, then the
// weights' sum (f32 over 8 of a thread, 64 bits beyond).
template <typename E>
__device__ __forceinline__ void piece_stats(const VerifyArgs &a, int t, int piece, float heat, Part *to) {
  constexpr int N = Vec<E>::N, U = PIECE / ST / N;
  __shared__ float tops[ST / 64];
  __shared__ double masses[ST / 64];
  __shared__ int bests[ST / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char *row = row_of<E>(a, t);
  const int first = first_of<E>(row, piece, PIECE);
  float x[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
    Vec<E>::unpack(block_of<E>(row, first + (u * ST + (int)threadIdx.x) * N, a.vocab), x[u]);
  float top = x[0][0];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) top = larger(top, x[u][i]);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = larger(top, exl3::xor_lanes(top, m));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) top = larger(top, tops[w]);
  if (heat == 0.0f) {  // the first place of the largest is what counts
    int best = INT32_MAX;
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (x[u][i] == top) best = first + (u * ST + (int)threadIdx.x) * N + i;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) best = min(best, across(best, m));
    if (lane == 0) bests[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < ST / 64; ++w) best = min(best, bests[w]);
      *to = Part{top, best, 0.0};
    }
    return;
  }
  const float rate = rate_of(heat), ref = top == -INFINITY ? 0.0f : top;
  double mass = 0.0;
#pragma unroll
  for (int u = 0; u < U * N / 8; ++u) {
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y += __builtin_amdgcn_exp2f((x[(8 * u + i) / N][(8 * u + i) % N] - ref) * rate);
    mass += (double)y;
  }
  mass = wave_sum(mass);
  if (lane == 0) masses[wave] = mass;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < ST / 64; ++w) mass += masses[w];
    *to = Part{top, 0, mass};
  }
}

// All rows' statistics, a piece a workgroup.  Bound by bytes.
template <typename E>
__global__ __launch_bounds__(ST) void verify_stats_kernel(VerifyArgs a) {
  const int t = blockIdx.x / a.pieces, piece = blockIdx.x - t * a.pieces;
  const int lane = threadIdx.x & 63;
  // the row's sequence: how many end at it or before
  int s = 0;
  for (int s0 = 0; s0 < a.st.seqs; s0 += 64)
    s += __popcll(__ballot(s0 + lane < a.st.seqs && a.st.cu[min(s0 + lane, a.st.seqs - 1) + 1] <= t));
  if (s >= a.st.seqs) return;
  if (piece == 0 && threadIdx.x == 0 && t == max(a.st.cu[s], 0)) a.arrived[s] = 0;
  piece_stats<E>(a, t, piece, a.temperature ? a.temperature[s] : 1.0f, a.part + (size_t)t * a.pieces + piece);
}

// ------------------------------------------------------------------- the walk

// e^x for x <= 0 in 64 bits: a power of two times the series of e^f, |f| <= ln(2) / 2,
// whose 14th term is below 2^-57 of the sum.
__device__ __forceinline__ double exp_of(double arg) {
  const bool there = arg > -746.0;  // else below the smallest number
  const double x = there ? arg : 0.0;
  const double n = __builtin_rint(x * 1.4426950408889634074);
  // ln(2) in two parts, the first with zeros behind its 32nd bit
  double f = fma(n, -0x1.62e42feep-1, x);
  f = fma(n, -0x1.a39ef35793c76p-33, f);
  double y = 1.0 / 6227020800.0;
  y = fma(y, f, 1.0 / 479001600.0);
  y = fma(y, f, 1.0 / 39916800.0);
  y = fma(y, f, 1.0 / 3628800.0);
  y = fma(y, f, 1.0 / 362880.0);
  y = fma(y, f, 1.0 / 40320.0);
  y = fma(y, f, 1.0 / 5040.0);
  y = fma(y, f, 1.0 / 720.0);
  y = fma(y, f, 1.0 / 120.0);
  y = fma(y, f, 1.0 / 24.0);
  y = fma(y, f, 1.0 / 6.0);
  y = fma(y, f, 0.5);
  y = fma(y, f, 1.0);
  y = fma(y, f, 1.0);
  return there ? __builtin_amdgcn_ldexp(y, (int)n) : 0.0;
}

// The share of q that p has lost after a refusal: by more than 64 bits' roundings of the two
// sides, so that a refused token has none left.
__device__ __forceinline__ double lost(double share, double step) {
  return (share + step) * (1.0 + 0x1p-48);
}

// A walk in LDS: N rows at most.
template <int N, bool DRAFT>
struct Walk {
  State st;
  double rest;  // what p~ has left after the last refusal
  double p[N], us[N];
  Part stat[N];  // rows' statistics, mass -1: none; not of lazy walks
  float q[DRAFT ? N : 1];
  int up[N], tok[N], next[N];
  double sums[ALONE / 64];
  float tops[ALONE / 64];
  int bests[ALONE / 64];
};

template <int N, bool DRAFT>
__device__ __forceinline__ void load_rows(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q) {
  for (int i = threadIdx.x; i < min(q.n, N); i += blockDim.x) {
    const int t = q.begin + i, x = a.parent ? a.parent[t] : i - 1;
    w.up[i] = x >= 0 && x < i ? x : -1;
    w.tok[i] = a.ids[t];
    w.us[i] = a.u[t];
    w.next[i] = -1;
  }
}

// A row's statistics, mass -1 where it has no distribution.
__device__ __forceinline__ Part stats_of(const Seq &q, float top, int best, double mass) {
  const bool whole = q.fit && (q.greedy ? top > -INFINITY : top > -INFINITY && top < INFINITY && mass > 0.0 && mass < INFINITY);
  return Part{top, best, !whole ? -1.0 : q.greedy ? 1.0 : mass};
}
__device__ __forceinline__ void enter(State &st, const Part &x) {
  st.top = x.top, st.best = x.best, st.mass = x.mass;
}
// A row's parts joined, by 16 lanes.
__device__ __forceinline__ Part join_parts(const VerifyArgs &a, const Seq &q, int row) {
  const Part *part = a.part + (size_t)(q.begin + row) * a.pieces;
  float hi = -INFINITY;
  int best = INT32_MAX;
  double m = 0.0;
  for (int k = threadIdx.x & 15; k < a.pieces; k += 16) {
    const Part y = part[k];
    const float now = larger(hi, y.top), ref = now == -INFINITY ? 0.0f : now;
    if (y.top > hi) best = y.best;
    if (!q.greedy)
      m = m * (double)__builtin_amdgcn_exp2f((hi - ref) * q.rate) +
          y.mass * (double)__builtin_amdgcn_exp2f((y.top - ref) * q.rate);
    hi = now;
  }
  float all = hi;
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) all = larger(all, across(all, x));
  const float ref = all == -INFINITY ? 0.0f : all;
  if (!q.greedy) m *= (double)__builtin_amdgcn_exp2f((hi - ref) * q.rate);
  best = hi == all ? best : INT32_MAX;
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) m += across(m, x), best = min(best, across(best, x));
  return stats_of(q, all, best, m);
}
// The statistics of the rows (of lazy walks: of the one that the walk is at) and what
// they give the tokens of their children.  Behind a barrier, and before one.
template <typename E, typename Q, bool DRAFT, int N>
__device__ __forceinline__ void take_rows(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q, bool joined) {
  const int n = min(q.n, N), at = w.st.at;
  if (!joined) {
    if (!a.lazy) {
      for (int i = threadIdx.x >> 4; i < n; i += blockDim.x / 16) {
        const Part x = join_parts(a, q, i);
        if ((threadIdx.x & 15) == 0) {
          w.stat[i] = x;
          if (i == at) enter(w.st, x);
        }
      }
    } else if (threadIdx.x < 16) {
      const Part x = join_parts(a, q, at);
      if (threadIdx.x == 0) enter(w.st, x);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x + 1; i < n; i += blockDim.x) {
    const int j = w.up[i];
    double p = 0.0;
    float d = 0.0f;
    if (j >= 0 && (j == at || !a.lazy) && !q.greedy && (uint32_t)w.tok[i] < (uint32_t)a.vocab) {
      const double mass = a.lazy ? w.st.mass : w.stat[j].mass;
      const float top = a.lazy ? w.st.top : w.stat[j].top;
      const size_t t = (size_t)(q.begin + j);
      if (mass > 0.0) {
        p = exp(((double)one_of<E>(a.logits, t * a.ls + w.tok[i]) - (double)top) * q.inv) / mass;
        if constexpr (DRAFT) d = one_of<Q>(a.draft, t * a.ds + w.tok[i]);
      }
    }
    w.p[i] = p;
    if constexpr (DRAFT) w.q[i] = d;
  }
  __syncthreads();
}

// The walk goes on from the row that it is at to its end or to what it needs next, by
// the first wave: the next child of a row is found among 64 rows a ballot.
//
// The refused tokens' probabilities, q given: p~ after refusals is max(p -
// share q, 0), share the sum of A_j / B_j over the refusals, A_j the sum of p~
// and B_j that of q~ (1, or what the refused ones leave of it).  A refused token
// has none left: u A_j / B_j q >= p~ says that p~ is below what is taken.
//
// A refusal that leaves nothing of p~ at all is roundings' alone: without them a u below 1 accepts
// a child or leaves something.  But a row's mass is a sum of 32-bit powers (no draft: the last
// token there is, as a child, is not quite certain), and a draft's numbers are rounded, to a
// sum above 1 perhaps, so that max(p - q, 0) may be 0 throughout.  The sampling would have to
// say a refused child's token, and whoever goes by the targets would go on to that child.  So
// the child that such a refusal refused is accepted after all; where p~ had nothing of its
// token, p~ stays as it was before.  Whether there is nothing is looked for where it can be:
// without a draft, where SCANT is left; with one, where step q is above p~ for every token, by
// no more than step (the sum of q - 1) in all, so by no more than that at the child.
template <typename Q>
__device__ __forceinline__ double above_one(int vocab) {  // the sum of a rounded q, less 1
  return sizeof(typename Q::T) == 4 ? SCANT : Q::EXP == F16::EXP ? 0x1p-10 + vocab * 0x1p-25 : 0x1p-7;
}
template <typename Q, bool DRAFT, int N>
__device__ __forceinline__ int walk_on(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q, bool less_now) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x, n = min(q.n, N);
    State st = w.st;
    st.need = END;
    if (DRAFT && less_now) st.share = lost(st.share, st.step), st.left = w.rest;  // (not read at a walk's end)
    // the next child of the row behind row `from`
    auto next = [&](int from) {
      for (int b = (from + 1) & ~63; b < n; b += 64) {
        const int i = b + lane;
        const uint64_t f = __ballot(i > from && i < n && w.up[min(i, n - 1)] == st.at);
        if (f != 0) return b + __builtin_ctzll(f);
      }
      return n;
    };
    int c = st.mass >= 0.0 ? next(max(st.seen, st.at)) : n;
    while (c < n) {
      bool hit;
      double less = 0.0, step = 0.0, mine = 0.0;
      if (q.greedy) {
        hit = w.tok[c] == st.best;
      } else if constexpr (DRAFT) {
        step = st.left / fmax(st.drawn, 0x1p-53);
        mine = fmax(w.p[c] - st.share * (double)w.q[c], 0.0);
        hit = w.us[c] * step * (double)w.q[c] < mine;
      } else {
        // a token that a sibling before it had is not there any more
        less = w.p[c];
        for (int b = 0; b < c; b += 64) {
          const int i = b + lane;
          if (__ballot(i > 0 && i < c && w.up[i] == st.at && w.tok[i] == w.tok[c]) != 0) less = 0.0;
        }
        hit = w.us[c] * st.left < less;
      }
      const int from = st.seen = c;
      if (hit) {
        if (lane == 0) w.next[st.at] = w.tok[c];
        st.at = c, st.left = 1.0, st.drawn = 1.0, st.share = 0.0, st.spare = NO_MATTER;
        if (a.lazy) {
          st.need = STATS;
          break;
        }
        enter(st, w.stat[c]);
        c = st.mass >= 0.0 ? next(c) : n;
        continue;
      }
      c = next(from);
      if (q.greedy) continue;
      const bool real = w.us[from] < 1.0;  // (not of numbers that are none)
      if constexpr (DRAFT) {
        st.spare = !real ? NO_MATTER : mine > 0.0 ? from : AS_BEFORE;
        st.step = step;
        if (a.distinct) st.drawn -= (double)w.q[from];
        if (c < n) {
          st.need = REST;
          break;
        }
        if (real && step * ((double)w.q[from] - above_one<Q>(a.vocab)) <= mine + SCANT)
          st.need = DOUBT;
        else
          st.share = lost(st.share, step);
      } else {
        st.left -= less;
        if (real && less > 0.0) st.spare = from;
        if (c >= n && st.spare >= 0 && st.left <= SCANT) st.need = DOUBT;
      }
    }
    if (lane == 0) w.st = st;
  }
  __syncthreads();
  return w.st.need;
}

// Whether refusals have left anything, where that is in doubt: of any token, in the sampling's
// own numbers (LEFT).  Usually the first elements that are looked at have something.  Where not,
// the walk is put as said above (PUT), for a row's statistics perhaps (WAITS).
enum Settled { LEFT, PUT, WAITS };
template <typename E, typename Q, bool DRAFT, int N>
__device__ __forceinline__ Settled settle(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q) {
  constexpr int V = Vec<E>::N;
  const int at = w.st.at, spare = w.st.spare, n = min(q.n, N);
  const double top = (double)w.st.top, share = lost(w.st.share, w.st.step) * w.st.mass;
  const char *row = row_of<E>(a, q.begin + at);
  bool any = false;
  for (int e = first_of<E>(row, 0, 0) + (int)threadIdx.x * V; e < a.vocab && !any; e += (int)blockDim.x * V) {
    float x[V], y[V];
    Vec<E>::unpack(block_of<E>(row, e, a.vocab), x);
    if constexpr (DRAFT)
      drafts_of<Q, V>(static_cast<const typename Q::T *>(a.draft) + (size_t)(q.begin + at) * a.ds, e, a.vocab, y);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double p = exp_of(((double)x[k] - top) * q.inv);
      if constexpr (DRAFT) {
        any |= p - share * (double)y[k] > 0.0;
      } else if (p > 0.0) {
        bool there = true;
        for (int i = at + 1; i < n; ++i) there &= w.up[i] != at || w.tok[i] != e + k;
        any |= there;
      }
    }
  }
  if (__syncthreads_or(any)) return LEFT;
  if (threadIdx.x == 0 && spare >= 0) {
    w.next[at] = w.tok[spare];
    w.st.at = w.st.seen = spare, w.st.left = 1.0, w.st.drawn = 1.0, w.st.share = 0.0, w.st.spare = NO_MATTER;
    w.st.need = STATS;
    if (!a.lazy) enter(w.st, w.stat[spare]);
  }
  __syncthreads();
  return a.lazy && spare >= 0 ? WAITS : PUT;
}
// The walk from a row whose statistics are there, or (rest) from behind a refusal whose rest is.
template <typename E, typename Q, bool DRAFT, int N>
__device__ __forceinline__ int walk_from(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q, bool rest) {
  bool doubt = false;
  if (rest) {
    doubt = w.st.spare != NO_MATTER && w.rest < SCANT;
    __syncthreads();  // all have read it: the walk goes on from there, by one wave
  }
  for (;;) {
    if (doubt) {
      const Settled how = settle<E, Q>(a, w, q);
      if (how == WAITS) return STATS;
      rest = how == LEFT;
    }
    const int need = walk_on<Q>(a, w, q, rest);
    if (need != DOUBT) return need;
    doubt = true;
  }
}

// What p~ has left at the row that the walk is at: of 8 elements, f32 but for the sum.
template <typename E, typename Q>
__device__ __forceinline__ double rest_of(const VerifyArgs &a, const State &st, const Seq &q, int begin, int end,
                                          int by) {
  constexpr int N = Vec<E>::N;
  const char *row = row_of<E>(a, q.begin + st.at);
  const typename Q::T *d = static_cast<const typename Q::T *>(a.draft) + (size_t)(q.begin + st.at) * a.ds;
  const float inv = (float)(1.0 / st.mass), share = (float)lost(st.share, st.step);
  double sum = 0.0;
#pragma unroll 4
  for (int e = begin; e < end; e += by) {
    float x[N], y[N], v = 0.0f;
    Vec<E>::unpack(block_of<E>(row, e, a.vocab), x);
    drafts_of<Q, N>(d, e, a.vocab, y);
#pragma unroll
    for (int k = 0; k < N; ++k)
      v += fmaxf(__builtin_amdgcn_exp2f((x[k] - st.top) * q.rate) * inv - share * y[k], 0.0f);
    sum += (double)v;
  }
  return sum;
}

// A walk's end: the tokens of its rows (the last one's is the sampling's, where there is one:
// another workgroup's to write) and what the sampling needs.
template <int N, bool DRAFT>
__device__ __forceinline__ Tip tip_of(const Walk<N, DRAFT> &w, const Seq &q) {
  const int row = w.st.at;
  if (!(w.st.mass >= 0.0) || q.greedy) return Tip{-1, row, 0.0f, 1.0f, 0.0, 0.0};
  return Tip{q.begin + row, row, w.st.top, q.heat, w.st.share * w.st.mass, w.us[0]};
}
// first: of this sequence nothing has been written yet.
template <int N, bool DRAFT>
__device__ __forceinline__ void write_rows(const VerifyArgs &a, const Walk<N, DRAFT> &w, const Seq &q, bool first,
                                           bool ended, const Tip &tip) {
  for (int i = threadIdx.x; i < min(q.n, N); i += blockDim.x) {
    int v = w.next[i];
    if (ended && i == w.st.at) {
      if (tip.row >= 0) continue;
      if (q.greedy && w.st.mass >= 0.0) v = w.st.best;
    }
    if (first || v >= 0) a.target[q.begin + i] = v;
  }
}

// A round: every workgroup of a sequence takes what the last round's have found, walks on,
// all alike, and forms its piece of what the walk needs next.  Rounds are launches, so
// nothing waits; a sequence whose walk has ended is left alone.  A chain of loads (state,
// parts, rows, children's logits, a piece): 6 us a round.
template <typename E, typename Q, bool DRAFT, int N>
__global__ __launch_bounds__(ST) void verify_round_kernel(VerifyArgs a, int round) {
  __shared__ Walk<N, DRAFT> w;
  const int s = blockIdx.x / a.pieces, piece = blockIdx.x - s * a.pieces;
  const Seq q = seq_of(a, s);
  if (round == 0 && piece == 0 && threadIdx.x == 0) {
    a.arrived[s] = 0, a.tip[s].row = -1;
    if (q.n <= 0) a.state[a.st.seqs + s].need = END;
  }
  if (q.n <= 0) return;
  const State had = round == 0 ? begun() : a.state[(size_t)(round & 1) * a.st.seqs + s];
  if (had.need == END) {
    if (piece == 0 && threadIdx.x == 0) a.state[(size_t)(~round & 1) * a.st.seqs + s].need = END;
    return;
  }
  // walks that need nothing are one workgroup's
  if (piece > 0 && !a.lazy && !(DRAFT && a.parent != nullptr && a.st.max_rows > 2)) return;
  load_rows(a, w, q);
  if (threadIdx.x == 0) w.st = had;
  __syncthreads();
  int need = STATS;
  if (round > 0 || !a.lazy) {
    if (had.need == REST) {
      if (threadIdx.x < 64) {
        const double *rest = a.rest + ((size_t)(round & 1) * a.st.seqs + s) * a.pieces;
        double left = 0.0;
        for (int k = threadIdx.x; k < a.pieces; k += 64) left += rest[k];
        left = wave_sum(left);
        if (threadIdx.x == 0) w.rest = left;
      }
    }
    take_rows<E, Q>(a, w, q, a.lazy && had.need == REST);
    need = walk_from<E, Q>(a, w, q, had.need == REST);
  }
  if (piece == 0) {
    const Tip tip = tip_of(w, q);
    write_rows(a, w, q, round == 0, need == END, tip);
    if (threadIdx.x == 0) {
      a.state[(size_t)(~round & 1) * a.st.seqs + s] = w.st;
      if (need == END) a.tip[s] = tip;
    }
  }
  if (need == STATS) {
    const int t = q.begin + w.st.at;
    piece_stats<E>(a, t, piece, q.fit ? q.heat : 1.0f, a.part + (size_t)t * a.pieces + piece);
  }
  if constexpr (DRAFT) {
    if (need == REST) {
      const int from = first_of<E>(row_of<E>(a, q.begin + w.st.at), piece, PIECE);
      constexpr int V = Vec<E>::N;
      const double sum = wave_sum(rest_of<E, Q>(a, w.st, q, from + (int)threadIdx.x * V, from + PIECE, ST * V));
      if ((threadIdx.x & 63) == 0) w.sums[threadIdx.x >> 6] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        double all = w.sums[0];
#pragma unroll
        for (int x = 1; x < ST / 64; ++x) all += w.sums[x];
        a.rest[((size_t)(~round & 1) * a.st.seqs + s) * a.pieces + piece] = all;
      }
    }
  }
}

// A row's statistics by one workgroup: each thread's own reference, moved once a sweep.
template <typename E, int N, bool DRAFT>
__device__ __forceinline__ void row_stats(const VerifyArgs &a, Walk<N, DRAFT> &w, const Seq &q) {
  constexpr int V = Vec<E>::N, U = 32 / V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char *row = row_of<E>(a, q.begin + w.st.at);
  constexpr int SWEEP = U * V * ALONE;
  float top = -INFINITY;
  double mass = 0.0;
  int best = INT32_MAX;
  for (int e0 = first_of<E>(row, 0, 0) + (int)threadIdx.x * V; e0 < a.vocab; e0 += SWEEP) {
    float x[U][V], now = top;
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<E>::unpack(block_of<E>(row, e0 + u * V * ALONE, a.vocab), x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) now = larger(now, x[u][k]);
    if (q.greedy) {
      if (now > top) {
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
#pragma unroll
          for (int k = V - 1; k >= 0; --k)
            if (x[u][k] == now) best = e0 + u * V * ALONE + k;
      }
    } else {
      const float ref = now == -INFINITY ? 0.0f : now;
      mass *= (double)__builtin_amdgcn_exp2f((top - ref) * q.rate);
#pragma unroll
      for (int u = 0; u < U * V / 8; ++u) {
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          y += __builtin_amdgcn_exp2f((x[(8 * u + k) / V][(8 * u + k) % V] - ref) * q.rate);
        mass += (double)y;
      }
    }
    top = now;
  }
  float all = top;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) all = larger(all, exl3::xor_lanes(all, m));
  if (lane == 0) w.tops[wave] = all;
  __syncthreads();
  for (int x = 0; x < ALONE / 64; ++x) all = larger(all, w.tops[x]);
  const float ref = all == -INFINITY ? 0.0f : all;
  mass = wave_sum(mass * (double)__builtin_amdgcn_exp2f((top - ref) * q.rate));
  best = top == all ? best : INT32_MAX;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) best = min(best, across(best, m));
  if (lane == 0) w.sums[wave] = mass, w.bests[wave] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int x = 1; x < ALONE / 64; ++x) mass += w.sums[x], best = min(best, w.bests[x]);
    enter(w.st, stats_of(q, all, best, mass));
  }
  __syncthreads();
}

// What the rounds have left of the walks, a workgroup a sequence: 10 to 13 us a row or a
// refusal at 152 thousand tokens, its exponentials.
template <typename E, typename Q, bool DRAFT>
__global__ __launch_bounds__(ALONE) void verify_alone_kernel(VerifyArgs a, int round) {
  __shared__ Walk<EXL3P_TREE_MAX, DRAFT> w;
  const int s = blockIdx.x;
  const Seq q = seq_of(a, s);
  const State had = a.state[(size_t)(round & 1) * a.st.seqs + s];
  if (q.n <= 0 || had.need == END) return;
  load_rows(a, w, q);
  if (threadIdx.x == 0) w.st = had;
  __syncthreads();
  // (the last round has formed the first row's parts)
  for (int need = had.need, first = 1; need != END; first = 0) {
    const bool joined = need == REST ? a.lazy : !first;
    if (need == STATS && !first) {
      row_stats<E>(a, w, q);
    } else if (DRAFT && need == REST) {
     if constexpr (DRAFT) {
      constexpr int V = Vec<E>::N;
      const int from = first_of<E>(row_of<E>(a, q.begin + w.st.at), 0, 0);
      const double sum = wave_sum(rest_of<E, Q>(a, w.st, q, from + (int)threadIdx.x * V, a.vocab, ALONE * V));
      if ((threadIdx.x & 63) == 0) w.sums[threadIdx.x >> 6] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        double all = w.sums[0];
        for (int x = 1; x < ALONE / 64; ++x) all += w.sums[x];
        w.rest = all;
      }
      __syncthreads();
     }
    }
    take_rows<E, Q>(a, w, q, joined);
    need = walk_from<E, Q>(a, w, q, need == REST);
    __syncthreads();  // all have read it
  }
  const Tip tip = tip_of(w, q);
  write_rows(a, w, q, false, true, tip);
  if (threadIdx.x == 0) a.tip[s] = tip;
}

// ------------------------------------------------------------------- sampling

// What p~ has left of a token, times the row's mass: exponents in 64 bits, since the
// cumulative sums lie next to u's border (f32 ones would give another token once in
// some thousand draws).
template <typename E, typename Q, bool DRAFT>
struct Rest {
  const VerifyArgs &a;
  Tip tip;
  double inv;
  size_t d;
  // of the workgroup: where no child was refused the draft's row is not read (nobody may have
  // filled it: a draft is not asked what follows its leaves)
  bool refused;
  __device__ __forceinline__ Rest(const VerifyArgs &args, const Tip &t)
      : a(args), tip(t), inv(1.0 / (double)t.heat), d((size_t)max(t.row, 0) * args.ds),
        refused(__builtin_amdgcn_readfirstlane(t.share != 0.0)) {}
  __device__ __forceinline__ int first(int piece) const {
    return first_of<E>(row_of<E>(a, max(tip.row, 0)), piece, DRAW);
  }
  // of p, and of p~, of the block at e; gone: bits of the piece that begins at `from`
  static constexpr int N = Vec<E>::N;
  __device__ __forceinline__ void of(int e, const uint32_t *gone, int from, double (&p)[N], double (&r)[N]) const {
    float x[N];
    Vec<E>::unpack(block_of<E>(row_of<E>(a, max(tip.row, 0)), e, a.vocab), x);
    float y[N];
    if constexpr (DRAFT)
      if (refused) drafts_of<Q, N>(static_cast<const typename Q::T *>(a.draft) + d, e, a.vocab, y);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      r[k] = p[k] = exp_of(((double)x[k] - (double)tip.top) * inv);
      if constexpr (!DRAFT)
        if (gone[(e + k - from) >> 5] >> ((e + k - from) & 31) & 1) r[k] = 0.0;
    }
    if constexpr (DRAFT)
      if (refused)
#pragma unroll
        for (int k = 0; k < N; ++k) r[k] = fmax(p[k] - tip.share * (double)y[k], 0.0);
  }
  // the tokens of the row's children, all refused
  __device__ __forceinline__ void mark(int s, int from, uint32_t *gone) const {
    if constexpr (!DRAFT) {
      for (int i = threadIdx.x; i < DRAW / 32; i += ST) gone[i] = 0;
      __syncthreads();
      const int begin = tip.row - tip.at;
      const int n = min(min(a.st.cu[s + 1], a.st.rows) - begin, min(a.st.max_rows, EXL3P_TREE_MAX));
      for (int i = tip.at + 1 + threadIdx.x; i < n; i += ST) {
        const int x = a.parent ? a.parent[begin + i] : i - 1;
        const int64_t e = (int64_t)a.ids[begin + i] - from;
        if (x == tip.at && e >= 0 && e < DRAW) atomicOr(&gone[e >> 5], 1u << (e & 31));
      }
      __syncthreads();
    }
  }
};

// Sum over the threads before this one; all threads', in `whole`.
__device__ __forceinline__ double before(double v, double (&waves)[ST / 64], double &whole) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double x = scan(v);
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  double base = 0.0;
  whole = 0.0;
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) {
    if (w < wave) base += waves[w];
    whole += waves[w];
  }
  return base + (x - v);
}
// The workgroup's least and largest.
__device__ __forceinline__ void ends(int &lo, int &hi, int (&waves)[2][ST / 64]) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) lo = min(lo, across(lo, m)), hi = max(hi, across(hi, m));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) waves[0][threadIdx.x >> 6] = lo, waves[1][threadIdx.x >> 6] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) lo = min(lo, waves[0][w]), hi = max(hi, waves[1][w]);
}

// The token that u says: the piece whose sum passes the border first, then the place in
// it.  sum_of(x, kind): piece x's sum; at(piece): its first element; of(e, kind, r): the
// block at e.  Kinds after the first stand in where all before them are 0 throughout.
template <int N, typename SUM, typename AT, typename OF>
__device__ __forceinline__ void choose(const VerifyArgs &a, int row, double u, int kinds, SUM &&sum_of, AT &&at,
                                       OF &&of) {
  __shared__ double waves[ST / 64], base;
  __shared__ int least[2][ST / 64];
  const int each = (a.draws + ST - 1) / ST, x0 = threadIdx.x * each, x1 = min(x0 + each, a.draws);
  double whole, run;
  int kind = 0;
  for (;; ++kind) {
    double own = 0.0;
    for (int x = x0; x < x1; ++x) own += sum_of(x, kind);
    run = before(own, waves, whole);
    if (whole > 0.0 || kind == kinds - 1) break;
  }
  const double border = u * whole;
  int found = INT32_MAX, last = -1;
  double under = 0.0;  // what lies before the piece found
  for (int x = x0; x < x1; ++x) {
    const double v = sum_of(x, kind);
    if (v > 0.0) {
      last = x;
      if (found == INT32_MAX && run + v > border) found = x, under = run;
    }
    run += v;
  }
  const int mine = found;
  ends(found, last, least);
  const bool passed = found != INT32_MAX;
  const int piece = passed ? found : max(last, 0);
  if (passed && mine == found) base = under;
  const int from = at(piece);
  __syncthreads();
  double r[DRAW / ST], own = 0.0;
#pragma unroll
  for (int k = 0; k < DRAW / ST / N; ++k) {
    double v[N];
    of(from + ((int)threadIdx.x * (DRAW / ST / N) + k) * N, kind, v);
#pragma unroll
    for (int i = 0; i < N; ++i) own += r[k * N + i] = v[i];
  }
  double sum;
  run = (passed ? base : -INFINITY) + before(own, waves, sum);
  found = INT32_MAX, last = -1;
#pragma unroll
  for (int k = 0; k < DRAW / ST; ++k) {
    run += r[k];
    const int e = from + (int)threadIdx.x * (DRAW / ST) + k;
    if (r[k] > 0.0) {
      last = e;
      if (found == INT32_MAX && run > border) found = e;
    }
  }
  ends(found, last, least);
  // (sums in another order may end a step short of the border: the last one then)
  if (threadIdx.x == 0) a.target[row] = found != INT32_MAX ? found : last;
}

// The sampling: sums of DRAW tokens a workgroup, and by the sequence's last one to
// arrive the token, the piece whose sum passes the border first, then the place in it.
// The sums go out and come in past the caches of an XCD (atomics of the device's scope), and
// a thread counts its piece once they are there: s_waitcnt says that of gfx950's stores, not the
// language of relaxed atomics.  A release and an acquire in its place write back and drop an
// XCD's whole L2, a workgroup each: 64 trees 91.8 us, not 60.9, 8 lines 20.0, not 18.6.
// OWN: the workgroups walk by themselves, all alike.
template <typename E, typename Q, bool DRAFT, bool OWN>
__global__ __launch_bounds__(ST) void verify_draw_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N;
  __shared__ Walk<OWN ? SHORT : 1, DRAFT> walked;
  __shared__ uint32_t gone[DRAW / 32];
  __shared__ double waves[ST / 64], whole_waves[ST / 64];
  __shared__ int order;
  const int s = blockIdx.x / a.draws, own_piece = blockIdx.x - s * a.draws;
  Tip tip;
  if constexpr (OWN) {
    const Seq q = seq_of(a, s);
    if (q.n <= 0) return;
    load_rows(a, walked, q);
    if (threadIdx.x == 0) walked.st = begun();
    __syncthreads();
    take_rows<E, Q>(a, walked, q, false);
    walk_from<E, Q>(a, walked, q, false);
    tip = tip_of(walked, q);
    if (own_piece == 0) write_rows(a, walked, q, true, true, tip);
  } else {
    tip = a.tip[s];
  }
  if (tip.row < 0) return;
  const Rest<E, Q, DRAFT> rest(a, tip);
  double *sums = a.sums + (size_t)s * a.draws * 2;
  {
    const int from = rest.first(own_piece);
    rest.mark(s, from, gone);
    double all = 0.0, left = 0.0;
#pragma unroll
    for (int k = 0; k < DRAW / ST / N; ++k) {
      double p[N], r[N];
      rest.of(from + (k * ST + (int)threadIdx.x) * N, gone, from, p, r);
#pragma unroll
      for (int i = 0; i < N; ++i) all += p[i], left += r[i];
    }
    all = wave_sum(all), left = wave_sum(left);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = left, whole_waves[threadIdx.x >> 6] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < ST / 64; ++w) left += waves[w], all += whole_waves[w];
      __hip_atomic_store(&sums[2 * own_piece], left, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&sums[2 * own_piece + 1], all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // both are there before the count
      order = __hip_atomic_fetch_add(&a.arrived[s], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (order != a.draws - 1) return;
  }
  // two kinds: where nothing is left of p~ (numbers that are none refused it), p in its place
  auto sum_of = [&](int x, int kind) {
    return __hip_atomic_load(&sums[2 * x + kind], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  int from = 0;
  auto at = [&](int piece) {
    from = rest.first(piece);
    rest.mark(s, from, gone);
    return from;
  };
  auto of = [&](int e, int kind, double (&v)[N]) {
    double p[N], left[N];
    rest.of(e, gone, from, p, left);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = kind == 1 ? p[i] : left[i];
  };
  choose<N>(a, tip.row, tip.u, 2, sum_of, at, of);
}

// A step of single rows has nothing to walk: each piece's largest logit and the sum of its
// powers below that one, in 64 bits at once, ...
template <typename E>
__global__ __launch_bounds__(ST) void verify_single_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N, U = DRAW / ST / N;
  __shared__ float tops[ST / 64];
  __shared__ double waves[ST / 64];
  const int s = blockIdx.x / a.draws, piece = blockIdx.x - s * a.draws;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Seq q = seq_of(a, s);
  if (q.n <= 0) return;
  const char *row = row_of<E>(a, q.begin);
  const int first = first_of<E>(row, piece, DRAW);
  float x[U][N];
#pragma unroll
  for (int k = 0; k < U; ++k)
    Vec<E>::unpack(block_of<E>(row, first + (k * ST + (int)threadIdx.x) * N, a.vocab), x[k]);
  float top = x[0][0];
#pragma unroll
  for (int k = 0; k < U; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) top = larger(top, x[k][i]);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = larger(top, exl3::xor_lanes(top, m));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) top = larger(top, tops[w]);
  // (greedy: minus the first place of it, the largest of which is looked for)
  double all = q.greedy ? -INFINITY : 0.0;
  if (q.greedy) {
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (x[k][i] == top) all = fmax(all, -(double)(first + (k * ST + (int)threadIdx.x) * N + i));
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) all = fmax(all, across(all, m));
  } else if (q.fit && top > -INFINITY && top < INFINITY) {
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) all += exp_of(((double)x[k][i] - (double)top) * q.inv);
    all = wave_sum(all);
  }
  if (lane == 0) waves[wave] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < ST / 64; ++w) all = q.greedy ? fmax(all, waves[w]) : all + waves[w];
    double *to = a.sums + ((size_t)s * a.draws + piece) * 2;
    to[0] = all, to[1] = (double)top;
  }
}
// ... and the token, a workgroup a sequence.
template <typename E>
__global__ __launch_bounds__(ST) void verify_single_draw_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N;
  __shared__ float tops[ST / 64];
  __shared__ int firsts[ST / 64];
  const int s = blockIdx.x;
  const Seq q = seq_of(a, s);
  if (q.n <= 0) return;
  const double *sums = a.sums + (size_t)s * a.draws * 2;
  float top = -INFINITY;
  for (int x = threadIdx.x; x < a.draws; x += ST) top = larger(top, (float)sums[2 * x + 1]);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = larger(top, exl3::xor_lanes(top, m));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) top = larger(top, tops[w]);
  if (!q.fit || !(top > -INFINITY) || (!q.greedy && top == INFINITY)) {
    if (threadIdx.x == 0) a.target[q.begin] = -1;
    return;
  }
  if (q.greedy) {
    int best = INT32_MAX;
    for (int x = threadIdx.x; x < a.draws; x += ST)
      if ((float)sums[2 * x + 1] == top) best = min(best, (int)-sums[2 * x]);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) best = min(best, across(best, m));
    if ((threadIdx.x & 63) == 0) firsts[threadIdx.x >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ST / 64; ++w) best = min(best, firsts[w]);
    if (threadIdx.x == 0) a.target[q.begin] = best;
    return;
  }
  const char *row = row_of<E>(a, q.begin);
  auto sum_of = [&](int x, int) { return sums[2 * x] * exp_of((sums[2 * x + 1] - (double)top) * q.inv); };
  auto at = [&](int piece) { return first_of<E>(row, piece, DRAW); };
  auto of = [&](int e, int, double (&v)[N]) {
    float x[N];
    Vec<E>::unpack(block_of<E>(row, e, a.vocab), x);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = exp_of(((double)x[k] - (double)top) * q.inv);
  };
  choose<N>(a, q.begin, a.u[q.begin], 1, sum_of, at, of);
}

// ------------------------------------------------------------------- host side

constexpr int VOCAB_MAX = 1 << 24;
// Needs of a walk that launches answer, behind a first round that forms the first: 2 us each where
// no walk has it, 10 to 13 us for the workgroup alone where one does.  4 trees of 24 rows of f16
// and 64 of 64 of bf16 (151936 tokens, before refusals that leave nothing were looked for):
// 36.6 and 65.5 us with 2, 40.7 and 61.8 with 4, 44.9 and 66.3 with 6.
constexpr int ROUNDS = 4;
constexpr int64_t LAZY = 1 << 25;  // bytes of logits

int pieces_of(int32_t vocab) { return (vocab + 7 + PIECE - 1) / PIECE; }
int draws_of(int32_t vocab) { return (vocab + 7 + DRAW - 1) / DRAW; }
size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }

exl3_verdict check_step(const exl3p_rows *r) {
  exl3p_cache any{};
  any.seqs = INT32_MAX;
  return check_rows(&any, r);
}

int size_of(int32_t dtype) {
  return dtype == EXL3_DT_F32 ? 4 : dtype == EXL3_DT_F16 || dtype == EXL3_DT_BF16 ? 2 : 0;
}

template <typename F>
void by_dtype(int32_t dtype, F &&f) {
  if (dtype == EXL3_DT_F32)
    f(F32{});
  else if (dtype == EXL3_DT_F16)
    f(F16{});
  else
    f(BF16{});
}

exl3_verdict check_probabilities(const void *p, int32_t dtype, int64_t stride, int32_t vocab) {
  const int size = size_of(dtype);
  if (size == 0)
    return refuse(EXL3_UNSUPPORTED, "PagedVerifyDtype: float32, float16 or bfloat16");
  if (!aligned(p, size))
    return refuse(EXL3_UNSUPPORTED, "PagedVerifyAlignment: elements on their own boundaries");
  if (stride < vocab) return refuse(EXL3_UNSUPPORTED, "PagedMatrixStride: rows overlap");
  return OK;
}

// Where the scratch's arrays lie: parts, states, rests, tips, sums, counters; its size.
size_t places(const exl3p_rows *r, int32_t vocab, size_t (&at)[6]) {
  const size_t seqs = r->seqs, pieces = pieces_of(vocab);
  const size_t bytes[6] = {(size_t)r->rows * pieces * sizeof(Part), 2 * seqs * sizeof(State),
                           2 * seqs * pieces * sizeof(double),      seqs * sizeof(Tip),
                           seqs * draws_of(vocab) * 2 * sizeof(double), seqs * sizeof(int)};
  size_t end = 0;
  for (int i = 0; i < 6; ++i) at[i] = end, end += up16(bytes[i]);
  return end;
}

}  // namespace

extern "C" {

size_t exl3p_verify_scratch_bytes(const exl3p_rows *r, int32_t vocab) {
  if (check_step(r).code != EXL3_OK || vocab <= 0 || vocab > VOCAB_MAX) return 0;
  size_t at[6];
  return places(r, vocab, at);
}

exl3_verdict exl3p_verify(const exl3p_rows *r, const int32_t *parent, const int32_t *ids,
                          int32_t vocab, const void *logits, int32_t logits_dtype,
                          int64_t logits_stride, const void *draft, int32_t draft_dtype,
                          int64_t draft_stride, int32_t distinct, const float *temperature,
                          const double *u, int32_t *target, void *scratch, size_t scratch_bytes,
                          exl3_stream s) {
  EXL3P_TRY(check_step(r));
  if (r->max_rows > EXL3P_TREE_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedTree: over 1024 rows of a sequence");
  if (vocab <= 0) return refuse(EXL3_UNSUPPORTED, "PagedVerifyVocab: tokens above 0");
  if (vocab > VOCAB_MAX) return refuse(EXL3_TOO_LARGE, "PagedVerifyVocab: over 2^24 tokens");
  EXL3P_TRY(check_probabilities(logits, logits_dtype, logits_stride, vocab));
  if (draft != nullptr) EXL3P_TRY(check_probabilities(draft, draft_dtype, draft_stride, vocab));
  if (r->rows == 0 || r->seqs == 0 || r->max_rows == 0) return OK;
  if (ids == nullptr || logits == nullptr || u == nullptr || target == nullptr)
    return refuse(EXL3_FAILED, "PagedVerify: a missing array");
  if (!aligned(u, 8))
    return refuse(EXL3_UNSUPPORTED, "PagedVerifyAlignment: elements on their own boundaries");
  const int pieces = pieces_of(vocab), draws = draws_of(vocab);
  if ((int64_t)r->rows * pieces > GRID_MAX || (int64_t)r->seqs * draws > GRID_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedVerify: too many rows and tokens for one call");
  const size_t need = exl3p_verify_scratch_bytes(r, vocab);
  if (scratch == nullptr || !aligned(scratch, 16) || scratch_bytes < need)
    return refuse(EXL3_FAILED, "PagedScratch: below exl3p_verify_scratch_bytes, or not aligned");
  const int64_t n = (int64_t)r->rows * 4;
  auto rows_of = [&](const void *p, int64_t stride, int32_t dtype) {
    return Span2D{p, p == nullptr ? 0 : r->rows, (int64_t)vocab * size_of(dtype), stride * size_of(dtype)};
  };
  EXL3P_TRY(check_apart({array(target, n), array(scratch, (int64_t)need)},
                        {array(r->cu, 4 * ((int64_t)r->seqs + 1)), array(parent, n), array(ids, n),
                         array(temperature, 4 * (int64_t)r->seqs), array(u, 2 * n),
                         rows_of(logits, logits_stride, logits_dtype),
                         rows_of(draft, draft_stride, draft_dtype)}));
  VerifyArgs a;
  a.logits = logits, a.ls = logits_stride, a.draft = draft, a.ds = draft_stride;
  a.st = step_of(r), a.vocab = vocab, a.pieces = pieces, a.draws = draws;
  a.parent = parent, a.ids = ids, a.temperature = temperature, a.u = u, a.target = target;
  a.distinct = distinct != 0;
  size_t at[6];
  places(r, vocab, at);
  char *const base = static_cast<char *>(scratch);
  a.part = reinterpret_cast<Part *>(base + at[0]);
  a.state = reinterpret_cast<State *>(base + at[1]);
  a.rest = reinterpret_cast<double *>(base + at[2]);
  a.tip = reinterpret_cast<Tip *>(base + at[3]);
  a.sums = reinterpret_cast<double *>(base + at[4]);
  a.arrived = reinterpret_cast<int *>(base + at[5]);
  const hipStream_t st = static_cast<hipStream_t>(s);
  // a refusal with a drafted sibling left wants a sum over the vocabulary
  const bool siblings = draft != nullptr && parent != nullptr && r->max_rows > 2;
  // Statistics when a walk gets there: of a tree, most of whose rows no walk gets to (a
  // line's are drafted to be accepted), where all rows' would take longer than the rounds
  // of the walks.  All and as the walks go, ragged batches, 151936 tokens where no other number
  // is given: 16 trees of up to 16 rows (bf16, 53 MB of logits) 26.5 and 35.9 us, 64 of 64
  // (32000 tokens, 139 MB) 46.8 and 44.7, 64 of 16 (167 MB) 60.3 and 59.3, 64 of 24 (259 MB) 74.7 and
  // 56.6, 16 of 64 (f32, 314 MB) 77.9 and 43.0.  Siblings that were drawn need rounds in any
  // case: 32 of 16 (88 MB) 66 and 83, 64 of 16 91 and 106, 12 of 64 (f32, 237 MB) 95.7 and
  // 99.8, 64 of 32 (355 MB) 138 and 134, 32 of 64 (f32, 589 MB) 167 and 122.  Lines that are
  // accepted whole lose: 64 of 8 (102 MB) 50.6 and 57.0.
  const int64_t read = (int64_t)r->rows * vocab * size_of(logits_dtype);
  const bool lazy = parent != nullptr && r->rows >= 4 * (int64_t)r->seqs && read > (siblings ? 8 : 5) * LAZY;
  const bool own = !lazy && !siblings && r->max_rows <= SHORT;
  a.lazy = lazy;
  // rounds: what walks usually need; the rest is for one workgroup a sequence
  const int needs = (lazy ? r->max_rows : 0) + (siblings ? r->max_rows - 2 : 0);
  const int rounds = needs < ROUNDS ? needs : ROUNDS;
  const dim3 all((unsigned)(r->seqs * draws)), each((unsigned)(r->seqs * pieces));
  auto after = [&](auto e, auto q, auto drafted) {
    typedef decltype(e) E;
    typedef decltype(q) Q;
    constexpr bool D = decltype(drafted)::value;
    if (own) {
      hipLaunchKernelGGL((verify_draw_kernel<E, Q, D, true>), all, dim3(ST), 0, st, a);
      return;
    }
    for (int k = 0; k <= rounds; ++k) {
      if (r->max_rows <= MIDDLE)
        hipLaunchKernelGGL((verify_round_kernel<E, Q, D, MIDDLE>), each, dim3(ST), 0, st, a, k);
      else
        hipLaunchKernelGGL((verify_round_kernel<E, Q, D, EXL3P_TREE_MAX>), each, dim3(ST), 0, st, a, k);
    }
    if (needs > rounds)
      hipLaunchKernelGGL((verify_alone_kernel<E, Q, D>), dim3(r->seqs), dim3(ALONE), 0, st, a, rounds + 1);
    hipLaunchKernelGGL((verify_draw_kernel<E, Q, D, false>), all, dim3(ST), 0, st, a);
  };
  by_dtype(logits_dtype, [&](auto e) {
    if (r->max_rows == 1) {
      hipLaunchKernelGGL((verify_single_kernel<decltype(e)>), all, dim3(ST), 0, st, a);
      hipLaunchKernelGGL((verify_single_draw_kernel<decltype(e)>), dim3(r->seqs), dim3(ST), 0, st, a);
      return;
    }
    if (!lazy)
      hipLaunchKernelGGL((verify_stats_kernel<decltype(e)>), dim3((unsigned)(r->rows * pieces)), dim3(ST), 0,
                         st, a);
    if (draft == nullptr)
      after(e, e, std::false_type{});
    else
      by_dtype(draft_dtype, [&](auto q) { after(e, q, std::true_type{}); });
  });
  return launched();
}

}  // extern "C"
