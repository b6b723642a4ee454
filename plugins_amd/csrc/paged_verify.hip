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
template <typename E>
__device__ __forceinline__ float one_of(const void *p, size_t i) {
  return (float)static_cast<const typename E::T *>(p)[i];
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr int ST = 256;       // threads of a statistics or sampling workgroup,
constexpr int PIECE = 8192;   // elements of a row that the first takes,
constexpr int DRAW = 4096;    // and the second
constexpr int WALK = 1024;    // the most threads of a walk
constexpr int SHORT = 32;     // rows of a sequence that the sampling walks by itself

// A piece's largest logit, the first place of it, and the sum of its weights
// 2^((logit - top) log2(e) / T).
struct Part {
  float top;
  int32_t best;
  double mass;
};

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
  Part *part;     // [rows][pieces]
  Tip *tip;       // [seqs]
  double *sums;   // [seqs][draws][2]: of what p has left, of p
  int *arrived;   // [seqs]: sampling workgroups that are done
};

// A temperature's factor of the logits, in powers of two, f32's largest at most.
__device__ __forceinline__ float rate_of(float heat) {
  return fminf(LOG2E / heat, 3.0e38f);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// ------------------------------------------------------------ rows' statistics

// A workgroup takes PIECE logits of a row into registers: the largest, then the
// weights' sum (f32 over 8 of a thread, 64 bits beyond).  Bound by bytes.  ROOTS:
// each sequence's first row alone.
template <typename E, bool ROOTS>
__global__ __launch_bounds__(ST) void verify_stats_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N, U = PIECE / ST / N;
  __shared__ float tops[ST / 64];
  __shared__ double masses[ST / 64];
  __shared__ int bests[ST / 64];
  const int item = blockIdx.x / a.pieces, piece = blockIdx.x - item * a.pieces;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int t = item, s = 0;
  if (ROOTS) {
    s = item, t = max(a.st.cu[s], 0);
    if (t >= min(a.st.cu[s + 1], a.st.rows)) return;
  } else {  // the row's sequence: how many end at it or before
    for (int s0 = 0; s0 < a.st.seqs; s0 += 64)
      s += __popcll(__ballot(s0 + lane < a.st.seqs && a.st.cu[min(s0 + lane, a.st.seqs - 1) + 1] <= t));
    if (s >= a.st.seqs) return;
  }
  if (piece == 0 && threadIdx.x == 0 && t == max(a.st.cu[s], 0)) a.arrived[s] = 0;
  const char *row = static_cast<const char *>(a.logits) + (int64_t)t * a.ls * sizeof(typename E::T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
  const int first = piece * PIECE - off;  // the first block's first element
  float x[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
    Vec<E>::unpack(block_of<E>(row, first + (u * ST + (int)threadIdx.x) * N, a.vocab), x[u]);
  float top = x[0][0];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) top = __builtin_elementwise_maximum(top, x[u][i]);  // NaN stays
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = __builtin_elementwise_maximum(top, exl3::xor_lanes(top, m));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) top = __builtin_elementwise_maximum(top, tops[w]);
  const float heat = a.temperature ? a.temperature[s] : 1.0f;
  Part *part = a.part + (size_t)item * a.pieces + piece;
  if (heat == 0.0f) {  // the first place of the largest is what counts
    int best = a.vocab;
#pragma unroll
    for (int u = U - 1; u >= 0; --u)
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (x[u][i] == top) best = first + (u * ST + (int)threadIdx.x) * N + i;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) best = min(best, __shfl_xor(best, m));
    if (lane == 0) bests[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < ST / 64; ++w) best = min(best, bests[w]);
      *part = Part{top, best, 0.0};
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
    *part = Part{top, 0, mass};
  }
}

// ------------------------------------------------------------------- the walk

// A wave's sequences of a walk in LDS: N rows at most.
template <int N, bool DRAFT>
struct Walk {
  double mass[N], p[N], us[N];  // mass -1: a row without a distribution
  float q[DRAFT ? N : 1], top[N];
  int up[N], tok[N], best[N], next[N];
  double left, drawn, share, sums[WALK / 64];
  float tops[WALK / 64];
  int bests[WALK / 64];
  int at, seen, more;
};
enum More { DONE, REST, ROW };  // a walk's next: nothing, what p~ has left, a row's statistics

// A row's statistics by one workgroup, for walks that look only at the rows on
// their way: each thread's own reference, moved once a sweep.
template <typename E, int N, bool DRAFT>
__device__ __forceinline__ void row_stats(const VerifyArgs &a, Walk<N, DRAFT> &w, int t, int i, float heat) {
  constexpr int V = Vec<E>::N, U = 32 / V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / 64;
  const float rate = rate_of(heat);
  const char *row = static_cast<const char *>(a.logits) + (int64_t)t * a.ls * sizeof(typename E::T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
  const int sweep = U * V * (int)blockDim.x;
  float top = -INFINITY;
  double mass = 0.0;
  int best = INT32_MAX;
  u32x4 raw[U];
  auto fetch = [&](int e0) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = block_of<E>(row, e0 + u * V * (int)blockDim.x, a.vocab);
  };
  int e0 = (int)threadIdx.x * V - off;
  fetch(e0);
  for (; e0 < a.vocab; e0 += sweep) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<E>::unpack(raw[u], x[u]);
    fetch(e0 + sweep);  // (-inf behind the last)
    float now = top;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) now = __builtin_elementwise_maximum(now, x[u][k]);
    if (heat == 0.0f) {
      if (now > top) {
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
#pragma unroll
          for (int k = V - 1; k >= 0; --k)
            if (x[u][k] == now) best = e0 + u * V * (int)blockDim.x + k;
      }
    } else {
      const float ref = now == -INFINITY ? 0.0f : now;
      mass *= (double)__builtin_amdgcn_exp2f((top - ref) * rate);
#pragma unroll
      for (int u = 0; u < U * V / 8; ++u) {
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          y += __builtin_amdgcn_exp2f((x[(8 * u + k) / V][(8 * u + k) % V] - ref) * rate);
        mass += (double)y;
      }
    }
    top = now;
  }
  float all = top;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) all = __builtin_elementwise_maximum(all, exl3::xor_lanes(all, m));
  if (lane == 0) w.tops[wave] = all;
  __syncthreads();
  for (int x = 0; x < waves; ++x) all = __builtin_elementwise_maximum(all, w.tops[x]);
  const float ref = all == -INFINITY ? 0.0f : all;
  mass = wave_sum(mass * (double)__builtin_amdgcn_exp2f((top - ref) * rate));
  best = top == all ? best : INT32_MAX;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) best = min(best, __shfl_xor(best, m));
  if (lane == 0) w.sums[wave] = mass, w.bests[wave] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int x = 1; x < waves; ++x) mass += w.sums[x], best = min(best, w.bests[x]);
    const bool whole = heat == 0.0f ? all > -INFINITY : all > -INFINITY && all < INFINITY && mass > 0.0 && mass < INFINITY;
    w.top[i] = all, w.best[i] = best, w.mass[i] = !whole ? -1.0 : heat == 0.0f ? 1.0 : mass;
  }
  __syncthreads();
}

// A sequence's walk, by a workgroup.  Each row's pieces are joined, or (LAZY) a
// row's logits looked at when the walk gets there; the tokens of rows get their
// probabilities under their parents, all at once; then one wave walks: the
// next child of a row is found among 64 rows a ballot.  Where a drafted sibling is
// left after a refusal, all threads sum max(p - share q, 0).
//
// The refused tokens' probabilities, q given: p~ after refusals is max(p -
// share q, 0), share the sum of A_j / B_j over the refusals, A_j the sum of p~
// and B_j that of q~ (1, or what the refused ones leave of it).  A refused token
// has none left: u A_j / B_j q >= p~ says that p~ is below what is taken.
template <typename E, typename Q, bool DRAFT, bool LAZY, int N>
__device__ __forceinline__ Tip walk(const VerifyArgs &a, Walk<N, DRAFT> &w, int s, bool writes) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int begin = min(max(a.st.cu[s], 0), a.st.rows), end = min(max(a.st.cu[s + 1], begin), a.st.rows);
  const int n = min(end - begin, min(a.st.max_rows, N));
  Tip tip{-1, 0, 0.0f, 1.0f, 0.0, 0.0};
  if (n <= 0) return tip;
  const float heat = a.temperature ? a.temperature[s] : 1.0f;
  const bool fit = heat >= 0.0f && heat < INFINITY, greedy = heat == 0.0f;
  const float rate = rate_of(heat);
  const double inv = 1.0 / (double)heat;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int t = begin + i;
    const int x = a.parent ? a.parent[t] : i - 1;
    w.up[i] = x >= 0 && x < i ? x : -1;
    w.tok[i] = a.ids[t];
    w.us[i] = a.u[t];
    w.p[i] = 0.0;
    if constexpr (DRAFT) w.q[i] = 0.0f;
    w.next[i] = -1;
  }
  // their statistics; of lazy walks only the first row's are there: 16 lanes a row
  {
    const int g = threadIdx.x & 15;
    for (int i = threadIdx.x >> 4; i < (LAZY ? 1 : n); i += blockDim.x / 16) {
      const Part *part = a.part + (size_t)(LAZY ? s : begin + i) * a.pieces;
      float hi = -INFINITY;
      int best = INT32_MAX;
      double m = 0.0;
      for (int k = g; k < a.pieces; k += 16) {
        const Part y = part[k];
        if (greedy) {
          if (y.top > hi) best = y.best;
          hi = __builtin_elementwise_maximum(hi, y.top);
        } else {
          const float now = __builtin_elementwise_maximum(hi, y.top), ref = now == -INFINITY ? 0.0f : now;
          m = m * (double)__builtin_amdgcn_exp2f((hi - ref) * rate) +
              y.mass * (double)__builtin_amdgcn_exp2f((y.top - ref) * rate);
          hi = now;
        }
      }
      float all = hi;
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) all = __builtin_elementwise_maximum(all, __shfl_xor(all, x, 16));
      const float ref = all == -INFINITY ? 0.0f : all;
      m *= (double)__builtin_amdgcn_exp2f((hi - ref) * rate);
      best = hi == all ? best : INT32_MAX;
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) m += __shfl_xor(m, x, 16), best = min(best, __shfl_xor(best, x, 16));
      if (g == 0) {
        const bool whole = fit && (greedy ? all > -INFINITY : all > -INFINITY && all < INFINITY && m > 0.0 && m < INFINITY);
        w.top[i] = all, w.best[i] = best, w.mass[i] = !whole ? -1.0 : greedy ? 1.0 : m;
      }
    }
  }
  if (threadIdx.x == 0) {
    w.at = 0, w.seen = 0, w.left = 1.0, w.drawn = 1.0, w.share = 0.0, w.more = ROW;
  }
  __syncthreads();
  // the children of `of` (-1: of any row) get their probabilities
  auto weigh_children = [&](int of) {
    for (int i = threadIdx.x + 1; i < n; i += blockDim.x) {
      const int j = w.up[i];
      if (j < 0 || (of >= 0 && j != of) || greedy || !(w.mass[j] > 0.0) || (uint32_t)w.tok[i] >= (uint32_t)a.vocab)
        continue;
      w.p[i] = exp(((double)one_of<E>(a.logits, (int64_t)(begin + j) * a.ls + w.tok[i]) - (double)w.top[j]) * inv) / w.mass[j];
      if constexpr (DRAFT) w.q[i] = one_of<Q>(a.draft, (int64_t)(begin + j) * a.ds + w.tok[i]);
    }
    __syncthreads();
  };
  int what = w.more;  // read between barriers: one wave writes it
  weigh_children(LAZY ? 0 : -1);
  while (what != DONE) {
    if (LAZY && what == ROW && w.at > 0) {
      row_stats<E>(a, w, begin + w.at, w.at, heat);
      weigh_children(w.at);
    }
    if (wave == 0) {
      // the next child of `row` behind row `from`
      auto next = [&](int row, int from) {
        for (int b = (from + 1) & ~63; b < n; b += 64) {
          const int i = b + lane;
          const uint64_t f = __ballot(i > from && i < n && w.up[min(i, n - 1)] == row);
          if (f != 0) return b + __builtin_ctzll(f);
        }
        return n;
      };
      int row = w.at, from = w.seen, then = DONE;
      double A = w.left, B = w.drawn, L = w.share;
      int c = w.mass[row] >= 0.0 ? next(row, from) : n;
      while (c < n) {
        bool hit;
        double less = 0.0, step = 0.0;
        if (greedy) {
          hit = w.tok[c] == w.best[row];
        } else if constexpr (DRAFT) {
          step = A / fmax(B, 0x1p-53);
          hit = w.us[c] * step * (double)w.q[c] < fmax(w.p[c] - L * (double)w.q[c], 0.0);
        } else {
          // a token that a sibling before it had is not there any more
          less = w.p[c];
          for (int b = 0; b < c; b += 64) {
            const int i = b + lane;
            if (__ballot(i > 0 && i < c && w.up[i] == row && w.tok[i] == w.tok[c]) != 0) less = 0.0;
          }
          hit = w.us[c] * A < less;
        }
        from = c;
        if (hit) {
          if (lane == 0) w.next[row] = w.tok[c];
          row = c, A = 1.0, B = 1.0, L = 0.0;
          if (LAZY) {
            then = ROW;
            break;
          }
          c = w.mass[row] >= 0.0 ? next(row, from) : n;
          continue;
        }
        c = next(row, from);
        if (greedy) continue;
        if constexpr (DRAFT) {
          L += step;
          if (a.distinct) B -= (double)w.q[from];
          if (c < n) {
            then = REST;
            break;
          }
        } else {
          A -= less;
        }
      }
      if (lane == 0) w.at = row, w.seen = from, w.more = then, w.left = A, w.drawn = B, w.share = L;
    }
    __syncthreads();
    what = w.more;
    if constexpr (DRAFT) {
      if (what == REST) {  // what p~ has left
        const int row = w.at;
        const float hi = w.top[row], by = (float)(1.0 / w.mass[row]), lost = (float)w.share;
        const size_t z = (size_t)(begin + row) * a.ls, d = (size_t)(begin + row) * a.ds;
        double sum = 0.0;
        for (int e0 = threadIdx.x; e0 < a.vocab; e0 += 16 * blockDim.x) {
          float x[16], y[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int e = e0 + k * blockDim.x;
            x[k] = -INFINITY, y[k] = 0.0f;
            if (e < a.vocab) x[k] = one_of<E>(a.logits, z + e), y[k] = one_of<Q>(a.draft, d + e);
          }
          float v = 0.0f;
#pragma unroll
          for (int k = 0; k < 16; ++k)
            v += fmaxf(__builtin_amdgcn_exp2f((x[k] - hi) * rate) * by - lost * y[k], 0.0f);
          sum += (double)v;
        }
        sum = wave_sum(sum);
        if (lane == 0) w.sums[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
          for (int x = 1; x < (int)blockDim.x / 64; ++x) sum += w.sums[x];
          w.left = sum;
        }
        __syncthreads();
      }
    }
  }
  const int row = w.at;
  const bool whole = w.mass[row] >= 0.0;
  tip.at = row;
  if (whole && !greedy) tip = Tip{begin + row, row, w.top[row], heat, w.share * w.mass[row], w.us[0]};
  // (the last row's is another workgroup's to write where it is sampled)
  if (writes)
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      if (i != row || tip.row < 0) a.target[begin + i] = i == row && whole ? w.best[row] : w.next[i];
  return tip;
}

template <typename E, typename Q, bool DRAFT, bool LAZY>
__global__ __launch_bounds__(WALK) void verify_walk_kernel(VerifyArgs a) {
  __shared__ Walk<EXL3P_TREE_MAX, DRAFT> w;
  const Tip tip = walk<E, Q, DRAFT, LAZY>(a, w, blockIdx.x, true);
  if (threadIdx.x == 0) a.tip[blockIdx.x] = tip, a.arrived[blockIdx.x] = 0;
}

// ------------------------------------------------------------------- sampling

// e^x for x <= 0 in 64 bits: a power of two times the series of e^f, |f| <= ln(2) / 2,
// whose 14th term is below 2^-57 of the sum.
__device__ __forceinline__ double exp_of(double x) {
  if (!(x > -746.0)) return x != x ? x : 0.0;  // below the smallest number
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
  return __builtin_amdgcn_ldexp(y, (int)n);
}

// What p~ has left of a token, times the row's mass: exponents in 64 bits, since the
// cumulative sums lie next to u's border (f32 ones would give another token once in
// some thousand draws).
template <typename E, typename Q, bool DRAFT>
struct Rest {
  const VerifyArgs &a;
  Tip tip;
  double inv;
  size_t z, d;
  __device__ __forceinline__ Rest(const VerifyArgs &args, const Tip &t)
      : a(args), tip(t), inv(1.0 / (double)t.heat), z((size_t)max(t.row, 0) * args.ls),
        d((size_t)max(t.row, 0) * args.ds) {}
  // the first element of a piece: its blocks of 16 bytes lie on their boundaries
  __device__ __forceinline__ int first(int piece) const {
    const char *row = static_cast<const char *>(a.logits) + z * sizeof(typename E::T);
    return piece * DRAW - (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
  }
  // of p, and of p~, of the block at e; gone: bits of the piece that begins at `from`
  static constexpr int N = Vec<E>::N;
  __device__ __forceinline__ void of(int e, const uint32_t *gone, int from, double (&p)[N], double (&r)[N]) const {
    float x[N];
    Vec<E>::unpack(block_of<E>(static_cast<const char *>(a.logits) + z * sizeof(typename E::T), e, a.vocab), x);
    float y[N];
    if constexpr (DRAFT) {
      typedef typename Q::T T;
      const T *q = static_cast<const T *>(a.draft) + d;
      if (e >= 0 && e + N <= a.vocab) {
        T t[N];
        __builtin_memcpy(t, q + e, sizeof(t));
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = (float)t[k];
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = e + k >= 0 && e + k < a.vocab ? (float)q[e + k] : 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      r[k] = p[k] = exp_of(((double)x[k] - (double)tip.top) * inv);
      if constexpr (DRAFT)
        r[k] = fmax(p[k] - tip.share * (double)y[k], 0.0);
      else if (gone[(e + k - from) >> 5] >> ((e + k - from) & 31) & 1)
        r[k] = 0.0;
    }
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
  double x = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
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
  for (int m = 1; m < 64; m <<= 1) lo = min(lo, __shfl_xor(lo, m)), hi = max(hi, __shfl_xor(hi, m));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) waves[0][threadIdx.x >> 6] = lo, waves[1][threadIdx.x >> 6] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) lo = min(lo, waves[0][w]), hi = max(hi, waves[1][w]);
}

// The sampling: sums of DRAW tokens a workgroup, and by the sequence's last one to
// arrive the token, the piece whose sum passes the border first, then the place in it.
// The sums go out and come in past the caches of an XCD.  OWN: the
// workgroups walk by themselves, all alike.
template <typename E, typename Q, bool DRAFT, bool OWN>
__global__ __launch_bounds__(ST) void verify_draw_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N;
  __shared__ Walk<OWN ? SHORT : 1, DRAFT> walked;
  __shared__ uint32_t gone[DRAW / 32];
  __shared__ double waves[ST / 64], whole_waves[ST / 64], base;
  __shared__ int least[2][ST / 64], order;
  const int s = blockIdx.x / a.draws, own_piece = blockIdx.x - s * a.draws;
  Tip tip;
  if constexpr (OWN)
    tip = walk<E, Q, DRAFT, false>(a, walked, s, own_piece == 0);
  else
    tip = a.tip[s];
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
  const int each = (a.draws + ST - 1) / ST, x0 = threadIdx.x * each, x1 = min(x0 + each, a.draws);
  auto sum_of = [&](int x, int kind) {
    return __hip_atomic_load(&sums[2 * x + kind], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  double whole, run;
  int kind = 0;  // 1: nothing is left of p~ (by rounding), p in its place
  for (;; kind = 1) {
    double own = 0.0;
    for (int x = x0; x < x1; ++x) own += sum_of(x, kind);
    run = before(own, waves, whole);
    if (whole > 0.0 || kind == 1) break;
  }
  const double border = tip.u * whole;
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
  const int piece = passed ? found : max(last, 0), from = rest.first(piece);
  if (passed && mine == found) base = under;
  rest.mark(s, from, gone);
  __syncthreads();
  double r[DRAW / ST], own = 0.0;
#pragma unroll
  for (int k = 0; k < DRAW / ST / N; ++k) {
    double p[N], left[N];
    rest.of(from + ((int)threadIdx.x * (DRAW / ST / N) + k) * N, gone, from, p, left);
#pragma unroll
    for (int i = 0; i < N; ++i) own += r[k * N + i] = kind == 1 ? p[i] : left[i];
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
  if (threadIdx.x == 0) a.target[tip.row] = found != INT32_MAX ? found : last;
}

// ------------------------------------------------------------------- host side

constexpr int VOCAB_MAX = 1 << 24;

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

}  // namespace

extern "C" {

size_t exl3p_verify_scratch_bytes(const exl3p_rows *r, int32_t vocab) {
  if (check_step(r).code != EXL3_OK || vocab <= 0 || vocab > VOCAB_MAX) return 0;
  return up16((size_t)r->rows * pieces_of(vocab) * sizeof(Part)) + up16((size_t)r->seqs * sizeof(Tip)) +
         (size_t)r->seqs * draws_of(vocab) * 2 * sizeof(double) + (size_t)r->seqs * sizeof(int);
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
  char *at = static_cast<char *>(scratch);
  a.part = reinterpret_cast<Part *>(at);
  at += up16((size_t)r->rows * pieces * sizeof(Part));
  a.tip = reinterpret_cast<Tip *>(at);
  at += up16((size_t)r->seqs * sizeof(Tip));
  a.sums = reinterpret_cast<double *>(at);
  a.arrived = reinterpret_cast<int *>(a.sums + (size_t)r->seqs * draws * 2);
  const hipStream_t st = static_cast<hipStream_t>(s);
  // rows that drafted siblings may follow: sums over the vocabulary within the walk
  const bool siblings = draft != nullptr && parent != nullptr;
  const bool lazy = r->rows > 500 && r->rows >= 4 * (int64_t)r->seqs;
  const bool own = !lazy && !siblings && r->max_rows <= SHORT;
  const dim3 all((unsigned)(r->seqs * draws));
  auto after = [&](auto e, auto q, auto drafted) {
    typedef decltype(e) E;
    typedef decltype(q) Q;
    constexpr bool D = decltype(drafted)::value;
    if (own) {
      hipLaunchKernelGGL((verify_draw_kernel<E, Q, D, true>), all, dim3(ST), 0, st, a);
      return;
    }
    if (lazy)
      hipLaunchKernelGGL((verify_walk_kernel<E, Q, D, true>), dim3(r->seqs), dim3(WALK), 0, st, a);
    else  // the sums after a refusal want many threads, the walk itself few
      hipLaunchKernelGGL((verify_walk_kernel<E, Q, D, false>), dim3(r->seqs), dim3(siblings ? WALK : ST), 0,
                         st, a);
    hipLaunchKernelGGL((verify_draw_kernel<E, Q, D, false>), all, dim3(ST), 0, st, a);
  };
  by_dtype(logits_dtype, [&](auto e) {
    if (!lazy)
      hipLaunchKernelGGL((verify_stats_kernel<decltype(e), false>), dim3((unsigned)(r->rows * pieces)),
                         dim3(ST), 0, st, a);
    else
      hipLaunchKernelGGL((verify_stats_kernel<decltype(e), true>), dim3((unsigned)(r->seqs * pieces)),
                         dim3(ST), 0, st, a);
    if (draft == nullptr)
      after(e, e, std::false_type{});
    else
      by_dtype(draft_dtype, [&](auto q) { after(e, q, std::true_type{}); });
  });
  return launched();
}

}  // extern "C"
