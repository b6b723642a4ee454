// paged_verify.hip -- sampled verification of drafted rows (exl3p_verify in
// include/exl3_paged.h) for MI355X (gfx950, wave64): the rows' softmax
// statistics, the walk down each sequence's tree, and the token sampled where it
// ends.
#include "paged_common.h"

namespace {

struct F32 {
  typedef float T;
};

// Elements of 16 bytes of a row as floats.
template <typename E>
struct Vec {
  static constexpr int N = 16 / sizeof(typename E::T);
  static __device__ __forceinline__ void unpack(u32x4 raw, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(typename E::T) == 4) {
        x[i] = __builtin_bit_cast(float, raw[i]);
      } else {
        x[2 * i] = to_f32<E>(raw[i] & 0xFFFFu);
        x[2 * i + 1] = to_f32<E>(raw[i] >> 16);
      }
    }
  }
};
template <typename E>
__device__ __forceinline__ float one_of(const void *p, size_t i) {
  return (float)static_cast<const typename E::T *>(p)[i];
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr int ST = 256;       // threads of a statistics workgroup,
constexpr int PIECE = 8192;   // elements of a row that it takes,
constexpr int DRAW = 2048;    // and that a workgroup of the sampling sums takes
constexpr int WALK = 1024;    // the most threads of a walk

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
  Part *part;    // [rows][pieces]
  Tip *tip;      // [seqs]
  double *sums;  // [seqs][draws][2]: of what p has left, of p
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
// weights' sum (f32 over 8 of a thread, 64 bits beyond).  Bound by bytes.
template <typename E>
__global__ __launch_bounds__(ST) void verify_stats_kernel(VerifyArgs a) {
  constexpr int N = Vec<E>::N, U = PIECE / ST / N;
  __shared__ float tops[ST / 64];
  __shared__ double masses[ST / 64];
  __shared__ int bests[ST / 64];
  const int t = blockIdx.x / a.pieces, piece = blockIdx.x - t * a.pieces;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the row's sequence: how many end at it or before
  int s = 0;
  for (int s0 = 0; s0 < a.st.seqs; s0 += 64)
    s += __popcll(__ballot(s0 + lane < a.st.seqs && a.st.cu[min(s0 + lane, a.st.seqs - 1) + 1] <= t));
  if (s >= a.st.seqs) return;
  const char *row = static_cast<const char *>(a.logits) + (int64_t)t * a.ls * sizeof(typename E::T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
  const int first = piece * PIECE - off;  // the first block's first element
  float x[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = first + (u * ST + (int)threadIdx.x) * N;
    if (e >= 0 && e + N <= a.vocab) {
      Vec<E>::unpack(*reinterpret_cast<const u32x4 *>(row + (int64_t)e * (int)sizeof(typename E::T)), x[u]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[u][i] = e + i >= 0 && e + i < a.vocab ? one_of<E>(row, e + i) : -INFINITY;
    }
  }
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
  Part *part = a.part + (size_t)t * a.pieces + piece;
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

// A workgroup a sequence.  Each row's pieces are joined, and each row's
// token gets its probabilities under its parent, all rows at once; then one
// wave walks: the next child of a row is found among 64 rows a ballot.  Where a
// drafted sibling is left after a refusal, all threads sum max(p - share q, 0).
//
// The refused tokens' probabilities, q given: with p~ after refusals = max(p -
// share q, 0), share the sum of A_j / B_j over the refusals, A_j the sum of p~
// and B_j that of q~ (1, or what the refused ones leave of it).  A refused token
// has none left: u A_j / B_j q >= p~ says that p~ is below what is taken.
template <typename E, typename Q, bool DRAFT>
__global__ __launch_bounds__(WALK) void verify_walk_kernel(VerifyArgs a) {
  __shared__ double mass[EXL3P_TREE_MAX], p[EXL3P_TREE_MAX], us[EXL3P_TREE_MAX];
  __shared__ float q[DRAFT ? EXL3P_TREE_MAX : 1], top[EXL3P_TREE_MAX];
  __shared__ int up[EXL3P_TREE_MAX], tok[EXL3P_TREE_MAX], best[EXL3P_TREE_MAX];
  __shared__ double left, drawn, share, sums[WALK / 64];
  __shared__ int at, seen, more;
  const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int begin = min(max(a.st.cu[s], 0), a.st.rows), end = min(max(a.st.cu[s + 1], begin), a.st.rows);
  const int n = min(end - begin, min(a.st.max_rows, EXL3P_TREE_MAX));
  if (n <= 0) {
    if (threadIdx.x == 0) a.tip[s].row = -1;
    return;
  }
  const float heat = a.temperature ? a.temperature[s] : 1.0f;
  const bool fit = heat >= 0.0f && heat < INFINITY, greedy = heat == 0.0f;
  const float rate = rate_of(heat);
  const double inv = 1.0 / (double)heat;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int t = begin + i;
    const int x = a.parent ? a.parent[t] : i - 1;
    up[i] = x >= 0 && x < i ? x : -1;
    tok[i] = a.ids[t];
    us[i] = a.u[t];
    a.target[t] = -1;
    const Part *part = a.part + (size_t)t * a.pieces;
    float hi = part[0].top;
    int where = part[0].best;
    double m = part[0].mass;
    for (int k = 1; k < a.pieces; ++k) {
      const Part y = part[k];
      if (greedy) {
        if (y.top > hi) where = y.best;
        hi = __builtin_elementwise_maximum(hi, y.top);
      } else {
        const float now = __builtin_elementwise_maximum(hi, y.top), ref = now == -INFINITY ? 0.0f : now;
        m = m * (double)__builtin_amdgcn_exp2f((hi - ref) * rate) +
            y.mass * (double)__builtin_amdgcn_exp2f((y.top - ref) * rate);
        hi = now;
      }
    }
    top[i] = hi;
    best[i] = where;
    // rows without a distribution: none of their tokens, and no walk past them
    const bool whole = fit && (greedy ? hi > -INFINITY : hi > -INFINITY && hi < INFINITY && m > 0.0 && m < INFINITY);
    mass[i] = whole ? m : -1.0;
  }
  if (threadIdx.x == 0) at = 0, seen = 0, left = 1.0, drawn = 1.0, share = 0.0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int j = up[i];
    double x = 0.0;
    float y = 0.0f;
    if (i > 0 && j >= 0 && !greedy && mass[j] > 0.0 && (uint32_t)tok[i] < (uint32_t)a.vocab) {
      x = exp(((double)one_of<E>(a.logits, (int64_t)(begin + j) * a.ls + tok[i]) - (double)top[j]) * inv) / mass[j];
      if constexpr (DRAFT) y = one_of<Q>(a.draft, (int64_t)(begin + j) * a.ds + tok[i]);
    }
    p[i] = x;
    if constexpr (DRAFT) q[i] = y;
  }
  __syncthreads();
  for (;;) {
    if (wave == 0) {
      // the next child of `row` behind row `from`
      auto next = [&](int row, int from) {
        for (int b = (from + 1) & ~63; b < n; b += 64) {
          const int i = b + lane;
          const uint64_t f = __ballot(i > from && i < n && up[min(i, n - 1)] == row);
          if (f != 0) return b + __builtin_ctzll(f);
        }
        return n;
      };
      int row = at, from = seen, need = 0;
      double A = left, B = drawn, L = share;
      int c = mass[row] >= 0.0 ? next(row, from) : n;
      while (c < n) {
        bool hit;
        double less = 0.0, step = 0.0;
        if (greedy) {
          hit = tok[c] == best[row];
        } else if constexpr (DRAFT) {
          step = A / fmax(B, 0x1p-53);
          hit = us[c] * step * (double)q[c] < fmax(p[c] - L * (double)q[c], 0.0);
        } else {
          // a token that a sibling before it had is not there any more
          less = p[c];
          for (int b = 0; b < c; b += 64) {
            const int i = b + lane;
            if (__ballot(i > 0 && i < c && up[i] == row && tok[i] == tok[c]) != 0) less = 0.0;
          }
          hit = us[c] * A < less;
        }
        from = c;
        if (hit) {
          if (lane == 0) a.target[begin + row] = tok[c];
          row = c, A = 1.0, B = 1.0, L = 0.0;
          c = mass[row] >= 0.0 ? next(row, from) : n;
          continue;
        }
        c = next(row, from);
        if (greedy) continue;
        if constexpr (DRAFT) {
          L += step;
          if (a.distinct) B -= (double)q[from];
          if (c < n) {
            need = 1;
            break;
          }
        } else {
          A -= less;
        }
      }
      if (lane == 0) at = row, seen = from, more = need, left = A, drawn = B, share = L;
    }
    __syncthreads();
    if (!DRAFT || !more) break;
    if constexpr (DRAFT) {  // what p~ has left
      const int row = at;
      const float hi = top[row], by = (float)(1.0 / mass[row]), lost = (float)share;
      const size_t z = (size_t)(begin + row) * a.ls, d = (size_t)(begin + row) * a.ds;
      double sum = 0.0;
      for (int e0 = threadIdx.x; e0 < a.vocab; e0 += 8 * blockDim.x) {
        float w = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = e0 + k * blockDim.x;
          if (e < a.vocab)
            w += fmaxf(__builtin_amdgcn_exp2f((one_of<E>(a.logits, z + e) - hi) * rate) * by -
                           lost * one_of<Q>(a.draft, d + e), 0.0f);
        }
        sum += (double)w;
      }
      sum = wave_sum(sum);
      if (lane == 0) sums[wave] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int w = 1; w < (int)blockDim.x / 64; ++w) sum += sums[w];
        left = sum;
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    const int row = at;
    Tip tip{-1, row, top[row], heat, share * mass[row], us[0]};
    if (mass[row] >= 0.0) {
      if (greedy)
        a.target[begin + row] = best[row];
      else
        tip.row = begin + row;
    }
    a.tip[s] = tip;
  }
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
  size_t z, d;
  __device__ __forceinline__ Rest(const VerifyArgs &args, int s)
      : a(args), tip(args.tip[s]), inv(1.0 / (double)tip.heat), z((size_t)max(tip.row, 0) * args.ls),
        d((size_t)max(tip.row, 0) * args.ds) {}
  // of p, and of p~; gone: bits of the piece that begins at `from`
  __device__ __forceinline__ void of(int e, const uint32_t *gone, int from, double &p, double &r) const {
    p = r = 0.0;
    if (e >= a.vocab) return;
    r = p = exp(((double)one_of<E>(a.logits, z + e) - (double)tip.top) * inv);
    if constexpr (DRAFT)
      r = fmax(p - tip.share * (double)one_of<Q>(a.draft, d + e), 0.0);
    else if (gone[(e - from) >> 5] >> ((e - from) & 31) & 1)
      r = 0.0;
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

// Sums of DRAW tokens a workgroup.
template <typename E, typename Q, bool DRAFT>
__global__ __launch_bounds__(ST) void verify_sums_kernel(VerifyArgs a) {
  __shared__ uint32_t gone[DRAW / 32];
  __shared__ double sums[2][ST / 64];
  const int s = blockIdx.x / a.draws, piece = blockIdx.x - s * a.draws, from = piece * DRAW;
  if (a.tip[s].row < 0) return;
  const Rest<E, Q, DRAFT> rest(a, s);
  rest.mark(s, from, gone);
  double all = 0.0, left = 0.0;
#pragma unroll
  for (int k = 0; k < DRAW / ST; ++k) {
    double p, r;
    rest.of(from + k * ST + (int)threadIdx.x, gone, from, p, r);
    all += p, left += r;
  }
  all = wave_sum(all), left = wave_sum(left);
  if ((threadIdx.x & 63) == 0) sums[0][threadIdx.x >> 6] = left, sums[1][threadIdx.x >> 6] = all;
  __syncthreads();
  if (threadIdx.x < 2) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < ST / 64; ++w) v += sums[threadIdx.x][w];
    a.sums[((size_t)s * a.draws + piece) * 2 + threadIdx.x] = v;
  }
}

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

// The token: the piece whose sum passes the border, then the place in it.
template <typename E, typename Q, bool DRAFT>
__global__ __launch_bounds__(ST) void verify_draw_kernel(VerifyArgs a) {
  __shared__ uint32_t gone[DRAW / 32];
  __shared__ double waves[ST / 64], base;
  __shared__ int found, last;
  const int s = blockIdx.x;
  if (a.tip[s].row < 0) return;
  const Rest<E, Q, DRAFT> rest(a, s);
  const double *sums = a.sums + (size_t)s * a.draws * 2;
  const int each = (a.draws + ST - 1) / ST, x0 = threadIdx.x * each, x1 = min(x0 + each, a.draws);
  if (threadIdx.x == 0) found = INT32_MAX, last = -1, base = 0.0;
  double whole, run;
  int kind = 0;  // 1: nothing is left of p~ (by rounding), p in its place
  for (;; kind = 1) {
    double own = 0.0;
    for (int x = x0; x < x1; ++x) own += sums[2 * x + kind];
    run = before(own, waves, whole);
    if (whole > 0.0 || kind == 1) break;
  }
  double border = rest.tip.u * whole;
  for (int x = x0; x < x1; ++x) {
    const double v = sums[2 * x + kind];
    run += v;
    if (!(v > 0.0)) continue;
    atomicMax(&last, x);
    if (run > border) {
      atomicMin(&found, x);
      break;
    }
  }
  __syncthreads();
  const bool passed = found != INT32_MAX;
  const int piece = passed ? found : max(last, 0);
  if (piece >= x0 && piece < x1) base = passed ? run - sums[2 * piece + kind] : -INFINITY;
  __syncthreads();
  if (threadIdx.x == 0) found = INT32_MAX, last = -1;
  const int from = piece * DRAW;
  rest.mark(s, from, gone);
  double r[DRAW / ST], own = 0.0;
#pragma unroll
  for (int k = 0; k < DRAW / ST; ++k) {
    double p;
    rest.of(from + (int)threadIdx.x * (DRAW / ST) + k, gone, from, p, r[k]);
    if (kind == 1) r[k] = p;
    own += r[k];
  }
  double sum;
  run = base + before(own, waves, sum);
  bool over = false;
#pragma unroll
  for (int k = 0; k < DRAW / ST; ++k) {
    run += r[k];
    const int e = from + (int)threadIdx.x * (DRAW / ST) + k;
    if (r[k] > 0.0) {
      atomicMax(&last, e);
      if (!over && run > border) atomicMin(&found, e), over = true;
    }
  }
  __syncthreads();
  // (sums in another order may end a step short of the border: the last one then)
  if (threadIdx.x == 0) a.target[rest.tip.row] = found != INT32_MAX ? found : last;
}

// ------------------------------------------------------------------- host side

constexpr int VOCAB_MAX = 1 << 24;

int pieces_of(int32_t vocab) { return (vocab + 7 + PIECE - 1) / PIECE; }
int draws_of(int32_t vocab) { return (vocab + DRAW - 1) / DRAW; }
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
         (size_t)r->seqs * draws_of(vocab) * 2 * sizeof(double);
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
  const hipStream_t st = static_cast<hipStream_t>(s);
  auto walk = [&](auto e, auto q, auto drafted) {
    typedef decltype(e) E;
    typedef decltype(q) Q;
    constexpr bool D = decltype(drafted)::value;
    // the sums after a refusal want many threads, the walk itself few
    hipLaunchKernelGGL((verify_walk_kernel<E, Q, D>), dim3(r->seqs), dim3(D && parent ? WALK : ST), 0,
                       st, a);
    hipLaunchKernelGGL((verify_sums_kernel<E, Q, D>), dim3((unsigned)(r->seqs * draws)), dim3(ST), 0, st, a);
    hipLaunchKernelGGL((verify_draw_kernel<E, Q, D>), dim3(r->seqs), dim3(ST), 0, st, a);
  };
  by_dtype(logits_dtype, [&](auto e) {
    hipLaunchKernelGGL((verify_stats_kernel<decltype(e)>), dim3((unsigned)(r->rows * pieces)), dim3(ST),
                       0, st, a);
    if (draft == nullptr)
      walk(e, e, std::false_type{});
    else
      by_dtype(draft_dtype, [&](auto q) { walk(e, q, std::true_type{}); });
  });
  return launched();
}

}  // extern "C"
