// paged_ops.hip -- the operators over a paged KV cache (include/exl3_paged.h)
// for MI355X (gfx950, wave64): tree plan, head norms + rotation + append,
// attention of new rows over pages, commit of accepted rows, page copies.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <new>
#include <type_traits>

#include "../../include/exl3_paged.h"
#include "exl3_device.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The element types of a cache: f32 conversions (to: one rounding, to nearest
// even), the exponent bits that mark infinities and NaN, the matrix product,
// and the power of two that softmax weights are scaled by (exponents below).
struct F16 {
  typedef _Float16 T;
  typedef half8 V8;
  static constexpr uint32_t EXP = 0x7C00u;
  // weights of 2^15 and less: one 2^-40 as large as the row's largest is still
  // not lost to f16's smallest number (2^-24)
  static constexpr float LIFT = 15.0f;
  static __device__ __forceinline__ f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
struct BF16 {
  typedef __bf16 T;
  typedef bf16x8 V8;
  static constexpr uint32_t EXP = 0x7F80u;
  static constexpr float LIFT = 0.0f;  // f32's exponents
  static __device__ __forceinline__ f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <typename E>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  return (float)__builtin_bit_cast(typename E::T, (uint16_t)bits);
}
template <typename E>
__device__ __forceinline__ uint32_t from_f32(float f) {
  return __builtin_bit_cast(uint16_t, (typename E::T)f);
}
template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return from_f32<E>(a) | (from_f32<E>(b) << 16);
}

// What the kernels need of a cache and of a step's rows.
struct Pool {
  char *k, *v;            // one layer's [pages][kv][page][dim]
  const int32_t *table;   // [seqs][max_pages]
  int32_t pages, kv, lp;  // lp: log2 of the page
  int32_t max_pages;
};
struct Step {
  const int32_t *cu, *len;
  int32_t seqs, rows, max_rows;
};

// The rows of a sequence, kept inside the step's tensors: first row, count.
struct Span {
  int row, n, len;
  bool bad;  // its keys do not fit its table
};
__device__ __forceinline__ Span span_of(const Step &st, int s, int64_t room) {
  const int a = min(max(st.cu[s], 0), st.rows);
  const int b = min(max(st.cu[s + 1], a), st.rows);
  Span sp;
  sp.row = a;
  sp.n = min(b - a, st.max_rows);
  sp.len = st.len[s];
  sp.bad = sp.len < 0 || (int64_t)sp.len + sp.n > room;
  if (sp.bad) sp.len = 0;
  return sp;
}

// The slot of a sequence's key, -1 where the table names no page of the pool.
__device__ __forceinline__ int slot_of(const Pool &p, int s, int key) {
  const uint32_t page = (uint32_t)p.table[(size_t)s * p.max_pages + (key >> p.lp)];
  return page < (uint32_t)p.pages ? (int)((page << p.lp) | (key & ((1 << p.lp) - 1))) : -1;
}

// ------------------------------------------------------------------ tree plan

// A workgroup a sequence, and one for the rows behind the last.  Each thread
// walks from its row to the root; the ancestors' numbers descend, so a word of
// the mask is finished when the walk leaves it.
constexpr int PLAN_THREADS = 256;

__global__ __launch_bounds__(PLAN_THREADS) void tree_plan_kernel(
    Pool pool, Step st, const int32_t *__restrict__ parent, int32_t *__restrict__ pos,
    int32_t *__restrict__ slot, uint64_t *__restrict__ mask, int words) {
  __shared__ int up[EXL3P_TREE_MAX];
  const int s = blockIdx.x;
  const int64_t room = (int64_t)pool.max_pages << pool.lp;
  if (s == st.seqs) {
    const int from = min(max(st.cu[st.seqs], 0), st.rows);
    for (int t = from + threadIdx.x; t < st.rows; t += PLAN_THREADS) {
      pos[t] = 0;
      slot[t] = -1;
      for (int w = 0; w < words; ++w) mask[(size_t)t * words + w] = 0;
    }
    return;
  }
  const Span sp = span_of(st, s, room);
  if (parent != nullptr) {
    for (int i = threadIdx.x; i < sp.n; i += PLAN_THREADS) {
      const int p = parent[sp.row + i];
      up[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
  }
  const int end = min(max(st.cu[s + 1], sp.row), st.rows) - sp.row;
  for (int i = threadIdx.x; i < end; i += PLAN_THREADS) {
    const size_t t = (size_t)sp.row + i;
    int depth = 0;
    if (i >= sp.n) {  // rows past max_rows
      for (int w = 0; w < words; ++w) mask[t * words + w] = 0;
    } else if (parent == nullptr) {
      depth = i;
      for (int w = 0; w < words; ++w)
        mask[t * words + w] = w < (i >> 6) ? ~0ull : w > (i >> 6) ? 0ull : ~0ull >> (63 - (i & 63));
    } else {
      for (int w = words - 1; w > (i >> 6); --w) mask[t * words + w] = 0;
      int word = i >> 6;
      uint64_t bits = 1ull << (i & 63);
      for (int j = up[i]; j >= 0; j = up[j], ++depth) {
        if (words > 0 && (j >> 6) != word) {
          mask[t * words + word] = bits;
          while (--word > (j >> 6)) mask[t * words + word] = 0;
          bits = 0;
        }
        bits |= 1ull << (j & 63);
      }
      if (words > 0) {
        mask[t * words + word] = bits;
        while (--word >= 0) mask[t * words + word] = 0;
      }
    }
    pos[t] = sp.len + depth;
    slot[t] = sp.bad || i >= sp.n ? -1 : slot_of(pool, s, sp.len + i);
  }
}

// ------------------------------------------------- norms, rotation and append

struct Rates {
  double turns[64];  // turns a position, theta^(-2 i / dim) / (2 pi)
};

// 4 elements of each half of a head a lane, dim / 8 lanes a head: a pair that
// turns together lies in one lane.
template <typename E, int D>
__global__ __launch_bounds__(256) void qkv_append_kernel(
    Pool pool, int rows, int nq, const uint16_t *__restrict__ q, int64_t qs,
    const uint16_t *__restrict__ k, int64_t ks, const uint16_t *__restrict__ v, int64_t vs,
    const uint16_t *__restrict__ qn, const uint16_t *__restrict__ kn,
    const int32_t *__restrict__ pos, const int32_t *__restrict__ slot, uint16_t *__restrict__ qo,
    int64_t os, float eps, Rates rates) {
  constexpr int LH = D / 8, HW = 64 / LH;  // lanes a head, heads a wave
  const int t = blockIdx.x;
  const int sl = slot[t];
  if (sl < 0 || sl >= (pool.pages << pool.lp)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & (LH - 1), sub = lane / LH;
  const int heads = nq + 2 * pool.kv;
  float co[4], si[4];
  const int p = pos[t];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double x = (double)p * rates.turns[4 * c + e];
    sincospif(2.0f * (float)(x - floor(x)), &si[e], &co[e]);
  }
  for (int h0 = wave * HW; h0 < heads; h0 += 4 * HW) {
    const int h = h0 + sub;
    if (h >= heads) break;  // the last heads of the row; no lane exchange follows for the others
    const bool isq = h < nq, isv = h >= nq + pool.kv;
    const int kvh = isq ? 0 : isv ? h - nq - pool.kv : h - nq;
    const uint16_t *src = isq ? q + t * qs + h * D : (isv ? v + t * vs : k + t * ks) + kvh * D;
    const size_t place = (((size_t)(sl >> pool.lp) * pool.kv + kvh) << pool.lp) +
                         (sl & ((1 << pool.lp) - 1));
    uint16_t *dst = isq ? qo + t * os + h * D
                        : reinterpret_cast<uint16_t *>(isv ? pool.v : pool.k) + place * D;
    const u32x2 a = *reinterpret_cast<const u32x2 *>(src + 4 * c);
    const u32x2 b = *reinterpret_cast<const u32x2 *>(src + D / 2 + 4 * c);
    u32x2 ra = a, rb = b;
    if (!isv) {
      float x[4], y[4], ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = to_f32<E>(a[e >> 1] >> (16 * (e & 1)));
        y[e] = to_f32<E>(b[e >> 1] >> (16 * (e & 1)));
        ss += x[e] * x[e] + y[e] * y[e];
      }
      const uint16_t *w = isq ? qn : kn;
      if (w != nullptr) {
#pragma unroll
        for (int m = 1; m < LH; m <<= 1) ss += __shfl_xor(ss, m, LH);
        const float r = 1.0f / sqrtf(ss / (float)D + eps);
        const u32x2 wa = *reinterpret_cast<const u32x2 *>(w + 4 * c);
        const u32x2 wb = *reinterpret_cast<const u32x2 *>(w + D / 2 + 4 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] *= r * to_f32<E>(wa[e >> 1] >> (16 * (e & 1)));
          y[e] *= r * to_f32<E>(wb[e >> 1] >> (16 * (e & 1)));
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ra[e] = pack2<E>(x[2 * e] * co[2 * e] - y[2 * e] * si[2 * e],
                         x[2 * e + 1] * co[2 * e + 1] - y[2 * e + 1] * si[2 * e + 1]);
        rb[e] = pack2<E>(y[2 * e] * co[2 * e] + x[2 * e] * si[2 * e],
                         y[2 * e + 1] * co[2 * e + 1] + x[2 * e + 1] * si[2 * e + 1]);
      }
    }
    *reinterpret_cast<u32x2 *>(dst + 4 * c) = ra;
    *reinterpret_cast<u32x2 *>(dst + D / 2 + 4 * c) = rb;
  }
}

// ------------------------------------------------------------------ attention

// What an attention workgroup does: rows r0 .. r0 + M - 1 of the (row, query
// head of the kv head) pairs of a sequence, keys k0 .. k1 - 1.
struct Work {
  int s;       // -1: nothing
  int r0;      // first pair
  int k0, k1;
  int first;   // the tile's first work item
  int splits;  // items of the tile
  Span sp;
};

struct Split {
  int group;   // query heads a kv head
  int tile;    // pairs a tile
  int target;  // items wanted, of a kv head
  int least;   // keys an item has at least
};

__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

__device__ __forceinline__ int tiles_of(const Span &sp, const Split &sl) {
  return (int)(((int64_t)sp.n * sl.group + sl.tile - 1) / sl.tile);
}
// 64-key units of a sequence
__device__ __forceinline__ int units_of(const Span &sp) { return (sp.len + sp.n + 63) >> 6; }

// Keys of an item, from all sequences: the units of all tiles over the target.
__device__ __forceinline__ int keys_of_item(const Step &st, const Split &sl, int64_t room) {
  const int lane = threadIdx.x & 63;
  // units up to 2^24 a sequence times its tiles: in double, exact and far from
  // overflow
  double units = 0.0;
  for (int s = lane; s < st.seqs; s += 64) {
    const Span sp = span_of(st, s, room);
    units += (double)tiles_of(sp, sl) * units_of(sp);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) units += __shfl_xor(units, m, 64);
  const double per = ceil(units / (double)sl.target);
  return max(sl.least, (int)fmin(per, (double)(1 << 24)) * 64);
}

// Item (ITEM) or tile (otherwise) number x among the sequences' ones.
template <bool ITEM>
__device__ __forceinline__ Work find_work(const Step &st, const Split &sl, int64_t room, int x) {
  const int lane = threadIdx.x & 63;
  const int chunk = keys_of_item(st, sl, room);
  Work w;
  w.s = -1;
  int items = 0, tiles = 0;  // of the sequences before
  for (int s0 = 0; s0 < st.seqs; s0 += 64) {
    const int s = s0 + lane;
    Span sp{0, 0, 0, false};
    int nt = 0, ns = 0;
    if (s < st.seqs) {
      sp = span_of(st, s, room);
      nt = tiles_of(sp, sl);
      ns = (int)(((int64_t)sp.len + sp.n + chunk - 1) / chunk);
    }
    // inclusive sums over the lanes
    int it = nt * ns, ti = nt;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int a = __shfl_up(it, m, 64), b = __shfl_up(ti, m, 64);
      if (lane >= m) it += a, ti += b;
    }
    const int mine = ITEM ? items + it : tiles + ti;
    const uint64_t past = __ballot(mine > x);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      const int s_ = s0 + l;
      sp = span_of(st, s_, room);
      nt = __shfl(nt, l, 64), ns = __shfl(ns, l, 64);
      const int before = items + __shfl(it, l, 64) - nt * ns;
      const int tbefore = tiles + __shfl(ti, l, 64) - nt;
      // the last tile first: a prompt's last rows see the most keys
      const int u = ITEM ? (x - before) / ns : nt - 1 - (x - tbefore);
      const int tile = ITEM ? nt - 1 - u : x - tbefore;
      w.s = s_;
      w.sp = sp;
      w.r0 = tile * sl.tile;
      w.first = before + (nt - 1 - tile) * ns;
      w.splits = ns;
      const int j = ITEM ? (x - before) % ns : 0;
      w.k0 = j * chunk;
      w.k1 = min(w.k0 + chunk, sp.len + sp.n);
      return w;
    }
    items += __shfl(it, 63, 64);
    tiles += __shfl(ti, 63, 64);
  }
  return w;
}

struct AttnArgs {
  Pool pool;
  Step st;
  Split sl;
  const uint16_t *q;
  int64_t qs;
  const uint64_t *mask;
  int words;
  float scale;  // times log2(e): weights are powers of two
  uint16_t *out;
  int64_t os;
  float *part;  // [items * kv][tile][D] sums, then [items * kv][tile][2] (max, sum)
  int slots;    // items * kv that part holds
};

// Bit `node` of a row's mask; without masks a row sees the rows up to itself.
__device__ __forceinline__ bool sees(const AttnArgs &a, const Span &sp, int i, int node) {
  if (node >= sp.n) return false;
  if (a.mask == nullptr) return node <= i;
  return (a.mask[(size_t)(sp.row + i) * a.words + (node >> 6)] >> (node & 63)) & 1;
}

constexpr int AW = 4;  // waves of an attention workgroup

// 16 pairs a workgroup; its waves take 32 keys in turn and join at the end.
// Scores are S^T = K q^T (rows keys, columns pairs), so a lane holds 8 keys'
// scores of one pair, in just the places where the second product, O^T = V^T
// P^T, wants its right operand if V's keys are taken in the same order: the
// weights never leave their lane.
template <typename E, int D>
__global__ __launch_bounds__(64 * AW) void attend_kernel(AttnArgs a) {
  constexpr int KK = D / 32;  // products of 32 dims a score
  constexpr int VH = D / 16;  // dims a lane loads of a value
  typedef typename std::conditional<VH == 8, u32x4, u32x2>::type VV;
  typedef typename E::V8 V8;
  __shared__ float so[AW][16][D + 4];
  __shared__ float sm[AW][16], sl[AW][16];
  __shared__ int sbad;
  const int head = blockIdx.x % a.pool.kv, item = blockIdx.x / a.pool.kv;
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.lp;
  Work w = find_work<true>(a.st, a.sl, room, item);
  if (w.s < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int G = a.sl.group, pairs = w.sp.n * G;
  const int pair = w.r0 + col, i = min(pair, pairs - 1) / G;
  const int hq = head * G + min(pair, pairs - 1) % G;
  const bool direct = w.splits == 1;
  // no row of the tile sees past its last row's own key without masks
  int last = w.sp.bad ? w.k0 : w.k1;
  if (a.mask == nullptr) last = min(last, w.sp.len + (min(w.r0 + 16, pairs) - 1) / G + 1);

  if (threadIdx.x == 0) sbad = w.sp.bad;
  __syncthreads();
  u32x4 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.sp.row + i) * a.qs + hq * D + 32 * kk + 8 * g);

  f32x4 acc[VH];
#pragma unroll
  for (int m = 0; m < VH; ++m) acc[m] = f32x4{0, 0, 0, 0};
  float top = -INFINITY, sum = 0.0f;
  bool bad = false;

  const int steps = last > w.k0 ? (last - w.k0 + 31) / 32 : 0;
  const int *trow = a.pool.table + (size_t)w.s * a.pool.max_pages;
  u32x4 kf[2][KK];
  VV vf[8];
  // where the two blocks of 16 keys of a step lie (elements from the layer's
  // first); blocks behind the last key read the last key's block
  size_t at[2];
  auto locate = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = min(w.k0 + step * 32 + 16 * t, (last - 1) & ~15);
      uint32_t page = (uint32_t)trow[key >> a.pool.lp];
      if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
      at[t] = ((((size_t)page * a.pool.kv + head) << a.pool.lp) + (key & ((1 << a.pool.lp) - 1))) * D;
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t *p = reinterpret_cast<const uint16_t *>(a.pool.k) + at[t] + col * D + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) kf[t][kk] = *reinterpret_cast<const u32x4 *>(p + 32 * kk);
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t *p = reinterpret_cast<const uint16_t *>(a.pool.v) + at[t] + 4 * g * D + VH * col;
#pragma unroll
      for (int r = 0; r < 4; ++r) vf[4 * t + r] = *reinterpret_cast<const VV *>(p + r * D);
    }
  };

  for (int step = wave; step < steps; step += AW) {
    const int kb = w.k0 + step * 32;
    locate(step);
    load_k();
    load_v();
    f32x4 s2[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s2[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        s2[t] = E::mma(__builtin_bit_cast(V8, kf[t][kk]), __builtin_bit_cast(V8, qf[kk]), s2[t]);
      s2[t] = s2[t] * a.scale;
    }
    const bool tail = kb + 32 > min(w.sp.len, last);
    bool odd = false;  // a value among the new rows that is not finite
    if (tail) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = kb + 16 * (e >> 2) + 4 * g + (e & 3);
        const bool in = key < last && (key < w.sp.len || sees(a, w.sp, i, key - w.sp.len));
        if (!in) s2[e >> 2][e & 3] = -INFINITY;
        // values behind the last key are nobody's
        if (key >= last) vf[e] = VV{};
#pragma unroll
        for (int x = 0; x < VH / 2; ++x)
          odd |= key >= w.sp.len && ((vf[e][x] & E::EXP) == E::EXP ||
                                     (vf[e][x] >> 16 & E::EXP) == E::EXP);
      }
    }
    float hi = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) hi = fmaxf(hi, s2[e >> 2][e & 3]);
    hi = fmaxf(hi, exl3::xor_lanes(hi, 16));
    hi = fmaxf(hi, exl3::xor_lanes(hi, 32));
    const float now = fmaxf(top, hi);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float alpha = __builtin_amdgcn_exp2f(top - ref);
    top = now;
    sum *= alpha;
#pragma unroll
    for (int m = 0; m < VH; ++m) acc[m] = acc[m] * alpha;
    uint32_t pw[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t b = pack2<E>(__builtin_amdgcn_exp2f(s2[e >> 2][e & 3] - ref + E::LIFT),
                                  __builtin_amdgcn_exp2f(s2[e >> 2][(e & 3) + 1] - ref + E::LIFT));
      pw[e >> 1] = b;
      // the sum of the rounded weights: they add up to one after the division
      sum += to_f32<E>(b) + to_f32<E>(b >> 16);
    }
    auto products = [&](const VV(&vv)[8], const uint32_t(&pp)[4], f32x4(&o)[VH]) {
      const V8 pb = __builtin_bit_cast(V8, u32x4{pp[0], pp[1], pp[2], pp[3]});
#pragma unroll
      for (int m = 0; m < VH; ++m) {
        const uint32_t sel = m & 1 ? 0x07060302u : 0x05040100u;
        u32x4 av;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          av[x] = __builtin_amdgcn_perm(vv[2 * x + 1][m >> 1], vv[2 * x][m >> 1], sel);
        o[m] = E::mma(__builtin_bit_cast(V8, av), pb, o[m]);
      }
    };
    if (!tail || __ballot(odd) == 0) {
      products(vf, pw, acc);
    } else {
      // a new row's value is infinite or NaN: a weight of zero would not keep
      // it from the rows that do not see it, so key by key, and only the pairs
      // that see the key take its product
      for (int x = 0; x < 32; ++x) {
        const int e = 4 * (x >> 4) + (x & 3);
        const bool mine = g == ((x >> 2) & 3);
        VV vx[8];
        uint32_t px[4];
#pragma unroll
        for (int y = 0; y < 8; ++y) vx[y] = y == e && mine ? vf[y] : VV{};
#pragma unroll
        for (int y = 0; y < 4; ++y)
          px[y] = y == e >> 1 && mine ? pw[y] & (e & 1 ? 0xFFFF0000u : 0xFFFFu) : 0;
        f32x4 o[VH];
#pragma unroll
        for (int m = 0; m < VH; ++m) o[m] = acc[m];
        products(vx, px, o);
        const int key = kb + x;
        const bool in = key < last && (key < w.sp.len || sees(a, w.sp, i, key - w.sp.len));
#pragma unroll
        for (int m = 0; m < VH; ++m)
          if (in) acc[m] = o[m];
      }
    }
  }
  if (bad) sbad = 1;
  sum += exl3::xor_lanes(sum, 16);
  sum += exl3::xor_lanes(sum, 32);
  if (g == 0) sm[wave][col] = top, sl[wave][col] = sum;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int m = 0; m < VH; ++m) so[wave][col][VH * (4 * g + r) + m] = acc[m][r];
  __syncthreads();
  // 16 lanes a pair, D / 16 dims each
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
  float all = -INFINITY;
#pragma unroll
  for (int x = 0; x < AW; ++x) all = fmaxf(all, sm[x][row]);
  const float ref = all == -INFINITY ? 0.0f : all;
  float o[VH], l = 0.0f;
#pragma unroll
  for (int m = 0; m < VH; ++m) o[m] = 0.0f;
#pragma unroll
  for (int x = 0; x < AW; ++x) {
    const float f = __builtin_amdgcn_exp2f(sm[x][row] - ref);
    l += f * sl[x][row];
#pragma unroll
    for (int m = 0; m < VH; ++m) o[m] += f * so[x][row][VH * c + m];
  }
  if (sbad) l = __builtin_nanf("");
  const int p = w.r0 + row;
  if (p >= pairs) return;
  if (direct) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *dst = a.out + (int64_t)(w.sp.row + p / G) * a.os + (head * G + p % G) * D + VH * c;
    VV b;
#pragma unroll
    for (int m = 0; m < VH; m += 2)
      b[m >> 1] = l == 0.0f ? 0u : pack2<E>(o[m] * inv, o[m + 1] * inv);
    *reinterpret_cast<VV *>(dst) = b;
  } else if ((int)blockIdx.x < a.slots) {
    float *dst = a.part + ((size_t)blockIdx.x * 16 + row) * D + VH * c;
#pragma unroll
    for (int m = 0; m < VH; m += 4)
      *reinterpret_cast<f32x4 *>(dst + m) = f32x4{o[m], o[m + 1], o[m + 2], o[m + 3]};
    float *ml = a.part + (size_t)a.slots * 16 * D + ((size_t)blockIdx.x * 16 + row) * 2;
    if (c == 0) ml[0] = all, ml[1] = l;
  }
}

// The items of a tile joined: 16 lanes a pair.
template <typename E, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a) {
  constexpr int VH = D / 16;
  typedef typename std::conditional<VH == 8, u32x4, u32x2>::type VV;
  const int head = blockIdx.x % a.pool.kv, tile = blockIdx.x / a.pool.kv;
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.lp;
  const Work w = find_work<false>(a.st, a.sl, room, tile);
  if (w.s < 0 || w.splits == 1) return;
  const int G = a.sl.group, row = threadIdx.x >> 4, c = threadIdx.x & 15;
  const int p = w.r0 + row;
  if (p >= w.sp.n * G) return;
  const float *ml = a.part + (size_t)a.slots * 16 * D;
  float all = -INFINITY;
  for (int x = 0; x < w.splits; ++x) {
    const int64_t slot = (int64_t)(w.first + x) * a.pool.kv + head;
    if (slot < a.slots) all = fmaxf(all, ml[(slot * 16 + row) * 2]);
  }
  const float ref = all == -INFINITY ? 0.0f : all;
  float o[VH], l = 0.0f;
#pragma unroll
  for (int m = 0; m < VH; ++m) o[m] = 0.0f;
  for (int x = 0; x < w.splits; ++x) {
    const int64_t slot = (int64_t)(w.first + x) * a.pool.kv + head;
    if (slot >= a.slots) continue;
    const float f = __builtin_amdgcn_exp2f(ml[(slot * 16 + row) * 2] - ref);
    l += f * ml[(slot * 16 + row) * 2 + 1];
    const float *src = a.part + (slot * 16 + row) * D + VH * c;
#pragma unroll
    for (int m = 0; m < VH; ++m) o[m] += f * src[m];
  }
  const float inv = 1.0f / l;
  uint16_t *dst = a.out + (int64_t)(w.sp.row + p / G) * a.os + (head * G + p % G) * D + VH * c;
  VV b;
#pragma unroll
  for (int m = 0; m < VH; m += 2) b[m >> 1] = l == 0.0f ? 0u : pack2<E>(o[m] * inv, o[m + 1] * inv);
  *reinterpret_cast<VV *>(dst) = b;
}

// --------------------------------------------------------------------- commit

// A workgroup a sequence, layer and array (keys or values).  Each walks the
// tree itself: the lowest fitting child of every row by an LDS minimum (the
// same whatever the order), then one link a step.  path ascends and path[j] >=
// j, so what row j's move overwrites no later row still reads; within a round
// all rows are read before any is written.
__global__ __launch_bounds__(256) void commit_kernel(
    Pool pool, Step st, size_t layer_bytes, int row_bytes, const int32_t *__restrict__ parent,
    const int32_t *__restrict__ ids, const int32_t *__restrict__ target, int32_t *__restrict__ path,
    int max_path, int32_t *__restrict__ count, int32_t *__restrict__ next,
    int32_t *__restrict__ new_len) {
  __shared__ int child[EXL3P_TREE_MAX], said[EXL3P_TREE_MAX], way[EXL3P_TREE_MAX];
  __shared__ int found, after;
  const int s = blockIdx.x;
  const Span sp = span_of(st, s, (int64_t)pool.max_pages << pool.lp);
  const int n = sp.bad ? 0 : sp.n;
  for (int i = threadIdx.x; i < n; i += 256) child[i] = INT32_MAX, said[i] = target[sp.row + i];
  __syncthreads();
  for (int i = threadIdx.x + 1; i < n; i += 256) {
    const int p = parent ? parent[sp.row + i] : i - 1;
    if (p >= 0 && p < i && ids[sp.row + i] == said[p]) atomicMin(&child[p], i);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0, c = 0;
    if (n > 0)
      for (;;) {
        way[c++] = at;
        const int to = child[at];
        if (to == INT32_MAX || c == max_path) break;
        at = to;
      }
    found = c;
    after = n > 0 ? said[at] : -1;
  }
  __syncthreads();
  const int c = found;
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < max_path; i += 256)
      path[(size_t)s * max_path + i] = i < c ? way[i] : -1;
    if (threadIdx.x == 0) {
      count[s] = c;
      next[s] = after;
      new_len[s] = (sp.bad ? st.len[s] : sp.len) + c;
    }
  }
  char *data = (blockIdx.y & 1 ? pool.v : pool.k) + (size_t)(blockIdx.y >> 1) * layer_bytes;
  const int lanes = row_bytes / 16;  // of a row of one head
  const int per = 256 / lanes;       // rows of one head a round
  const int x = threadIdx.x % lanes, y = threadIdx.x / lanes;
  const int todo = c * pool.kv;
  for (int b = 0; b < todo; b += per) {
    const int j = (b + y) / pool.kv, h = (b + y) % pool.kv;
    u32x4 val{};
    size_t to = 0;
    bool go = false;
    if (b + y < todo && way[j] != j) {
      const int from = slot_of(pool, s, sp.len + way[j]), dst = slot_of(pool, s, sp.len + j);
      if (from >= 0 && dst >= 0) {
        const int m = (1 << pool.lp) - 1;
        const size_t src = (((size_t)(from >> pool.lp) * pool.kv + h) << pool.lp) + (from & m);
        to = ((((size_t)(dst >> pool.lp) * pool.kv + h) << pool.lp) + (dst & m)) * row_bytes + 16 * x;
        val = *reinterpret_cast<const u32x4 *>(data + src * row_bytes + 16 * x);
        go = true;
      }
    }
    __syncthreads();
    if (go) *reinterpret_cast<u32x4 *>(data + to) = val;
  }
}

// ---------------------------------------------------------------- page copies

constexpr int COPY_PAIRS = 256;  // a launch's pairs travel in its arguments
struct Pairs {
  int32_t src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ __launch_bounds__(256) void copy_pages_kernel(char *k, char *v, size_t layer_bytes,
                                                         size_t page_bytes, Pairs pairs) {
  char *data = (blockIdx.z & 1 ? v : k) + (size_t)(blockIdx.z >> 1) * layer_bytes;
  const char *src = data + (size_t)pairs.src[blockIdx.y] * page_bytes;
  char *dst = data + (size_t)pairs.dst[blockIdx.y] * page_bytes;
  for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 16; i < page_bytes;
       i += (size_t)gridDim.x * 256 * 16)
    *reinterpret_cast<u32x4 *>(dst + i) = *reinterpret_cast<const u32x4 *>(src + i);
}

// ----------------------------------------------------------------- host checks

constexpr exl3_verdict OK{EXL3_OK, ""};
exl3_verdict refuse(int32_t code, const char *why) { return exl3_verdict{code, why}; }

exl3_verdict launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OK : refuse(EXL3_FAILED, hipGetErrorString(e));
}

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

exl3_verdict check_cache(const exl3p_cache *c) {
  if (c == nullptr || c->size != sizeof(exl3p_cache))
    return refuse(EXL3_FAILED, "PagedCache: no cache, or another version's");
  if (c->dtype != EXL3_DT_F16 && c->dtype != EXL3_DT_BF16)
    return refuse(EXL3_UNSUPPORTED, "PagedCacheDtype: float16 or bfloat16");
  if (c->k == nullptr || c->v == nullptr || c->table == nullptr)
    return refuse(EXL3_FAILED, "PagedCache: a missing array");
  if (!aligned(c->k, 16) || !aligned(c->v, 16))
    return refuse(EXL3_UNSUPPORTED, "PagedCacheAlignment: k and v on 16-byte boundaries");
  if (c->dim != 64 && c->dim != 128)
    return refuse(EXL3_UNSUPPORTED, "PagedCacheDim: heads of 64 or 128");
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)) != 0)
    return refuse(EXL3_UNSUPPORTED, "PagedCachePage: a power of two from 16 to 256");
  if (c->layers <= 0 || c->pages <= 0 || c->kv_heads <= 0 || c->seqs <= 0 || c->max_pages <= 0)
    return refuse(EXL3_UNSUPPORTED, "PagedCacheShape: sizes above 0");
  if ((int64_t)c->pages * c->page > INT32_MAX || (int64_t)c->max_pages * c->page > INT32_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedCacheShape: 2^31 keys or more");
  if (c->kv_heads > 65535 || c->layers > 32767)
    return refuse(EXL3_TOO_LARGE, "PagedCacheShape: over 65535 kv heads or 32767 layers");
  return OK;
}

exl3_verdict check_rows(const exl3p_cache *c, const exl3p_rows *r) {
  if (r == nullptr || r->size != sizeof(exl3p_rows))
    return refuse(EXL3_FAILED, "PagedRows: no rows, or another version's");
  if (r->seqs < 0 || r->rows < 0 || r->max_rows < 0 || r->max_rows > r->rows)
    return refuse(EXL3_UNSUPPORTED, "PagedRows: sizes below 0, or more rows a sequence than rows");
  if (r->seqs > c->seqs) return refuse(EXL3_UNSUPPORTED, "PagedRows: more sequences than the cache's");
  if (r->cu == nullptr || r->len == nullptr)
    return refuse(EXL3_FAILED, "PagedRows: a missing array");
  return OK;
}

exl3_verdict check_layer(const exl3p_cache *c, int32_t layer) {
  return layer >= 0 && layer < c->layers ? OK
                                         : refuse(EXL3_UNSUPPORTED, "PagedLayer: no such layer");
}

int log2_of(int v) { return 31 - __builtin_clz((unsigned)v); }

size_t page_bytes(const exl3p_cache *c) { return (size_t)c->kv_heads * c->page * c->dim * 2; }
size_t layer_bytes(const exl3p_cache *c) { return (size_t)c->pages * page_bytes(c); }

Pool pool_of(const exl3p_cache *c, int32_t layer) {
  const size_t at = (size_t)layer * layer_bytes(c);
  return Pool{static_cast<char *>(c->k) + at, static_cast<char *>(c->v) + at, c->table, c->pages,
              c->kv_heads, log2_of(c->page), c->max_pages};
}
Step step_of(const exl3p_rows *r) { return Step{r->cu, r->len, r->seqs, r->rows, r->max_rows}; }

// A matrix of rows: base and stride such that 16-byte accesses are whole.
exl3_verdict check_matrix(const void *p, int64_t stride, int64_t width) {
  if (p == nullptr) return refuse(EXL3_FAILED, "PagedMatrix: a missing array");
  if (!aligned(p, 16) || stride % 8 != 0)
    return refuse(EXL3_UNSUPPORTED,
                  "PagedMatrixAlignment: a 16-byte base and a row stride that 8 divides");
  if (stride < width) return refuse(EXL3_UNSUPPORTED, "PagedMatrixStride: rows overlap");
  return OK;
}

#define EXL3P_TRY(x)                     \
  do {                                   \
    const exl3_verdict v_ = (x);         \
    if (v_.code != EXL3_OK) return v_;   \
  } while (0)

// The device's compute units, read once per device.
int device_cus() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cached[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
    cached[dev] = n;
  }
  return cached[dev];
}

Split split_of(const exl3p_cache *c, int32_t heads) {
  Split sl;
  sl.group = heads / c->kv_heads;
  sl.tile = 16;
  sl.least = 32 * AW;
  const int n = (2 * device_cus() + c->kv_heads - 1) / c->kv_heads;
  sl.target = n > 1 ? n : 1;
  return sl;
}

// Tiles of a kv head that the rows can make, and items: a sequence's last tile
// and a tile's last item may be short.
int64_t most_tiles(const exl3p_rows *r, const Split &sl) {
  return (int64_t)r->rows * sl.group / sl.tile + r->seqs;
}
int64_t most_items(const exl3p_rows *r, const Split &sl) { return most_tiles(r, sl) + sl.target; }

template <typename F>
exl3_verdict by_type(const exl3p_cache *c, F &&f) {
  if (c->dtype == EXL3_DT_F16)
    c->dim == 64 ? f(F16{}, std::integral_constant<int, 64>{})
                 : f(F16{}, std::integral_constant<int, 128>{});
  else
    c->dim == 64 ? f(BF16{}, std::integral_constant<int, 64>{})
                 : f(BF16{}, std::integral_constant<int, 128>{});
  return launched();
}

exl3_verdict check_heads(const exl3p_cache *c, int32_t heads) {
  if (heads <= 0 || heads % c->kv_heads != 0)
    return refuse(EXL3_UNSUPPORTED, "PagedHeads: a multiple of the cache's kv heads");
  if (heads > 65535) return refuse(EXL3_TOO_LARGE, "PagedHeads: over 65535 heads");
  return OK;
}

}  // namespace

extern "C" {

exl3_verdict exl3p_tree_plan(const exl3p_cache *c, const exl3p_rows *r, const int32_t *parent,
                             int32_t *pos, int32_t *slot, uint64_t *mask, int32_t words,
                             exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_rows(c, r));
  if (words < 0 || (mask == nullptr) != (words == 0) || (mask != nullptr && (int64_t)words * 64 < r->max_rows))
    return refuse(EXL3_UNSUPPORTED, "PagedMask: 64 * words below the rows of a sequence");
  if (parent != nullptr && r->max_rows > EXL3P_TREE_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedTree: over 1024 rows of a sequence");
  if (r->rows == 0) return OK;
  if (pos == nullptr || slot == nullptr) return refuse(EXL3_FAILED, "PagedPlan: a missing array");
  hipLaunchKernelGGL(tree_plan_kernel, dim3(r->seqs + 1), dim3(PLAN_THREADS), 0,
                     static_cast<hipStream_t>(s), pool_of(c, 0), step_of(r), parent, pos, slot, mask,
                     words);
  return launched();
}

exl3_verdict exl3p_qkv_append(const exl3p_cache *c, int32_t layer, int32_t rows, int32_t heads,
                              const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                              const void *v, int64_t v_stride, const void *q_norm,
                              const void *k_norm, const int32_t *pos, const int32_t *slot,
                              void *q_out, int64_t out_stride, float eps, double theta,
                              exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_layer(c, layer));
  EXL3P_TRY(check_heads(c, heads));
  if (rows < 0) return refuse(EXL3_UNSUPPORTED, "PagedRows: sizes below 0");
  if (!(theta > 0.0) || !(theta < INFINITY))
    return refuse(EXL3_UNSUPPORTED, "PagedTheta: a rotation's base is positive and finite");
  if (rows == 0) return OK;
  const int64_t wq = (int64_t)heads * c->dim, wk = (int64_t)c->kv_heads * c->dim;
  EXL3P_TRY(check_matrix(q, q_stride, wq));
  EXL3P_TRY(check_matrix(k, k_stride, wk));
  EXL3P_TRY(check_matrix(v, v_stride, wk));
  EXL3P_TRY(check_matrix(q_out, out_stride, wq));
  if (pos == nullptr || slot == nullptr) return refuse(EXL3_FAILED, "PagedAppend: a missing array");
  if (!aligned(q_norm, 8) || !aligned(k_norm, 8))
    return refuse(EXL3_UNSUPPORTED, "PagedMatrixAlignment: norm weights on an 8-byte boundary");
  Rates rates{};
  const double ratio = pow(theta, -2.0 / c->dim);
  double turn = 1.0 / 6.283185307179586476925287;
  for (int i = 0; i < c->dim / 2; ++i, turn *= ratio) rates.turns[i] = turn;
  return by_type(c, [&](auto e, auto d) {
    hipLaunchKernelGGL((qkv_append_kernel<decltype(e), d>), dim3(rows), dim3(256), 0,
                       static_cast<hipStream_t>(s), pool_of(c, layer), rows, heads,
                       static_cast<const uint16_t *>(q), q_stride, static_cast<const uint16_t *>(k),
                       k_stride, static_cast<const uint16_t *>(v), v_stride,
                       static_cast<const uint16_t *>(q_norm), static_cast<const uint16_t *>(k_norm),
                       pos, slot, static_cast<uint16_t *>(q_out), out_stride, eps, rates);
  });
}

size_t exl3p_attend_scratch_bytes(const exl3p_cache *c, const exl3p_rows *r, int32_t heads) {
  if (check_cache(c).code != EXL3_OK || check_rows(c, r).code != EXL3_OK ||
      check_heads(c, heads).code != EXL3_OK)
    return 0;
  const Split sl = split_of(c, heads);
  return (size_t)most_items(r, sl) * c->kv_heads * sl.tile * (c->dim + 2) * sizeof(float);
}

exl3_verdict exl3p_attend(const exl3p_cache *c, int32_t layer, const exl3p_rows *r, int32_t heads,
                          const void *q, int64_t q_stride, const uint64_t *mask, int32_t words,
                          float scale, void *out, int64_t out_stride, void *scratch,
                          size_t scratch_bytes, exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_layer(c, layer));
  EXL3P_TRY(check_rows(c, r));
  EXL3P_TRY(check_heads(c, heads));
  if (words < 0 || (mask == nullptr) != (words == 0) || (mask != nullptr && (int64_t)words * 64 < r->max_rows))
    return refuse(EXL3_UNSUPPORTED, "PagedMask: 64 * words below the rows of a sequence");
  if (r->rows == 0 || r->seqs == 0 || r->max_rows == 0) return OK;
  const int64_t wq = (int64_t)heads * c->dim;
  EXL3P_TRY(check_matrix(q, q_stride, wq));
  EXL3P_TRY(check_matrix(out, out_stride, wq));
  const Split sl = split_of(c, heads);
  if ((int64_t)r->max_rows * sl.group > INT32_MAX / 2 || most_items(r, sl) * c->kv_heads > INT32_MAX / 16)
    return refuse(EXL3_TOO_LARGE, "PagedAttend: too many rows and heads for one call");
  if (scratch == nullptr || !aligned(scratch, 16) ||
      scratch_bytes < exl3p_attend_scratch_bytes(c, r, heads))
    return refuse(EXL3_FAILED, "PagedScratch: below exl3p_attend_scratch_bytes, or not aligned");
  AttnArgs a;
  a.pool = pool_of(c, layer), a.st = step_of(r), a.sl = sl;
  a.q = static_cast<const uint16_t *>(q), a.qs = q_stride, a.mask = mask, a.words = words;
  a.scale = scale * 1.4426950408889634f;
  a.out = static_cast<uint16_t *>(out), a.os = out_stride;
  a.part = static_cast<float *>(scratch);
  a.slots = (int)(most_items(r, sl) * c->kv_heads);
  const hipStream_t st = static_cast<hipStream_t>(s);
  return by_type(c, [&](auto e, auto d) {
    hipLaunchKernelGGL((attend_kernel<decltype(e), d>), dim3((unsigned)a.slots), dim3(64 * AW), 0, st,
                       a);
    hipLaunchKernelGGL((attend_join_kernel<decltype(e), d>),
                       dim3((unsigned)(most_tiles(r, sl) * c->kv_heads)), dim3(256), 0, st, a);
  });
}

exl3_verdict exl3p_commit(const exl3p_cache *c, const exl3p_rows *r, const int32_t *parent,
                          const int32_t *ids, const int32_t *target, int32_t *path,
                          int32_t max_path, int32_t *count, int32_t *next, int32_t *new_len,
                          exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_rows(c, r));
  if (r->max_rows > EXL3P_TREE_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedTree: over 1024 rows of a sequence");
  if (max_path <= 0) return refuse(EXL3_UNSUPPORTED, "PagedPath: max_path above 0");
  if (r->seqs == 0) return OK;
  if (path == nullptr || count == nullptr || next == nullptr || new_len == nullptr ||
      (r->rows > 0 && (ids == nullptr || target == nullptr)))
    return refuse(EXL3_FAILED, "PagedCommit: a missing array");
  if (new_len == r->len) return refuse(EXL3_UNSUPPORTED, "PagedCommit: new_len over len itself");
  hipLaunchKernelGGL(commit_kernel, dim3(r->seqs, 2 * c->layers), dim3(256), 0,
                     static_cast<hipStream_t>(s), pool_of(c, 0), step_of(r), layer_bytes(c),
                     c->dim * 2, parent, ids, target, path, max_path, count, next, new_len);
  return launched();
}

exl3_verdict exl3p_copy_pages(const exl3p_cache *c, const int32_t *src, const int32_t *dst,
                              int32_t count, exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  if (count < 0) return refuse(EXL3_UNSUPPORTED, "PagedCopy: a count below 0");
  if (count == 0) return OK;
  if (src == nullptr || dst == nullptr) return refuse(EXL3_FAILED, "PagedCopy: a missing array");
  if (count > c->pages) return refuse(EXL3_UNSUPPORTED, "PagedCopy: a page written twice");
  // one bit a page: read, written
  uint8_t *seen = new (std::nothrow) uint8_t[(size_t)c->pages]();
  if (seen == nullptr) return refuse(EXL3_FAILED, "PagedCopy: out of host memory");
  const char *why = nullptr;
  for (int32_t i = 0; i < count && why == nullptr; ++i) {
    if (src[i] < 0 || src[i] >= c->pages || dst[i] < 0 || dst[i] >= c->pages) {
      why = "PagedCopy: a page outside the cache";
      break;
    }
    if (seen[dst[i]] & 2) why = "PagedCopy: a page written twice";
    seen[dst[i]] |= 2;
    seen[src[i]] |= 1;
  }
  for (int32_t i = 0; i < count && why == nullptr; ++i)
    if (seen[dst[i]] & 1) why = "PagedCopy: a page both read and written";
  delete[] seen;
  if (why != nullptr) return refuse(EXL3_UNSUPPORTED, why);
  const size_t bytes = page_bytes(c);
  const unsigned wgs = (unsigned)((bytes + 32767) / 32768);
  for (int32_t at = 0; at < count; at += COPY_PAIRS) {
    const int n = count - at < COPY_PAIRS ? count - at : COPY_PAIRS;
    Pairs p;
    for (int i = 0; i < n; ++i) p.src[i] = src[at + i], p.dst[i] = dst[at + i];
    hipLaunchKernelGGL(copy_pages_kernel, dim3(wgs, n, 2 * c->layers), dim3(256), 0,
                       static_cast<hipStream_t>(s), static_cast<char *>(c->k),
                       static_cast<char *>(c->v), layer_bytes(c), bytes, p);
    EXL3P_TRY(launched());
  }
  return OK;
}

}  // extern "C"
