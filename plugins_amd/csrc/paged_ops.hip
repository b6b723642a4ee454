// paged_ops.hip -- the operators over a paged KV cache (include/exl3_paged.h)
// for MI355X (gfx950, wave64): tree plan, head norms + rotation + append,
// attention of new rows over pages, commit of accepted rows, page copies.
#include <new>

#include "paged_common.h"

namespace {

// A row's reference for its weights follows its running maximum only in steps of
// more than SLACK (powers of two): what has been summed is rarely scaled again.
constexpr float SLACK = 4.0f;
// Up to a reference of FAR a weight's exponent is one multiply-add of score, scale
// and (LIFT - reference).  Beyond, the product's rounding that the reference has
// and the sum has not, and the sum's own, are whole powers of two (at 2^20 they
// are 2^-4 of one): such a wave multiplies its scores first, and what is far is
// not lifted.
constexpr float FAR = 0x1p20f;

// ------------------------------------------------------------------ tree plan

// A workgroup a sequence, and one for the rows behind the last.  Each thread
// walks from its row to the root; the ancestors' numbers descend, so a word of
// the mask is finished when the walk leaves it.  A launch's time and a chain of
// loads (lengths, table), not bytes: one tree of 60 rows 2.9 us, 128 trees of up
// to 64 rows 3.8.
constexpr int PLAN_THREADS = 256;

__global__ __launch_bounds__(PLAN_THREADS) void tree_plan_kernel(
    Pool pool, Step st, const int32_t *__restrict__ parent, int32_t *__restrict__ pos,
    int32_t *__restrict__ slot, uint64_t *__restrict__ mask, int words) {
  __shared__ int up[EXL3P_TREE_MAX];
  const int s = blockIdx.x;
  const int64_t room = (int64_t)pool.max_pages << pool.lp;
  if (s == st.seqs) {
    const int from = min(max(st.cu[st.seqs], 0), st.rows), first = st.cu[0];
    for (int t = threadIdx.x; t < st.rows; t += PLAN_THREADS) {
      if (t >= first && t < from) continue;
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
// turns together lies in one lane, the squares are summed over the head's lanes,
// and a row's angles, in 64 bits until they are less than a turn, are formed once
// for the heads that a wave takes.  Bound by bytes: 4428 rows of 48 heads of 128
// 21.9 us, 5.0 TB/s read and written.
template <typename E, int D>
__global__ __launch_bounds__(256) void qkv_append_kernel(
    Pool pool, int rows, int nq, const uint16_t *q, int64_t qs,
    const uint16_t *__restrict__ k, int64_t ks, const uint16_t *__restrict__ v, int64_t vs,
    const uint16_t *__restrict__ qn, const uint16_t *__restrict__ kn,
    const int32_t *__restrict__ pos, const int32_t *__restrict__ slot, uint16_t *qo, int64_t os,
    float eps, Rates rates) {
  constexpr int LH = D / 8, HW = 64 / LH;  // lanes a head, heads a wave
  const int t = blockIdx.x;
  const int sl = slot[t];
  if (sl < 0 || sl >= (pool.pages << pool.lp)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & (LH - 1), sub = lane / LH;
  const int heads = nq + 2 * pool.kv, step = gridDim.y * 4 * HW;
  // a head's elements, loaded before the angles and before the head before it is
  // worked on
  u32x2 a{}, b{};
  auto fetch = [&](int h) {
    if (h >= heads) return;
    const uint16_t *src = h < nq              ? q + t * qs + h * D
                          : h < nq + pool.kv ? k + t * ks + (h - nq) * D
                                             : v + t * vs + (h - nq - pool.kv) * D;
    a = *reinterpret_cast<const u32x2 *>(src + 4 * c);
    b = *reinterpret_cast<const u32x2 *>(src + D / 2 + 4 * c);
  };
  int h = (blockIdx.y * 4 + wave) * HW + sub;
  fetch(h);
  float co[4], si[4];
  const int p = pos[t];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double x = (double)p * rates.turns[4 * c + e];
    sincospif(2.0f * (float)(x - floor(x)), &si[e], &co[e]);
  }
  // (the last heads of a row leave lanes behind: exchanges stay inside a head)
  for (; h < heads; h += step) {
    const bool isq = h < nq, isv = h >= nq + pool.kv;
    const int kvh = isq ? 0 : isv ? h - nq - pool.kv : h - nq;
    const size_t place = (((size_t)(sl >> pool.lp) * pool.kv + kvh) << pool.lp) +
                         (sl & ((1 << pool.lp) - 1));
    uint16_t *dst = isq ? qo + t * os + h * D
                        : reinterpret_cast<uint16_t *>(isv ? pool.v : pool.k) + place * D;
    u32x2 ra = a, rb = b;
    fetch(h + step);
    if (!isv) {
      float x[4], y[4], ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = to_f32<E>(ra[e >> 1] >> (16 * (e & 1)));
        y[e] = to_f32<E>(rb[e >> 1] >> (16 * (e & 1)));
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
  int splits;  // items of the tile; where there are several:
  int first;   // the place of the tile's first item in the scratch
  int place;   // of this one: items of a tile lie side by side
  int index;   // of the tile among those that are split
  int total;   // of those, where asked for
  Span sp;
};

// What the join needs of a split tile, left for it in the scratch by the tile's
// first item; the number of them stands before the first.
struct Joint {
  int row;     // the sequence's first row
  int pairs;   // of the sequence
  int r0;
  int first, splits;
  int pad[3];
};

// How keys are split into items, by what the host knows; the lengths decide on
// the device.  A tile (pairs of a row and a query head) has items of equal length.
struct Split {
  int group;    // query heads a kv head
  int tile;     // pairs a tile, a power of two: log2 of it
  int least;    // 64-key units that an item has at least; 4 behind `few`
  float round;  // items of a kv head that fill the CUs once, two each
  float few;    // up to so many tiles, a round less the tiles is the target,
  float most;   // else so many items
  float whole, more;  // no tile is split whose units are at most whole * all + more
};

__device__ __forceinline__ int tiles_of(const Span &sp, const Split &sl) {
  return (int)((uint32_t)(sp.n * sl.group + (1 << sl.tile) - 1) >> sl.tile);
}

// Item number x among the sequences' ones.  Every workgroup finds its own: no
// plan on the device or the host depends on the lengths, so a captured call
// follows them.  A tile of u units has ceil(u / c) items, c the units of all tiles
// over the target, plus what 32-bit sums may be short of: items are never more
// than target + tiles.  (Lane exchanges by DPP and scalars: 1 us of a launch less
// than through LDS, with 64-bit divisions.)
__device__ __forceinline__ Work find_work(const Step &st, const Split &sl, int64_t room, int x) {
  const int lane = threadIdx.x & 63;
  Span sp{0, 0, 0, false, false};
  float units = 0.0f, all = 0.0f, longest = 0.0f;
  bool back = false;
  auto units_of = [](const Span &v) { return (uint32_t)(v.len + v.n + 63) >> 6; };
  for (int s = lane; s < st.seqs; s += 64) {
    sp = span_of(st, s, room);
    const float t = (float)tiles_of(sp, sl);
    units += t * (float)units_of(sp);
    all += t;
    longest = fmaxf(longest, t > 0.0f ? (float)units_of(sp) : 0.0f);
    back |= sp.back;
  }
  // The launch and the scratch are sized for no more rows than the step has: a
  // step whose sequences share rows does nothing.
  Work w;
  w.s = -1;
  w.total = 0;
  if (__ballot(back) != 0) return w;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    units += exl3::xor_lanes(units, m);
    all += exl3::xor_lanes(all, m);
    longest = fmaxf(longest, exl3::xor_lanes(longest, m));
  }
  // 65535 sequences are 1024 sums a lane, each off by 2^-24 at most
  const float target = all <= sl.few ? sl.round - all : sl.most;
  // Items of up to 16 units are made so long that half a round holds them: a
  // workgroup alone on a CU takes a unit in little more than half the time, and
  // the join has half to read (64 rows behind 8000 keys 34.3 us -> 28.8, two single
  // tokens of 5000 14.8 -> 12.5).  Else a tile's first 16 items may be short; more
  // of them are 8 units at least, since the join's time goes with their number.
  const float spare = floorf(0.5f * sl.round) - all;
  const float half = ceilf(units * __builtin_amdgcn_rcpf(spare));
  const float least =
      fmaxf((float)(all <= sl.few ? sl.least : 4),
            spare > 0.0f && half <= 16.0f
                ? half
                : fminf(8.0f, floorf(units * 0.0625f * __builtin_amdgcn_rcpf(fmaxf(all, 1.0f)))));
  // Whole tiles where the longest of them ends soon after a full round would (its
  // parts' way through memory and the join cost more): four prompts of up to 500
  // rows 50.8 us -> 31.0, one of 2000 73.9 -> 58.3, 64 single rows over up to 500
  // keys 22.6 -> 18.9.
  const float chunk_of = longest <= sl.whole * units + sl.more
                             ? (float)(1 << 25)
                             : ceilf(units * (1.0f + 0x1p-12f) / target);
  const uint32_t chunk = __builtin_amdgcn_readfirstlane(
      (int)fminf(fmaxf(chunk_of, least), (float)(1 << 25)));
  int items = 0, tiles = 0, parts = 0;  // of the sequences before: all, and split ones'
  for (int s0 = 0; s0 < st.seqs; s0 += 64) {
    const int s = s0 + lane;
    int nt = 0, ns = 0;
    uint32_t each = 1;
    if (s < st.seqs) {
      if (st.seqs > 64) sp = span_of(st, s, room);
      nt = tiles_of(sp, sl);
      const uint32_t u = units_of(sp);
      if (nt > 0) {
        ns = (int)((u + chunk - 1) / chunk);
        each = (u + ns - 1) / ns;  // the last items may be empty
      }
    }
    const int mi = nt * ns, mt = ns > 1 ? nt : 0, mp = ns > 1 ? mi : 0;
    const int it = scan(mi), ti = scan(mt), pi = scan(mp);
    const uint64_t past = __ballot(items + it > x);
    if (w.s < 0 && past != 0) {
      const int l = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int n_t = of(nt), n_s = of(ns), keys = of((int)each) * 64;
      const int before = items + of(it - mi);
      // Tiles that read the same keys side by side, the last tile first: a prompt's
      // last rows see the most keys, and items behind a tile's last key come last
      // (a tile's items side by side: 1000 rows of 2 kv heads 25.0 us against 24.0,
      // four prompts of up to 300 rows over up to 4000 keys 62.8 against 60.5).
      const int j = (x - before) / n_t, u = (x - before) - j * n_t;
      w.s = s0 + l;
      w.sp = Span{of(sp.row), of(sp.n), of(sp.len), (bool)of(sp.bad), false};
      w.r0 = (n_t - 1 - u) << sl.tile;
      w.first = parts + of(pi - mp) + u * n_s;
      w.place = w.first + j;
      w.splits = n_s;
      w.index = tiles + of(ti - mt) + u;
      const uint32_t end = w.sp.len + w.sp.n, from = (uint32_t)j * (uint32_t)keys;
      w.k0 = (int)min(from, end);
      w.k1 = (int)min(from + keys, end);
      if (x > 0) return w;  // the first item looks at all sequences
    }
    items += __builtin_amdgcn_readlane(it, 63);
    tiles += __builtin_amdgcn_readlane(ti, 63);
    parts += __builtin_amdgcn_readlane(pi, 63);
  }
  w.total = tiles;
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
  float scale;    // |scale| log2(e): weights are powers of two
  uint32_t flip;  // 0x80008000 where the scale is negative: q's sign bits
  uint16_t *out;
  int64_t os;
  Joint *joint;  // [0].row: how many; [1 + i]: the split tiles
  int joints;    // that joint holds
  float *part;   // [parts * kv][tile][D] sums, then [parts * kv][tile][2] (max, sum)
  int slots;     // parts * kv that part holds: items of split tiles
};

// The scratch's head, from the workgroups that find it.
__device__ __forceinline__ void leave_joint(const AttnArgs &a, const Work &w, int item) {
  if (blockIdx.x % a.pool.kv != 0 || threadIdx.x != 0) return;
  if (item == 0) a.joint[0].row = min(w.total, a.joints);
  if (w.s >= 0 && w.splits > 1 && w.place == w.first && w.index < a.joints)
    a.joint[1 + w.index] = Joint{w.sp.row, w.sp.n * a.sl.group, w.r0, w.first, w.splits, {}};
}

// Which of keys kb .. kb + 63 (below `last`) row i of a sequence sees, a bit a
// key: the context's, and of the rows those in its mask, or up to itself.
__device__ __forceinline__ uint64_t seen64(const AttnArgs &a, const Span &sp, int i, int kb,
                                           int last) {
  const int lim = a.mask == nullptr ? min(last, sp.len + i + 1) : min(last, sp.len + sp.n);
  if (lim <= kb) return 0;
  uint64_t v = lim - kb >= 64 ? ~0ull : ~0ull >> (64 - (lim - kb));
  if (a.mask != nullptr && lim > sp.len) {
    const uint64_t *m = a.mask + (size_t)(sp.row + i) * a.words;
    const int j = kb - sp.len;  // the first key's number among the rows
    const uint64_t lo = j >= 0 && (j >> 6) < a.words ? m[j >> 6] >> (j & 63) : 0;
    const int next = j >= 0 ? (j >> 6) + 1 : 0, by = j >= 0 ? 64 - (j & 63) : -j;
    const uint64_t hi = by < 64 && next < a.words ? m[next] << by : 0;
    v &= j >= 0 ? lo | hi : j > -64 ? hi | ~(~0ull << -j) : ~0ull;
  }
  return v;
}

constexpr int AW = 4;      // waves of an attention workgroup
constexpr int FEW = 32;    // the most pairs of a tile of attend_few (16 or 32),
constexpr int MANY = 128;  // a tile of attend_many's

// A wave's softmax over the keys it has seen: the reference of each pair's
// weights, the sum of them and their lift: 2^(score * scale + lift - reference).
struct Soft {
  float ref, sum, lift;
  // from some pair's first far reference on: the wave's scores are multiplied by
  // AttnArgs' scale before all else, and scale is 1
  bool far;
  float scale;
};

// The larger, NaN if either is: without the canonicalizing instructions that
// fmaxf takes for each operand.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// The running maximum `hi` (of scores times so.scale) of each lane's pair joins
// its reference; the factor for what has been summed so far is 1 (false) unless
// some pair of the wave outgrew its reference by more than SLACK.  turned: the
// wave's first far reference (-inf, nothing seen, is none).
template <typename E>
__device__ __forceinline__ bool outgrown(Soft &so, float hi, float &alpha, bool &turned) {
  turned = false;
  if (__ballot(hi - so.ref > SLACK) == 0) return false;
  const float now = fmaxf(so.ref, hi);
  alpha = __builtin_amdgcn_exp2f(so.ref - (now == -INFINITY ? 0.0f : now));
  so.ref = now;
  turned = !so.far && __ballot(fabsf(now) > FAR && now != -INFINITY) != 0;
  if (turned) so.far = true, so.scale = 1.0f;
  if (so.far && E::LIFT > 0.0f) {
    const float to = fabsf(now) > FAR ? 0.0f : E::LIFT;
    alpha *= __builtin_amdgcn_exp2f(to - so.lift);
    so.lift = to;
  }
  so.sum *= alpha;
  return true;
}

// A new row's value that is infinite or NaN would reach, times a weight of zero,
// the rows that do not see it.  Such elements are taken out of the products
// (finite(): zero in their place), and added afterwards to the rows that see
// them: they are so whatever their weight.
template <typename E>
__device__ __forceinline__ uint32_t finite(uint32_t two) {
  if ((two & E::EXP) == E::EXP) two &= 0xFFFF0000u;
  if (((two >> 16) & E::EXP) == E::EXP) two &= 0xFFFFu;
  return two;
}
// element e of a pair of elements where it is not finite, else 0
template <typename E>
__device__ __forceinline__ float not_finite(uint32_t two, int e) {
  const uint32_t one = e ? two >> 16 : two & 0xFFFFu;
  return (one & E::EXP) == E::EXP ? to_f32<E>(one) : 0.0f;
}
// a key's value row, for the rare rows above (nullptr: no page)
__device__ __forceinline__ const uint16_t *value_row(const Pool &p, int s, int head, int key, int D) {
  const int sl = slot_of(p, s, key);
  if (sl < 0) return nullptr;
  const size_t row = (((size_t)(sl >> p.lp) * p.kv + head) << p.lp) + (sl & ((1 << p.lp) - 1));
  return reinterpret_cast<const uint16_t *>(p.v) + row * D;
}

// Keys below this every row of the work's tile sees: its first row's.
__device__ __forceinline__ int clear_of(const AttnArgs &a, const Work &w, int last) {
  return min(last, a.mask == nullptr ? w.sp.len + w.r0 / a.sl.group + 1 : w.sp.len);
}

// 16 NT pairs a workgroup; its waves take 32 keys in turn and join at the end.
// Scores are S^T = K q^T (rows keys, columns pairs), so a lane holds 8 keys'
// scores of one pair, in just the places where the second product, O^T = V^T
// P^T, wants its right operand if V's keys are taken in the same order: the
// weights never leave their lane, and no load passes through LDS (16 bytes a lane,
// the next step's keys on their way while the weights form).  Bound by bytes: trees
// of 8 rows over 4 contexts of up to 65536 keys 138 us, 5.5 TB/s (a read alone of 2
// GiB: 6.3); one token over 2048 keys 7.4 us, its chain of loads.
//
// Weights are rounded to the cache's type, since the second product takes both
// operands in it (in 32 bits it would run at a sixteenth of the rate), and summed
// as rounded, so that they add up to one: a value is off by half a step of its
// type, at most, beside the output's own half: 1.2 to 1.4 times the error of 32-bit
// weights.  References, sums and joins are of 32 bits.
template <typename E, int D, int NT>
__global__ __launch_bounds__(64 * AW, NT == 1 ? 3 : 2) void attend_few_kernel(AttnArgs a) {
  constexpr int KK = D / 32;  // products of 32 dims a score
  constexpr int VH = D / 16;  // dims a lane loads of a value
  constexpr int ROWS = 16 * NT;
  typedef typename std::conditional<VH == 8, u32x4, u32x2>::type VV;
  typedef typename E::V8 V8;
  __shared__ float so[AW][16][D + 4];
  __shared__ float sm[AW][16], sl[AW][16];
  __shared__ int sbad;
  const int head = blockIdx.x % a.pool.kv, item = blockIdx.x / a.pool.kv;
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.lp;
  const Work w = find_work(a.st, a.sl, room, item);
  leave_joint(a, w, item);
  if (w.s < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int G = a.sl.group, pairs = w.sp.n * G;
  // no row of the tile sees past its last row's own key without masks
  int last = w.sp.bad ? w.k0 : w.k1;
  if (a.mask == nullptr) last = min(last, w.sp.len + (min(w.r0 + ROWS, pairs) - 1) / G + 1);
  const int clear = clear_of(a, w, last);
  if (threadIdx.x == 0) sbad = w.sp.bad;

  const int steps = last > w.k0 ? (last - w.k0 + 31) / 32 : 0;
  const int *trow = a.pool.table + (size_t)w.s * a.pool.max_pages;
  const uint16_t *pk = reinterpret_cast<const uint16_t *>(a.pool.k) + col * D + 8 * g;
  const uint16_t *pv = reinterpret_cast<const uint16_t *>(a.pool.v) + 4 * g * D + VH * col;
  bool bad = false;
  u32x4 kf[2][KK];
  VV vf[8];
  uint32_t ids[2];
  size_t at[2];
  // the pages of a step's two blocks of 16 keys; blocks behind the last key
  // stand for the last key's
  auto key_of = [&](int step, int t) {
    return min(w.k0 + step * 32 + 16 * t, (last - 1) & ~15);
  };
  auto fetch = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) ids[t] = (uint32_t)trow[key_of(step, t) >> a.pool.lp];
  };
  // where the blocks lie (elements from the layer's first)
  auto locate = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t page = __builtin_amdgcn_readfirstlane(ids[t]);
      if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
      at[t] = ((((size_t)page * a.pool.kv + head) << a.pool.lp) +
               (key_of(step, t) & ((1 << a.pool.lp) - 1))) * D;
    }
  };
  auto load_k = [&] {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        kf[t][kk] = *reinterpret_cast<const u32x4 *>(pk + at[t] + 32 * kk);
  };
  auto load_v = [&] {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        vf[4 * t + r] = *reinterpret_cast<const VV *>(pv + at[t] + r * D);
  };

  u32x4 qf[NT][KK];
  int row_of[NT];  // a lane's pairs' rows of the sequence
  if (wave < steps) fetch(wave);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int pair = min(w.r0 + 16 * n + col, pairs - 1);
    row_of[n] = pair / G;
    const uint16_t *src = a.q + (w.sp.row + row_of[n]) * a.qs +
                          (head * G + pair - row_of[n] * G) * D + 8 * g;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[n][kk] = *reinterpret_cast<const u32x4 *>(src + 32 * kk) ^ a.flip;
  }
  if (wave < steps) {
    locate(wave);
    load_k();
    load_v();
    if (wave + AW < steps) fetch(wave + AW);
  }
  f32x4 acc[NT][VH];
  Soft sf[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sf[n] = Soft{-INFINITY, 0.0f, E::LIFT, false, a.scale};
#pragma unroll
    for (int m = 0; m < VH; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
  }

  auto turn = [&](int step, auto MORE) {
    constexpr bool more = decltype(MORE)::value;
    const int kb = w.k0 + step * 32;
    f32x4 s2[NT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s2[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          s2[n][t] = E::mma(__builtin_bit_cast(V8, kf[t][kk]), __builtin_bit_cast(V8, qf[n][kk]),
                            s2[n][t]);
      }
    if constexpr (more) {
      locate(step + AW);
      load_k();
      fetch(min(step + 2 * AW, steps - 1));
    }
    const bool tail = kb + 32 > clear;
    uint32_t seen[NT];
    uint32_t odd = 0;  // keys among the new rows with a value that is not finite
    if (tail) {
#pragma unroll
      for (int n = 0; n < NT; ++n) seen[n] = (uint32_t)seen64(a, w.sp, row_of[n], kb, last);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int x = 16 * (e >> 2) + 4 * g + (e & 3);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (!(seen[n] >> x & 1)) s2[n][e >> 2][e & 3] = -INFINITY;
        // values behind the last key are nobody's
        if (kb + x >= last) vf[e] = VV{};
        bool bad_value = false;
        if (kb + x >= w.sp.len) {
#pragma unroll
          for (int y = 0; y < VH / 2; ++y) {
            const uint32_t f = finite<E>(vf[e][y]);
            bad_value |= f != vf[e][y];
            vf[e][y] = f;
          }
        }
        const uint64_t lanes = __ballot(bad_value);
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (lanes >> (16 * z) & 0xFFFFu) odd |= 1u << (16 * (e >> 2) + 4 * z + (e & 3));
      }
    }
    u32x4 pw[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (sf[n].far) s2[n][0] *= a.scale, s2[n][1] *= a.scale;
      float hi = larger(s2[n][0][0], s2[n][0][1]);
#pragma unroll
      for (int e = 2; e < 8; ++e) hi = larger(hi, s2[n][e >> 2][e & 3]);
      hi = larger(hi, exl3::xor_lanes(hi, 16));
      hi = larger(hi, exl3::xor_lanes(hi, 32));
      float alpha;
      bool turned;
      if (outgrown<E>(sf[n], hi * sf[n].scale, alpha, turned)) {
        if (turned) s2[n][0] *= a.scale, s2[n][1] *= a.scale;
#pragma unroll
        for (int m = 0; m < VH; ++m) acc[n][m] = acc[n][m] * alpha;
      }
      const float by = sf[n].lift - (sf[n].ref == -INFINITY ? 0.0f : sf[n].ref);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float(&x)[2] = {fmaf(s2[n][e >> 2][e & 3], sf[n].scale, by),
                              fmaf(s2[n][e >> 2][(e & 3) + 1], sf[n].scale, by)};
        pw[n][e >> 1] = pack2<E>(__builtin_amdgcn_exp2f(x[0]), __builtin_amdgcn_exp2f(x[1]));
        // the sum of the rounded weights: they add up to one after the division
        sf[n].sum = E::add2(pw[n][e >> 1], sf[n].sum);
      }
    }
#pragma unroll
    for (int m = 0; m < VH; ++m) {
      const uint32_t sel = m & 1 ? 0x07060302u : 0x05040100u;
      u32x4 av;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        av[x] = __builtin_amdgcn_perm(vf[2 * x + 1][m >> 1], vf[2 * x][m >> 1], sel);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        acc[n][m] = E::mma(__builtin_bit_cast(V8, av), __builtin_bit_cast(V8, pw[n]), acc[n][m]);
    }
    for (; odd != 0; odd &= odd - 1) {
      const int x = __builtin_ctz(odd);
      const uint16_t *row = value_row(a.pool, w.s, head, kb + x, D);
      if (row == nullptr) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const VV b = *reinterpret_cast<const VV *>(row + VH * (4 * g + r));
#pragma unroll
        for (int m = 0; m < VH; ++m) {
          const float v = not_finite<E>(b[m >> 1], m & 1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (seen[n] >> x & 1) acc[n][m][r] += v;
        }
      }
    }
    if constexpr (more) load_v();
  };
  int step = wave;
  for (; step + AW < steps; step += AW) turn(step, std::true_type{});
  if (step < steps) turn(step, std::false_type{});

  __syncthreads();
  if (bad) sbad = 1;
  // the waves' sums join, 16 pairs at a time: 16 lanes a pair, D / 16 dims each
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n > 0) __syncthreads();
    if (sf[n].far) {  // lifted as all other sums are
      const float by = __builtin_amdgcn_exp2f(E::LIFT - sf[n].lift);
      sf[n].sum *= by;
#pragma unroll
      for (int m = 0; m < VH; ++m) acc[n][m] = acc[n][m] * by;
    }
    float sum = sf[n].sum;
    sum += exl3::xor_lanes(sum, 16);
    sum += exl3::xor_lanes(sum, 32);
    if (g == 0) sm[wave][col] = sf[n].ref, sl[wave][col] = sum;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int m = 0; m < VH; ++m) so[wave][col][VH * (4 * g + r) + m] = acc[n][m][r];
    __syncthreads();
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
    const int p = w.r0 + 16 * n + row;
    if (p >= pairs) continue;
    if (w.splits == 1) {
      const float inv = 1.0f / l;
      uint16_t *dst = a.out + (int64_t)(w.sp.row + p / G) * a.os + (head * G + p % G) * D + VH * c;
      VV b;
#pragma unroll
      for (int m = 0; m < VH; m += 2)
        b[m >> 1] = l == 0.0f ? 0u : pack2<E>(o[m] * inv, o[m + 1] * inv);
      *reinterpret_cast<VV *>(dst) = b;
    } else if (w.place * a.pool.kv + head < a.slots) {
      const size_t to = ((size_t)w.place * a.pool.kv + head) * ROWS + 16 * n + row;
      float *dst = a.part + to * D + VH * c;
#pragma unroll
      for (int m = 0; m < VH; m += 4)
        *reinterpret_cast<f32x4 *>(dst + m) = f32x4{o[m], o[m + 1], o[m + 2], o[m + 3]};
      float *ml = a.part + (size_t)a.slots * ROWS * D + to * 2;
      if (c == 0) ml[0] = all, ml[1] = l;
    }
  }
}

// A barrier that orders LDS alone: loads in flight stay so.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// 128 pairs a workgroup, 32 a wave; tiles of 64 keys and values pass through
// LDS, two of them so that one is loaded while the other is used.  The products
// are those of attend_few with 32 x 32 tiles: a lane holds 32 keys' scores of
// one pair and feeds its weights to the second product as they are.  A row of
// LDS holds a key's 16-byte pieces at places q ^ f(row) (the lanes that load
// choose their pieces so): pieces of one number of 16 rows of keys lie in 16
// places of the 64 banks, and so do the 4 rows by 64 bytes of values that 32
// lanes of a transposing read take.  Two workgroups a CU, each one's products
// beside the other's softmax.  Prompts of 2048 rows (222 GFLOP) 239 us, 0.75 of a
// large product's rate; of an earlier 250, 221 without the softmax, 212 without the
// loads, 184 without both (times only): what is left lies between the pipes.  16
// trees of up to 64 rows over up to 8192 keys 68 us, 3.3 TB/s: a tile's loads are one
// tile ahead, and the longest item is 1.23 times the mean.  Heads of 64 have LDS and,
// held to 128, registers for four workgroups (prompts 157.3 us -> 156.1, 16 trees 46.3
// -> 46.0).
template <typename E, int D>
__global__ __launch_bounds__(64 * AW, D == 64 ? 4 : 2) void attend_many_kernel(AttnArgs a) {
  constexpr int KK = D / 16, ND = D / 32;
  constexpr int ROW = D * 2;          // bytes of a key
  constexpr int ARR = 64 * ROW;       // of a tile's keys, or values
  constexpr int LOADS = 16 * ROW / 1024;  // a wave loads 16 keys, 1 KiB an instruction
  constexpr int LR = 1024 / ROW;          // rows an instruction loads
  typedef typename E::V8 V8;
  __shared__ __align__(1024) char lds[4 * ARR];  // [buffer][keys, values]
  __shared__ int sbad;
  __shared__ uint32_t sodd[AW];  // rows of a tile whose values are not all finite
  const int head = blockIdx.x % a.pool.kv, item = blockIdx.x / a.pool.kv;
  const int64_t room = (int64_t)a.pool.max_pages << a.pool.lp;
  const Work w = find_work(a.st, a.sl, room, item);
  leave_joint(a, w, item);
  if (w.s < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int G = a.sl.group, pairs = w.sp.n * G;
  const int r0 = w.r0 + 32 * wave;
  const int pair = min(r0 + col, pairs - 1), i = pair / G, hq = head * G + pair % G;
  // the last key that the workgroup's, and the wave's, rows see
  int last = w.sp.bad ? w.k0 : w.k1, mine = last;
  if (a.mask == nullptr) {
    last = min(last, w.sp.len + (min(w.r0 + MANY, pairs) - 1) / G + 1);
    mine = min(last, w.sp.len + (min(r0 + 32, pairs) - 1) / G + 1);
  }
  if (r0 >= pairs) mine = w.k0;
  const int clear = clear_of(a, w, last);
  if (threadIdx.x == 0) sbad = w.sp.bad;

  const int steps = last > w.k0 ? (last - w.k0 + 63) / 64 : 0;
  const int *trow = a.pool.table + (size_t)w.s * a.pool.max_pages;
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
  // a lane's pieces of a load: row LR u + lane / (64 / LR), place lane % (64 / LR)
  uint32_t voff[2][LOADS];  // keys, values
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int row = LR * u + lane / (ROW / 16), place = lane % (ROW / 16);
    voff[0][u] = row * ROW + (place ^ (D == 128 ? row & 15 : (row >> 1) & 7)) * 16;
    voff[1][u] = row * ROW + (place ^ (D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1))) * 16;
  }
  bool bad = false;
  auto key_of = [&](int step) { return min(w.k0 + step * 64 + 16 * wave, (last - 1) & ~15); };
  uint32_t id = 0;
  auto fetch = [&](int step) { id = (uint32_t)trow[key_of(step) >> a.pool.lp]; };
  auto load = [&](int step) {
    uint32_t page = __builtin_amdgcn_readfirstlane(id);
    if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
    const size_t at = ((((size_t)page * a.pool.kv + head) << a.pool.lp) +
                       (key_of(step) & ((1 << a.pool.lp) - 1))) * ROW;
    const uint32_t to = base + (step & 1) * 2 * ARR + 16 * wave * ROW;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) exl3::lds_dma16(a.pool.k + at, voff[0][u], to + u * 1024);
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      exl3::lds_dma16(a.pool.v + at, voff[1][u], to + ARR + u * 1024);
  };
  if (steps > 0) {
    fetch(0);
    load(0);
    if (steps > 1) fetch(1);
  }
  u32x4 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.sp.row + i) * a.qs + hq * D + 16 * kk + 8 * h);
    qf[kk] = qf[kk] ^ a.flip;
  }
  // byte addresses in a tile: piece 2 kk + h of row `col`; the values' 4 keys by
  // 4 dims of a transposing read (16 lanes: keys 4 h + 0 .. 3, dims 16 u + 0 .. 15)
  const int ti = lane & 15, tu = (lane >> 4) & 1;
  // (a product's piece number only changes bits that an exclusive or reaches; the
  // compiler may not spread the addresses over registers)
  uint32_t ka = col * ROW + 16 * (h ^ (D == 128 ? col & 15 : (col >> 1) & 7));
  uint32_t va = (4 * h + (ti >> 2)) * ROW + 64 * (D == 128 ? ti >> 2 : ti >> 3) + 32 * tu + 8 * (ti & 3);
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  Soft sf{-INFINITY, 0.0f, E::LIFT, false, a.scale};

  auto turn = [&](int step, auto TAIL) {
    constexpr bool tail = decltype(TAIL)::value;
    const int kb = w.k0 + step * 64;
    const char *tk = lds + (step & 1) * 2 * ARR;
    const char *tv = tk + ARR;
    asm volatile("" : "+v"(ka), "+v"(va));
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        s[b] = E::mma(*reinterpret_cast<const V8 *>(tk + (ka ^ (32 * kk)) + b * 32 * ROW),
                      __builtin_bit_cast(V8, qf[kk]), s[b]);
    }
    // element r of block b: key 32 b + 8 (r / 4) + 4 h + r % 4
    uint64_t seen = ~0ull;
    if constexpr (tail) {
      seen = seen64(a, w.sp, i, kb, last);
      const uint64_t my = seen >> (4 * h);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((uint32_t)(my >> (32 * b)) >> (8 * (r >> 2) + (r & 3)) & 1)) s[b][r] = -INFINITY;
    }
    if (sf.far) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] *= a.scale;
    }
    float hi = larger(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) hi = larger(larger(hi, s[0][r]), s[1][r]);
    hi = larger(hi, exl3::xor_lanes(hi, 32));
    float alpha;
    bool turned;
    if (outgrown<E>(sf, hi * sf.scale, alpha, turned)) {
      if (turned) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] *= a.scale;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    const float by = sf.lift - (sf.ref == -INFINITY ? 0.0f : sf.ref);
    u32x4 pw[4];  // of 16 keys each
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const uint32_t x = pack2<E>(__builtin_amdgcn_exp2f(fmaf(s[b][r], sf.scale, by)),
                                    __builtin_amdgcn_exp2f(fmaf(s[b][r + 1], sf.scale, by)));
        pw[2 * b + (r >> 3)][(r & 7) >> 1] = x;
        sf.sum = E::add2(x, sf.sum);
      }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        typedef __attribute__((address_space(3))) s16x4 *lptr;
        s16x4 v[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          v[c] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lptr)(tv + (va ^ (64 * d)) + (16 * b + 8 * c) * ROW));
        u32x4 av = {__builtin_bit_cast(u32x2, v[0])[0], __builtin_bit_cast(u32x2, v[0])[1],
                    __builtin_bit_cast(u32x2, v[1])[0], __builtin_bit_cast(u32x2, v[1])[1]};
        acc[d] = E::mma(__builtin_bit_cast(V8, av), __builtin_bit_cast(V8, pw[b]), acc[d]);
      }
    if constexpr (tail) {
      for (int x16 = 0; x16 < 4; ++x16)
        for (int odd = __builtin_amdgcn_readfirstlane(sodd[x16]); odd != 0; odd &= odd - 1) {
          const int x = 16 * x16 + __builtin_ctz(odd);
          const uint16_t *row = value_row(a.pool, w.s, head, kb + x, D);
          if (row == nullptr || !(seen >> x & 1)) continue;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const u32x2 v = *reinterpret_cast<const u32x2 *>(row + 32 * d + 8 * y + 4 * h);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[d][4 * y + e] += not_finite<E>(v[e >> 1], e & 1);
            }
        }
    }
  };
  // The wave's 16 rows of a tile's values that reaches behind the context:
  // zeros behind the last key (nobody's), and in place of what is not finite.
  auto mend = [&](int step) {
    const int kb = w.k0 + step * 64 + 16 * wave;
    char *tv = lds + (step & 1) * 2 * ARR + ARR + 16 * wave * ROW;
    uint32_t odd = 0;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int key = kb + LR * u + lane / (ROW / 16);
      u32x4 *p = reinterpret_cast<u32x4 *>(tv + u * 1024 + lane * 16);
      bool bad_value = false;
      if (key >= last) {
        *p = u32x4{0, 0, 0, 0};
      } else if (key >= w.sp.len) {
        u32x4 v = *p;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t f = finite<E>(v[y]);
          bad_value |= f != v[y];
          v[y] = f;
        }
        if (bad_value) *p = v;
      }
      const uint64_t lanes = __ballot(bad_value);
#pragma unroll
      for (int j = 0; j < LR; ++j)
        if (lanes >> (j * (ROW / 16)) & ((1ull << (ROW / 16)) - 1)) odd |= 1u << (LR * u + j);
    }
    if (lane == 0) sodd[wave] = odd;
  };
  // this wave's loads of the tile are in LDS, and so are, behind the barrier,
  // the others'; all have read the tile before, whose buffer is loaded next
  auto begin = [&](int step) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + 1 < steps) {
      load(step + 1);
      if (step + 2 < steps) fetch(step + 2);
    }
  };
  const int whole = max(0, clear - w.k0) / 64;  // tiles that every row sees whole
  int step = 0;
  for (; step < whole; ++step) {
    begin(step);
    if (r0 < pairs) turn(step, std::false_type{});
  }
  for (; step < steps; ++step) {
    begin(step);
    mend(step);
    lds_barrier();
    if (w.k0 + step * 64 < mine) turn(step, std::true_type{});
  }
  __syncthreads();
  if (bad) sbad = 1;
  __syncthreads();
  if (sf.far) {  // lifted as all other sums are
    const float by = __builtin_amdgcn_exp2f(E::LIFT - sf.lift);
    sf.sum *= by;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= by;
  }
  float l = sf.sum;
  l += exl3::xor_lanes(l, 32);
  if (sbad) l = __builtin_nanf("");
  if (r0 + col >= pairs) return;
  // a lane's dims: 32 d + 8 x + 4 h + 0 .. 3
  if (w.splits == 1) {
    const float inv = 1.0f / l;
    uint16_t *dst = a.out + (int64_t)(w.sp.row + i) * a.os + hq * D + 4 * h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        u32x2 b = {pack2<E>(acc[d][4 * x] * inv, acc[d][4 * x + 1] * inv),
                   pack2<E>(acc[d][4 * x + 2] * inv, acc[d][4 * x + 3] * inv)};
        if (l == 0.0f) b = u32x2{0, 0};
        *reinterpret_cast<u32x2 *>(dst + 32 * d + 8 * x) = b;
      }
  } else if (w.place * a.pool.kv + head < a.slots) {
    const size_t row = ((size_t)w.place * a.pool.kv + head) * MANY + 32 * wave + col;
    float *dst = a.part + row * D + 4 * h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f32x4 *>(dst + 32 * d + 8 * x) =
            f32x4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]};
    float *ml = a.part + (size_t)a.slots * MANY * D + row * 2;
    if (h == 0) ml[0] = sf.ref, ml[1] = l;
  }
}

// The items of a tile joined, 16 pairs a workgroup, 16 lanes a group of threads.
// Where the tile has fewer pairs (one token's query heads), several groups take a
// share of a pair's items each.  A group's lanes hold 16 items' references and
// sums, so the loop over the items has no load that another waits for.
template <typename E, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a) {
  constexpr int VH = D / 16;
  typedef typename std::conditional<VH == 8, u32x4, u32x2>::type VV;
  __shared__ float so[16][D];
  __shared__ float sm[16][2];
  const int rows = 1 << a.sl.tile, parts = rows / 16;
  const int head = blockIdx.x % a.pool.kv, tile = blockIdx.x / a.pool.kv / parts;
  const Joint w = a.joint[1 + tile];
  if (tile >= a.joint[0].row) return;
  const int row0 = 16 * ((blockIdx.x / a.pool.kv) % parts);
  const int left = w.pairs - w.r0 - row0;
  if (left <= 0) return;
  const int n = min(w.splits, a.slots / a.pool.kv - w.first);
  // log2 of the pairs' groups (shares for more than 8 items, what a group has in
  // flight at once); a group's pair and its share of the items
  const int lp = left >= 16 || n <= 8 ? 4 : left > 1 ? 32 - __builtin_clz(left - 1) : 0;
  const int G = a.sl.group, c = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int row = row0 + (group & ((1 << lp) - 1)), share = group >> lp;
  const int p = w.r0 + row;
  const float *ml = a.part + (size_t)a.slots * rows * D;
  const int each = (n + (16 >> lp) - 1) >> (4 - lp);
  const int begin = min(n, share * each), end = p < w.pairs ? min(n, begin + each) : begin;
  float top = -INFINITY, o[VH], l = 0.0f;
#pragma unroll
  for (int m = 0; m < VH; ++m) o[m] = 0.0f;
  for (int x0 = begin; x0 < end; x0 += 16) {
    // 16 items a round, one a lane; the first 8 items' sums are on their way before
    // the references are
    const int e = min(16, end - x0);
    const float *src = a.part + (((size_t)(w.first + x0) * a.pool.kv + head) * rows + row) * D + VH * c;
    const size_t stride = (size_t)a.pool.kv * rows * D;
    f32x4 y[8][VH / 4];
    auto fetch = [&](int x) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int m = 0; m < VH / 4; ++m)
          y[u][m] = *reinterpret_cast<const f32x4 *>(src + min(x + u, e - 1) * stride + 4 * m);
    };
    fetch(0);
    float ref = -INFINITY, sum = 0.0f;
    if (x0 + c < end) {
      const size_t slot = (size_t)(w.first + x0 + c) * a.pool.kv + head;
      const f32x2 v = *reinterpret_cast<const f32x2 *>(ml + (slot * rows + row) * 2);
      ref = v[0], sum = v[1];
    }
    float hi = ref;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) hi = fmaxf(hi, __shfl_xor(hi, m, 16));
    const float now = fmaxf(top, hi), to = now == -INFINITY ? 0.0f : now;
    const float alpha = __builtin_amdgcn_exp2f(top - to), f = __builtin_amdgcn_exp2f(ref - to);
    top = now;
    float part = f * sum;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) part += __shfl_xor(part, m, 16);
    l = l * alpha + part;
#pragma unroll
    for (int m = 0; m < VH; ++m) o[m] *= alpha;
    for (int x = 0; x < e; x += 8) {
      if (x > 0) fetch(x);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float fx = __shfl(f, min(x + u, 15), 16);
        if (x + u < e) {
#pragma unroll
          for (int m = 0; m < VH; ++m) o[m] += fx * y[u][m >> 2][m & 3];
        }
      }
    }
  }
  if (lp < 4) {  // the shares, in their order
#pragma unroll
    for (int m = 0; m < VH; ++m) so[group][VH * c + m] = o[m];
    if (c == 0) sm[group][0] = top, sm[group][1] = l;
    __syncthreads();
    if (share > 0) return;
    float all = top;
    for (int x = 1; x < 16 >> lp; ++x) all = fmaxf(all, sm[(x << lp) + group][0]);
    const float ref = all == -INFINITY ? 0.0f : all;
    l = 0.0f;
#pragma unroll
    for (int m = 0; m < VH; ++m) o[m] = 0.0f;
    for (int x = 0; x < 16 >> lp; ++x) {
      const int from = (x << lp) + group;
      const float f = __builtin_amdgcn_exp2f(sm[from][0] - ref);
      l += f * sm[from][1];
#pragma unroll
      for (int m = 0; m < VH; ++m) o[m] += f * so[from][VH * c + m];
    }
  }
  if (p >= w.pairs) return;
  const float inv = 1.0f / l;
  uint16_t *dst = a.out + (int64_t)(w.row + p / G) * a.os + (head * G + p % G) * D + VH * c;
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
// all rows are read before any is written.  A round holds MOVES rows of a head a
// thread group, so a usual path is one round: its time is a chain of loads
// (tree, table, rows), not bytes.
constexpr int MOVES = 4;

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
  // slots of the rows that move, where child and said were: -1 for the others
  for (int j = threadIdx.x; j < c; j += 256) {
    const int from = way[j] != j ? slot_of(pool, s, sp.len + way[j]) : -1;
    const int to = from >= 0 ? slot_of(pool, s, sp.len + j) : -1;
    child[j] = to >= 0 ? from : -1;
    said[j] = to;
  }
  __syncthreads();
  char *data = (blockIdx.y & 1 ? pool.v : pool.k) + (size_t)(blockIdx.y >> 1) * layer_bytes;
  const int lanes = row_bytes / 16;  // of a row of one head
  const int per = 256 / lanes;       // rows of one head at once
  const int x = threadIdx.x % lanes, y = threadIdx.x / lanes;
  const int todo = c * pool.kv, m = (1 << pool.lp) - 1;
  for (int b = 0; b < todo; b += MOVES * per) {
    u32x4 val[MOVES];
    char *to[MOVES];
#pragma unroll
    for (int u = 0; u < MOVES; ++u) {
      const int e = b + u * per + y, j = min(e, todo - 1) / pool.kv, h = e % pool.kv;
      const int from = e < todo ? child[j] : -1, dst = said[j];
      to[u] = nullptr;
      if (from >= 0) {
        const size_t src = (((size_t)(from >> pool.lp) * pool.kv + h) << pool.lp) + (from & m);
        val[u] = *reinterpret_cast<const u32x4 *>(data + src * row_bytes + 16 * x);
        to[u] = data + ((((size_t)(dst >> pool.lp) * pool.kv + h) << pool.lp) + (dst & m)) * row_bytes + 16 * x;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MOVES; ++u)
      if (to[u] != nullptr) *reinterpret_cast<u32x4 *>(to[u]) = val[u];
  }
}

// ---------------------------------------------------------------- page copies

// 16 bytes a thread, and no more: as many loads in flight as the CUs hold, each
// written as it comes (2, 4, 8 of them a thread: 200 pages of 8 layers, 839 MB
// moved, 158, 164, 218 us against 145; one page of 36 layers 4.5, 5.0, 6.9
// against 4.6).  5.8 TB/s of reads and writes: a large copy's rate and more,
// the Infinity Cache taking part.
constexpr int COPY_PAIRS = 256;  // a launch's pairs travel in its arguments
struct Pairs {
  int32_t src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ __launch_bounds__(256) void copy_pages_kernel(char *k, char *v, size_t layer_bytes,
                                                         size_t page_bytes, Pairs pairs) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (i >= page_bytes) return;
  char *data = (blockIdx.z & 1 ? v : k) + (size_t)(blockIdx.z >> 1) * layer_bytes + i;
  *reinterpret_cast<u32x4 *>(data + (size_t)pairs.dst[blockIdx.y] * page_bytes) =
      *reinterpret_cast<const u32x4 *>(data + (size_t)pairs.src[blockIdx.y] * page_bytes);
}

// ----------------------------------------------------------------- host side

// Tiles of a kv head that the rows can make: a sequence's last one may be short.
int64_t most_tiles(const exl3p_rows *r, const Split &sl) {
  return ((int64_t)r->rows * sl.group >> sl.tile) + r->seqs;
}

// The tile by the most pairs that a sequence has, and how many items its keys are
// split into; n workgroups of a kv head fill the CUs with two each.  With few
// tiles one round holds all items (n less the tiles, since a tile's items are
// rounded up); with more, items are several rounds, for sequences of unlike
// lengths: 4 n of few pairs, 1.5 n of 128, whose joins cost more.  A tile stays
// whole up to 0.9 or 1.4 times a workgroup's share of all units and some more (128
// pairs 1 + 8 and 1.8 + 8 the same, 2.5 + 8 prompts of 300 over 4000 92 us -> 102;
// few pairs 1.4 + 8 one row over 300 keys 10.1 -> 11.2, 128 over up to 4096 keys
// 205 -> 215).
Split split_of(const exl3p_cache *c, const exl3p_rows *r, int32_t heads) {
  Split sl;
  sl.group = heads / c->kv_heads;
  const int64_t pairs = (int64_t)r->max_rows * sl.group;
  sl.tile = log2_of(pairs <= 16 ? 16 : pairs <= FEW ? FEW : MANY);
  sl.least = pairs <= FEW ? 32 * AW / 64 : 4;
  const int n = (2 * device_cus() + c->kv_heads - 1) / c->kv_heads;
  sl.round = (float)n;
  sl.few = (float)(pairs <= FEW ? n / 2 : 3 * n / 8);
  sl.most = (float)(pairs <= FEW ? 4 * n : n + n / 2);
  sl.whole = (pairs <= FEW ? 0.9f : 1.4f) / (float)n;
  sl.more = pairs <= FEW ? 4.5f : 8.0f;
  return sl;
}

// Items of a kv head, and tiles that are split (each has more units than an item
// has at most, so they are fewer than the target).
int64_t most_items(const exl3p_rows *r, const Split &sl) {
  const int64_t tiles = most_tiles(r, sl);
  return (float)tiles <= sl.few ? (int64_t)sl.round : tiles + (int64_t)sl.most;
}
int64_t most_split(const exl3p_rows *r, const Split &sl) {
  const int64_t tiles = most_tiles(r, sl);
  const int64_t target = (float)tiles <= sl.few ? (int64_t)sl.round : (int64_t)sl.most;
  return tiles < target ? tiles : target;
}
// Items of those: only they leave sums for the join, so that the scratch does not
// grow with the rows (131072 rows of 32 over 8 heads: 102 MB, for all items 2.2 GB).
int64_t most_parts(const exl3p_rows *r, const Split &sl) {
  return (float)most_tiles(r, sl) <= sl.few ? (int64_t)sl.round
                                            : (int64_t)sl.most + most_split(r, sl);
}

}  // namespace

extern "C" {

exl3_verdict exl3p_tree_plan(const exl3p_cache *c, const exl3p_rows *r, const int32_t *parent,
                             int32_t *pos, int32_t *slot, uint64_t *mask, int32_t words,
                             exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_rows(c, r));
  EXL3P_TRY(check_mask(r, mask, words));
  if (parent != nullptr && r->max_rows > EXL3P_TREE_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedTree: over 1024 rows of a sequence");
  if (r->rows == 0) return OK;
  if (pos == nullptr || slot == nullptr) return refuse(EXL3_FAILED, "PagedPlan: a missing array");
  const int64_t n = (int64_t)r->rows * 4;
  EXL3P_TRY(check_apart({array(pos, n), array(slot, n), array(mask, 2 * n * words)},
                        {array(r->cu, 4 * ((int64_t)r->seqs + 1)), array(r->len, 4 * (int64_t)r->seqs),
                         array(parent, n), table_of(c)}));
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
  if (rows > GRID_MAX) return refuse(EXL3_TOO_LARGE, "PagedRows: 2^24 rows or more in one call");
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
  // workgroups take rows and heads in any order: what one writes no other reads
  const Span2D out = matrix(q_out, out_stride, wq, rows), in = matrix(q, q_stride, wq, rows);
  const Span2D reads[] = {matrix(k, k_stride, wk, rows), matrix(v, v_stride, wk, rows),
                          array(q_norm, c->dim * 2),     array(k_norm, c->dim * 2),
                          array(pos, (int64_t)rows * 4), array(slot, (int64_t)rows * 4)};
  const Pool pool = pool_of(c, layer);
  const Span2D kv[] = {array(pool.k, layer_bytes(c)), array(pool.v, layer_bytes(c))};
  if (!(q_out == q && (out_stride == q_stride || rows == 1)) && meet(out, in))
    return refuse(EXL3_UNSUPPORTED, "PagedOverlap: q_out over q, and not q itself");
  for (const Span2D &x : reads)
    if (meet(out, x)) return refuse(EXL3_UNSUPPORTED, "PagedOverlap: q_out over another input");
  for (const Span2D &y : kv) {
    if (meet(out, y) || meet(in, y))
      return refuse(EXL3_UNSUPPORTED, "PagedOverlap: q or q_out over the layer's pages");
    for (const Span2D &x : reads)
      if (meet(x, y)) return refuse(EXL3_UNSUPPORTED, "PagedOverlap: an input over the layer's pages");
  }
  if ((q_norm != nullptr || k_norm != nullptr) && !(eps >= 0.0f && eps < INFINITY))
    return refuse(EXL3_UNSUPPORTED, "PagedEps: a norm's eps is finite and not below 0");
  if (meet(kv[0], kv[1])) return refuse(EXL3_UNSUPPORTED, "PagedOverlap: keys over values");
  Rates rates{};
  const double ratio = pow(theta, -2.0 / c->dim);
  double turn = 1.0 / 6.283185307179586476925287;
  for (int i = 0; i < c->dim / 2; ++i, turn *= ratio) rates.turns[i] = turn;
  // A wave's angles serve all heads that it takes: one workgroup a row, or, where
  // rows are few, as many as the heads fill (8 rows 4.7 -> 3.4 us, 256 5.2 -> 4.3;
  // 1500 rows 10.7 with one, 12.2 with all).
  const int all = (heads + 2 * c->kv_heads) * c->dim / 512;  // waves of a row's heads
  const int y = rows < 512 ? (all + 3) / 4 : 1;
  return by_type(c, [&](auto e, auto d) {
    hipLaunchKernelGGL((qkv_append_kernel<decltype(e), d>), dim3(rows, y > 1 ? y : 1), dim3(256), 0,
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
  const Split sl = split_of(c, r, heads);
  return (size_t)(1 + most_split(r, sl)) * sizeof(Joint) +
         (size_t)most_parts(r, sl) * c->kv_heads * ((size_t)1 << sl.tile) * (c->dim + 2) * sizeof(float);
}

exl3_verdict exl3p_attend(const exl3p_cache *c, int32_t layer, const exl3p_rows *r, int32_t heads,
                          const void *q, int64_t q_stride, const uint64_t *mask, int32_t words,
                          float scale, void *out, int64_t out_stride, void *scratch,
                          size_t scratch_bytes, exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_layer(c, layer));
  EXL3P_TRY(check_rows(c, r));
  EXL3P_TRY(check_heads(c, heads));
  EXL3P_TRY(check_mask(r, mask, words));
  if (!(fabsf(scale) * 1.4426950408889634f < INFINITY))
    return refuse(EXL3_UNSUPPORTED, "PagedScale: finite, also times log2(e)");
  if (r->rows == 0 || r->seqs == 0 || r->max_rows == 0) return OK;
  const int64_t wq = (int64_t)heads * c->dim;
  EXL3P_TRY(check_matrix(q, q_stride, wq));
  EXL3P_TRY(check_matrix(out, out_stride, wq));
  const Split sl = split_of(c, r, heads);
  if ((int64_t)r->max_rows * sl.group > INT32_MAX / 2 ||
      most_items(r, sl) * c->kv_heads > GRID_MAX ||
      most_split(r, sl) * c->kv_heads << (sl.tile - 4) > GRID_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedAttend: too many rows and heads for one call");
  if (scratch == nullptr || !aligned(scratch, 16) ||
      scratch_bytes < exl3p_attend_scratch_bytes(c, r, heads))
    return refuse(EXL3_FAILED, "PagedScratch: below exl3p_attend_scratch_bytes, or not aligned");
  // a workgroup reads its pairs' q before it writes their out, the join writes when
  // all have read: out may be q
  const Span2D to = matrix(out, out_stride, wq, r->rows), from = matrix(q, q_stride, wq, r->rows),
               held = array(scratch, (int64_t)exl3p_attend_scratch_bytes(c, r, heads));
  const Pool pool = pool_of(c, layer);
  EXL3P_TRY(check_apart({to, held}, {array(pool.k, layer_bytes(c)), array(pool.v, layer_bytes(c)),
                                     array(mask, 8 * (int64_t)r->rows * words),
                                     array(r->cu, 4 * ((int64_t)r->seqs + 1)),
                                     array(r->len, 4 * (int64_t)r->seqs), table_of(c)}));
  if (meet(held, from) || (!(out == q && (out_stride == q_stride || r->rows == 1)) && meet(to, from)))
    return refuse(EXL3_UNSUPPORTED, "PagedOverlap: scratch over q, or out over q and not q itself");
  AttnArgs a;
  a.pool = pool, a.st = step_of(r), a.sl = sl;
  a.q = static_cast<const uint16_t *>(q), a.qs = q_stride, a.mask = mask, a.words = words;
  // at least f32's smallest, so that a hidden key's -inf times it stays -inf
  a.scale = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.17549435e-38f);
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.out = static_cast<uint16_t *>(out), a.os = out_stride;
  a.joint = static_cast<Joint *>(scratch), a.joints = (int)most_split(r, sl);
  a.part = reinterpret_cast<float *>(a.joint + 1 + most_split(r, sl));
  a.slots = (int)(most_parts(r, sl) * c->kv_heads);
  const dim3 items((unsigned)(most_items(r, sl) * c->kv_heads));
  const hipStream_t st = static_cast<hipStream_t>(s);
  return by_type(c, [&](auto e, auto d) {
    if (sl.tile == 4)
      hipLaunchKernelGGL((attend_few_kernel<decltype(e), d, 1>), items,
                         dim3(64 * AW), 0, st, a);
    else if (sl.tile == 5)
      hipLaunchKernelGGL((attend_few_kernel<decltype(e), d, 2>), items,
                         dim3(64 * AW), 0, st, a);
    else
      hipLaunchKernelGGL((attend_many_kernel<decltype(e), d>), items,
                         dim3(64 * AW), 0, st, a);
    hipLaunchKernelGGL((attend_join_kernel<decltype(e), d>),
                       dim3((unsigned)(most_split(r, sl) * c->kv_heads << (sl.tile - 4))), dim3(256),
                       0, st, a);
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
  // every workgroup of a sequence walks its tree, whatever the others have written
  const int64_t n = (int64_t)r->seqs * 4, t = (int64_t)r->rows * 4;
  const int64_t pool = (int64_t)layer_bytes(c) * c->layers;
  EXL3P_TRY(check_apart({array(path, n * max_path), array(count, n), array(next, n),
                         array(new_len, n), array(c->k, pool), array(c->v, pool)},
                        {array(r->cu, n + 4), array(r->len, n), array(parent, t), array(ids, t),
                         array(target, t), table_of(c)}));
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
  const unsigned wgs = (unsigned)((bytes + 4095) / 4096);
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
