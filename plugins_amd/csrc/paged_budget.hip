// paged_budget.hip -- a budget of keys for a paged KV cache (include/exl3_paged.h)
// for MI355X (gfx950, wave64): the attention weight that every key gets, and
// eviction of the keys that have least of it.
#include "paged_common.h"

namespace {

// ------------------------------------------------------------ weights of keys

struct WeighArgs {
  Pool pool;
  Step st;
  int group, window;
  const uint16_t *q;
  int64_t qs;
  const uint64_t *mask;
  int words;
  float scale;  // log2(e) times the scale: weights are powers of two
  float decay;
  const int32_t *base;
  float *score;
  int room;
  float target;  // items of a kv head
  float least;   // 64-key units of one, at least
  int slots;     // items * kv that part holds
  f32x2 *part;   // [items * kv][TILE]: an item's reference and sum of each pair
  f32x2 *ref;    // [kv][rows * group]: a pair's reference, and one over its sum
  float *t;      // few pairs: [seqs][kv][most][wide] scores, in place of ref
  int most, wide;
};

constexpr int WW = 4;       // waves of a workgroup
constexpr int TILE = 128;   // pairs of a row and a query head that an item has
constexpr int FEW = 16;     // or, where no sequence has more, this many
constexpr int KEYS = 128;   // keys that a workgroup adds up weights for
constexpr float SLACK = 4.0f;  // a reference follows its maximum in steps of more (powers of two)

// A sequence's rows that count and its keys.
struct Watch {
  int row, n, len;  // as Span
  int lo;           // the first row that counts
  int pairs;        // of a kv head; 0: nothing to do
  int keys;
  bool back;
};
__device__ __forceinline__ Watch watch_of(const WeighArgs &a, int s) {
  const Span sp = span_of(a.st, s, (int64_t)a.pool.max_pages << a.pool.lp);
  Watch w{sp.row, sp.n, sp.len, 0, 0, 0, sp.back};
  if (sp.bad || sp.n == 0 || (int64_t)sp.len + sp.n > a.room) return w;
  const int rows = a.window > 0 ? min(sp.n, a.window) : sp.n;
  w.lo = sp.n - rows;
  w.pairs = rows * a.group;
  w.keys = sp.len + sp.n;
  return w;
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int scan(int v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int y = __shfl_up(v, m);
    if ((int)(threadIdx.x & 63) >= m) v += y;
  }
  return v;
}

enum Kind { ITEM, PAIRS, SPAN };  // (tile, part of the keys); tile; KEYS keys
struct Find {
  int s;       // -1: nothing
  int u, j;    // tile of pairs, part of the keys
  int first;   // the tile's first item
  int parts;   // items of a tile
  int each;    // 64-key units of one
  Watch w;
};

// Number x among the sequences' items, tiles or spans of keys.  A tile of u units of
// 64 keys has ceil(u / c) items, c the units of all tiles over the target, and
// what a 32-bit sum may be short of: items are never more than target + tiles.
template <Kind KIND>
__device__ __forceinline__ Find find(const WeighArgs &a, int x) {
  const int lane = threadIdx.x & 63;
  Find f;
  f.s = -1;
  Watch w{};
  float units = 0.0f;
  bool back = false;
  for (int s = lane; s < a.st.seqs; s += 64) {
    w = watch_of(a, s);
    back |= w.back;
    units += (float)((w.pairs + TILE - 1) / TILE) * (float)((w.keys + 63) >> 6);
  }
  if (__ballot(back) != 0) return f;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) units += exl3::xor_lanes(units, m);
  const int chunk = __builtin_amdgcn_readfirstlane(
      (int)fminf(fmaxf(ceilf(units * (1.0f + 0x1p-12f) / a.target), a.least), (float)(1 << 25)));
  int before = 0, items = 0;
  for (int s0 = 0; s0 < a.st.seqs; s0 += 64) {
    const int s = s0 + lane;
    int tiles = 0, ns = 0, each = 1, count = 0;
    if (s < a.st.seqs) {
      if (a.st.seqs > 64) w = watch_of(a, s);
      if (w.pairs > 0) {
        const int u = (w.keys + 63) >> 6;
        tiles = (w.pairs + TILE - 1) / TILE;
        ns = (u + chunk - 1) / chunk;
        each = (u + ns - 1) / ns;  // the last items may be empty
        count = KIND == ITEM ? tiles * ns : KIND == PAIRS ? tiles : (w.keys + KEYS - 1) / KEYS;
      }
    }
    const int ct = scan(count), it = KIND == SPAN ? 0 : scan(tiles * ns);
    const uint64_t past = __ballot(before + ct > x);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int y = x - before - of(ct - count), nt = of(tiles), n_s = of(ns);
      f.s = s0 + l;
      f.w = Watch{of(w.row), of(w.n), of(w.len), of(w.lo), of(w.pairs), of(w.keys), false};
      f.parts = n_s;
      f.each = of(each);
      // tiles that read the same keys side by side
      f.j = KIND == ITEM ? y / nt : 0;
      f.u = KIND == ITEM ? y - f.j * nt : y;
      f.first = items + of(it - tiles * ns) + f.u * n_s;
      return f;
    }
    before += __builtin_amdgcn_readlane(ct, 63);
    if (KIND != SPAN) items += __builtin_amdgcn_readlane(it, 63);
  }
  return f;
}

// Which of keys kb .. kb + 63 row i of a sequence sees, a bit a key.
__device__ __forceinline__ uint64_t seen64(const WeighArgs &a, const Watch &w, int i, int kb) {
  const int lim = a.mask == nullptr ? w.len + i + 1 : w.keys;
  if (lim <= kb) return 0;
  uint64_t v = lim - kb >= 64 ? ~0ull : ~0ull >> (64 - (lim - kb));
  if (a.mask != nullptr && kb + 64 > w.len) {
    const uint64_t *m = a.mask + (size_t)(w.row + i) * a.words;
    const int j = kb - w.len;  // the first key's number among the rows
    const uint64_t lo = j >= 0 && (j >> 6) < a.words ? m[j >> 6] >> (j & 63) : 0;
    const int next = j >= 0 ? (j >> 6) + 1 : 0, by = j >= 0 ? 64 - (j & 63) : -j;
    const uint64_t hi = by < 64 && next < a.words ? m[next] << by : 0;
    v &= j >= 0 ? lo | hi : hi | ~(~0ull << -j);
  }
  return v;
}

// 16 bytes a lane from its own address to LDS at `lds` + 16 * lane.
__device__ __forceinline__ void lds_dma16_at(const void *p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p)
               : "memory");
}

// The places of a row's 16-byte pieces in LDS: those of one number of 16 rows lie in
// 16 places of the banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}

// A score that a row does not see, where scores are kept: its weight is none, also
// where the row's sum is NaN.
constexpr float UNSEEN = -0x1.fffffep127f;

// Two parts of a pair's keys: the reference and the sum of weights of both.
__device__ __forceinline__ void join(float &ref, float &sum, float other, float more) {
  const float now = __builtin_elementwise_maximum(ref, other), from = now == -INFINITY ? 0.0f : now;
  sum = sum * __builtin_amdgcn_exp2f(ref - from) + more * __builtin_amdgcn_exp2f(other - from);
  ref = now;
}
// What the second pass wants of them: a pair that sees nothing has no weights, a NaN
// stays in the factor.
__device__ __forceinline__ f32x2 ended(float ref, float sum) {
  return f32x2{ref == -INFINITY || ref != ref ? 0.0f : ref,
               sum == 0.0f ? 0.0f : ref != ref ? ref : 1.0f / sum};
}

// The first pass: each pair's reference (its largest score, or less by SLACK at
// most) and the sum of its weights over an item's keys.  128 pairs a workgroup, 32
// a wave; tiles of 64 keys pass through LDS, the next loaded while one is used.
// Scores are S^T = K q^T (rows keys, columns pairs): a lane holds 32 keys' scores
// of one pair.
template <typename E, int D>
__global__ __launch_bounds__(64 * WW, 2) void weigh_sums_kernel(WeighArgs a) {
  constexpr int KK = D / 16, ROW = D * 2, ARR = 64 * ROW;
  constexpr int LOADS = 16 * ROW / 1024, LR = 1024 / ROW;
  typedef typename E::V8 V8;
  __shared__ __align__(1024) char lds[2 * ARR];
  __shared__ int sbad;
  const int head = blockIdx.x % a.pool.kv;
  const Find f = find<ITEM>(a, blockIdx.x / a.pool.kv);
  if (f.s < 0) return;
  const Watch &w = f.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int G = a.group;
  const int r0 = f.u * TILE + 32 * wave;
  const int pair = min(r0 + col, w.pairs - 1), i = w.lo + pair / G, hq = head * G + pair % G;
  const int k0 = (int)min((int64_t)f.j * f.each * 64, (int64_t)w.keys);
  const int k1 = (int)min((int64_t)k0 + (int64_t)f.each * 64, (int64_t)w.keys);
  // the last key that the workgroup's, and the wave's, rows see
  int last = k1, mine = k1;
  if (a.mask == nullptr) {
    last = min(last, w.len + w.lo + (min(f.u * TILE + TILE, w.pairs) - 1) / G + 1);
    mine = min(last, w.len + w.lo + (min(r0 + 32, w.pairs) - 1) / G + 1);
  }
  if (r0 >= w.pairs) mine = k0;
  // keys below this every row of the wave sees
  const int clear = a.mask == nullptr ? w.len + w.lo + r0 / G + 1 : w.len;
  if (threadIdx.x == 0) sbad = 0;
  const int steps = last > k0 ? (last - k0 + 63) / 64 : 0;
  const int *trow = a.pool.table + (size_t)f.s * a.pool.max_pages;
  const uint32_t lbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
  uint32_t voff[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int row = LR * u + lane / (ROW / 16), place = lane % (ROW / 16);
    voff[u] = row * ROW + (place ^ swizzle<D>(row)) * 16;
  }
  bool bad = false;
  auto key_of = [&](int step) { return min(k0 + step * 64 + 16 * wave, (last - 1) & ~15); };
  uint32_t id = 0;
  auto fetch = [&](int step) { id = (uint32_t)trow[key_of(step) >> a.pool.lp]; };
  auto load = [&](int step) {
    uint32_t page = __builtin_amdgcn_readfirstlane(id);
    if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
    const size_t at = ((((size_t)page * a.pool.kv + head) << a.pool.lp) +
                       (key_of(step) & ((1 << a.pool.lp) - 1))) * ROW;
    const uint32_t to = lbase + (step & 1) * ARR + 16 * wave * ROW;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) exl3::lds_dma16(a.pool.k + at, voff[u], to + u * 1024);
  };
  if (steps > 0) {
    fetch(0);
    load(0);
    if (steps > 1) fetch(1);
  }
  u32x4 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.row + i) * a.qs + hq * D + 16 * kk + 8 * h);
  uint32_t ka = col * ROW + 16 * (h ^ swizzle<D>(col));
  float ref = -INFINITY, sum = 0.0f;
  for (int step = 0; step < steps; ++step) {
    // this wave's loads of the tile are in LDS, and so are, behind the barrier, the
    // others'; all have read the tile before, whose buffer is loaded next
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + 1 < steps) {
      load(step + 1);
      if (step + 2 < steps) fetch(step + 2);
    }
    const int kb = k0 + step * 64;
    if (kb >= mine) continue;
    const char *tk = lds + (step & 1) * ARR;
    asm volatile("" : "+v"(ka));
    f32x16 t[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) t[b][r] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        t[b] = E::mma(*reinterpret_cast<const V8 *>(tk + (ka ^ (32 * kk)) + b * 32 * ROW),
                      __builtin_bit_cast(V8, qf[kk]), t[b]);
#pragma unroll
      for (int r = 0; r < 16; ++r) t[b][r] *= a.scale;
    }
    if (kb + 64 > clear || kb + 64 > last) {
      // element r of block b: key 32 b + 8 (r / 4) + 4 h + r % 4
      uint64_t my = seen64(a, w, i, kb);
      if (last - kb < 64) my &= ~0ull >> (64 - (last - kb));
      my >>= 4 * h;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((uint32_t)(my >> (32 * b)) >> (8 * (r >> 2) + (r & 3)) & 1)) t[b][r] = -INFINITY;
    }
    float hi = t[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) hi = __builtin_elementwise_maximum(hi, t[b][r]);
    if (__ballot(!(hi - ref <= SLACK)) != 0) {
      const float now = __builtin_elementwise_maximum(ref, hi);
      sum *= __builtin_amdgcn_exp2f(ref - (now == -INFINITY ? 0.0f : now));
      ref = now;
    }
    const float from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(t[b][r] - from);
  }
  __syncthreads();
  if (bad) sbad = 1;
  __syncthreads();
  // the two halves of a pair's keys
  join(ref, sum, exl3::xor_lanes(ref, 32), exl3::xor_lanes(sum, 32));
  if (sbad) sum = __builtin_nanf("");
  const int64_t slot = (int64_t)(f.first + f.j) * a.pool.kv + head;
  if (h == 0 && r0 + col < w.pairs && slot < a.slots) a.part[slot * TILE + 32 * wave + col] = f32x2{ref, sum};
}

// A tile's items joined, a pair a thread.
__global__ __launch_bounds__(TILE) void weigh_join_kernel(WeighArgs a) {
  const int head = blockIdx.x % a.pool.kv;
  const Find f = find<PAIRS>(a, blockIdx.x / a.pool.kv);
  const int pair = f.u * TILE + (int)threadIdx.x;
  if (f.s < 0 || pair >= f.w.pairs) return;
  float ref = -INFINITY, sum = 0.0f;
  for (int j = 0; j < f.parts; ++j) {
    const int64_t slot = (int64_t)(f.first + j) * a.pool.kv + head;
    if (slot >= a.slots) break;
    const f32x2 v = a.part[slot * TILE + threadIdx.x];
    join(ref, sum, v[0], v[1]);
  }
  a.ref[(int64_t)head * a.st.rows * a.group + (int64_t)(f.w.row + f.w.lo) * a.group + pair] = ended(ref, sum);
}

// The second pass: KEYS keys a workgroup, 32 a wave in registers; the pairs pass
// through LDS 32 at a time, the next loaded while one tile is used.  A lane adds
// up the weights of 16 keys over the pairs of its column; the columns join at the end.
template <typename E, int D>
__global__ __launch_bounds__(64 * WW, 2) void weigh_keys_kernel(WeighArgs a) {
  constexpr int KK = D / 16, ROW = D * 2, ARR = 32 * ROW;
  constexpr int LOADS = 8 * ROW / 1024, LR = 1024 / ROW;
  typedef typename E::V8 V8;
  __shared__ __align__(1024) char lds[2 * ARR];
  const int head = blockIdx.x % a.pool.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int G = a.group;
  const uint32_t lbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
  uint32_t qa = col * ROW + 16 * (h ^ swizzle<D>(col));
  for (int x = blockIdx.x / a.pool.kv;; x += gridDim.x / a.pool.kv) {
    const Find f = find<SPAN>(a, x);
    if (f.s < 0) return;
    const Watch &w = f.w;
    const int kb0 = f.u * KEYS, kb = kb0 + 32 * wave;
    // pairs before this one see no key of the span
    const int p0 = a.mask == nullptr ? max(0, kb0 - w.len - w.lo) * G & ~31 : 0;
    const int steps = (w.pairs - p0 + 31) / 32;
    auto load = [&](int step) {
      const uint32_t to = lbase + (step & 1) * ARR + 8 * wave * ROW;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int row = 8 * wave + LR * u + lane / (ROW / 16), place = lane % (ROW / 16);
        const int pair = min(p0 + step * 32 + row, w.pairs - 1), i = pair / G;
        lds_dma16_at(a.q + (w.row + w.lo + i) * a.qs + (head * G + pair - i * G) * D +
                         (place ^ swizzle<D>(row)) * 8,
                     to + u * 1024);
      }
    };
    if (steps > 0) load(0);
    // (a key behind the last, or of no page, stands for one that is there: its
    // weights are not kept, or are NaN)
    const int key = min(kb + col, w.keys - 1);
    const int sl = max(slot_of(a.pool, f.s, key), 0);
    const char *kp = a.pool.k + ((((size_t)(sl >> a.pool.lp) * a.pool.kv + head) << a.pool.lp) +
                                 (sl & ((1 << a.pool.lp) - 1))) * ROW + 16 * h;
    u32x4 kf[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) kf[kk] = *reinterpret_cast<const u32x4 *>(kp + 32 * kk);
    const f32x2 *refs = a.ref + (int64_t)head * a.st.rows * G + (int64_t)(w.row + w.lo) * G;
    float acc[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
    for (int step = 0; step < steps; ++step) {
      const int p = p0 + step * 32, pair = min(p + col, w.pairs - 1);
      const f32x2 ref = refs[pair];
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (step + 1 < steps) load(step + 1);
      const char *tq = lds + (step & 1) * ARR;
      asm volatile("" : "+v"(qa));
      f32x16 t;
#pragma unroll
      for (int r = 0; r < 16; ++r) t[r] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        t = E::mma(__builtin_bit_cast(V8, kf[kk]),
                   *reinterpret_cast<const V8 *>(tq + (qa ^ (32 * kk))), t);
      const bool whole = p + 32 <= w.pairs &&
                         kb + 32 <= (a.mask == nullptr ? w.len + w.lo + p / G + 1 : w.len);
      if (whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[r] = fmaf(__builtin_amdgcn_exp2f(t[r] * a.scale - ref[0]), ref[1], acc[r]);
      } else {
        // element r: key 8 (r / 4) + 4 h + r % 4.  What a row does not see it
        // leaves alone, NaN or not.
        const uint32_t seen = p + col < w.pairs ? (uint32_t)seen64(a, w, w.lo + pair / G, kb) >> (4 * h) : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = fmaf(__builtin_amdgcn_exp2f(t[r] * a.scale - ref[0]), ref[1], acc[r]);
          if (seen >> (8 * (r >> 2) + (r & 3)) & 1) acc[r] = e;
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the next span's tiles
    float mine = 0.0f;  // column r's lane keeps element r
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v = acc[r];
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) v += exl3::xor_lanes(v, m);
      if (col == r) mine = v;
    }
    const int to = kb + 8 * (col >> 2) + 4 * h + (col & 3);
    if (col < 16 && to < w.keys) {
      float *score = a.score + ((int64_t)f.s * a.pool.kv + head) * a.room + to;
      const int base = a.base ? a.base[f.s] : w.len;
      *score = to < base ? a.decay * *score + mine : mine;
    }
  }
}

// Few pairs (single tokens): their scores are kept in 32 bits from the first pass
// to the second, 4 bytes a pair beside a key's 2 D, so that keys are read
// once.  The first pass: 16 x 16 products, a lane has 4 keys' scores of one pair; a wave
// takes 32 keys in turn, the next ones on their way while the sums form.
template <typename E, int D>
__global__ __launch_bounds__(64 * WW, 4) void weigh_few_sums_kernel(WeighArgs a) {
  constexpr int KK = D / 32;
  typedef typename E::V8 V8;
  __shared__ f32x2 so[WW][FEW];
  __shared__ int sbad;
  const int head = blockIdx.x % a.pool.kv;
  const Find f = find<ITEM>(a, blockIdx.x / a.pool.kv);
  if (f.s < 0) return;
  const Watch &w = f.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int pair = min(col, w.pairs - 1), i = w.lo + pair / a.group, hq = head * a.group + pair % a.group;
  const int k0 = (int)min((int64_t)f.j * f.each * 64, (int64_t)w.keys);
  const int k1 = (int)min((int64_t)k0 + (int64_t)f.each * 64, (int64_t)w.keys);
  const int steps = (k1 - k0 + 31) / 32;
  // keys below this every row that counts sees
  const int clear = a.mask == nullptr ? w.len + w.lo + 1 : w.len;
  if (threadIdx.x == 0) sbad = 0;
  const int *trow = a.pool.table + (size_t)f.s * a.pool.max_pages;
  const uint16_t *pk = reinterpret_cast<const uint16_t *>(a.pool.k) + col * D + 8 * g;
  bool bad = false;
  uint32_t ids[2];
  u32x4 kf[2][KK];
  // blocks behind the last key stand for the last key's
  auto key_of = [&](int step, int t) { return min(k0 + step * 32 + 16 * t, (k1 - 1) & ~15); };
  auto fetch = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) ids[t] = (uint32_t)trow[key_of(step, t) >> a.pool.lp];
  };
  auto load = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t page = __builtin_amdgcn_readfirstlane(ids[t]);
      if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
      const size_t at = ((((size_t)page * a.pool.kv + head) << a.pool.lp) +
                         (key_of(step, t) & ((1 << a.pool.lp) - 1))) * D;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        kf[t][kk] = *reinterpret_cast<const u32x4 *>(pk + at + 32 * kk);
    }
  };
  if (wave < steps) fetch(wave);
  u32x4 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.row + i) * a.qs + hq * D + 32 * kk + 8 * g);
  if (wave < steps) {
    load(wave);
    fetch(min(wave + WW, steps - 1));
  }
  float *to = a.t + (((int64_t)f.s * a.pool.kv + head) * a.most + col) * a.wide + 4 * g;
  float ref = -INFINITY, sum = 0.0f;
  for (int step = wave; step < steps; step += WW) {
    const int kb = k0 + step * 32;
    f32x4 t[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      t[b] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        t[b] = E::mma(__builtin_bit_cast(V8, kf[b][kk]), __builtin_bit_cast(V8, qf[kk]), t[b]);
    }
    if (step + WW < steps) {
      load(step + WW);
      fetch(min(step + 2 * WW, steps - 1));
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) t[b] *= a.scale;
    f32x4 kept[2] = {t[0], t[1]};
    if (kb + 32 > clear || kb + 32 > k1) {
      uint32_t seen = (uint32_t)seen64(a, w, i, kb);
      if (k1 - kb < 32) seen &= ~0u >> (32 - (k1 - kb));
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(seen >> (16 * b + 4 * g + r) & 1)) t[b][r] = -INFINITY, kept[b][r] = UNSEEN;
    }
    if (col < w.pairs) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (kb + 16 * b < k1) *reinterpret_cast<f32x4 *>(to + kb + 16 * b) = kept[b];
    }
    float hi = t[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) hi = __builtin_elementwise_maximum(hi, t[e >> 2][e & 3]);
    if (__ballot(!(hi - ref <= SLACK)) != 0) {
      const float now = __builtin_elementwise_maximum(ref, hi);
      sum *= __builtin_amdgcn_exp2f(ref - (now == -INFINITY ? 0.0f : now));
      ref = now;
    }
    const float from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f(t[e >> 2][e & 3] - from);
  }
#pragma unroll
  for (int m = 16; m < 64; m <<= 1) join(ref, sum, exl3::xor_lanes(ref, m), exl3::xor_lanes(sum, m));
  __syncthreads();
  if (bad) sbad = 1;
  if (g == 0) so[wave][col] = f32x2{ref, sum};
  __syncthreads();
  const int64_t slot = (int64_t)(f.first + f.j) * a.pool.kv + head;
  if (threadIdx.x < FEW && slot < a.slots) {
    ref = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < WW; ++x) join(ref, sum, so[x][threadIdx.x][0], so[x][threadIdx.x][1]);
    if (sbad) sum = __builtin_nanf("");
    a.part[slot * FEW + threadIdx.x] = f32x2{ref, sum};
  }
}

// The second pass: the same keys' scores again, 4 keys a thread, once the
// items of the sequence are joined.
__global__ __launch_bounds__(64 * WW) void weigh_few_keys_kernel(WeighArgs a) {
  __shared__ f32x2 so[16][FEW];
  const int head = blockIdx.x % a.pool.kv;
  const Find f = find<ITEM>(a, blockIdx.x / a.pool.kv);
  if (f.s < 0) return;
  const Watch &w = f.w;
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  float ref = -INFINITY, sum = 0.0f;
  for (int j = row; j < f.parts; j += 16) {
    const int64_t slot = (int64_t)(f.first + j) * a.pool.kv + head;
    if (slot >= a.slots) break;
    const f32x2 v = a.part[slot * FEW + col];
    join(ref, sum, v[0], v[1]);
  }
  so[row][col] = f32x2{ref, sum};
  __syncthreads();
  if (threadIdx.x < FEW) {
    for (int x = 1; x < 16; ++x) join(ref, sum, so[x][col][0], so[x][col][1]);
    so[0][col] = ended(ref, sum);
  }
  __syncthreads();
  const int k0 = (int)min((int64_t)f.j * f.each * 64, (int64_t)w.keys);
  const int k1 = (int)min((int64_t)k0 + (int64_t)f.each * 64, (int64_t)w.keys);
  const float *from = a.t + ((int64_t)f.s * a.pool.kv + head) * a.most * a.wide;
  float *score = a.score + ((int64_t)f.s * a.pool.kv + head) * a.room;
  const int base = a.base ? a.base[f.s] : w.len;
  for (int k = k0 + 4 * (int)threadIdx.x; k < k1; k += 256 * WW) {
    f32x4 acc{0, 0, 0, 0};
    for (int p = 0; p < w.pairs; ++p) {
      const f32x4 t = *reinterpret_cast<const f32x4 *>(from + (int64_t)p * a.wide + k);
      const f32x2 r = so[0][p];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = fmaf(__builtin_amdgcn_exp2f(t[e] - r[0]), r[1], acc[e]);
        if (t[e] != UNSEEN) acc[e] = x;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < k1) score[k + e] = k + e < base ? a.decay * score[k + e] + acc[e] : acc[e];
  }
}

// ------------------------------------------------------------------- eviction

struct EvictArgs {
  Pool pool;  // layer 0's
  size_t layer_bytes;
  int layers, seqs;
  const int32_t *len;
  const float *score;
  int room;
  const int32_t *keep;
  int most, first, last;
  int32_t *kept;
  float *new_score;
  int32_t *new_len;
};

constexpr int PICK = 1024;   // threads that pick a head's keys
constexpr int BINS = 2048;
constexpr int HELD = 32768;  // scores of a head in LDS
constexpr int FEWEST = 512;  // keys whose border is found by rank

// Keys that a sequence keeps, or -1: it stays as it is.
__device__ __forceinline__ int budget_of(const EvictArgs &a, int s, int len) {
  int b = a.most;
  if (a.keep != nullptr) {
    b = min(a.keep[s], a.most);
    if (b < 0) return -1;
  }
  return len > b && len <= a.room && len <= (int64_t)a.pool.max_pages << a.pool.lp ? b : -1;
}

// Scores in the order of whole numbers; NaN below all, zeros alike.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return x != x ? 0u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Sum over the workgroup's threads before this one, and over all.
__device__ __forceinline__ uint32_t before(uint32_t v, uint32_t (&waves)[PICK / 64], uint32_t &whole) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  uint32_t base = 0;
  whole = 0;
#pragma unroll
  for (int w = 0; w < PICK / 64; ++w) {
    if (w < wave) base += waves[w];
    whole += waves[w];
  }
  return base + x - v;
}

// A workgroup a sequence, layer and kv head.  The budget's border is found by
// counting: the range of the scores in BINS bins, then the bin that holds the
// border in BINS again, three rounds at most (32 bits of order), or, once a bin
// holds few keys, by each one's rank among them.  Bins divide the range that
// the scores have, so that few of them fall into one and the counters in LDS are
// rarely fought over.  Then the keys above the border, and as many of those on
// it as are left, earliest first, get their places by counting again.  Scores
// stay in LDS, HELD of them; where there are more they are read again.
__global__ __launch_bounds__(PICK) void evict_pick_kernel(EvictArgs a, int held) {
  extern __shared__ float scores[];
  __shared__ uint32_t bins[BINS], waves[PICK / 64];
  __shared__ uint32_t lows[PICK / 64], highs[PICK / 64];
  __shared__ uint32_t rows[HELD / 64];
  __shared__ int chosen, above, holds, count, found_ties;
  __shared__ uint32_t found;
  uint32_t *const cand = bins;  // FEWEST keys, then their numbers
  const int heads = a.layers * a.pool.kv;
  const int s = blockIdx.x / heads, lh = blockIdx.x - s * heads;
  const int layer = lh / a.pool.kv, h = lh - layer * a.pool.kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = a.len[s];
  const int b = budget_of(a, s, len);
  const size_t at = ((size_t)layer * a.seqs + s) * a.pool.kv + h;
  const float *score = a.score + at * a.room;
  float *to_score = a.new_score + at * a.room;
  int32_t *kept = a.kept + at * a.most;
  // a thread reads what it has written: keys tid, tid + PICK, ... of a block
  const int blocks = b < 0 ? 0 : (len + held - 1) / held;
  auto read = [&](int blk) {
    const int n = min(held, len - blk * held);
#pragma unroll 8
    for (int i = tid; i < n; i += PICK) scores[i] = score[blk * held + i];
    return n;
  };
  if (blocks == 1) read(0);
  bool bad = b < 0;
  if (!bad)
    for (int x = tid; x < (len + (1 << a.pool.lp) - 1) >> a.pool.lp; x += PICK)
      bad |= (uint32_t)a.pool.table[(size_t)s * a.pool.max_pages + x] >= (uint32_t)a.pool.pages;
  bad = __syncthreads_or(bad);
  if (tid == 0 && lh == 0) a.new_len[s] = bad ? len : b;
  for (int x = (bad ? 0 : b) + tid; x < a.most; x += PICK) kept[x] = -1;
  if (bad || b == 0) return;
  const int head = min(a.first, b), tail = min(a.last, b - head);  // those that stay anyway
  const int lo = head, hi = len - tail;                            // the others
  int need = b - head - tail;
  // f(key, its number) for the thread's keys among the others
  auto each = [&](auto &&f) {
    for (int blk = 0; blk < blocks; ++blk) {
      const int n = blocks > 1 ? read(blk) : len, from = blk * held;
#pragma unroll 4
      for (int i = tid; i < n; i += PICK)
        if (from + i >= lo && from + i < hi) f(ordered(scores[i]), from + i);
    }
  };
  // the border: keys of more than `border` stay, and the first `ties` on it
  uint32_t border = ~0u;
  int ties = 0;
  if (need > 0) {
    uint32_t low = ~0u, high = 0;
    each([&](uint32_t k, int) { low = min(low, k), high = max(high, k); });
#pragma unroll
    for (int m = 1; m < 64; m <<= 1)
      low = min(low, (uint32_t)__shfl_xor((int)low, m)), high = max(high, (uint32_t)__shfl_xor((int)high, m));
    if (lane == 0) lows[wave] = low, highs[wave] = high;
    for (int i = tid; i < BINS; i += PICK) bins[i] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PICK / 64; ++w) low = min(low, lows[w]), high = max(high, highs[w]);
    uint32_t width = high - low;  // the range: low .. low + width
    for (;;) {
      const int shift = max(0, 32 - (width ? __builtin_clz(width) : 32) - 11);
      each([&](uint32_t k, int) {
        if (k - low <= width) atomicAdd(&bins[(k - low) >> shift], 1u);
      });
      if (tid == 0) count = 0;
      __syncthreads();
      // a thread's two bins, the highest first
      const int top = BINS - 1 - 2 * tid;
      const uint32_t n1 = bins[top], n0 = bins[top - 1];
      uint32_t whole;
      const uint32_t over = before(n1 + n0, waves, whole);
      if (over < (uint32_t)need && over + n1 + n0 >= (uint32_t)need) {
        const bool second = over + n1 < (uint32_t)need;
        chosen = top - second;
        above = (int)(over + (second ? n1 : 0));
        holds = (int)(second ? n0 : n1);
      }
      __syncthreads();
      const int bin = chosen, n = holds;
      need -= above;
      low += (uint32_t)bin << shift;
      width = min((1u << shift) - 1, width - ((uint32_t)bin << shift));
      border = low, ties = need;
      if (shift == 0) break;
      if (n <= FEWEST) {
        each([&](uint32_t k, int i) {
          if (k - low > width) return;
          const int c = atomicAdd(&count, 1);
          cand[c] = k, cand[FEWEST + c] = i;
        });
        __syncthreads();
        if (tid < n) {
          const uint32_t k = cand[tid], i = cand[FEWEST + tid];
          int more = 0, same = 0;  // before this one: of higher keys, of the same and an earlier number
          for (int c = 0; c < n; ++c) {
            more += cand[c] > k;
            same += cand[c] == k && cand[FEWEST + c] < i;
          }
          if (more + same == need - 1) found = k, found_ties = need - more;
        }
        __syncthreads();
        border = found, ties = found_ties;
        break;
      }
      for (int i = tid; i < BINS; i += PICK) bins[i] = 0;
      __syncthreads();
    }
  }
  // places: what stays whatever the ties are, and the ties, before each key
  uint32_t sure0 = 0, tie0 = 0;  // of the blocks before
  for (int blk = 0; blk < blocks; ++blk) {
    const int n = blocks > 1 ? read(blk) : len, from = blk * held;
    const int turns = (n + PICK - 1) / PICK;
    auto kind = [&](int e, uint64_t &bs, uint64_t &bt) {
      const int i = e * PICK + tid, key = from + i;
      const uint32_t k = i < n ? ordered(scores[i]) : 0;
      const bool other = key >= lo && key < hi;
      bs = __ballot(i < n && (!other || k > border));
      bt = __ballot(i < n && other && k == border);
    };
    for (int e = 0; e < turns; ++e) {
      uint64_t bs, bt;
      kind(e, bs, bt);
      if (lane == 0) rows[e * (PICK / 64) + wave] = (uint32_t)__popcll(bs) | (uint32_t)__popcll(bt) << 16;
    }
    __syncthreads();
    uint32_t whole;
    const bool has = tid < turns * (PICK / 64);
    const uint32_t pre = before(has ? rows[tid] : 0, waves, whole);
    if (has) rows[tid] = pre;
    __syncthreads();
    for (int e = 0; e < turns; ++e) {
      uint64_t bs, bt;
      kind(e, bs, bt);
      const uint64_t under = (1ull << lane) - 1;
      const uint32_t r = rows[e * (PICK / 64) + wave];
      const uint32_t ns = sure0 + (r & 0xFFFFu) + __popcll(bs & under);
      const uint32_t nt = tie0 + (r >> 16) + __popcll(bt & under);
      if (bs >> lane & 1 || (bt >> lane & 1 && nt < (uint32_t)ties)) {
        const uint32_t place = ns + min(nt, (uint32_t)ties);
        kept[place] = from + e * PICK + tid;
        to_score[place] = scores[e * PICK + tid];
      }
    }
    sure0 += whole & 0xFFFFu;
    tie0 += whole >> 16;
    __syncthreads();
  }
}

// Rows move to the front, in their order.  A workgroup takes all rows of a sequence,
// layer, kv head and array, 128 bytes of each: places ascend and no row moves
// back, so what a tile of rows overwrites only tiles up to it read: its stores
// wait for its loads, all threads', and the next tile's loads are on their way
// meanwhile.  The pieces of a row keep out of each other's way, so a row is split
// between workgroups.
constexpr int MV = 256, MU = 8;          // threads, 16-byte pieces of a tile a thread
constexpr int TROWS = MV / 8 * MU;       // rows of a tile
constexpr int BATCH = 8 * TROWS;         // rows whose places are looked up at once

template <int D>
__global__ __launch_bounds__(MV) void evict_move_kernel(EvictArgs a) {
  constexpr int PARTS = D / 64, ROW = D * 2;
  __shared__ int src[BATCH], dst[BATCH];
  const int part = blockIdx.x % (2 * PARTS), rest = blockIdx.x / (2 * PARTS);
  const int heads = a.layers * a.pool.kv;
  const int s = rest / heads, lh = rest - s * heads;
  const int layer = lh / a.pool.kv, h = lh - layer * a.pool.kv;
  const int32_t *kept = a.kept + (((size_t)layer * a.seqs + s) * a.pool.kv + h) * a.most;
  const int n = budget_of(a, s, a.len[s]);
  if (n <= 0 || kept[0] < 0) return;
  char *data = (part & 1 ? a.pool.v : a.pool.k) + layer * a.layer_bytes + (part >> 1) * 128 +
               (threadIdx.x & 7) * 16;
  const int m = (1 << a.pool.lp) - 1, r = threadIdx.x >> 3;
  auto row_at = [&](int sl) {
    return data + ((((size_t)(sl >> a.pool.lp) * a.pool.kv + h) << a.pool.lp) + (sl & m)) * ROW;
  };
  for (int b0 = 0; b0 < n; b0 += BATCH) {
    const int count = min(BATCH, n - b0);
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += MV) {
      const int from = kept[b0 + i];
      const bool moves = from != b0 + i;
      src[i] = moves ? slot_of(a.pool, s, from) : -1;
      dst[i] = moves ? slot_of(a.pool, s, b0 + i) : -1;
    }
    __syncthreads();
    u32x4 v[2][MU];
    const int tiles = (count + TROWS - 1) / TROWS;
    auto load = [&](int t, u32x4 (&to)[MU]) {
#pragma unroll
      for (int u = 0; u < MU; ++u) {
        const int i = t * TROWS + u * (MV / 8) + r;
        to[u] = u32x4{};
        if (i < count && src[i] >= 0) to[u] = *reinterpret_cast<const u32x4 *>(row_at(src[i]));
      }
    };
    auto store = [&](int t, u32x4 (&of)[MU]) {
#pragma unroll
      for (int u = 0; u < MU; ++u) asm volatile("" : "+v"(of[u]));  // in its registers
      asm volatile("s_barrier" ::: "memory");
#pragma unroll
      for (int u = 0; u < MU; ++u) {
        const int i = t * TROWS + u * (MV / 8) + r;
        if (i < count && src[i] >= 0 && dst[i] >= 0) *reinterpret_cast<u32x4 *>(row_at(dst[i])) = of[u];
      }
    };
    load(0, v[0]);
    for (int t = 0; t < tiles; t += 2) {
      if (t + 1 < tiles) load(t + 1, v[1]);
      store(t, v[0]);
      if (t + 1 >= tiles) break;
      if (t + 2 < tiles) load(t + 2, v[0]);
      store(t + 1, v[1]);
    }
  }
}

// ------------------------------------------------------------------- host side

constexpr float LOG2E = 1.4426950408889634f;
size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }

// Rows of all sequences that may count, at most.
int64_t rows_watched(const exl3p_rows *r, int32_t window) {
  const int64_t by = window > 0 ? (int64_t)window * r->seqs : r->rows;
  return by < r->rows ? by : r->rows;
}
// Workgroups of a kv head that fill the CUs: four of the first pass each.
int64_t target_of(const exl3p_cache *c) { return (4 * device_cus() + c->kv_heads - 1) / c->kv_heads; }
int64_t most_tiles(const exl3p_rows *r, int group, int32_t window) {
  return rows_watched(r, window) * group / TILE + r->seqs;
}
size_t refs_bytes(const exl3p_cache *c, const exl3p_rows *r, int group) {
  return up16((size_t)r->rows * group * c->kv_heads * sizeof(f32x2));
}

// How the weights are formed, by what the host knows.  Pairs whose scores are
// kept read the keys once and the scores (4 bytes a pair and key) twice; others
// read the keys twice.
struct Plan {
  int group;
  int64_t tiles, items;  // at most
  int few;               // pairs whose scores are kept, 0: none
  int wide;              // of a row of them
  size_t parts, rest;    // bytes
};
constexpr size_t KEPT_MAX = (size_t)1 << 30;
Plan plan_of(const exl3p_cache *c, const exl3p_rows *r, int32_t heads, int32_t window, int32_t room) {
  Plan p;
  p.group = heads / c->kv_heads;
  const int64_t rows = window > 0 && window < r->max_rows ? window : r->max_rows;
  p.wide = (room + 15) & ~15;
  p.tiles = most_tiles(r, p.group, window);
  p.items = target_of(c) + p.tiles;
  p.few = rows * p.group <= FEW ? (int)(rows * p.group) : 0;
  p.rest = (size_t)r->seqs * c->kv_heads * p.few * p.wide * sizeof(float);
  if (p.rest > KEPT_MAX) p.few = 0;
  if (p.few == 0) p.rest = refs_bytes(c, r, p.group);
  p.parts = (size_t)p.items * c->kv_heads * (p.few ? FEW : TILE) * sizeof(f32x2);
  return p;
}

exl3_verdict check_score(const void *p, int32_t room) {
  if (p == nullptr) return refuse(EXL3_FAILED, "PagedScore: a missing array");
  if (!aligned(p, 4)) return refuse(EXL3_UNSUPPORTED, "PagedScore: elements on their own boundaries");
  if (room <= 0) return refuse(EXL3_UNSUPPORTED, "PagedScore: room for keys above 0");
  return OK;
}

}  // namespace

extern "C" {

size_t exl3p_weigh_scratch_bytes(const exl3p_cache *c, const exl3p_rows *r, int32_t heads,
                                 int32_t window, int32_t room) {
  if (check_cache(c).code != EXL3_OK || check_rows(c, r).code != EXL3_OK ||
      check_heads(c, heads).code != EXL3_OK || window < 0 || room <= 0)
    return 0;
  const Plan p = plan_of(c, r, heads, window, room);
  return p.parts + p.rest;
}

exl3_verdict exl3p_weigh(const exl3p_cache *c, int32_t layer, const exl3p_rows *r, int32_t heads,
                         const void *q, int64_t q_stride, const uint64_t *mask, int32_t words,
                         float scale, int32_t window, float decay, const int32_t *base,
                         float *score, int32_t room, void *scratch, size_t scratch_bytes,
                         exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  EXL3P_TRY(check_layer(c, layer));
  EXL3P_TRY(check_rows(c, r));
  EXL3P_TRY(check_heads(c, heads));
  EXL3P_TRY(check_mask(r, mask, words));
  if (!(fabsf(scale) * LOG2E < INFINITY))
    return refuse(EXL3_UNSUPPORTED, "PagedScale: finite, also times log2(e)");
  if (!(fabsf(decay) < INFINITY)) return refuse(EXL3_UNSUPPORTED, "PagedDecay: finite");
  if (window < 0) return refuse(EXL3_UNSUPPORTED, "PagedWindow: rows from 0 (all of them)");
  if (r->rows == 0 || r->seqs == 0 || r->max_rows == 0) return OK;
  EXL3P_TRY(check_score(score, room));
  EXL3P_TRY(check_matrix(q, q_stride, (int64_t)heads * c->dim));
  const Plan p = plan_of(c, r, heads, window, room);
  if ((int64_t)r->rows * p.group > INT32_MAX / 2 || p.items * c->kv_heads > GRID_MAX)
    return refuse(EXL3_TOO_LARGE, "PagedWeigh: too many rows and heads for one call");
  const size_t need = exl3p_weigh_scratch_bytes(c, r, heads, window, room);
  if (scratch == nullptr || !aligned(scratch, 16) || scratch_bytes < need)
    return refuse(EXL3_FAILED, "PagedScratch: below exl3p_weigh_scratch_bytes, or not aligned");
  const Pool pool = pool_of(c, layer);
  EXL3P_TRY(check_apart({array(score, (int64_t)r->seqs * c->kv_heads * room * 4), array(scratch, (int64_t)need)},
                        {array(pool.k, layer_bytes(c)), matrix(q, q_stride, (int64_t)heads * c->dim, r->rows),
                         array(mask, 8 * (int64_t)r->rows * words),
                         array(r->cu, 4 * ((int64_t)r->seqs + 1)), array(r->len, 4 * (int64_t)r->seqs),
                         array(base, 4 * (int64_t)r->seqs), table_of(c)}));
  WeighArgs a;
  a.pool = pool, a.st = step_of(r), a.group = p.group, a.window = window;
  a.q = static_cast<const uint16_t *>(q), a.qs = q_stride, a.mask = mask, a.words = words;
  a.scale = scale * LOG2E, a.decay = decay, a.base = base, a.score = score, a.room = room;
  a.target = (float)target_of(c), a.slots = (int)(p.items * c->kv_heads);
  a.least = p.few ? 2.0f : 4.0f;
  a.part = static_cast<f32x2 *>(scratch);
  a.ref = reinterpret_cast<f32x2 *>(static_cast<char *>(scratch) + p.parts);
  a.t = reinterpret_cast<float *>(a.ref), a.most = p.few, a.wide = p.wide;
  const hipStream_t st = static_cast<hipStream_t>(s);
  const dim3 items((unsigned)(p.items * c->kv_heads));
  return by_type(c, [&](auto e, auto d) {
    if (p.few) {
      hipLaunchKernelGGL((weigh_few_sums_kernel<decltype(e), d>), items, dim3(64 * WW), 0, st, a);
      hipLaunchKernelGGL(weigh_few_keys_kernel, items, dim3(64 * WW), 0, st, a);
      return;
    }
    hipLaunchKernelGGL((weigh_sums_kernel<decltype(e), d>), items, dim3(64 * WW), 0, st, a);
    hipLaunchKernelGGL(weigh_join_kernel, dim3((unsigned)(p.tiles * c->kv_heads)), dim3(TILE), 0, st, a);
    hipLaunchKernelGGL((weigh_keys_kernel<decltype(e), d>), dim3((unsigned)(2 * target_of(c) * c->kv_heads)),
                       dim3(64 * WW), 0, st, a);
  });
}

exl3_verdict exl3p_evict(const exl3p_cache *c, int32_t seqs, const int32_t *len,
                         const float *score, int32_t room, const int32_t *keep, int32_t most,
                         int32_t first, int32_t last, int32_t *kept, float *new_score,
                         int32_t *new_len, exl3_stream s) {
  EXL3P_TRY(check_cache(c));
  if (seqs < 0 || seqs > c->seqs)
    return refuse(EXL3_UNSUPPORTED, "PagedEvict: more sequences than the cache's");
  if (most <= 0 || first < 0 || last < 0)
    return refuse(EXL3_UNSUPPORTED, "PagedEvict: most above 0, first and last from 0");
  if (seqs == 0) return OK;
  EXL3P_TRY(check_score(score, room));
  EXL3P_TRY(check_score(new_score, room));
  if (len == nullptr || kept == nullptr || new_len == nullptr)
    return refuse(EXL3_FAILED, "PagedEvict: a missing array");
  const int64_t n = (int64_t)c->layers * seqs * c->kv_heads;
  const int parts = 2 * c->dim / 64;
  if (n * 4 > GRID_MAX)  // of 1024 threads, and of 256
    return refuse(EXL3_TOO_LARGE, "PagedEvict: too many layers, sequences and heads for one call");
  const Span2D from = array(score, n * room * 4), to = array(new_score, n * room * 4);
  const int64_t pool = (int64_t)layer_bytes(c) * c->layers;
  EXL3P_TRY(check_apart({array(kept, n * most * 4), to, array(new_len, 4 * (int64_t)seqs),
                         array(c->k, pool), array(c->v, pool)},
                        {array(len, 4 * (int64_t)seqs), array(keep, 4 * (int64_t)seqs), table_of(c)}));
  // a workgroup reads a head's scores before it writes them: new_score may be score
  EXL3P_TRY(check_apart({array(kept, n * most * 4), array(new_len, 4 * (int64_t)seqs), array(c->k, pool),
                         array(c->v, pool)}, {from}));
  if (new_score != score && meet(from, to))
    return refuse(EXL3_UNSUPPORTED, "PagedOverlap: new_score over score, and not score itself");
  EvictArgs a;
  a.pool = pool_of(c, 0), a.layer_bytes = layer_bytes(c), a.layers = c->layers, a.seqs = seqs;
  a.len = len, a.score = score, a.room = room, a.keep = keep, a.most = most;
  a.first = first, a.last = last, a.kept = kept, a.new_score = new_score, a.new_len = new_len;
  const hipStream_t st = static_cast<hipStream_t>(s);
  const int held = room < HELD ? (room + PICK - 1) / PICK * PICK : HELD;
  hipLaunchKernelGGL(evict_pick_kernel, dim3((unsigned)n), dim3(PICK), held * sizeof(float), st, a, held);
  if (c->dim == 64)
    hipLaunchKernelGGL(evict_move_kernel<64>, dim3((unsigned)(n * parts)), dim3(MV), 0, st, a);
  else
    hipLaunchKernelGGL(evict_move_kernel<128>, dim3((unsigned)(n * parts)), dim3(MV), 0, st, a);
  return launched();
}

}  // extern "C"
