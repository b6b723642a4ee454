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
  float scale;    // |scale| log2(e): weights are powers of two
  uint32_t flip;  // 0x80008000 where the scale is negative: q's sign bits
  float decay;
  const int32_t *base;
  float *score;
  int room;
  float target;  // items of a kv head
  float least;   // 64-key units of one, at least,
  float fill, some;  // and as many as leave `fill` items of a kv head, up to `some`
  int slots;     // items * kv that part holds
  int tile;      // pairs of an item
  f32x2 *part;   // [items * kv][tile]: an item's reference and sum of each pair
  float *ref, *inv;  // [kv][rows * group]: a pair's reference and 1 / sum of its weights below it
  float *t;      // few pairs: [seqs][kv][most][wide] scores, in place of these
  int most, wide;
  int deal;      // pairs that an item of the second pass adds up, whole tiles
  int deals;     // such items of a key, at most; where there are several:
  float *sums;   // [seqs][kv][deals][room]: their sums
};

constexpr int WW = 4;       // waves of a workgroup
constexpr int TILE = 128;   // pairs of a row and a query head that an item has,
constexpr int FEW = 16;     // or where scores are kept, this many or twice as many,
constexpr int PART = 4096;  // keys of an item of the second pass, at most
constexpr float SLACK = 4.0f;  // a reference follows its maximum in steps of more (powers of two)
// Up to references of FAR a weight's exponent is one multiply-add of score, scale
// and reference; beyond, the reference's rounding is whole powers of two, and
// scores are multiplied first.
constexpr float FAR = 0x1p20f;

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

enum Kind { ITEM, PAIRS, DEAL };  // part of a tile's keys; a tile; part of a deal's keys
struct Find {
  int s;       // -1: nothing
  int u, j;    // tile or deal of pairs, part of the keys
  int first;   // the tile's first item
  int parts;   // items of a tile or deal
  int each;    // 64-key units of one
  int tiles;   // tiles or deals of the sequence
  Watch w;
};

// Numbers among the sequences' items.  A tile (or deal of tiles) of u units of 64 keys
// has ceil(u / c) items, c the units of all over the target, and what a 32-bit sum may
// be short of: items are never more than target + tiles (deals: where their parts are
// not cut short at PART).  A lane keeps a sequence, of up to 64.
template <Kind KIND>
struct Finder {
  const WeighArgs &a;
  Watch w{};
  int chunk = 1;
  bool none = false;
  __device__ __forceinline__ int tiles_of(const Watch &v) const {
    const int t = KIND == DEAL ? a.deal : a.tile;
    return (v.pairs + t - 1) / t;
  }
  __device__ __forceinline__ explicit Finder(const WeighArgs &args) : a(args) {
    float units = 0.0f;
    bool back = false;
    for (int s = threadIdx.x & 63; s < a.st.seqs; s += 64) {
      w = watch_of(a, s);
      back |= w.back;
      units += (float)tiles_of(w) * (float)((w.keys + 63) >> 6);
    }
    none = __ballot(back) != 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) units += exl3::xor_lanes(units, m);
    chunk = __builtin_amdgcn_readfirstlane((int)fminf(fmaxf(fmaxf(ceilf(units * (1.0f + 0x1p-12f) / a.target), a.least),
                                                            fminf(ceilf(units / a.fill), a.some)),
                                                      KIND == DEAL ? (float)(PART / 64) : (float)(1 << 25)));
  }
  __device__ __forceinline__ Find at(int x) {
    Find f;
    f.s = -1;
    if (none) return f;
    int before = 0, items = 0;
    for (int s0 = 0; s0 < a.st.seqs; s0 += 64) {
      const int s = s0 + (int)(threadIdx.x & 63);
      int tiles = 0, ns = 0, each = 1, count = 0;
      if (s < a.st.seqs) {
        if (a.st.seqs > 64) w = watch_of(a, s);
        if (w.pairs > 0) {
          const int u = (w.keys + 63) >> 6;
          tiles = tiles_of(w);
          ns = (u + chunk - 1) / chunk;
          each = (u + ns - 1) / ns;  // the last items may be empty
          count = KIND == PAIRS ? tiles : tiles * ns;
        }
      }
      const int ct = scan(count), it = KIND == PAIRS ? scan(tiles * ns) : ct;
      const uint64_t past = __ballot(before + ct > x);
      if (past != 0) {
        const int l = __builtin_ctzll(past);
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        const int y = x - before - of(ct - count), nt = of(tiles), n_s = of(ns);
        f.s = s0 + l;
        f.w = Watch{of(w.row), of(w.n), of(w.len), of(w.lo), of(w.pairs), of(w.keys), false};
        f.parts = n_s;
        f.each = of(each);
        f.tiles = nt;
        // tiles that read the same keys side by side, the last, whose rows see most, first
        f.j = KIND == PAIRS ? 0 : y / nt;
        f.u = nt - 1 - (y - f.j * nt);
        f.first = items + of(it - tiles * ns) + f.u * n_s;
        return f;
      }
      before += __builtin_amdgcn_readlane(ct, 63);
      items += __builtin_amdgcn_readlane(it, 63);
    }
    return f;
  }
};

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

// The places of a row's 16-byte pieces in LDS: those of one number of 16 rows lie in
// 16 places of the banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}

// The larger, NaN if either is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A score that a row does not see, where scores are kept: its weight is none, also
// where the row's sum is NaN.
constexpr float UNSEEN = -0x1.fffffep127f;

// Two parts of a pair's keys: the reference and the sum of weights of both.
__device__ __forceinline__ void join(float &ref, float &sum, float other, float more) {
  const float now = larger(ref, other), from = now == -INFINITY ? 0.0f : now;
  sum = sum * __builtin_amdgcn_exp2f(ref - from) + more * __builtin_amdgcn_exp2f(other - from);
  ref = now;
}
// What the second pass wants of them: a pair that sees nothing has no weights, a NaN
// stays in the factor.
__device__ __forceinline__ f32x2 ended(float ref, float sum) {
  return f32x2{ref == -INFINITY || ref != ref ? 0.0f : ref,
               sum == 0.0f ? 0.0f : ref != ref ? ref : 1.0f / sum};
}

// An item's keys, tiles of 64 of which pass through LDS, the next loaded while one is
// used: 16 a wave, by direct loads.
template <typename E, int D>
struct Keys {
  static constexpr int ROW = D * 2, ARR = 64 * ROW;
  static constexpr int LOADS = 16 * ROW / 1024, LR = 1024 / ROW;  // loads a wave, rows a load
  typedef typename E::V8 V8;
  const WeighArgs &a;
  int k0, last, wave, head;
  const int *trow;
  const char *lds;
  uint32_t lbase, ka, id = 0, voff[LOADS];
  bool bad = false;
  __device__ __forceinline__ Keys(const WeighArgs &args, const char *to, int s, int head_, int from, int end)
      : a(args), k0(from), last(end), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), head(head_),
        trow(args.pool.table + (size_t)s * args.pool.max_pages), lds(to),
        lbase(__builtin_amdgcn_readfirstlane(
            (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)to)) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
    ka = col * ROW + 16 * (h ^ swizzle<D>(col));
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int row = LR * u + lane / (ROW / 16), place = lane % (ROW / 16);
      voff[u] = row * ROW + (place ^ swizzle<D>(row)) * 16;
    }
  }
  // blocks behind the last key stand for the last key's
  __device__ __forceinline__ int key_of(int step) const {
    return min(k0 + step * 64 + 16 * wave, (last - 1) & ~15);
  }
  __device__ __forceinline__ void fetch(int step) { id = (uint32_t)trow[key_of(step) >> a.pool.lp]; }
  __device__ __forceinline__ void load(int step, int buffer) {
    uint32_t page = __builtin_amdgcn_readfirstlane(id);
    if (page >= (uint32_t)a.pool.pages) bad = true, page = 0;
    const size_t at = ((((size_t)page * a.pool.kv + head) << a.pool.lp) +
                       (key_of(step) & ((1 << a.pool.lp) - 1))) * ROW;
    const uint32_t to = lbase + buffer * ARR + 16 * wave * ROW;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) exl3::lds_dma16(a.pool.k + at, voff[u], to + u * 1024);
  }
  // This wave's loads of the tile are in LDS, and so are, behind the barrier, the
  // others'; all have read the tile before, whose place is loaded next.
  __device__ __forceinline__ void arrive() const {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  // 8 elements of key 32 b + column, from element 16 kk + 8 h on
  __device__ __forceinline__ V8 piece(int buffer, int b, int kk) {
    return *reinterpret_cast<const V8 *>(lds + buffer * ARR + (ka ^ (32 * kk)) + b * 32 * ROW);
  }
  __device__ __forceinline__ void anew() { asm volatile("" : "+v"(ka)); }
};

// A tile's products, of 64 keys and 32 pairs.  Four pieces of keys are on their way from LDS
// while four are multiplied (the compiler's own order waits for each piece right after it
// has asked for it: 287 us, not 270, for 3 prompts of up to 2048 rows).  64 pairs a wave,
// which reads half as much of LDS, leave two waves a SIMD: 286 us.
template <typename E, int D, typename MMA>
__device__ __forceinline__ void products(Keys<E, D> &keys, int buffer, f32x16 (&t)[2], MMA &&mma) {
  constexpr int KK = D / 16, AT = 4, GROUPS = 2 * KK / AT;
  typename E::V8 kf[2][AT];
  auto read = [&](int g) {
#pragma unroll
    for (int x = 0; x < AT; ++x) kf[g & 1][x] = keys.piece(buffer, (g * AT + x) / KK, (g * AT + x) % KK);
  };
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) t[b][r] = 0.0f;
  read(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    if (g + 1 < GROUPS) read(g + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < AT; ++x) {
      const int b = (g * AT + x) / KK, kk = (g * AT + x) % KK;
      t[b] = mma(kf[g & 1][x], kk, t[b]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The first pass: each pair's reference (its largest score, or less by SLACK at
// most) and the sum of its weights over an item's keys.  128 pairs a workgroup, 32 a
// wave; scores are S^T = K q^T (rows keys, columns pairs): a lane holds 32 keys' scores
// of one pair.
template <typename E, int D>
__global__ __launch_bounds__(64 * WW, 2) void weigh_sums_kernel(WeighArgs a) {
  constexpr int KK = D / 16;
  typedef typename E::V8 V8;
  __shared__ __align__(1024) char lds[2 * Keys<E, D>::ARR];
  const int head = blockIdx.x % a.pool.kv;
  const Find f = Finder<ITEM>(a).at(blockIdx.x / a.pool.kv);
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
    last = min(last, w.len + w.lo + (min((f.u + 1) * TILE, w.pairs) - 1) / G + 1);
    mine = min(last, w.len + w.lo + (min(r0 + 32, w.pairs) - 1) / G + 1);
  }
  if (r0 >= w.pairs) mine = k0;
  // keys below this every row of the wave sees
  const int clear = min(last, a.mask == nullptr ? w.len + w.lo + r0 / G + 1 : w.len);
  const int steps = last > k0 ? (last - k0 + 63) / 64 : 0;
  Keys<E, D> keys(a, lds, f.s, head, k0, last);
  if (steps > 0) {
    keys.fetch(0);
    keys.load(0, 0);
    if (steps > 1) keys.fetch(1);
  }
  u32x4 qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.row + i) * a.qs + hq * D + 16 * kk + 8 * h) ^ a.flip;
  float ref = -INFINITY, sum = 0.0f, scale = a.scale;
  bool far = false;  // of the wave: its scores are multiplied first, and scale is 1
  auto turn = [&](int step, auto TAIL) {
    keys.arrive();
    if (step + 1 < steps) {
      keys.load(step + 1, (step + 1) & 1);
      if (step + 2 < steps) keys.fetch(step + 2);
    }
    const int kb = k0 + step * 64;
    if (kb >= mine) return;
    keys.anew();
    f32x16 t[2];
    products<E, D>(keys, step & 1, t,
                   [&](V8 kf, int kk, f32x16 c) { return E::mma(kf, __builtin_bit_cast(V8, qf[kk]), c); });
    if constexpr (decltype(TAIL)::value) {
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
    auto multiply = [&] {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) t[b][r] *= a.scale;
    };
    if (far) multiply();
    float hi = larger(t[0][0], t[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) hi = larger(larger(hi, t[0][r]), t[1][r]);
    hi *= scale;
    if (__ballot(!(hi - ref <= SLACK)) != 0) {
      const float now = larger(ref, hi);
      sum *= __builtin_amdgcn_exp2f(ref - (now == -INFINITY ? 0.0f : now));
      ref = now;
      if (!far && __ballot(fabsf(now) > FAR && now != -INFINITY) != 0) {
        far = true, scale = 1.0f;
        multiply();
      }
    }
    const float from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(t[b][r], scale, -from));
  };
  // tiles that every row of the wave sees whole, then the others
  const int whole = min(max(clear - k0, 0) / 64, steps);
  int step = 0;
  for (; step < whole; ++step) turn(step, std::false_type{});
  for (; step < steps; ++step) turn(step, std::true_type{});
  __syncthreads();
  // (no more LDS than the tiles' own: five workgroups a CU)
  int *const sbad = reinterpret_cast<int *>(lds);
  if (threadIdx.x == 0) *sbad = 0;
  __syncthreads();
  if (keys.bad) *sbad = 1;
  __syncthreads();
  // the two halves of a pair's keys
  join(ref, sum, exl3::xor_lanes(ref, 32), exl3::xor_lanes(sum, 32));
  if (*sbad) sum = __builtin_nanf("");
  const int64_t slot = (int64_t)(f.first + f.j) * a.pool.kv + head;
  if (h == 0 && r0 + col < w.pairs && slot < a.slots) a.part[slot * TILE + 32 * wave + col] = f32x2{ref, sum};
}

// A tile's items joined, 256 / SHARE pairs a workgroup, whose items are shared out to SHARE
// threads each.
template <int SHARE>
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighArgs a) {
  constexpr int OF = 256 / SHARE;
  __shared__ f32x2 so[SHARE][OF];
  const int head = blockIdx.x % a.pool.kv, rest = blockIdx.x / a.pool.kv;
  const Find f = Finder<PAIRS>(a).at(rest / (a.tile / OF));
  const int col = threadIdx.x % OF, row = threadIdx.x / OF;
  const int in = rest % (a.tile / OF) * OF + col;
  if (f.s < 0 || f.u * a.tile + in - col >= f.w.pairs) return;
  float ref = -INFINITY, sum = 0.0f;
  for (int j = row; j < f.parts; j += SHARE) {
    const int64_t slot = (int64_t)(f.first + j) * a.pool.kv + head;
    if (slot >= a.slots) break;
    const f32x2 v = a.part[slot * a.tile + in];
    join(ref, sum, v[0], v[1]);
  }
  so[row][col] = f32x2{ref, sum};
  __syncthreads();
  const int pair = f.u * a.tile + in;
  if (row > 0 || pair >= f.w.pairs) return;
  for (int x = 1; x < SHARE; ++x) join(ref, sum, so[x][col][0], so[x][col][1]);
  // (two numbers: the logarithm of what a row's weights sum to would be rounded as a score of
  // its size is, all of the row's weights by one factor, 1 % at scores of 2^18)
  const f32x2 both = ended(ref, sum);
  const int64_t at = (int64_t)head * a.st.rows * a.group + (int64_t)(f.w.row + f.w.lo) * a.group + pair;
  a.ref[at] = both[0], a.inv[at] = both[1];
}

// A key's score: what it had, and the weights of this step.
__device__ __forceinline__ void add_score(const WeighArgs &a, const Find &f, int head, int key, float more) {
  float *score = a.score + ((int64_t)f.s * a.pool.kv + head) * a.room + key;
  const int base = a.base ? a.base[f.s] : f.w.len;
  *score = key < base ? a.decay * *score + more : more;
}

// The second pass: each key's weights over a deal of pairs.  The deal's tiles take
// their turns, each in registers (32 pairs a wave) while the item's keys pass
// through LDS as in the first pass.  Scores are S = q K^T here (rows pairs, columns
// keys), so that a lane adds up its key's weights over 16 pairs of a product by
// itself; the waves' sums join through LDS, one tile of keys behind.  Several deals of a
// key (many pairs) leave their sums for the next kernel.
template <typename E, int D>
__global__ __launch_bounds__(64 * WW, 2) void weigh_keys_kernel(WeighArgs a) {
  constexpr int KK = D / 16;
  typedef typename E::V8 V8;
  __shared__ __align__(1024) char lds[2 * Keys<E, D>::ARR];
  __shared__ float joint[2][WW][64];
  __shared__ float total[PART];
  __shared__ __align__(16) float invs[WW][32];
  const int head = blockIdx.x % a.pool.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int G = a.group;
  Finder<DEAL> finder(a);
  for (int x = blockIdx.x / a.pool.kv;; x += gridDim.x / a.pool.kv) {
    const Find f = finder.at(x);
    if (f.s < 0) return;
    const Watch &w = f.w;
    const int k0 = (int)min((int64_t)f.j * f.each * 64, (int64_t)w.keys);
    const int k1 = (int)min((int64_t)k0 + (int64_t)f.each * 64, (int64_t)w.keys);
    const int p1 = min((f.u + 1) * a.deal, w.pairs);
    for (int k = threadIdx.x; k < k1 - k0; k += 64 * WW) total[k] = 0.0f;
    const int64_t pairs0 = (int64_t)head * a.st.rows * G + (int64_t)(w.row + w.lo) * G;
    int count = 0;  // tiles of keys done: their places in LDS
    auto finish = [&](int step) {
      if (wave > 0) return;
      float v = 0.0f;
#pragma unroll
      for (int y = 0; y < WW; ++y) v += joint[(count - 1) & 1][y][lane];
      total[step * 64 + lane] += v;
    };
    for (int p0 = f.u * a.deal; p0 < p1; p0 += TILE) {
      // keys that the tile's rows see
      const int last = a.mask != nullptr ? k1 : min(k1, w.len + w.lo + (min(p0 + TILE, w.pairs) - 1) / G + 1);
      if (last <= k0) continue;
      const int steps = (last - k0 + 63) / 64;
      const int r0 = p0 + 32 * wave;
      const bool any = r0 < w.pairs;
      const int clear = min(last, a.mask == nullptr ? w.len + w.lo + r0 / G + 1 : w.len);
      Keys<E, D> keys(a, lds, f.s, head, k0, last);
      keys.fetch(0);
      __syncthreads();  // the tile before is read, and its last sums are joined below
      keys.load(0, count & 1);
      if (steps > 1) keys.fetch(1);
      const int pair = min(r0 + col, w.pairs - 1), i = w.lo + pair / G;
      u32x4 qf[KK];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.row + i) * a.qs + (head * G + pair % G) * D + 16 * kk +
                                                  8 * h) ^ a.flip;
      // element r: pair 8 (r / 4) + 4 h + r % 4; its 1 / sum is read from LDS where it is needed
      // (16 more registers would leave two waves a SIMD).  A pair behind the last is that one's
      // copy: no weight, but for a NaN that it gives too.
      float ref[16];
      bool far = false;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        ref[r] = a.ref[pairs0 + min(r0 + 8 * (r >> 2) + 4 * h + (r & 3), w.pairs - 1)];
        far |= fabsf(ref[r]) > FAR;
      }
      far = __ballot(far) != 0;
      if (h == 0) invs[wave][col] = r0 + col < w.pairs ? a.inv[pairs0 + pair] : 0.0f;
      auto inv4 = [&](int r) { return *reinterpret_cast<const f32x4 *>(&invs[wave][8 * (r >> 2) + 4 * h]); };
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+v"(qf[kk]));  // (the sign is not turned in each tile)
      const float scale = far ? 1.0f : a.scale;
      for (int step = 0; step < steps; ++step, ++count) {
        keys.arrive();
        if (step > 0) finish(step - 1);
        if (step + 1 < steps) {
          keys.load(step + 1, (count + 1) & 1);
          if (step + 2 < steps) keys.fetch(step + 2);
        }
        const int kb = k0 + step * 64;
        float v[2] = {0.0f, 0.0f};
        if (any) {
          keys.anew();
          f32x16 t[2];
          products<E, D>(keys, count & 1, t,
                         [&](V8 kf, int kk, f32x16 c) { return E::mma(__builtin_bit_cast(V8, qf[kk]), kf, c); });
          if (far) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int r = 0; r < 16; ++r) t[b][r] *= a.scale;
          }
          if (kb + 64 <= clear) {
#pragma unroll
            for (int r4 = 0; r4 < 16; r4 += 4) {
              const f32x4 inv = inv4(r4);
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = r4; r < r4 + 4; ++r)
                  v[b] = fmaf(__builtin_amdgcn_exp2f(fmaf(t[b][r], scale, -ref[r])), inv[r - r4], v[b]);
            }
          } else {
            // what each of the wave's pairs sees, a pair a lane.  What a row does not see it
            // leaves alone, NaN or not.
            const uint64_t seen = r0 + col < w.pairs ? seen64(a, w, i, kb) : 0;
#pragma unroll
            for (int r4 = 0; r4 < 16; r4 += 4) {
              const f32x4 inv = inv4(r4);
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = r4; r < r4 + 4; ++r) {
                  const uint32_t of = __shfl((int)(uint32_t)(seen >> (32 * b)), 8 * (r >> 2) + 4 * h + (r & 3));
                  const float y = fmaf(__builtin_amdgcn_exp2f(fmaf(t[b][r], scale, -ref[r])), inv[r - r4], v[b]);
                  if (of >> col & 1) v[b] = y;
                }
            }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) v[b] += exl3::xor_lanes(v[b], 32);
        }
        joint[count & 1][wave][lane] = h ? v[1] : v[0];
      }
      __syncthreads();
      finish(steps - 1);
    }
    __syncthreads();
    float *to = a.sums + (((int64_t)f.s * a.pool.kv + head) * a.deals + f.u) * a.room;
    for (int k = threadIdx.x; k < k1 - k0; k += 64 * WW) {
      if (f.tiles == 1)
        add_score(a, f, head, k0 + k, total[k]);
      else if (f.u < a.deals)
        to[k0 + k] = total[k];
    }
    __syncthreads();
  }
}

// The deals of a key added up, 64 keys a workgroup, a share of the deals a wave.
__global__ __launch_bounds__(64 * WW) void weigh_deals_kernel(WeighArgs a) {
  __shared__ float joint[WW][64];
  const int spans = (a.room + 63) / 64;
  const int head = blockIdx.x % a.pool.kv, rest = blockIdx.x / a.pool.kv;
  Find f;
  f.s = rest / spans;
  f.w = watch_of(a, f.s);
  const int tiles = min((f.w.pairs + a.deal - 1) / a.deal, a.deals);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key = rest % spans * 64 + lane;
  if (tiles < 2 || key - lane >= f.w.keys) return;
  bool back = false;  // (of a step whose cu goes back nothing is done)
  for (int s = lane; s < a.st.seqs; s += 64) back |= watch_of(a, s).back;
  if (__ballot(back) != 0) return;
  const float *from = a.sums + ((int64_t)f.s * a.pool.kv + head) * a.deals * a.room + min(key, f.w.keys - 1);
  const int each = (tiles + WW - 1) / WW;
  float v = 0.0f;
#pragma unroll 8
  for (int j = wave * each; j < min(tiles, (wave + 1) * each); ++j) v += from[(int64_t)j * a.room];
  joint[wave][lane] = v;
  __syncthreads();
  if (wave > 0 || key >= f.w.keys) return;
#pragma unroll
  for (int y = 1; y < WW; ++y) v += joint[y][lane];
  add_score(a, f, head, key, v);
}

// Few pairs (single tokens, small trees): their scores are kept in 32 bits from the first
// pass to the second, 4 bytes a pair beside a key's 2 D, so that keys are read
// once.  The first pass: 16 x 16 products, a lane has 4 keys' scores of each of NB pairs; a
// wave takes 32 keys in turn, the next ones on their way while the sums form.
template <typename E, int D, int NB>
__global__ __launch_bounds__(64 * WW, 4) void weigh_few_sums_kernel(WeighArgs a) {
  constexpr int KK = D / 32, TILE = FEW * NB;
  typedef typename E::V8 V8;
  __shared__ f32x2 so[WW][TILE];
  __shared__ int sbad;
  const int head = blockIdx.x % a.pool.kv;
  const Find f = Finder<ITEM>(a).at(blockIdx.x / a.pool.kv);
  if (f.s < 0) return;
  const Watch &w = f.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
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
  int i[NB];
  u32x4 qf[NB][KK];
  float ref[NB], sum[NB];
#pragma unroll
  for (int p = 0; p < NB; ++p) {
    const int pair = min(FEW * p + col, w.pairs - 1), hq = head * a.group + pair % a.group;
    i[p] = w.lo + pair / a.group;
    ref[p] = -INFINITY, sum[p] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[p][kk] = *reinterpret_cast<const u32x4 *>(a.q + (w.row + i[p]) * a.qs + hq * D + 32 * kk + 8 * g) ^ a.flip;
  }
  if (wave < steps) {
    load(wave);
    fetch(min(wave + WW, steps - 1));
  }
  float *to = a.t + (((int64_t)f.s * a.pool.kv + head) * a.most + col) * a.wide + 4 * g;
  for (int step = wave; step < steps; step += WW) {
    const int kb = k0 + step * 32;
    f32x4 t[NB][2];
#pragma unroll
    for (int p = 0; p < NB; ++p)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        t[p][b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          t[p][b] = E::mma(__builtin_bit_cast(V8, kf[b][kk]), __builtin_bit_cast(V8, qf[p][kk]), t[p][b]);
      }
    if (step + WW < steps) {
      load(step + WW);
      fetch(min(step + 2 * WW, steps - 1));
    }
    float hi[NB];
    bool moves = false;
#pragma unroll
    for (int p = 0; p < NB; ++p) {
#pragma unroll
      for (int b = 0; b < 2; ++b) t[p][b] *= a.scale;
      f32x4 kept[2] = {t[p][0], t[p][1]};
      if (kb + 32 > clear || kb + 32 > k1) {
        uint32_t seen = (uint32_t)seen64(a, w, i[p], kb);
        if (k1 - kb < 32) seen &= ~0u >> (32 - (k1 - kb));
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(seen >> (16 * b + 4 * g + r) & 1)) t[p][b][r] = -INFINITY, kept[b][r] = UNSEEN;
      }
      if (FEW * p + col < w.pairs) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
          if (kb + 16 * b < k1)
            *reinterpret_cast<f32x4 *>(to + (int64_t)FEW * p * a.wide + kb + 16 * b) = kept[b];
      }
      hi[p] = t[p][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) hi[p] = larger(hi[p], t[p][e >> 2][e & 3]);
      moves |= !(hi[p] - ref[p] <= SLACK);
    }
    if (__ballot(moves) != 0) {
#pragma unroll
      for (int p = 0; p < NB; ++p) {
        const float now = larger(ref[p], hi[p]);
        sum[p] *= __builtin_amdgcn_exp2f(ref[p] - (now == -INFINITY ? 0.0f : now));
        ref[p] = now;
      }
    }
#pragma unroll
    for (int p = 0; p < NB; ++p) {
      const float from = ref[p] == -INFINITY ? 0.0f : ref[p];
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[p] += __builtin_amdgcn_exp2f(t[p][e >> 2][e & 3] - from);
    }
  }
#pragma unroll
  for (int p = 0; p < NB; ++p)
#pragma unroll
    for (int m = 16; m < 64; m <<= 1)
      join(ref[p], sum[p], exl3::xor_lanes(ref[p], m), exl3::xor_lanes(sum[p], m));
  __syncthreads();
  if (bad) sbad = 1;
#pragma unroll
  for (int p = 0; p < NB; ++p)
    if (g == 0) so[wave][FEW * p + col] = f32x2{ref[p], sum[p]};
  __syncthreads();
  const int64_t slot = (int64_t)(f.first + f.j) * a.pool.kv + head;
  if (threadIdx.x < TILE && slot < a.slots) {
    float all = -INFINITY, whole = 0.0f;
#pragma unroll
    for (int x = 0; x < WW; ++x) join(all, whole, so[x][threadIdx.x][0], so[x][threadIdx.x][1]);
    if (sbad) whole = __builtin_nanf("");
    a.part[slot * TILE + threadIdx.x] = f32x2{all, whole};
  }
}

// The second pass: the same keys' scores again, 4 keys a thread, once the items of the
// sequence are joined.  Four pairs' scores are asked for at once, the first ones ahead of the
// joining, since a load's latency is all that a thread waits for.
template <int NB>
__global__ __launch_bounds__(64 * WW) void weigh_few_keys_kernel(WeighArgs a) {
  constexpr int AT = 4, BY = 256 * WW, TILE = FEW * NB, ROWS = 64 * WW / TILE;
  __shared__ f32x2 so[ROWS][TILE];
  const int head = blockIdx.x % a.pool.kv;
  const Find f = Finder<ITEM>(a).at(blockIdx.x / a.pool.kv);
  if (f.s < 0) return;
  const Watch &w = f.w;
  const int k0 = (int)min((int64_t)f.j * f.each * 64, (int64_t)w.keys);
  const int k1 = (int)min((int64_t)k0 + (int64_t)f.each * 64, (int64_t)w.keys);
  const float *from = a.t + ((int64_t)f.s * a.pool.kv + head) * a.most * a.wide;
  float *score = a.score + ((int64_t)f.s * a.pool.kv + head) * a.room;
  const int base = a.base ? a.base[f.s] : w.len;
  f32x4 t[AT];
  float had[4];
  auto load = [&](int k, int p) {
#pragma unroll
    for (int x = 0; x < AT; ++x)
      if (p + x < w.pairs) t[x] = *reinterpret_cast<const f32x4 *>(from + (int64_t)(p + x) * a.wide + k);
    if (p > 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) had[e] = k + e < min(k1, base) ? score[k + e] : 0.0f;
  };
  int k = k0 + 4 * (int)threadIdx.x;
  if (k < k1) load(k, 0);
  const int col = threadIdx.x % TILE, row = threadIdx.x / TILE;
  float ref = -INFINITY, sum = 0.0f;
  for (int j = row; j < f.parts; j += ROWS) {
    const int64_t slot = (int64_t)(f.first + j) * a.pool.kv + head;
    if (slot >= a.slots) break;
    const f32x2 v = a.part[slot * TILE + col];
    join(ref, sum, v[0], v[1]);
  }
  so[row][col] = f32x2{ref, sum};
  __syncthreads();
  if (threadIdx.x < TILE) {
    for (int x = 1; x < ROWS; ++x) join(ref, sum, so[x][col][0], so[x][col][1]);
    so[0][col] = ended(ref, sum);
  }
  __syncthreads();
  for (; k < k1; k += BY) {
    f32x4 acc{0, 0, 0, 0};
    for (int p = 0;;) {
#pragma unroll
      for (int x = 0; x < AT; ++x) {
        if (p + x >= w.pairs) break;
        const f32x2 r = so[0][p + x];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = fmaf(__builtin_amdgcn_exp2f(t[x][e] - r[0]), r[1], acc[e]);
          if (t[x][e] != UNSEEN) acc[e] = y;
        }
      }
      p += AT;
      if (p >= w.pairs) break;
      load(k, p);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < k1) score[k + e] = k + e < base ? a.decay * had[e] + acc[e] : acc[e];
    if (k + BY < k1) load(k + BY, 0);
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

constexpr int BINS = 2048;
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

// Scores in the order of whole numbers, between NEVER and ALWAYS; NaN below all, zeros alike.
constexpr uint32_t NEVER = 0, ALWAYS = ~0u;
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return x != x ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Bits of the lanes below this one, and `more`.
__device__ __forceinline__ uint32_t below(uint64_t bits, uint32_t more) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(bits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bits, more));
}
// Of the waves' numbers: the sum of those before this wave, and of all.  (By lanes: P / 64
// numbers in registers would be too many beside the scores.)
template <int P>
__device__ __forceinline__ uint32_t before_wave(const uint32_t (&waves)[P / 64], uint32_t &whole) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t v = lane < P / 64 ? waves[lane] : 0, x = (uint32_t)scan((int)v);
  whole = __builtin_amdgcn_readlane(x, 63);
  return __builtin_amdgcn_readlane(x - v, wave);
}
// Sum over the workgroup's threads before this one, and over all.
template <int P>
__device__ __forceinline__ uint32_t before(uint32_t v, uint32_t (&waves)[P / 64], uint32_t &whole) {
  const uint32_t x = (uint32_t)scan((int)v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = x;
  __syncthreads();
  return before_wave<P>(waves, whole) + x - v;
}

// P threads a sequence, layer and kv head, N scores of each in registers (where there
// are more than P N they are read again in each pass).  The budget's border is found by
// counting: the range of the scores in BINS bins, then the bin that holds the
// border in BINS again, three rounds at most (32 bits of order), or, once a bin
// holds few keys, by each one's rank among them.  Bins divide the range that
// the scores have, so that few of them fall into one and the counters in LDS are
// rarely fought over.  Then the keys above the border, and as many of those on
// it as are left, earliest first, get their places by counting: a wave's keys lie
// side by side, so that the waves' counts join once.
template <int P, int N, bool MANY>
__global__ __launch_bounds__(P) void evict_pick_kernel(EvictArgs a) {
  constexpr int HELD = P * N, WAVES = P / 64;
  // the keys that stay meet in LDS, where a turn's few of a wave cost less than stores
  constexpr int STAGED = HELD < 4096 ? HELD : 4096;
  __shared__ int places[STAGED];
  // few keys: of their order, and the earlier one above the later
  __shared__ __align__(16) union { uint32_t bins[BINS]; uint64_t cand[FEWEST + 1]; } m;
  __shared__ uint32_t waves[WAVES], lows[WAVES], highs[WAVES];
  __shared__ int chosen, above, holds, count, found_ties;
  __shared__ uint32_t found;
  const int heads = a.layers * a.pool.kv;
  const int s = blockIdx.x / heads, lh = blockIdx.x - s * heads;
  const int layer = lh / a.pool.kv, h = lh - layer * a.pool.kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = a.len[s];
  const int b = budget_of(a, s, len);
  const size_t at = ((size_t)layer * a.seqs + s) * a.pool.kv + h;
  const float *score = a.score + at * a.room;
  float *to_score = a.new_score + at * a.room;
  int32_t *kept = a.kept + at * a.most;
  const int head = min(a.first, max(b, 0)), tail = min(a.last, max(b, 0) - head);  // those that stay anyway
  const int lo = head, hi = len - tail;                                            // the others
  const int blocks = b < 0 ? 0 : MANY ? (len + HELD - 1) / HELD : 1;
  // key number k0 + 64 e in turn e; those that are not among the others ALWAYS, those behind
  // the wave's keys (in turns that a short sequence does not need) NEVER
  uint32_t key[N];
  int k0 = 0;
  auto read = [&](int blk) __attribute__((always_inline)) {
    const int each = 64 * ((min(HELD, len - blk * HELD) + P - 1) / P);
    k0 = blk * HELD + wave * each + lane;
    const int end = min(blk * HELD + (wave + 1) * each, len);
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = score[min(k0 + 64 * e, len - 1)];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int k = k0 + 64 * e;
      key[e] = k >= end ? NEVER : (uint32_t)(k - lo) < (uint32_t)(hi - lo) ? ordered(x[e]) : ALWAYS;
    }
  };
  auto each = [&](auto &&f) __attribute__((always_inline)) {
    for (int blk = 0; blk < blocks; ++blk) {
      if (MANY) read(blk);
      asm volatile("" : "+v"(k0));  // (N numbers of keys are not kept)
#pragma unroll
      for (int e = 0; e < N; ++e) f(key[e], k0 + 64 * e);
    }
  };
  if (!MANY && b >= 0) read(0);
  uint32_t low = ALWAYS, past = 0;  // the others' range: low + 1 .. past - 1
  bool bad = b < 0;
  if (!bad) {
#pragma unroll 4
    for (int y = tid; y < (len + (1 << a.pool.lp) - 1) >> a.pool.lp; y += P)
      bad |= (uint32_t)a.pool.table[(size_t)s * a.pool.max_pages + y] >= (uint32_t)a.pool.pages;
    each([&](uint32_t k, int) { low = min(low, k - 1), past = max(past, k + 1); });
  }
#pragma unroll
  for (int y = 1; y < 64; y <<= 1)
    low = min(low, (uint32_t)__shfl_xor((int)low, y)), past = max(past, (uint32_t)__shfl_xor((int)past, y));
  if (lane == 0) lows[wave] = low, highs[wave] = past;
  for (int i = tid; i < BINS; i += P) m.bins[i] = 0;
  bad = __syncthreads_or(bad);
  if (tid == 0 && lh == 0) a.new_len[s] = bad ? len : b;
  for (int y = (bad ? 0 : b) + tid; y < a.most; y += P) kept[y] = -1;
  if (bad || b == 0) return;
  int need = b - head - tail;
  // the border: keys of more than `border` stay, and the first `ties` on it
  uint32_t border = ALWAYS - 1;
  int ties = 0;
  if (need > 0) {
    low = lows[lane % WAVES], past = highs[lane % WAVES];
#pragma unroll
    for (int y = 1; y < WAVES; y <<= 1)
      low = min(low, (uint32_t)__shfl_xor((int)low, y)), past = max(past, (uint32_t)__shfl_xor((int)past, y));
    uint32_t width = past - 2 - low;  // the range: low .. low + width
    ++low;
    for (;;) {
      const int shift = max(0, 32 - (width ? __builtin_clz(width) : 32) - 11);
      each([&](uint32_t k, int) {
        if (k - low <= width) atomicAdd(&m.bins[(k - low) >> shift], 1u);
      });
      if (tid == 0) count = 0;
      __syncthreads();
      // a thread's bins, the highest first
      constexpr int B = BINS / P;
      uint32_t own[B], all = 0, whole;
#pragma unroll
      for (int e = 0; e < B; ++e) all += own[e] = m.bins[BINS - 1 - B * tid - e];
      uint32_t over = before<P>(all, waves, whole);
      if (over < (uint32_t)need && over + all >= (uint32_t)need) {
#pragma unroll
        for (int e = 0; e < B; ++e) {
          if (over < (uint32_t)need && over + own[e] >= (uint32_t)need)
            chosen = BINS - 1 - B * tid - e, above = (int)over, holds = (int)own[e];
          over += own[e];
        }
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
          if (k - low <= width) m.cand[atomicAdd(&count, 1)] = (uint64_t)k << 32 | ~(uint32_t)i;
        });
        if (tid == 0) m.cand[n] = 0;
        __syncthreads();
        for (int y = tid; y < n; y += P) {
          const uint64_t own_key = m.cand[y];
          int more = 0, higher = 0;  // before this one, and those of them of higher scores
#pragma unroll 4
          for (int c = 0; c < n; c += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(m.cand + c);
            more += (two.x > own_key) + (two.y > own_key);
            higher += (uint32_t)(two.x >> 32) > (uint32_t)(own_key >> 32);
            higher += (uint32_t)(two.y >> 32) > (uint32_t)(own_key >> 32);
          }
          if (more == need - 1) found = (uint32_t)(own_key >> 32), found_ties = need - higher;
        }
        __syncthreads();
        border = found, ties = found_ties;
        break;
      }
      for (int i = tid; i < BINS; i += P) m.bins[i] = 0;
      __syncthreads();
    }
  }
  // places: what stays whatever the ties are, and the ties, before each key
  const bool staged = b <= STAGED;
  uint32_t sure0 = 0, tie0 = 0;  // of the blocks before
  for (int blk = 0; blk < blocks; ++blk) {
    if (MANY) read(blk);
    uint32_t sure = 0, tie = 0;  // the wave's
    asm volatile("" : "+v"(k0));
#pragma unroll
    for (int e = 0; e < N; ++e) {
      sure += __popcll(__ballot(key[e] > border));
      tie += __popcll(__ballot(key[e] == border));
    }
    // (of a wave and of a block, neither is more than 16 bits hold)
    __syncthreads();
    if (lane == 0) waves[wave] = sure | tie << 16;
    __syncthreads();
    uint32_t whole;
    const uint32_t both = before_wave<P>(waves, whole);
    uint32_t ns = sure0 + (both & 0xFFFFu), nt = tie0 + (both >> 16);
    sure0 += whole & 0xFFFFu, tie0 += whole >> 16;
    auto place = [&](auto &&put) __attribute__((always_inline)) {
      if (tie == 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          asm volatile("" : "+v"(border), "+v"(k0));  // (compared again, not kept from before)
          const uint64_t bs = __ballot(key[e] > border);
          if (key[e] > border) put(below(bs, ns + min(nt, (uint32_t)ties)), e);
          ns += __popcll(bs);
        }
        return;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        asm volatile("" : "+v"(border), "+v"(k0));
        const bool on = key[e] == border;
        const uint64_t bs = __ballot(key[e] > border), bt = __ballot(on);
        const uint32_t t = below(bt, nt);
        if (key[e] > border || (on && t < (uint32_t)ties)) put(below(bs, ns) + min(t, (uint32_t)ties), e);
        ns += __popcll(bs), nt += __popcll(bt);
      }
    };
    if (staged)
      place([&](uint32_t to, int e) { places[to] = k0 + 64 * e; });
    else
      place([&](uint32_t to, int e) { kept[to] = k0 + 64 * e; });
  }
  // places ascend and no key moves back: what a turn overwrites only turns up to it read
  for (int y0 = 0; y0 < b; y0 += 4 * P) {
    __syncthreads();
    int from[4];
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int y = min(y0 + P * i + tid, b - 1);
      from[i] = staged ? places[y] : kept[y];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = score[from[i]];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(x[i]));  // in its register
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int y = y0 + P * i + tid;
      if (y < b) {
        if (staged) kept[y] = from[i];
        to_score[y] = x[i];
      }
    }
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
// Of every pair's reference, and as many of its 1 / sum.
size_t refs_bytes(const exl3p_cache *c, const exl3p_rows *r, int group) {
  return up16((size_t)r->rows * group * c->kv_heads * sizeof(float));
}

// How the weights are formed, by what the host knows.  Pairs whose scores are
// kept read the keys once and the scores (4 bytes a pair and key) twice; others
// read the keys twice, in a launch or two more.  32 pairs (trees of 8 rows, 4 query heads of
// 128), kept and not: over 2000 keys 14.7 and 20.6 us, 16 sequences over up to 4000 keys 39 and
// 56, 48 over up to 3000 57 and 79, but one over 40000 43.7 and 40.6.  64 pairs kept would be 21.9
// and 21.2 over 2000 keys, 69 and 42 over 40000.
struct Plan {
  int group;
  int tile;              // pairs
  int64_t tiles, items;  // at most
  int few;               // pairs whose scores are kept, 0: none
  int wide;              // of a row of them
  int deal, deals;       // pairs of an item of the second pass, such items of a key at most
  size_t parts, rest, sums;  // bytes
};
constexpr size_t KEPT_MAX = (size_t)1 << 30;
// A deal is a tile, so that its pairs stay in registers, until the deals' sums would
// take more than this.
constexpr size_t SUMS_MAX = (size_t)1 << 28;
// Items of many pairs, in first passes' workgroups: 264 us for 3 prompts of up to 2048 rows
// with 2, 270 with 3, 305 and more with 4; 315 with 1, some of which are long after others (one
// number a pair between the passes then, 4 us less than two).
constexpr int ROUNDS = 2;
Plan plan_of(const exl3p_cache *c, const exl3p_rows *r, int32_t heads, int32_t window, int32_t room) {
  Plan p;
  p.group = heads / c->kv_heads;
  const int64_t rows = window > 0 && window < r->max_rows ? window : r->max_rows, pairs = rows * p.group;
  p.wide = (room + 15) & ~15;
  p.few = pairs <= 2 * FEW ? (int)pairs : 0;
  p.rest = (size_t)r->seqs * c->kv_heads * p.few * p.wide * sizeof(float);
  if (p.rest > KEPT_MAX) p.few = 0;
  if (p.few == 0) p.rest = 2 * refs_bytes(c, r, p.group);
  p.tile = p.few > FEW ? 2 * FEW : p.few ? FEW : TILE;
  p.tiles = rows_watched(r, window) * p.group / p.tile + r->seqs;
  p.items = target_of(c) * (p.few ? 1 : ROUNDS) + p.tiles;
  for (p.deal = p.tile;; p.deal *= 2) {
    p.deals = p.few ? 1 : (int)((pairs + p.deal - 1) / p.deal);
    p.sums = p.deals > 1 ? up16((size_t)r->seqs * c->kv_heads * p.deals * room * sizeof(float)) : 0;
    if (p.sums <= SUMS_MAX || p.deals == 2) break;
  }
  p.parts = (size_t)p.items * c->kv_heads * p.tile * sizeof(f32x2);
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
  return p.parts + p.rest + p.sums;
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
  // items of a deal and a part of the keys are counted in 32 bits, spans of 64 keys are a grid
  const int64_t spans = r->seqs * (((int64_t)room + 63) / 64);
  if ((int64_t)r->rows * p.group > INT32_MAX / 2 || p.items * c->kv_heads * (p.tile / 16) > GRID_MAX ||
      (r->seqs * ((int64_t)room / PART + 1) + p.items) * p.deals > INT32_MAX / 2 ||
      (p.deals > 1 && spans * c->kv_heads > GRID_MAX))
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
  // at least f32's smallest, so that a hidden key's -inf times it stays -inf
  a.scale = fmaxf(fabsf(scale) * LOG2E, 1.17549435e-38f), a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.decay = decay, a.base = base, a.score = score, a.room = room;
  a.target = (float)(p.items - p.tiles), a.slots = (int)(p.items * c->kv_heads);
  a.least = p.few ? 2.0f : 4.0f;
  // An item's start (its place among the items, its pairs' 32 KB of q) costs as much as some tiles
  // of keys: up to 16 units while half the first pass' workgroups are left.  A window of 128
  // pairs over 32048 keys and one over 24456: 78.5 us with 4 units at least, 72.7 while all of them are
  // left, 67.7 so, 66.7 up to 24 units, 77.4 up to 32 and a quarter of them.
  a.fill = 0.5f * (float)target_of(c), a.some = p.few ? 0.0f : 16.0f;
  a.part = static_cast<f32x2 *>(scratch);
  a.t = a.ref = reinterpret_cast<float *>(static_cast<char *>(scratch) + p.parts);
  a.inv = a.ref + refs_bytes(c, r, p.group) / sizeof(float);
  a.most = p.few, a.wide = p.wide;
  a.sums = reinterpret_cast<float *>(static_cast<char *>(scratch) + p.parts + p.rest);
  a.tile = p.tile, a.deal = p.deal, a.deals = p.deals;
  const hipStream_t st = static_cast<hipStream_t>(s);
  const dim3 items((unsigned)(p.items * c->kv_heads));
  return by_type(c, [&](auto e, auto d) {
    if (p.few) {
      auto blocks = [&](auto nb) {
        hipLaunchKernelGGL((weigh_few_sums_kernel<decltype(e), d, nb>), items, dim3(64 * WW), 0, st, a);
        hipLaunchKernelGGL((weigh_few_keys_kernel<nb>), items, dim3(64 * WW), 0, st, a);
      };
      if (p.tile == FEW)
        blocks(std::integral_constant<int, 1>{});
      else
        blocks(std::integral_constant<int, 2>{});
      return;
    }
    // the second pass' items: as many as its target may make, or round again
    const dim3 parts((unsigned)((target_of(c) * ROUNDS + p.tiles) * c->kv_heads));

    hipLaunchKernelGGL((weigh_sums_kernel<decltype(e), d>), items, dim3(64 * WW), 0, st, a);
    // few tiles have many items each
    if (p.tiles * 8 <= p.items)
      hipLaunchKernelGGL(weigh_join_kernel<16>, dim3((unsigned)(p.tiles * c->kv_heads * (p.tile / 16))),
                         dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL(weigh_join_kernel<2>, dim3((unsigned)(p.tiles * c->kv_heads * (p.tile / 128))),
                         dim3(256), 0, st, a);
    hipLaunchKernelGGL((weigh_keys_kernel<decltype(e), d>), parts, dim3(64 * WW), 0, st, a);
    if (p.deals > 1)
      hipLaunchKernelGGL(weigh_deals_kernel, dim3((unsigned)(spans * c->kv_heads)), dim3(64 * WW), 0, st, a);
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
  if (n * 4 > GRID_MAX)  // of 1024 threads, and `parts` of 256
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
  auto pick = [&](auto threads, auto each, auto many) {
    hipLaunchKernelGGL((evict_pick_kernel<decltype(threads)::value, decltype(each)::value, decltype(many)::value>),
                       dim3((unsigned)n), dim3(decltype(threads)::value), 0, st, a);
  };
  // as few turns and threads as the room asks for (a turn is work whether it has keys or
  // not): 9.4 us for 1100 keys of 288 heads with 16 turns of 256 threads, 7.9 with 8; 12.8 for
  // 4096 of 1024 heads with 16 of 256, 11.2 with 8 of 512, 16.6 with 4 of 1024; 18 for 32768
  // of 64 heads, 36 with the scores in LDS instead
  typedef std::integral_constant<int, 8> Few;
  typedef std::integral_constant<int, 32> Many;
  typedef std::integral_constant<int, 1024> Wide;
  if (room <= 256 * 8)
    pick(std::integral_constant<int, 256>{}, Few{}, std::false_type{});
  else if (room <= 512 * 8)
    pick(std::integral_constant<int, 512>{}, Few{}, std::false_type{});
  else if (room <= 1024 * 8)
    pick(Wide{}, Few{}, std::false_type{});
  else if (room <= 1024 * 32)
    pick(Wide{}, Many{}, std::false_type{});
  else
    pick(Wide{}, Many{}, std::true_type{});
  if (c->dim == 64)
    hipLaunchKernelGGL(evict_move_kernel<64>, dim3((unsigned)(n * parts)), dim3(MV), 0, st, a);
  else
    hipLaunchKernelGGL(evict_move_kernel<128>, dim3((unsigned)(n * parts)), dim3(MV), 0, st, a);
  return launched();
}

}  // extern "C"
