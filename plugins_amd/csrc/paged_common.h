// paged_common.h -- what the operators over a paged KV cache share: element types,
// a cache and a step's rows as the kernels see them, and the host's checks.
#ifndef EXL3_PAGED_COMMON_H
#define EXL3_PAGED_COMMON_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "../../include/exl3_paged.h"
#include "exl3_device.h"

namespace {


typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The element types of a cache: f32 conversions (to: one rounding, to nearest
// even), the exponent bits that mark infinities and NaN, the matrix product,
// and the power of two that softmax weights are scaled by (exponents below).
struct F16 {
  typedef _Float16 T;
  typedef half2_t T2;
  typedef half8 V8;
  static constexpr uint32_t EXP = 0x7C00u;
  // weights of 2^(11 + SLACK) and less: one 2^-35 as large as the row's largest
  // is still not lost to f16's smallest number (2^-24)
  static constexpr float LIFT = 11.0f;
  static __device__ __forceinline__ f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // c plus both elements
  static __device__ __forceinline__ float add2(uint32_t v, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, v), half2_t{1, 1}, c, false);
  }
};
struct BF16 {
  typedef __bf16 T;
  typedef bf16x2 T2;
  typedef bf16x8 V8;
  static constexpr uint32_t EXP = 0x7F80u;
  static constexpr float LIFT = 0.0f;  // f32's exponents
  static __device__ __forceinline__ f32x4 mma(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(uint32_t v, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{1, 1}, c, false);
  }
};
template <typename E>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  return (float)__builtin_bit_cast(typename E::T, (uint16_t)bits);
}
template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), typename E::T2));
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
  bool bad;   // its keys do not fit its table
  bool back;  // cu goes back here: sequences may share rows, and have more than all
};
__device__ __forceinline__ Span span_of(const Step &st, int s, int64_t room) {
  const int a = min(max(st.cu[s], 0), st.rows);
  const int to = min(max(st.cu[s + 1], 0), st.rows), b = max(to, a);
  Span sp;
  sp.row = a;
  sp.n = min(b - a, st.max_rows);
  sp.len = st.len[s];
  sp.bad = sp.len < 0 || (int64_t)sp.len + sp.n > room;
  sp.back = to < a;
  if (sp.bad) sp.len = 0;
  return sp;
}

// The slot of a sequence's key, -1 where the table names no page of the pool.
__device__ __forceinline__ int slot_of(const Pool &p, int s, int key) {
  const uint32_t page = (uint32_t)p.table[(size_t)s * p.max_pages + (key >> p.lp)];
  return page < (uint32_t)p.pages ? (int)((page << p.lp) | (key & ((1 << p.lp) - 1))) : -1;
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // 1, 2, 4, 8 lanes down a row
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // a row's last lane to the next
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // the second row's to both after
  return v;
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
  if ((int64_t)c->pages * c->page > INT32_MAX || (int64_t)c->max_pages * c->page > 1 << 30)
    return refuse(EXL3_TOO_LARGE, "PagedCacheShape: 2^31 keys or more, or over 2^30 of a sequence");
  if (c->kv_heads > 65535 || c->layers > 32767)
    return refuse(EXL3_TOO_LARGE, "PagedCacheShape: over 65535 kv heads or 32767 layers");
  return OK;
}

exl3_verdict check_rows(const exl3p_cache *c, const exl3p_rows *r) {
  if (r == nullptr || r->size != sizeof(exl3p_rows))
    return refuse(EXL3_FAILED, "PagedRows: no rows, or another version's");
  if (r->seqs < 0 || r->rows < 0 || r->max_rows < 0 || r->max_rows > r->rows)
    return refuse(EXL3_UNSUPPORTED, "PagedRows: sizes below 0, or more rows a sequence than rows");
  if (r->seqs > 65535) return refuse(EXL3_TOO_LARGE, "PagedRows: over 65535 sequences");
  if (r->rows > 1 << 30) return refuse(EXL3_TOO_LARGE, "PagedRows: over 2^30 rows");
  if (r->seqs > c->seqs) return refuse(EXL3_UNSUPPORTED, "PagedRows: more sequences than the cache's");
  if (r->cu == nullptr || (r->len == nullptr && r->seqs > 0))
    return refuse(EXL3_FAILED, "PagedRows: a missing array");
  return OK;
}

exl3_verdict check_mask(const exl3p_rows *r, const void *mask, int32_t words) {
  // (of no rows it may lie nowhere)
  if (words < 0 || (r->rows > 0 && (mask == nullptr) != (words == 0)) ||
      (mask != nullptr && (int64_t)words * 64 < r->max_rows))
    return refuse(EXL3_UNSUPPORTED, "PagedMask: 64 * words below the rows of a sequence");
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

// A grid's workgroups of 256 threads in one dimension: the launch counts threads
// in 32 bits.
constexpr int64_t GRID_MAX = ((int64_t)1 << 24) - 1;

// Memory of a tensor: `rows` pieces of `width` bytes, `stride` apart (rows that
// do not overlap one another).
struct Span2D {
  const void *p;
  int64_t rows, width, stride;
};
Span2D array(const void *p, int64_t bytes) { return Span2D{p, bytes > 0, bytes, bytes}; }
Span2D matrix(const void *p, int64_t stride, int64_t width, int64_t rows) {
  return Span2D{p, rows, 2 * width, 2 * stride};
}

// Whether a byte lies in both: exact for slices of one matrix too, whose rows
// interleave.
bool meet(Span2D x, Span2D y) {
  typedef __int128 wide;
  if (x.p == nullptr || y.p == nullptr || x.rows <= 0 || y.rows <= 0) return false;
  const wide d = (wide) reinterpret_cast<uintptr_t>(y.p) - reinterpret_cast<uintptr_t>(x.p);
  auto end = [](const Span2D &v) { return (wide)(v.rows - 1) * v.stride + v.width; };
  if (d >= end(x) || -d >= end(y)) return false;
  // row i of x against the last row of y that begins before it ends
  auto row = [&](int64_t i) {
    const wide from = (wide)i * x.stride - d, last = from + x.width - 1;
    if (last < 0) return false;
    const wide j = last / y.stride < y.rows - 1 ? last / y.stride : y.rows - 1;
    return j * y.stride + y.width > from;
  };
  if (x.rows > 1 && y.rows > 1 && x.stride == y.stride) {
    // every row lies alike among the other's, but for where those begin and end:
    // row i meets row i + k, k the number below or the one before it
    wide k = x.width - 1 - d;
    k = k >= 0 ? k / x.stride : -((-k + x.stride - 1) / x.stride);
    for (int u = 0; u < 2; ++u, --k)
      if (k > -x.rows && k < y.rows && d + k * x.stride < x.width && d + k * x.stride > -(wide)y.width)
        return true;
    return false;
  }
  if (x.rows > y.rows) return meet(y, x);
  for (int64_t i = 0; i < x.rows; ++i)
    if (row(i)) return true;
  return false;
}

// What a call writes lies over nothing that it reads and over nothing else that it
// writes: workgroups come in any order.
exl3_verdict check_apart(std::initializer_list<Span2D> writes, std::initializer_list<Span2D> reads) {
  for (const Span2D &w : writes)
    for (const Span2D &x : reads)
      if (meet(w, x)) return refuse(EXL3_UNSUPPORTED, "PagedOverlap: an output over an input");
  for (auto w = writes.begin(); w != writes.end(); ++w)
    for (auto x = writes.begin(); x != w; ++x)
      if (meet(*w, *x)) return refuse(EXL3_UNSUPPORTED, "PagedOverlap: an output over another");
  return OK;
}
Span2D table_of(const exl3p_cache *c) { return array(c->table, (int64_t)c->seqs * c->max_pages * 4); }

// The device's compute units, read once per device.
int device_cus() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

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

#endif  // EXL3_PAGED_COMMON_H
