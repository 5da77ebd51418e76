// What the kernels of the paged cache share: how a position finds its row, and the host checks of a cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "apart.h"
#include "div.h"
#include "fcr.h"

namespace fcr_detail {
int fail(int code, const char* what);      // fcr.hip: the error text of this thread
int launched(const char* what);            // fcr.hip: the launch's status as a return code
int chip_cus_of_current_device();
}  // namespace fcr_detail

namespace fcr_paged {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int64_t kMaxBlocks = 1ll << 24;   // of 256 threads: the runtime refuses launches of 2^32 threads or more

// One side (keys or values) of a cache: strides of pages, heads and rows in bytes, those of scales (a head's page has consecutive ones)
// in elements.
struct Side {
  char* rows;
  float* scale;
  int64_t page, head, row;
  int64_t s_page, s_head;
};
struct Pages {
  Side side[2];
  const int32_t* table;
  int64_t table_stride;
  int table_pages, pages, H;
  Div page_size;
  int64_t capacity;      // positions that a row of the table names
};
struct Lengths {          // an int32 per sequence, or per sequence and head
  const int32_t* at;
  int64_t sb, sh;
  __device__ __forceinline__ int of(int b, int h) const;
};

// Words that no kernel writes while others read them: read by the scalar unit where every lane asks for the same one.
__device__ __forceinline__ int constant_at(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

__device__ __forceinline__ int Lengths::of(int b, int h) const { return constant_at(at + b * sb + h * sh); }

// The page of position `pos` (0 <= pos < capacity), or -1 where it is not there.
__device__ __forceinline__ int page_of(const Pages& c, int b, uint32_t pos, uint32_t& row) {
  const uint32_t i = c.page_size.of(pos);
  row = pos - i * c.page_size.d;
  const int page = constant_at(c.table + b * c.table_stride + i);
  return (uint32_t)page < (uint32_t)c.pages ? page : -1;
}

inline int element_bytes(int dtype) {
  return dtype == FCR_DTYPE_F32 ? 4 : dtype == FCR_DTYPE_F16 || dtype == FCR_DTYPE_BF16 ? 2 : 1;
}
inline bool has_codes(int dtype) { return dtype == FCR_DTYPE_INT8 || dtype == FCR_DTYPE_E4M3; }

// (tests without a device reach these: nothing here calls HIP)
inline int check_cache(const fcr_cache* c, const char* name) {
  using fcr_detail::fail;
  char text[160];
  if (!c || !c->k || !c->v) return fail(FCR_E_NULL, "null pointer argument");
  if (c->dtype != FCR_DTYPE_F16 && c->dtype != FCR_DTYPE_BF16 && !has_codes(c->dtype))
    return fail(FCR_E_DTYPE, "a cache holds FCR_DTYPE_F16, FCR_DTYPE_BF16, FCR_DTYPE_INT8 or FCR_DTYPE_E4M3");
  if (has_codes(c->dtype) && (!c->k_scale || !c->v_scale)) return fail(FCR_E_NULL, "a cache of codes needs its scales");
  if (c->pages < 1 || c->H < 1 || c->page_size < 16 || c->page_size % 16 != 0 || c->D < 16 || c->D > 256 || c->D % 16 != 0) {
    snprintf(text, sizeof(text), "%s: pages and H must be >= 1, page_size a positive multiple of 16, D a multiple of 16 in [16, 256]", name);
    return fail(FCR_E_SHAPE, text);
  }
  // (the stride of a dimension of size one is never used: torch reports any value there)
  const int e = element_bytes(c->dtype);
  const int sizes[3] = {c->pages, c->H, c->page_size};
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? c->v_strides : c->k_strides;
    bool ok = (reinterpret_cast<uintptr_t>(i ? c->v : c->k) & 15) == 0 && s[2] >= c->D && s[2] * e < (1 << 25);
    for (int j = 0; j < 3; ++j) ok = ok && (sizes[j] == 1 || (s[j] >= 0 && s[j] < (1ll << 40) && s[j] * e % 16 == 0));
    if (!ok) {
      snprintf(text, sizeof(text), "%s: 16-byte aligned pointers, strides in multiples of 16 bytes, rows that do not overlap and lie less than 2^25 bytes apart", name);
      return fail(FCR_E_STRIDE, text);
    }
    if (!has_codes(c->dtype)) continue;
    const int64_t* f = i ? c->v_scale_strides : c->k_scale_strides;
    ok = (reinterpret_cast<uintptr_t>(i ? c->v_scale : c->k_scale) & 15) == 0 && f[2] == 1;
    for (int j = 0; j < 2; ++j) ok = ok && (sizes[j] == 1 || (f[j] >= 0 && f[j] < (1ll << 40) && f[j] % 4 == 0));
    if (!ok) {
      snprintf(text, sizeof(text), "%s: scales of a head's page are consecutive, pages and heads 16-byte aligned", name);
      return fail(FCR_E_STRIDE, text);
    }
  }
  return 0;
}

// A cache that is written: no two of its rows share memory.
inline int check_written(const fcr_cache& c, const char* name) {
  char text[128];
  Dimension rows[2][3], scales[2][2];
  for (int i = 0; i < 2; ++i) {
    const int64_t *s = i ? c.v_strides : c.k_strides, *f = i ? c.v_scale_strides : c.k_scale_strides;
    rows[i][0] = Dimension{c.pages, s[0]}, rows[i][1] = Dimension{c.H, s[1]}, rows[i][2] = Dimension{c.page_size, s[2]};
    scales[i][0] = Dimension{c.pages, f[0]}, scales[i][1] = Dimension{c.H, f[1]};
  }
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if (rows_apart(c.D, rows[0], at(c.k), rows[1], at(c.v), 3, element_bytes(c.dtype)) &&
      (!has_codes(c.dtype) || rows_apart(c.page_size, scales[0], at(c.k_scale), scales[1], at(c.v_scale), 2, 4)))
    return 0;
  snprintf(text, sizeof(text), "%s: rows that share memory (of an expanded view, of keys and values) cannot be written", name);
  return fcr_detail::fail(FCR_E_STRIDE, text);
}

inline int check_table(const int32_t* table, int64_t stride, int pages, int page_size, int B) {
  using fcr_detail::fail;
  if (!table) return fail(FCR_E_NULL, "null pointer argument");
  if (B < 1 || pages < 1 || (int64_t)pages * page_size > (1 << 30))
    return fail(FCR_E_SHAPE, "B and the table's pages must be >= 1, and name at most 2^30 positions");
  if (stride < 0 || (reinterpret_cast<uintptr_t>(table) & 3) != 0) return fail(FCR_E_STRIDE, "the table's stride must be >= 0");
  return 0;
}

inline Pages pages_of(const fcr_cache& c, const int32_t* table, int64_t stride, int table_pages) {
  Pages p;
  const int e = element_bytes(c.dtype);
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? c.v_strides : c.k_strides;
    const int64_t* f = i ? c.v_scale_strides : c.k_scale_strides;
    const bool codes = has_codes(c.dtype);
    p.side[i] = Side{static_cast<char*>(i ? c.v : c.k), codes ? (i ? c.v_scale : c.k_scale) : nullptr,
                     c.pages > 1 ? s[0] * e : 0, c.H > 1 ? s[1] * e : 0, s[2] * e,
                     codes && c.pages > 1 ? f[0] : 0, codes && c.H > 1 ? f[1] : 0};
  }
  p.table = table;
  p.table_stride = stride;
  p.table_pages = table_pages;
  p.pages = c.pages;
  p.H = c.H;
  p.page_size.set((uint32_t)c.page_size);
  p.capacity = (int64_t)table_pages * c.page_size;
  return p;
}

// Elements and codes -------------------------------------------------------------------------------------------------

__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return (float)__builtin_bit_cast(f16x2, w)[i];
}
__device__ __forceinline__ float bf16_of(uint32_t w, int i) {
  return __builtin_bit_cast(float, i ? (w & 0xffff0000u) : (w << 16));
}
template <int DT>
__device__ __forceinline__ float element(uint32_t w, int i) {   // element i of the two in w
  if constexpr (DT == FCR_DTYPE_F16) return half_of(w, i);
  else return bf16_of(w, i);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {   // nearest, ties to even
  if constexpr (DT == FCR_DTYPE_F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// The four values that a word of codes stands for, without their scale.
template <int DT>
__device__ __forceinline__ void values_of(uint32_t w, float* x) {
  if constexpr (DT == FCR_DTYPE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((int32_t)(w << (24 - 8 * i)) >> 24);
  } else {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  }
}

}  // namespace fcr_paged
