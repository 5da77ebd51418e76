// The paged cache of keys and values: written (quantised or not), read back, and pruned by a keep-mask.
//
// Codes.  A row x of D elements is held as D codes of 8 bits and one fp32 scale, with a = max |x_d|:
//   int8   s = a / 127,  c_d = rint(127 x_d / a)      (ties to even)
//   e4m3   s = a / 448,  c_d = e4m3(448 x_d / a)      (ties to even)
// and stands for c_d s.  The largest element is the largest code, nothing saturates.  A row of zeros has s = 0; a row with an element
// that is not finite has s = NaN and codes 0, so codes are finite always and such a row reads as NaN.
// The quotient of 16-bit elements is formed so that the code is the one that exact arithmetic gives (see quotient).
//
// All three kernels are bound by memory: 16 elements per lane, 16 bytes and more per load and store.  Measured per call, D = 128 (a large copy
// reaches 4.95 TB/s): 32 x 8192 rows fp16 to e4m3 49 us (4.1 TB/s), fp32 to int8 80 (4.2); 8 x 32 heads of 9001 bf16 rows into a bf16 cache 472 us
// (5.0 TB/s) and back 441 (5.4), up to 9001 e4m3 rows to bf16 333 (4.9); half of up to 4 x 8 x 32768 bf16 rows kept 67 to 101 us by the drawn lengths
// (4.5 TB/s; rows of 256 bytes with gaps between them); one token of 64 sequences 4.6 us, one launch.

#include "paged.h"

namespace {
using namespace fcr_paged;
using fcr_detail::fail;
using fcr_detail::launched;

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// 16 elements as floats, from 2 (16-bit) or 4 loads of 16 bytes.
template <int DT>
__device__ __forceinline__ void load16(const char* at, float (&x)[16]) {
  const u32x4* w = reinterpret_cast<const u32x4*>(at);
  if constexpr (DT == FCR_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 v = w[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = __builtin_bit_cast(float, (uint32_t)v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 v = w[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * i + j] = element<DT>(v[j / 2], j & 1);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store16(char* at, const float (&x)[16]) {
  u32x4* w = reinterpret_cast<u32x4*>(at);
  if constexpr (DT == FCR_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(uint32_t, x[4 * i + j]);
      w[i] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = pack2<DT>(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
      w[i] = v;
    }
  }
}

// top * x / a.  For 16-bit x the product with top (7 significant bits, x at most 11) is exact, and one correction of the product with the
// reciprocal gives a quotient that is right to about half a step of fp32, and exact where the quotient is an fp32 value: ties of the
// rounding to codes stay ties.  Any other quotient is at least 2^-19 of its value away from a tie (top x / a = t / 2 with x = X 2^i,
// a = A 2^j and X, A < 2^11: the two sides of 2 top X 2^i = t A 2^j are integers times a power of two), where fp32 errs by 2^-23.
template <int IN, int CODE>
__device__ __forceinline__ float quotient(float x, float a, float inverse) {
  constexpr float top = CODE == FCR_DTYPE_INT8 ? 127.0f : 448.0f;
  const float n = x * top;
  if constexpr (IN == FCR_DTYPE_F32) {
    return n / a;
  } else {
    const float q = n * inverse;
    return __builtin_fmaf(__builtin_fmaf(-q, a, n), inverse, q);
  }
}

struct WriteArgs {
  Pages c;
  Lengths start, counts;
  const char* x[2];               // keys, values
  int64_t xb[2], xh[2], xt[2];    // strides in bytes
  Div T, H;
  uint32_t rows;                  // B * H * T
  int lanes_log2;                 // lanes per row
  int used;                       // of them, those with elements: D / 16
};

// L lanes take a row of keys or of values (blockIdx.y), 16 elements each; the largest element is found by log2 L exchanges.
template <int IN, int CODE>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(WriteArgs p) {
  const int which = blockIdx.y;
  const Side side = p.c.side[which];
  const int L = 1 << p.lanes_log2;
  const int lane = threadIdx.x & (L - 1);
  const uint32_t r = (blockIdx.x * kThreads + threadIdx.x) >> p.lanes_log2;
  if (r >= p.rows) return;                       // (the lanes of a row go together)
  const uint32_t bh = p.T.of(r), t = r - bh * p.T.d;
  const uint32_t b = p.H.of(bh), h = bh - b * p.H.d;
  if (p.counts.at && (int)t >= p.counts.of(b, h)) return;
  const int64_t pos = (int64_t)p.start.of(b, h) + t;
  if (pos < 0 || pos >= p.c.capacity) return;
  uint32_t row;
  const int page = page_of(p.c, b, (uint32_t)pos, row);
  if (page < 0) return;
  const char* from = p.x[which] + b * p.xb[which] + h * p.xh[which] + t * p.xt[which];
  char* to = side.rows + page * side.page + h * side.head + row * side.row;
  constexpr int in_bytes = IN == FCR_DTYPE_F32 ? 64 : 32;
  const bool live = lane < p.used;
  if constexpr (CODE == IN) {
    if (live) {
      const u32x4 a = reinterpret_cast<const u32x4*>(from + lane * 32)[0], z = reinterpret_cast<const u32x4*>(from + lane * 32)[1];
      reinterpret_cast<u32x4*>(to + lane * 32)[0] = a;
      reinterpret_cast<u32x4*>(to + lane * 32)[1] = z;
    }
    return;
  }
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.0f;
  if (live) load16<IN>(from + lane * in_bytes, x);
  if constexpr (CODE == FCR_DTYPE_F16 || CODE == FCR_DTYPE_BF16) {
    if (live) store16<CODE>(to + lane * 32, x);
    return;
  } else {
    // the largest magnitude, as bits: an infinity is above every number, a NaN above it
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, abs_bits(x[i]));
    for (int o = 1; o < L; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
    constexpr float top = CODE == FCR_DTYPE_INT8 ? 127.0f : 448.0f;
    float a = __builtin_bit_cast(float, most);
    const float scale = most >= 0x7f800000u ? __builtin_nanf("") : a / top;
    uint32_t w[4] = {0, 0, 0, 0};
    if (most < 0x7f800000u && most != 0) {
      // (a power of two keeps products and the reciprocal of the very large and the very small in range)
      const float by = a < 0x1p-64f ? 0x1p64f : a > 0x1p64f ? 0x1p-64f : 1.0f;
      a *= by;
      const float inverse = __builtin_amdgcn_rcpf(a);
      float q[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) q[i] = quotient<IN, CODE>(x[i] * by, a, inverse);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (CODE == FCR_DTYPE_INT8) {
          // 1.5 * 2^23 in front: the sum's last bits are the integer, rounded to nearest even
          uint32_t e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = __builtin_bit_cast(uint32_t, q[4 * i + j] + 12582912.0f);
          w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(e[3], e[2], 0x0c0c0400u), __builtin_amdgcn_perm(e[1], e[0], 0x0c0c0400u), 0x05040100u);
        } else {
          int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
          w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], v, true);
        }
      }
    }
    if (live) *reinterpret_cast<u32x4*>(to + lane * 16) = u32x4{w[0], w[1], w[2], w[3]};
    if (lane == 0) side.scale[page * side.s_page + h * side.s_head + row] = scale;
  }
}

struct ReadArgs {
  Pages c;
  Lengths lengths;
  char* out[2];
  Div N, H;
  uint32_t rows;       // B * H * N
  int lanes_log2, used, D;
};

template <int CODE, int OUT>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(ReadArgs p) {
  const int which = blockIdx.y;
  const Side side = p.c.side[which];
  const int L = 1 << p.lanes_log2;
  const int lane = threadIdx.x & (L - 1);
  const uint32_t r = (blockIdx.x * kThreads + threadIdx.x) >> p.lanes_log2;
  if (r >= p.rows || lane >= p.used) return;
  const uint32_t bh = p.N.of(r), j = r - bh * p.N.d;
  const uint32_t b = p.H.of(bh), h = bh - b * p.H.d;
  constexpr int out_bytes = OUT == FCR_DTYPE_F32 ? 4 : 2;
  char* to = p.out[which] + ((int64_t)r * p.D + lane * 16) * out_bytes;
  uint32_t row = 0;
  const int page = (int)j < p.lengths.of(b, h) && j < p.c.capacity ? page_of(p.c, b, j, row) : -1;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.0f;
  if (page >= 0) {
    const char* from = side.rows + page * side.page + h * side.head + row * side.row;
    if constexpr (CODE == FCR_DTYPE_F16 || CODE == FCR_DTYPE_BF16) {
      if constexpr (CODE == OUT) {
        const u32x4 a = reinterpret_cast<const u32x4*>(from + lane * 32)[0], z = reinterpret_cast<const u32x4*>(from + lane * 32)[1];
        reinterpret_cast<u32x4*>(to)[0] = a;
        reinterpret_cast<u32x4*>(to)[1] = z;
        return;
      }
      load16<CODE>(from + lane * 32, x);
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(from + lane * 16);
      const float scale = side.scale[page * side.s_page + h * side.s_head + row];
#pragma unroll
      for (int i = 0; i < 4; ++i) values_of<CODE>(w[i], x + 4 * i);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= scale;
    }
  }
  store16<OUT>(to, x);
}

struct KeepArgs {
  Pages c, into;
  Lengths lengths;
  const uint8_t* keep;   // [B, H, N]
  int32_t* counts;       // [B, H]
  int N, chunk;
  Div chunks, H, pieces; // by chunks of N, by heads, by 16-byte pieces of a row
};

// 16 bytes of a mask as 16 bits.
__device__ __forceinline__ uint32_t bits_of(const uint8_t* at) {
  u32x4 w;
  __builtin_memcpy(&w, at, 16);   // (any alignment)
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // any bit of a byte, moved to its lowest; then the four of them side by side
    uint32_t v = w[i];
    v |= v >> 4, v |= v >> 2, v |= v >> 1;
    v &= 0x01010101u;
    bits |= ((v * 0x01020408u) >> 24) << (4 * i);
  }
  return bits;
}
// Which of the 16 rows from `first` on stay: kept, shorter than the length, and on a page that is there.  The rows lie in one page (`first`
// and the page size are multiples of 16).
__device__ __forceinline__ uint32_t kept16(const KeepArgs& p, const uint8_t* keep, int b, int first, int n, int& page, uint32_t& row) {
  page = -1, row = 0;
  if (first >= n) return 0;
  page = page_of(p.c, b, (uint32_t)first, row);
  uint32_t bits = 0;
  if (first + 16 <= n) {
    bits = bits_of(keep + first);
  } else {
    for (int i = 0; first + i < n; ++i) bits |= (keep[first + i] != 0 ? 1u : 0u) << i;
  }
  return page < 0 ? 0 : bits;
}

// A workgroup takes `chunk` rows of one (batch, head): it counts the kept rows in front of them (the mask is read again by every
// chunk, at a byte per row next to the 2 D bytes of a kept one), lists where its own lie and go, and copies them, codes and scales as they are.
constexpr int kKeepRows = 512;   // rows listed at once

__global__ void __launch_bounds__(kThreads) cache_keep_kernel(KeepArgs p) {
  __shared__ int counted[kThreads / 64];
  __shared__ int4 list[kKeepRows];         // page and row, from and to; a page to go to below 0: none
  const int bh = (int)p.chunks.of(blockIdx.x), part = blockIdx.x - bh * p.chunks.d;
  const int b = (int)p.H.of((uint32_t)bh), h = bh - b * p.H.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int n = p.lengths.of(b, h);
  n = min(n, p.N);
  n = (int)min((int64_t)n, p.c.capacity);
  const uint8_t* keep = p.keep + (int64_t)bh * p.N;
  const int begin = part * p.chunk, end = min(begin + p.chunk, n);

  int before = 0, page;
  uint32_t row;
  const int whole = min(begin, max(n, 0) & ~15);
#pragma unroll 4
  for (int i = tid * 16; i < whole; i += kThreads * 16) {
    const uint32_t bits = bits_of(keep + i);
    before += page_of(p.c, b, (uint32_t)i, row) < 0 ? 0 : __popc(bits);
  }
  if (tid == 0 && whole < begin) before += __popc(kept16(p, keep, b, whole, n, page, row));
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if (lane == 0) counted[wave] = before;
  __syncthreads();
  int at = counted[0] + counted[1] + counted[2] + counted[3];

  for (int first = begin; first < end; first += kKeepRows) {
    // rows of this turn: at most 16 per thread for the first kKeepRows / 16 threads
    __syncthreads();
    const int mine0 = first + tid * 16;
    uint32_t bits = tid < kKeepRows / 16 && mine0 < end ? kept16(p, keep, b, mine0, n, page, row) : 0;
    int mine = __popc(bits), sum = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 63) counted[wave] = sum;
    __syncthreads();
    int place = sum - mine;
    for (int i = 0; i < wave; ++i) place += counted[i];
    const int total = counted[0] + counted[1] + counted[2] + counted[3];
    while (bits) {
      const int i = __ffs(bits) - 1;
      bits &= bits - 1;
      list[place++] = int4{page, (int)row + i, -1, 0};
    }
    __syncthreads();
    for (int k = tid; k < total; k += kThreads) {
      uint32_t to_row = 0;
      list[k].z = at + k < p.into.capacity ? page_of(p.into, b, at + k, to_row) : -1;
      list[k].w = (int)to_row;
    }
    __syncthreads();
    const Side ks = p.c.side[0], vs = p.c.side[1], kd = p.into.side[0], vd = p.into.side[1];
    for (int i = tid; i < total * (int)p.pieces.d; i += kThreads) {
      const int k = (int)p.pieces.of((uint32_t)i), piece = i - k * p.pieces.d;
      const int4 l = list[k];
      if (l.z < 0) continue;
      const u32x4 x = *reinterpret_cast<const u32x4*>(ks.rows + l.x * ks.page + h * ks.head + l.y * ks.row + piece * 16);
      const u32x4 y = *reinterpret_cast<const u32x4*>(vs.rows + l.x * vs.page + h * vs.head + l.y * vs.row + piece * 16);
      *reinterpret_cast<u32x4*>(kd.rows + l.z * kd.page + h * kd.head + l.w * kd.row + piece * 16) = x;
      *reinterpret_cast<u32x4*>(vd.rows + l.z * vd.page + h * vd.head + l.w * vd.row + piece * 16) = y;
    }
    if (ks.scale) {
      for (int k = tid; k < total; k += kThreads) {
        const int4 l = list[k];
        if (l.z < 0) continue;
        kd.scale[l.z * kd.s_page + h * kd.s_head + l.w] = ks.scale[l.x * ks.s_page + h * ks.s_head + l.y];
        vd.scale[l.z * vd.s_page + h * vd.s_head + l.w] = vs.scale[l.x * vs.s_page + h * vs.s_head + l.y];
      }
    }
    at += total;
  }
  if (part == (int)p.chunks.d - 1 && tid == 0) p.counts[bh] = (int)min((int64_t)at, p.into.capacity);
}

int check_lengths(const int32_t* at, const int64_t strides[2], const char* what) {
  if (!at || !strides) return fail(FCR_E_NULL, "null pointer argument");
  if (strides[0] < 0 || strides[1] < 0 || (reinterpret_cast<uintptr_t>(at) & 3) != 0) return fail(FCR_E_STRIDE, what);
  return 0;
}
Lengths lengths_of(const int32_t* at, const int64_t s[2]) { return Lengths{at, at ? s[0] : 0, at ? s[1] : 0}; }

int lanes_log2_of(int D) {
  int l = 0;
  while ((16 << l) < D) ++l;
  return l;
}

// Lanes of a launch over heads * n rows of keys; another as many take the values, and a launch has fewer than 2^32.
constexpr int64_t kMostLanes = (kMaxBlocks / 2 - 1) * kThreads;
bool too_many_rows(int64_t heads, int64_t n, int D) { return heads * n > (kMostLanes >> lanes_log2_of(D)); }   // (each at most 2^30)

template <int IN>
void launch_write(int code, const WriteArgs& p, dim3 grid, hipStream_t s) {
  switch (code) {
    case FCR_DTYPE_F16: hipLaunchKernelGGL((cache_write_kernel<IN, FCR_DTYPE_F16>), grid, dim3(kThreads), 0, s, p); break;
    case FCR_DTYPE_BF16: hipLaunchKernelGGL((cache_write_kernel<IN, FCR_DTYPE_BF16>), grid, dim3(kThreads), 0, s, p); break;
    case FCR_DTYPE_INT8: hipLaunchKernelGGL((cache_write_kernel<IN, FCR_DTYPE_INT8>), grid, dim3(kThreads), 0, s, p); break;
    default: hipLaunchKernelGGL((cache_write_kernel<IN, FCR_DTYPE_E4M3>), grid, dim3(kThreads), 0, s, p); break;
  }
}
template <int CODE>
void launch_read(int out, const ReadArgs& p, dim3 grid, hipStream_t s) {
  switch (out) {
    case FCR_DTYPE_F16: hipLaunchKernelGGL((cache_read_kernel<CODE, FCR_DTYPE_F16>), grid, dim3(kThreads), 0, s, p); break;
    case FCR_DTYPE_BF16: hipLaunchKernelGGL((cache_read_kernel<CODE, FCR_DTYPE_BF16>), grid, dim3(kThreads), 0, s, p); break;
    default: hipLaunchKernelGGL((cache_read_kernel<CODE, FCR_DTYPE_F32>), grid, dim3(kThreads), 0, s, p); break;
  }
}
bool tensor_dtype(int d) { return d == FCR_DTYPE_F16 || d == FCR_DTYPE_BF16 || d == FCR_DTYPE_F32; }

}  // namespace

extern "C" {

int fcr_cache_write(const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages, const int32_t* start,
                    const int64_t start_strides[2], const int32_t* counts, const int64_t counts_strides[2], const void* key,
                    const void* value, int dtype, int B, int T, const int64_t key_strides[4], const int64_t value_strides[4],
                    void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc) return rc;
  if ((rc = check_table(table, table_stride, table_pages, cache->page_size, B))) return rc;
  if ((rc = check_lengths(start, start_strides, "start: strides must be >= 0"))) return rc;
  if (counts && (rc = check_lengths(counts, counts_strides, "counts: strides must be >= 0"))) return rc;
  if (!key || !value || !key_strides || !value_strides) return fail(FCR_E_NULL, "null pointer argument");
  if (!tensor_dtype(dtype)) return fail(FCR_E_DTYPE, "dtype must be FCR_DTYPE_F16, FCR_DTYPE_BF16 or FCR_DTYPE_F32");
  const int H = cache->H;
  if (T < 1 || T > (1 << 30) || (int64_t)B * H > (1 << 30) || too_many_rows((int64_t)B * H, T, cache->D))
    return fail(FCR_E_SHAPE, "T must be >= 1 and B*H*T*L at most 2^31 - 256, L being D / 16 rounded up to a power of two");
  WriteArgs p;
  const int e = element_bytes(dtype);
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? value_strides : key_strides;
    const void* x = i ? value : key;
    bool ok = s[3] == 1 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const int sizes[3] = {B, H, T};
    for (int j = 0; j < 3; ++j) ok = ok && (sizes[j] == 1 || (s[j] >= 0 && s[j] * e % 16 == 0 && s[j] < (1ll << 40)));
    if (!ok) return fail(FCR_E_STRIDE, "key, value: unit stride of the last dimension, 16-byte aligned rows");
    p.x[i] = static_cast<const char*>(x);
    p.xb[i] = B > 1 ? s[0] * e : 0;
    p.xh[i] = H > 1 ? s[1] * e : 0;
    p.xt[i] = T > 1 ? s[2] * e : 0;
  }
  p.c = pages_of(*cache, table, table_stride, table_pages);
  p.start = lengths_of(start, start_strides);
  p.counts = lengths_of(counts, counts_strides);
  p.T.set((uint32_t)T);
  p.H.set((uint32_t)H);
  p.rows = (uint32_t)((int64_t)B * H * T);
  p.lanes_log2 = lanes_log2_of(cache->D);
  p.used = cache->D / 16;
  const int64_t blocks = (((int64_t)p.rows << p.lanes_log2) + kThreads - 1) / kThreads;
  if ((rc = check_written(*cache, "cache"))) return rc;
  const dim3 grid((unsigned)blocks, 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FCR_DTYPE_F16) launch_write<FCR_DTYPE_F16>(cache->dtype, p, grid, s);
  else if (dtype == FCR_DTYPE_BF16) launch_write<FCR_DTYPE_BF16>(cache->dtype, p, grid, s);
  else launch_write<FCR_DTYPE_F32>(cache->dtype, p, grid, s);
  return launched("cache_write_kernel");
}

int fcr_cache_read(const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages, const int32_t* lengths,
                   const int64_t lengths_strides[2], void* key, void* value, int out_dtype, int B, int N, void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc) return rc;
  if ((rc = check_table(table, table_stride, table_pages, cache->page_size, B))) return rc;
  if ((rc = check_lengths(lengths, lengths_strides, "lengths: strides must be >= 0"))) return rc;
  if (!key || !value) return fail(FCR_E_NULL, "null pointer argument");
  if (!tensor_dtype(out_dtype)) return fail(FCR_E_DTYPE, "out_dtype must be FCR_DTYPE_F16, FCR_DTYPE_BF16 or FCR_DTYPE_F32");
  if (((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) != 0)
    return fail(FCR_E_STRIDE, "key, value: 16-byte aligned pointers");
  const int H = cache->H;
  if (N < 1 || N > (1 << 30) || (int64_t)B * H > (1 << 30) || too_many_rows((int64_t)B * H, N, cache->D))
    return fail(FCR_E_SHAPE, "N must be >= 1 and B*H*N*L at most 2^31 - 256, L being D / 16 rounded up to a power of two");
  ReadArgs p;
  p.c = pages_of(*cache, table, table_stride, table_pages);
  p.lengths = lengths_of(lengths, lengths_strides);
  p.out[0] = static_cast<char*>(key);
  p.out[1] = static_cast<char*>(value);
  p.N.set((uint32_t)N);
  p.H.set((uint32_t)H);
  p.rows = (uint32_t)((int64_t)B * H * N);
  p.lanes_log2 = lanes_log2_of(cache->D);
  p.used = cache->D / 16;
  p.D = cache->D;
  const int64_t blocks = (((int64_t)p.rows << p.lanes_log2) + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)blocks, 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (cache->dtype) {
    case FCR_DTYPE_F16: launch_read<FCR_DTYPE_F16>(out_dtype, p, grid, s); break;
    case FCR_DTYPE_BF16: launch_read<FCR_DTYPE_BF16>(out_dtype, p, grid, s); break;
    case FCR_DTYPE_INT8: launch_read<FCR_DTYPE_INT8>(out_dtype, p, grid, s); break;
    default: launch_read<FCR_DTYPE_E4M3>(out_dtype, p, grid, s); break;
  }
  return launched("cache_read_kernel");
}

int fcr_cache_keep(const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages, const int32_t* lengths,
                   const int64_t lengths_strides[2], const uint8_t* keep, int N, const fcr_cache* into, const int32_t* into_table,
                   int64_t into_table_stride, int into_table_pages, int32_t* counts, int B, void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc || (rc = check_cache(into, "into"))) return rc;
  if ((rc = check_table(table, table_stride, table_pages, cache->page_size, B))) return rc;
  if ((rc = check_table(into_table, into_table_stride, into_table_pages, into->page_size, B))) return rc;
  if ((rc = check_lengths(lengths, lengths_strides, "lengths: strides must be >= 0"))) return rc;
  if (!keep || !counts) return fail(FCR_E_NULL, "null pointer argument");
  if (into->dtype != cache->dtype) return fail(FCR_E_DTYPE, "both caches must hold the same type");
  if (into->H != cache->H || into->D != cache->D) return fail(FCR_E_SHAPE, "both caches must have the same heads and D");
  if (N < 1 || N > (1 << 30) || (int64_t)B * cache->H > (1 << 22)) return fail(FCR_E_SHAPE, "N must be in [1, 2^30], B*H at most 2^22");
  KeepArgs p;
  p.c = pages_of(*cache, table, table_stride, table_pages);
  p.into = pages_of(*into, into_table, into_table_stride, into_table_pages);
  p.lengths = lengths_of(lengths, lengths_strides);
  p.keep = keep;
  p.counts = counts;
  p.N = N;
  p.pieces.set((uint32_t)(cache->D * element_bytes(cache->dtype) / 16));
  p.H.set((uint32_t)cache->H);
  // short ranges, but a mask is counted again by every range behind, so no more than 128 of them (4 x 8 x 32768 rows of bf16, the kernel alone: 79 us; with 64
  // all workgroups count at one time and copy at another, 85; with 256 80)
  int chunk = 128;
  while ((N + chunk - 1) / chunk > 128) chunk *= 2;
  p.chunk = chunk;
  p.chunks.set((uint32_t)((N + chunk - 1) / chunk));
  const int64_t blocks = (int64_t)B * cache->H * p.chunks.d;
  if (blocks >= kMaxBlocks) return fail(FCR_E_SHAPE, "B*H and N are too many for one call");
  if ((rc = check_written(*into, "into"))) return rc;
  hipLaunchKernelGGL(cache_keep_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
  return launched("cache_keep_kernel");
}

}  // extern "C"
