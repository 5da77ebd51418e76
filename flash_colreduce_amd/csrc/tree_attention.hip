// Attention of drafted tokens over a paged cache of keys and values, quantised or not.
//
// T tokens of a sequence have been drafted (a single one in plain decoding, a chain, or a tree whose nodes share their prefixes) and their
// keys and values written behind the sequence's `context` rows.  A query row is a (token, query head of the key head) pair; it
// sees every key of the context, and of the drafted tokens those that the tree's mask names:
//   s_j = scale log2(e) <q, c_j> ks_j,   p_j = 2^(s_j - m),   o = sum_j p_j vs_j v_j / sum_j p_j,   lse2 = m + log2 sum_j p_j.
//
// The G query heads of a key head and the drafted tokens are the columns of the matrix instructions, 16 to a tile, in one of two kernels
// (form_of has the rule, with both sides measured).  Both form
//   S^T = K Q^T   so that a lane owns one query (lane & 15) and keys 4 g + i of a 16-key tile (g = lane / 16, register i), and
//   O^T = V^T P^T in which that query stays in the lane.  The 8 keys that a lane feeds to one instruction are keys 4 g + i of two tiles,
//                 which is what it holds of P: probabilities never leave their lane, softmax statistics are one scalar per lane.
//                 V^T is formed from rows of V with byte permutes that convert codes on the way.
// tree_attention_kernel (few rows): bound by reading the cache.  Each wave takes 32 keys of a block of 128, from global memory into
//   registers without a stop in LDS, and 16 rows; the four waves' results are joined at the end.  32 ragged sequences of up to 16384 e4m3 keys, 8 heads
//   of 4 queries, D = 128: 154 to 164 us by the drawn lengths, 5.3 TB/s; 8 tokens over 4 x 32 heads of 9001 fp16 keys of 64 elements: 51 us,
//   5.8 TB/s; one token over 1000 keys 10.7 us, two launches and a chain of loads: lengths, table, keys.
// tall_attention_kernel (many rows): bound by how far the vector instructions of the softmax (half of a SIMD's time) run beside the products (a third)
//   and not behind them.  Each wave takes 32 rows (of
//   more than 128 elements 16) and all keys; the operands of a block are converted once, by all waves, and lie in LDS as the matrix instructions take them.  64 drafted tokens of 4
//   query heads over 8 x 8 heads of 32768 int8 keys, D = 128: 273 us, 760 TFLOP/s (1049 with operands formed by every wave from global memory, 341
//   with one stage in LDS); over 4 x 8 heads of 8192 keys 63 us, a quarter of it what runs once per workgroup.
//
// Codes are multiplied in fp16, where each of them is exact: bf16 rows of queries are scaled by a power of two to fit, of their own or (many rows)
// of rows that are up to 2^16 larger (an element keeps its 8 bits down to 2^-15 of its row's largest, and is off by 2^-23 of that at most
// below), the keys' scales multiply the scores, the values' scales the probabilities, in 32 bits, before these are rounded to 11 bits, as
// the matrix instructions take them.  16-bit caches are multiplied in their own type (probabilities against bf16 values have 8 bits).  The reference m
// of a row is what its weights p_j vs_j ask for, so that they fit fp16 whatever the scales are, the largest near its upper end (see weights); sums and
// statistics are in 32 bits.
//
// Distribution: the (batch, head, row tile) items are cut into blocks of 128 keys, laid end to end, and every workgroup takes the same
// number of blocks, found from the lengths on the device; or, where that takes little longer, one piece of one item.  Parts of an item that
// was cut are joined by tree_join_kernel, in the order of the keys.

#include <math.h>

#include <algorithm>

#include "deal.h"
#include "paged.h"

#ifndef FCR_PART
#define FCR_PART -1
#endif
#define FCR_HAS(part) (FCR_PART == -1 || FCR_PART == (part))

namespace fcr_tree {
using namespace fcr_paged;

struct Args {
  const char* q;
  int64_t qb, qh, qt;          // strides in bytes
  Pages c;
  Lengths context;
  const int32_t* tree_lengths; // [B] or null
  const uint8_t* mask;         // [T, T] per sequence or shared; null: the drafted tokens are a chain
  int64_t mask_b;
  char* out;                   // [B, H G, T, D]
  float* lse;                  // [B, H G, T] or null
  int32_t* first;              // [4]: blocks of a workgroup; [items][2]: the first workgroup that has a part of an item, blocks of others
  float* part;                 // [2 workgroups][rows of a tile][D + 4]: reference, sum, 2 unused, weighted values
  int B, H, T, D, rows, row_tiles, bf16;
  Div G, per_head, heads, all; // by G, by row_tiles, by H, by wgs
  float scale2;
  int wgs;                     // workgroups of the launch
  int positions;               // that a row of the table names
};
// form: see form_of.  false: there is no such kernel
bool attention_f16(const Args& a, int w, int form, hipStream_t s);
bool attention_bf16(const Args& a, int w, int form, hipStream_t s);
bool attention_int8(const Args& a, int w, int form, hipStream_t s);
bool attention_e4m3(const Args& a, int w, int form, hipStream_t s);
}  // namespace fcr_tree

namespace {
using namespace fcr_tree;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The kernel's arguments, read again where they are used: kept for the whole kernel they would not fit the scalar registers, and their
// spills take vector registers and instructions of the inner loops.  (Args is the only parameter of the kernels that call this.)
__device__ __forceinline__ const Args& arguments() {
  typedef const __attribute__((address_space(4))) Args* Pointer;
  Pointer p = (Pointer)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

constexpr int kFirst = 4;                    // words in front of the items in Args::first
constexpr int kNoPower = 200;                // of a row without a finite element but zeros; above all others
constexpr float kNone = -3.0e38f;            // reference of a row that has seen no key
constexpr float kMostWeight = 65504.0f;      // weights above this (fp16's largest number) raise the reference
constexpr float kRaised = 9.0f;              // fp16: to where the largest is in (2^8, 2^9]
constexpr float kMostSum = 0x1p110f;         // and so do sums above this

// Keys of a sequence: those of the context, then those of the drafted tokens.
__device__ __forceinline__ void keys_of(const Args& a, int b, int h, int& context, int& n) {
  const int tree = a.tree_lengths ? min(max(constant_at(a.tree_lengths + b), 0), a.T) : a.T;
  context = max(a.context.of(b, h), 0);
  n = (int)min((uint32_t)context + (uint32_t)tree, (uint32_t)a.positions);   // (each below 2^31)
}

// The sum over the wave's lanes up to this one: within rows of 16 lanes, then each row's last sum to the rows behind.  (Lanes exchange
// within the vector unit; exchanges by way of LDS take ten times as long.)
__device__ __forceinline__ int sum_up_to(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15, to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31, to rows 2 and 3
  return x;
}
// The least over 16 lanes that lie together.
__device__ __forceinline__ int least_of_row(int x) {
  x = min(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));   // row_ror:8
  x = min(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
  return min(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));
}

// Over the four lanes that share a query, those of the four rows of 16: a swap of two copies leaves one row's values in the one and its
// neighbour's in the other.
template <class T, class Op>
__device__ __forceinline__ T across(T x, Op op) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto rows = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t c = __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(T, (uint32_t)rows[0]), __builtin_bit_cast(T, (uint32_t)rows[1])));
  const auto halves = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return op(__builtin_bit_cast(T, (uint32_t)halves[0]), __builtin_bit_cast(T, (uint32_t)halves[1]));
}
__device__ __forceinline__ float across(float x, bool largest) {
  return across(x, [&](float y, float z) { return largest ? fmaxf(y, z) : y + z; });
}

template <bool BF16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two bytes above 1024 in fp16 (0x64 in front) are the codes + 128: less 1152 they are the codes.
__device__ __forceinline__ uint32_t centred(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f});
}
template <bool HI>
__device__ __forceinline__ uint32_t halves_of_e4m3(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
}

// 1 in the bytes that are e4m3's NaNs, 0x7f and 0xff, else 0.
__device__ __forceinline__ uint32_t nans_of_e4m3(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; }

// W: D / 64, rounded up.
template <int CD_, int W>
struct Form {
  static constexpr int CD = CD_;
  static constexpr bool codes = CD == FCR_DTYPE_INT8 || CD == FCR_DTYPE_E4M3;
  static constexpr bool bf16 = CD == FCR_DTYPE_BF16;
  static constexpr bool finite = CD == FCR_DTYPE_INT8;   // no element of a row is an infinity or a NaN
  static constexpr int KS = 2 * W;                // k-steps of 32 elements
  static constexpr int DT = 4 * W;                // 16-element tiles of the output; a lane's elements are consecutive
  static constexpr int KL = codes ? W : 2 * W;    // 16-byte loads of a key
  static constexpr int VW = codes ? W : 2 * W;    // words that a lane has of a value row
};

// Where a sequence's keys of one head lie: what a tile's address is formed from, and nothing else that would be kept in scalar registers.
struct Source {
  const char* rows[2];
  const float* scale[2];
  int64_t page[2], s_page[2];     // bytes; elements
  int row[2];                     // bytes
  const int32_t* table;
  Div page_size;
  int pages, n;
  __device__ __forceinline__ Source(const Args& a, int b, int h, int n_) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Side& s = a.c.side[i];
      rows[i] = s.rows + h * s.head;
      scale[i] = s.scale + h * s.s_head;
      page[i] = s.page, s_page[i] = s.s_page, row[i] = (int)s.row;
    }
    table = a.c.table + b * a.c.table_stride;
    page_size = a.c.page_size;
    pages = a.c.pages, n = n_;
  }
};
// Where the 16-key tile from position `pos` on lies: page (not below Source::pages: not there, or behind the last key) and first row in it.
struct Place {
  int page, row;
  __device__ __forceinline__ Place() {}
  __device__ __forceinline__ Place(const Source& s, int pos) : page(-1), row(0) {
    if (pos < s.n) {
      const uint32_t i = s.page_size.of((uint32_t)pos);
      row = pos - (int)(i * s.page_size.d);
      page = constant_at(s.table + i);
    }
  }
  __device__ __forceinline__ bool there(const Source& s) const { return (uint32_t)page < (uint32_t)s.pages; }
};

// The lane's places in a 16-key tile: of keys (row lane & 15; 16-byte pieces; those behind a row's end, where
// queries are zeros, are its last one, or with ZEROS are read as zeros, at a place that no view has) and of values (rows 4 g + i, elements from
// elements_of(col) on, where behind the row's end there are elements that another lane has as well).
template <class F>
struct Lane {
  static constexpr uint32_t kBytes = F::codes ? 1 : 2;
  static constexpr uint32_t kOutside = 0x7ffff000u;      // (views have at most 2^29 bytes)
  int lane, g, col;
  __device__ __forceinline__ Lane(int lane_) : lane(lane_), g(lane_ >> 4), col(lane_ & 15) {}
  __device__ __forceinline__ Lane again() const {        // (what is derived from it is formed again, not kept in registers)
    int l = lane;
    asm volatile("" : "+v"(l));
    return Lane(l);
  }
  // Whether the lane's piece i lies behind the row's end (D > 64 (W - 1): the last two may).
  __device__ __forceinline__ bool behind(int i, int D) const { return i >= F::KL - 2 && 64 * i + 16 * g >= (int)kBytes * D; }
  template <bool ZEROS>
  __device__ __forceinline__ uint32_t key(const Source& s, int i, int D) const {
    const uint32_t at = (uint32_t)(col * s.row[0]) + min(64u * i + 16u * g, (uint32_t)D * kBytes - 16u);
    return ZEROS && behind(i, D) ? kOutside : at;
  }
  __device__ __forceinline__ uint32_t value(const Source& s, int D) const { return (uint32_t)(4 * g * s.row[1]) + (uint32_t)elements_of(D, col) * kBytes; }
  __device__ __forceinline__ static int elements_of(int D, int col) { return min(col * F::DT, D - F::DT); }
};

// A tile's rows, or its scales, as a view that reads as zeros where its page is not there: the loads need no branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const Source& s, int side, const Place& p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(s.rows[side]) + p.page * s.page[side] + (int64_t)p.row * s.row[side], 0,
                                           p.there(s) ? 16 * s.row[side] : 0, 0x00020000);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t scales_of(const Source& s, int side, const Place& p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(s.scale[side]) + p.page * s.s_page[side] + p.row, 0, p.there(s) ? 64 : 0, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t v, uint32_t at) { return __builtin_amdgcn_raw_buffer_load_b128(v, (int)at, 0, 0); }

template <int N>
__device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t v, uint32_t at, int row, uint32_t (&w)[N]) {
  // (a lane's part of a row is 4 N bytes: aligned to 16 where N is a multiple of 4, to 8 where it is even)
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(v, (int)at + 16 * i, row, 0);
      w[4 * i] = x[0], w[4 * i + 1] = x[1], w[4 * i + 2] = x[2], w[4 * i + 3] = x[3];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(v, (int)at + 8 * i, row, 0);
      w[2 * i] = x[0], w[2 * i + 1] = x[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_raw_buffer_load_b32(v, (int)at + 4 * i, row, 0);
  }
}

// A 16-key tile as the lane loads it, and its scales of keys 4 g + i.
template <class F>
struct Keys {
  u32x4 w[F::KL];
  f32x4 scale;
  // ZEROS: of rows of 16-bit elements, whose infinities must not meet the queries' zeros.  (Codes are finite, or the row's scores are NaNs anyway.)
  template <bool ZEROS>
  __device__ __forceinline__ void load(const Source& s, int D, const Place& p, const Lane<F>& at) {
    const __amdgpu_buffer_rsrc_t rows = rows_of(s, 0, p);
#pragma unroll
    for (int i = 0; i < F::KL; ++i) w[i] = load16(rows, at.template key<ZEROS && !F::codes>(s, i, D));
    if constexpr (F::codes) scale = __builtin_bit_cast(f32x4, load16(scales_of(s, 0, p), 16 * at.g));
  }
  // k-steps 2 i and 2 i + 1 (codes) or i (16-bit) of load i
  __device__ __forceinline__ u32x4 operand(int ks) const {
    if constexpr (F::CD == FCR_DTYPE_INT8) {
      u32x4 f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = w[ks / 2][2 * (ks & 1) + j] ^ 0x80808080u;
        f[2 * j] = centred(__builtin_amdgcn_perm(0x64646464u, x, 0x04010400u));
        f[2 * j + 1] = centred(__builtin_amdgcn_perm(0x64646464u, x, 0x04030402u));
      }
      return f;
    } else if constexpr (F::CD == FCR_DTYPE_E4M3) {
      u32x4 f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = w[ks / 2][2 * (ks & 1) + j];
        f[2 * j] = halves_of_e4m3<false>(x);
        f[2 * j + 1] = halves_of_e4m3<true>(x);
      }
      return f;
    } else {
      return w[ks];
    }
  }
};

template <class F>
struct Values {
  uint32_t w[4][F::VW];
  f32x4 scale;
  __device__ __forceinline__ void load(const Source& s, int D, const Place& p, const Lane<F>& at) {
    const __amdgpu_buffer_rsrc_t rows = rows_of(s, 1, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_words(rows, at.value(s, D), i * s.row[1], w[i]);
    if constexpr (F::codes) scale = __builtin_bit_cast(f32x4, load16(scales_of(s, 1, p), 16 * at.g));
  }
  // Keys that are not there: bits of `there` from bit 0 on.  What their rows hold is not looked at.
  __device__ __forceinline__ void drop(uint32_t there) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!((there >> i) & 1u)) {
#pragma unroll
        for (int j = 0; j < F::VW; ++j) w[i][j] = 0;
        if constexpr (F::codes) scale[i] = 0.0f;
      }
  }
  // Elements that are not finite become 0 (see add_not_finite); returns whether there was one.  (Codes: e4m3's NaNs.)
  __device__ __forceinline__ bool clean() {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < F::VW; ++j) {
        uint32_t bad;
        if constexpr (F::codes) {
          bad = nans_of_e4m3(w[i][j]) * 0xffu;
        } else {
          constexpr uint32_t e = F::bf16 ? 0x7f80u : 0x7c00u;
          bad = ((w[i][j] & e) == e ? 0xffffu : 0u) | (((w[i][j] >> 16) & e) == e ? 0xffff0000u : 0u);
        }
        found |= bad;
        w[i][j] &= ~bad;
      }
    return found != 0;
  }
  // Element d (of the lane's DT) of the four rows, as four fp16 or bf16.
  __device__ __forceinline__ u32x2 operand(int d) const {
    u32x2 f;
    if constexpr (F::CD == FCR_DTYPE_INT8) {
      const uint32_t pick = 0x0c040c00u + 0x00010001u * (d & 3);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[j] = centred(__builtin_amdgcn_perm(w[2 * j + 1][d / 4] ^ 0x80808080u, w[2 * j][d / 4] ^ 0x80808080u, pick) | 0x64006400u);
    } else if constexpr (F::CD == FCR_DTYPE_E4M3) {
      const uint32_t pick = (d & 2) ? 0x07030602u : 0x05010400u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = __builtin_amdgcn_perm(w[2 * j + 1][d / 4], w[2 * j][d / 4], pick);
        f[j] = (d & 1) ? halves_of_e4m3<true>(x) : halves_of_e4m3<false>(x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[j] = __builtin_amdgcn_perm(w[2 * j + 1][d / 2], w[2 * j][d / 2], (d & 1) ? 0x07060302u : 0x05040100u);
    }
    return f;
  }
};
__device__ __forceinline__ u32x4 joined_operand(u32x2 a, u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }

// What a lane knows of the query of each of its column tiles.
template <class F, int RT>
struct State {
  f32x4 o[RT][F::DT];   // sum 2^(s - m) vs v
  float m[RT];          // reference exponent, a whole number; kNone before the first key
  float l[RT];          // this lane's part of sum 2^(s - m)
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = kNone, l[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < F::DT; ++d) o[r][d] = f32x4{0, 0, 0, 0};
    }
  }
};

// A product that is not joined with the sum it goes into.
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}

// The weights of 32 keys from their products with the queries: 2^(k_scale s - m) v_scale.  MASKED: seen[r] holds the keys that a row
// sees, bit 4 t + i; else every key is seen.  Bound by the vector unit: per score an fma, an exponential (four slots), the sum, the product
// with the value's scale and half a conversion.  Returns whether some row's reference has to be raised, because a weight might not fit fp16 (the
// sum of the lane's probabilities times most_v, the largest scale of the 32 values: nothing asks for a maximum of weights) or a sum fp32.
// A few of the first steps ask for it and hardly any later one: a weight may be 2^7 times the one that the reference was raised for, 2^4 where
// all eight of a lane are as large.
// In fp16 a row's largest weight is above 2^8 (of scores below 2^24 and scales from 2^-90 to 2^90): others keep their 11 bits down to 2^-22 of it, and what is lost of those below is 2^-33 of it each.
// (Many keys of little weight share what a few large ones leave: 65536 of them a thousandth, from weights of 2^-26.  Raised to 1 the
// reference had them lose nine tenths of that.  256 rows over 4 x 8 heads of 8192 keys of 128 elements: 67 us fp16, 72 int8 either way for scores
// that spread by 1.4 in base 2; 68 -> 74 and 74 -> 84 where they spread by 5.8 and references rise more often.)  bf16 has weights of any size, and
// the reference is raised to the largest.
template <bool MASKED, class F, int RT>
__device__ __forceinline__ bool weights(const f32x4 (&k_scale)[2], const f32x4 (&v_scale)[2], float most_v, const f32x4 (&s)[RT][2],
                                        const uint32_t (&seen)[RT], const State<F, RT>& st, float (&sum)[RT], u32x4 (&p)[RT]) {
  bool raise = false;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float x[8], part[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (of scores whose last bit is worth more than a weight's exponent, the rounded one is at the reference that `raise` chose; one rounding
      // less may put it far above, which raises the reference again and comes here)
      x[e] = MASKED ? rounded(s[r][e / 4][e % 4] * k_scale[e / 4][e % 4]) - st.m[r]
                    : __builtin_fmaf(s[r][e / 4][e % 4], k_scale[e / 4][e % 4], -st.m[r]);
      if (MASKED) x[e] = (seen[r] >> e) & 1u ? x[e] : -INFINITY;
      x[e] = __builtin_amdgcn_exp2f(x[e]);
      part[e & 1] = e < 2 ? x[e] : part[e & 1] + x[e];
      if constexpr (F::codes) {
        x[e] *= v_scale[e / 4][e % 4];
        if (MASKED) x[e] = (seen[r] >> e) & 1u ? x[e] : 0.0f;      // (a hidden value's scale may be a NaN)
      }
    }
    part[0] += part[1];
    sum[r] = st.l[r] + part[0];
    raise = raise || part[0] * most_v > kMostWeight || !(sum[r] < kMostSum);
#pragma unroll
    for (int j = 0; j < 4; ++j) p[r][j] = F::bf16 ? pack2<FCR_DTYPE_BF16>(x[2 * j], x[2 * j + 1]) : pack2<FCR_DTYPE_F16>(x[2 * j], x[2 * j + 1]);
  }
  return __any(raise);
}

// Raises references so that the largest weight of these keys is in (2^8, 2^9] (fp16) or (1/2, 1] (bf16).
template <class F, int RT>
__device__ __forceinline__ void raise(const f32x4 (&k_scale)[2], const f32x4 (&v_scale)[2], const f32x4 (&s)[RT][2], const uint32_t (&seen)[RT],
                                      State<F, RT>& st) {
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float of_weights = -INFINITY, of_sum = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = rounded(s[r][e / 4][e % 4] * k_scale[e / 4][e % 4]);
      x = (seen[r] >> e) & 1u ? x : -INFINITY;
      of_sum = fmaxf(of_sum, x);
      if constexpr (F::codes) {
        // (an infinite scale does not count: a reference of infinity would leave the row no weights at all)
        const float of_scale = __builtin_amdgcn_logf(fabsf(v_scale[e / 4][e % 4]));
        x += of_scale < 200.0f ? of_scale : 0.0f;
      }
      of_weights = fmaxf(of_weights, x);
    }
    // (a reference above 2^24 is not followed by 9: its last bit may be worth 16 and more)
    if constexpr (!F::bf16) of_weights -= fabsf(of_weights) < 0x1p24f ? kRaised : 0.0f;
    const float top = across(fmaxf(of_weights, of_sum - 100.0f), true);
    const float m = top > st.m[r] ? ceilf(top) : st.m[r];
    const float shrink = __builtin_amdgcn_exp2f(st.m[r] - m);
    st.m[r] = m;
    st.l[r] *= shrink;
#pragma unroll
    for (int d = 0; d < F::DT; ++d) st.o[r][d] *= shrink;
  }
}

template <class F, int RT>
__device__ __forceinline__ void weigh(const f32x4 (&k_scale)[2], const f32x4 (&v_scale)[2], float most_v, const f32x4 (&s)[RT][2], bool masked,
                                      const uint32_t (&seen)[RT], State<F, RT>& st, u32x4 (&p)[RT]) {
  float sum[RT];
  const bool up = masked ? weights<true, F, RT>(k_scale, v_scale, most_v, s, seen, st, sum, p)
                         : weights<false, F, RT>(k_scale, v_scale, most_v, s, seen, st, sum, p);
  if (__builtin_expect(up, 0)) {
    raise<F, RT>(k_scale, v_scale, s, seen, st);
    weights<true, F, RT>(k_scale, v_scale, most_v, s, seen, st, sum, p);
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) st.l[r] = sum[r];
}

// O^T += V^T P^T of 32 keys, for the lane's elements [D0, D1).
template <class F, int RT, int D0, int D1>
__device__ __forceinline__ void add_values(const u32x4 (&v)[F::DT], const u32x4 (&p)[RT], State<F, RT>& st) {
#pragma unroll
  for (int d = D0; d < D1; ++d)
#pragma unroll
    for (int r = 0; r < RT; ++r) st.o[r][d] = mma<F::bf16>(v[d], p[r], st.o[r][d]);
}
// Values that are not finite, at keys that only some rows see: in a matrix product 0 * inf would reach the others.  They are 0 there, and
// come here from the cache: p v for the rows that see the key, which for e4m3 is always a NaN.  (pos: the first of the 32 keys.  Rare, and as short as can be.)
template <class F, int RT>
__device__ __forceinline__ void add_not_finite(const Source& src, int D, int pos, const u32x4 (&p)[RT], const uint32_t (&seen)[RT], const Lane<F>& at,
                                               State<F, RT>& st) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const Place place(src, pos + 16 * t);
    if (!place.there(src)) continue;
    const char* row = src.rows[1] + place.page * src.page[1] + (int64_t)place.row * src.row[1];
#pragma unroll 1
    for (int k = 0; k < 16; ++k, row += src.row[1]) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int from = 16 * (k >> 2) + at.col;                             // the lane that has this key's weight
        const bool see = (__shfl((int)seen[r], from) >> (4 * t + (k & 3))) & 1;
        if constexpr (F::codes) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t* const from_row = reinterpret_cast<const uint32_t*>(row + Lane<F>::elements_of(D, 4 * at.again().g + i));
#pragma unroll
            for (int j = 0; j < F::VW; ++j) {
              uint32_t x = from_row[j];
              x = see ? nans_of_e4m3(x) : 0;
#pragma unroll
              for (int d = 0; d < 4; ++d)      // (a NaN or 0 is added)
                st.o[r][4 * j + d][i] += __builtin_bit_cast(float, (uint32_t)((int32_t)(x << (31 - 8 * d)) >> 31) & 0x7fc00000u);
            }
          }
          continue;
        }
        const uint32_t two = (uint32_t)__shfl((int)(k & 2 ? p[r][2 * t + 1] : p[r][2 * t]), from);
        const float w = element<F::CD>(k & 1 ? two >> 16 : two, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < F::DT; ++d) {
            const uint32_t x = *reinterpret_cast<const uint16_t*>(row + 2 * (Lane<F>::elements_of(D, 4 * at.g + i) + d));
            constexpr uint32_t e = F::bf16 ? 0x7f80u : 0x7c00u;
            if (see && (x & e) == e) st.o[r][d][i] += w * element<F::CD>(x, 0);
          }
      }
    }
  }
}

// The queries of column tiles from row `row0` on: row t G + g is token t and head g of the key head's.  Elements in the order in which
// the lane has those of a key.
template <class F, int RT>
struct Queries {
  u32x4 w[RT][F::KS];
  // Waits for the loads here: a loop that is entered with them on the way would wait, in every turn, for all that it has on the way itself.
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < F::KS; ++c) asm volatile("" : "+v"(w[r][c]));
  }
  __device__ __forceinline__ void load(const Args& a, int b, int h, int row0, const Lane<F>& at) {
    constexpr int mine = F::codes ? 16 : 8;   // elements that lanes are apart
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + 16 * r + at.col;
      const uint32_t t = a.G.of((uint32_t)row), head = (uint32_t)row - t * a.G.d;
      const char* from = a.q + b * a.qb + (int64_t)(h * (int)a.G.d + (int)head) * a.qh + t * a.qt + 2 * mine * at.g;
#pragma unroll
      for (int s = 0; s < F::KS; ++s) w[r][s] = u32x4{0, 0, 0, 0};
      if (row < a.rows) {
        const int d0 = mine * at.g;
        if (a.D == 64 * (F::KS / 2)) {
#pragma unroll
          for (int s = 0; s < F::KS; ++s) w[r][s] = *reinterpret_cast<const u32x4*>(from + 2 * element(s));
        } else {
#pragma unroll
          for (int s = 0; s < F::KS; ++s)
            if (d0 + element(s) < a.D) w[r][s] = *reinterpret_cast<const u32x4*>(from + 2 * element(s));
        }
      }
    }
  }
  // The power of two that takes the largest finite element of the lane's row r of bf16 to [2^14, 2^15), kNoPower for a row without one.
  __device__ __forceinline__ int power(int r) const {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 most = {0, 0};
    // magnitudes with 0x80 added: as signed halves bf16's infinities and NaNs are below all others
#pragma unroll
    for (int s = 0; s < F::KS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        most = __builtin_elementwise_max(most, __builtin_bit_cast(s16x2, (w[r][s][j] & 0x7fff7fffu) + 0x00800080u));
    int x = max((int)most[0], (int)most[1]) - 0x80;
    x = across(x, [](int y, int z) { return max(y, z); });
    return x <= 0 ? kNoPower : 14 - ((x >> 7) - 127);
  }
  // Where in a row the lanes' first elements of k-step s are.
  __device__ __forceinline__ static constexpr int element(int s) { return F::codes ? 64 * (s / 2) + 8 * (s & 1) : 32 * s; }
  // Row r from bf16 to fp16, times 2^up.
  __device__ __forceinline__ void scale(int r, int up) {
#pragma unroll
    for (int s = 0; s < F::KS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[r][s][j] = pack2<FCR_DTYPE_F16>(__builtin_amdgcn_ldexpf(bf16_of(w[r][s][j], 0), up), __builtin_amdgcn_ldexpf(bf16_of(w[r][s][j], 1), up));
  }
};

// Which of the lane's keys from position `pos` on (a 32-key step: bits 4 t + i) the query of a row sees.  (Rows that are none are given
// token 0.  Bytes in front of the mask's row, for keys of the context, and behind it, for keys that are not there, do not count.)
__device__ __forceinline__ uint32_t seen_by(const Args& a, int b, int row, int pos, int context, uint32_t there, int g) {
  const int token = row < a.rows ? (int)a.G.of((uint32_t)row) : 0;
  const int u = pos + 4 * g - context;   // which drafted token the lane's first key is; below 0: of the context
  uint32_t seen = 0;
  if (a.mask) {
    const __amdgpu_buffer_rsrc_t mask = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.mask) + b * a.mask_b, 0, a.T * a.T, 0x00020000);
    uint32_t is[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) is[e] = __builtin_amdgcn_raw_buffer_load_b8(mask, token * a.T + u + 16 * (e / 4) + e % 4, 0, 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) seen |= u + 16 * (e / 4) + e % 4 < 0 || (is[e] & 0xffu) ? 1u << e : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) seen |= u + 16 * (e / 4) + e % 4 <= token ? 1u << e : 0u;
  }
  return seen & there;
}
// Which of the lane's keys are there: in front of n, on a page that is.  Bits 4 t + i.
__device__ __forceinline__ uint32_t there_of(int pos, int n, bool page0, bool page1, int g) {
  uint32_t there = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) there |= pos + 16 * (e / 4) + 4 * g + e % 4 < n && (e < 4 ? page0 : page1) ? 1u << e : 0u;
  return there;
}

// A query row's place in the outputs.
struct Output {
  int64_t row;
  bool live, none;     // there is such a row; the sequence has no such token, or it sees nothing
  __device__ __forceinline__ Output(const Args& a, int b, int h, int r, float l) : live(r < a.rows) {
    const int token = (int)a.G.of((uint32_t)r);
    none = (a.tree_lengths && token >= a.tree_lengths[live ? b : 0]) || l == 0.0f;
    row = ((int64_t)b * a.H * a.G.d + (int64_t)h * a.G.d + (r - token * (int)a.G.d)) * a.T + token;
  }
};
// DT consecutive elements of a row, from d0 (a multiple of 4) on: its result, or its part of one (`to` is the row's in the part).
template <class F>
__device__ __forceinline__ void emit(const Args& a, const Output& out, int d0, const float (&x)[F::DT], float inverse) {
  uint32_t* const o = reinterpret_cast<uint32_t*>(a.out + (out.row * a.D + d0) * 2);
#pragma unroll
  for (int d = 0; d < F::DT; d += 4) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = out.none ? 0.0f : x[d + j] * inverse;
    *reinterpret_cast<u32x2*>(o + d / 2) = a.bf16 ? u32x2{pack2<FCR_DTYPE_BF16>(y[0], y[1]), pack2<FCR_DTYPE_BF16>(y[2], y[3])}
                                                  : u32x2{pack2<FCR_DTYPE_F16>(y[0], y[1]), pack2<FCR_DTYPE_F16>(y[2], y[3])};
  }
}
template <class F>
__device__ __forceinline__ void emit_part(float* to, int d0, const float (&x)[F::DT]) {
#pragma unroll
  for (int d = 0; d < F::DT; d += 4) *reinterpret_cast<f32x4*>(to + 4 + d0 + d) = f32x4{x[d], x[d + 1], x[d + 2], x[d + 3]};
}

// The blocks of a workgroup, as pieces of items.  Lengths are known on the device only: every workgroup adds them up.  Lengths of
// sequences (not of heads): an entry is all heads of one.
template <int THREADS, bool TALL>
struct Deal {
  int at, end, b, h, tile, blk, nb, context, n;
  // (Short on purpose: this and what else runs once per workgroup costs about 200 cycles per 64 bytes of instructions, which come
  // from memory at that point.)
  __device__ __forceinline__ bool start(const Args& a, int wg, int* scan) {   // scan: THREADS / 64 + 2 words of LDS
    constexpr int waves = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool by_head = a.context.sh != 0;
    const int entries = by_head ? a.B * a.H : a.B;
    const int weight = by_head ? a.row_tiles : a.H * a.row_tiles;
    const auto entry_blocks = [&](int e) {
      if (e >= entries) return 0;
      int eb = e, eh = 0, context, n;
      if (by_head) eb = (int)a.heads.of((uint32_t)e), eh = e - eb * a.H;
      keys_of(a, eb, eh, context, n);
      return blocks_of(n) * weight;
    };
    const auto in_front = [&](int x, int& sum) {        // of this thread; the sum over all
      const int upto = sum_up_to(x);
      if (lane == 63) scan[wave] = upto;
      __syncthreads();
      sum = 0;
      int before = upto - x;
#pragma unroll
      for (int i = 0; i < waves; ++i) {
        before += i < wave ? scan[i] : 0;
        sum += scan[i];
      }
      return before;
    };
    int mine = entry_blocks(tid), round, total;         // a round: as many entries as there are threads
    int start = in_front(mine, round);
    total = round;
    if (__builtin_expect(entries > THREADS, 0)) {
      int rest = 0;
      for (int e = tid + THREADS; e < entries; e += THREADS) rest += entry_blocks(e);
      __syncthreads();
      in_front(rest, total);
      total += round;
    }
    const int per = (int)a.all.of((uint32_t)(total + a.wgs - 1));
    int most = 0;
    if (pieces_are_tried(entries, THREADS, per, a.row_tiles, TALL)) {
      const int blocks = tid < entries ? mine / weight : 0;
      int pieces, before, sum;
      most = most_of(per, most_allowed(per, a.row_tiles, TALL), [&](int p) {
        pieces = pieces_of(blocks, p) * weight;
        __syncthreads();
        before = in_front(pieces, sum);
        return __builtin_amdgcn_readfirstlane(sum) <= a.wgs;
      });
      if (most) mine = pieces, start = before, round = total = sum;
    }
    const int unit = most ? 1 : per;
    if (wg == 0 && tid == 0) a.first[0] = most ? most : per;
    at = wg * unit;                                     // (wgs * per is total + wgs at most: checked by the host to fit)
    end = min(at + unit, total);
    if (at >= end) return false;
    int base = 0;
    for (int before = round; __builtin_expect(at >= before, 0); before += round) {
      base += THREADS;
      if (base >= entries) return false;                // (only if lengths change under the call)
      __syncthreads();
      mine = entry_blocks(base + tid);
      start = before + in_front(mine, round);
    }
    if (at >= start && at < start + mine) {             // the entry that holds `at`, and its first block
      scan[waves] = base + tid;
      scan[waves + 1] = start;
    }
    __syncthreads();
    const int entry = __builtin_amdgcn_readfirstlane(scan[waves]);
    const int in = at - __builtin_amdgcn_readfirstlane(scan[waves + 1]);
    b = by_head ? (int)a.heads.of((uint32_t)entry) : entry;
    h = by_head ? entry - b * a.H : 0;
    look(a);
    const int pieces = most ? pieces_of(nb, most) : nb;
    int item_of_entry = (int)((uint32_t)in / (uint32_t)pieces);
    blk = in - item_of_entry * pieces;
    if (most) {
      const int length = piece_length(nb, pieces);
      blk *= length;
      at = 0, end = min(length, nb - blk);
    }
    if (!by_head) h = (int)a.per_head.of((uint32_t)item_of_entry), item_of_entry -= h * a.row_tiles;
    tile = item_of_entry;
    return true;
  }
  __device__ __forceinline__ void look(const Args& a) {
    keys_of(a, b, h, context, n);
    context = __builtin_amdgcn_readfirstlane(context);
    n = __builtin_amdgcn_readfirstlane(n);
    nb = blocks_of(n);
  }
  __device__ __forceinline__ int stop() const { return min(nb, blk + (end - at)); }   // blocks [blk, stop) of this item
  __device__ __forceinline__ int item(const Args& a) const { return (b * a.H + h) * a.row_tiles + tile; }
  // For the join, by the workgroup that has an item's first part.
  __device__ __forceinline__ void tell(const Args& a, int wg) const {
    int32_t* const to = a.first + kFirst + 2 * (int64_t)item(a);
    to[0] = wg;
    to[1] = nb - (end - at);
  }
  // To the next piece; false: there is none.
  __device__ __forceinline__ bool next(const Args& a) {
    at += stop() - blk;
    if (at >= end) return false;
    blk = 0;
    if (++tile == a.row_tiles) {
      tile = 0;
      if (++h == a.H) h = 0, ++b;
      look(a);
    }
    return true;
  }
};
// workgroups are dealt to 8 dies in turn: consecutive ranges of blocks, whose row tiles share keys, go to one die
__device__ __forceinline__ int range_of(const Args& a, int block) { return (block & 7) * (a.wgs >> 3) + (block >> 3); }

template <int CD, int W>
__global__ void __launch_bounds__(256, (W <= 2 || Form<CD, W>::codes) ? 2 : 1) tree_attention_kernel(Args args) {
  using F = Form<CD, W>;
  constexpr int kWaves = 4;
  __shared__ float joined[kWaves * 4 * F::DT * 64];     // [wave][register][tile][lane]
  __shared__ float stats[kWaves][16][2];                // m, l
  __shared__ int scan[kWaves + 2];
  const int wg = range_of(args, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Lane<F> at(threadIdx.x & 63);
  Deal<256, false> deal;
  if (!deal.start(arguments(), wg, scan)) return;
  do {
    const Args& a = arguments();
    const int b = deal.b, h = deal.h, n = deal.n, context = deal.context, stop = deal.stop();
    const int row = deal.tile * 16 + at.col;
    Keys<F> k[2];
    Values<F> v[2];
    // (places are a block further ahead than the loads, which need them)
    const Source src(a, b, h, n);
    Place here[2], next[2], then[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) here[t] = Place(src, deal.blk * kBlock + wave * 32 + 16 * t);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      k[t].template load<true>(src, a.D, here[t], at);
      v[t].load(src, a.D, here[t], at);
      next[t] = Place(src, (deal.blk + 1) * kBlock + wave * 32 + 16 * t);
    }
    Queries<F, 1> q;
    float by = a.scale2;
    q.load(a, b, h, deal.tile * 16, at);
    if (F::codes && a.bf16) {
      int up = q.power(0);
      up = up == kNoPower ? 0 : up;
      q.scale(0, up);
      by = __builtin_amdgcn_ldexpf(by, -up);            // (of the lane's row)
    }
    q.arrive();
    State<F, 1> st;
    st.clear();
    for (int i = deal.blk; i < stop; ++i) {
      const int pos = i * kBlock + wave * 32;
      if (pos >= n) break;                              // (a wave's later blocks lie behind this one)
#pragma unroll
      for (int t = 0; t < 2; ++t) then[t] = Place(src, pos + 2 * kBlock + 16 * t);
      f32x4 s[1][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[0][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < F::KS; ++c) s[0][t] = mma<F::bf16>(k[t].operand(c), q.w[0][c], s[0][t]);
      }
      f32x4 k_scale[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) k_scale[t] = F::codes ? k[t].scale * by : f32x4{by, by, by, by};
      if (i + 1 < stop) {
#pragma unroll
        for (int t = 0; t < 2; ++t) k[t].template load<true>(src, a.D, next[t], at);
      }
      u32x4 p[1];
      uint32_t seen[1] = {0xff};
      const bool there0 = here[0].there(src), there1 = here[1].there(src);
      const bool masked = pos + 32 > min(context, n) || !there0 || !there1;
      bool not_finite = false;
      if (masked) {
        const uint32_t there = there_of(pos, n, there0, there1, at.g);
        v[0].drop(there);
        v[1].drop(there >> 4);
        if constexpr (!F::finite) {
          if (pos + 32 > context) not_finite = v[0].clean() | v[1].clean();
          not_finite = __any(not_finite);
        }
        seen[0] = seen_by(a, b, row, pos, context, there, at.g);
      }
      const f32x4 v_scale[2] = {v[0].scale, v[1].scale};
      float most_v = F::codes ? 0.0f : 1.0f;
      if constexpr (F::codes) {
#pragma unroll
        for (int e = 0; e < 8; ++e) most_v = fmaxf(most_v, fabsf(v_scale[e / 4][e % 4]));
      }
      weigh<F, 1>(k_scale, v_scale, most_v, s, masked, seen, st, p);
#pragma unroll
      for (int d = 0; d < F::DT; ++d) st.o[0][d] = mma<F::bf16>(joined_operand(v[0].operand(d), v[1].operand(d)), p[0], st.o[0][d]);
      if constexpr (!F::finite) {
        if (__builtin_expect(not_finite, 0)) add_not_finite<F, 1>(src, arguments().D, pos, p, seen, at, st);
      }
      if (i + 1 < stop) {
#pragma unroll
        for (int t = 0; t < 2; ++t) v[t].load(src, a.D, next[t], at);
      }
      here[0] = next[0], here[1] = next[1];
      next[0] = then[0], next[1] = then[1];
    }

    // join the four waves
    const Args& a_end = arguments();
    const bool final = deal.blk == 0 && stop == deal.nb;
    float* const slot = a_end.part + (int64_t)(2 * wg + (deal.blk == 0 ? 1 : 0)) * 16 * (a_end.D + 4);
    if (deal.blk == 0 && threadIdx.x == 0) deal.tell(a_end, wg);
    __syncthreads();
    const float sum = across(st.l[0], false);
    if (at.g == 0) stats[wave][at.col][0] = st.m[0], stats[wave][at.col][1] = sum;
    __syncthreads();
    float m = stats[0][at.col][0], l = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, stats[w][at.col][0]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) l += stats[w][at.col][1] * __builtin_amdgcn_exp2f(stats[w][at.col][0] - m);
    const float shrink = __builtin_amdgcn_exp2f(st.m[0] - m);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < F::DT; ++d) joined[((wave * 4 + i) * F::DT + d) * 64 + at.lane] = st.o[0][d][i] * shrink;
    __syncthreads();
    // wave w writes register w of every tile: query col, the elements of lane 4 g + w
    float x[F::DT];
#pragma unroll
    for (int d = 0; d < F::DT; ++d) {
      x[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x[d] += joined[((w * 4 + wave) * F::DT + d) * 64 + at.lane];
    }
    const int d0 = Lane<F>::elements_of(a_end.D, 4 * at.g + wave);
    const bool first = wave == 0 && at.g == 0;
    if (row < a_end.rows) {
      if (final) {
        const Output out(a_end, b, h, row, l);
        emit<F>(a_end, out, d0, x, 1.0f / l);
        if (a_end.lse && first) a_end.lse[out.row] = out.none ? -INFINITY : m + __builtin_amdgcn_logf(l);
      } else {
        float* const to = slot + (int64_t)at.col * (a_end.D + 4);
        emit_part<F>(to, d0, x);
        if (first) to[0] = m, to[1] = l;
      }
    }
    __syncthreads();
  } while (deal.next(arguments()));
}

// Keys of a stage: two stages in LDS, of one workgroup of eight waves, or of two of four.
constexpr int tall_keys(int w, int waves) { return w == 1 || (w == 2 && waves == 8) ? 128 : 64; }

// A stage holds the operands of its keys: of every 16-key tile the KS key operands, of every 32 keys the DT value operands, 16 bytes per
// lane, and the scales.  The waves share its conversion.  While one stage is used the next one is written.
// A SIMD has two waves.  While one forms weights (vector unit) the other one multiplies, values with weights and the next keys with the
// queries (matrix unit, at a higher priority: where both ask for it the one that multiplies goes on, and they part).  The later half of the
// waves converts later in the stage, for the same reason.
// One barrier per stage, before the products of its last step, which read the first keys of the next stage: that has been written by then, and
// the stage before, whose place it takes, was last read before the last such barrier.
template <int CD, int W, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) tall_attention_kernel(Args args) {
  using F = Form<CD, W>;
  constexpr int RT = tall_tiles(W), kKeys = tall_keys(W, WAVES), kSteps = kKeys / 32, kTiles = kKeys / 16;
  constexpr int kMine = kTiles > WAVES ? kTiles / WAVES : 1;             // 16-key tiles that a wave converts
  constexpr bool kApart = kTiles < WAVES;                                // a wave converts a tile's keys or its values
  constexpr int kValues = kTiles * F::KS * 64;                           // where the values begin, in 16 bytes
  constexpr int kStage = kValues + kSteps * F::DT * 64;
  // Rows of 256 elements leave no registers for both halves of a step's values, or for keys next to them.
  constexpr bool kLean = W == 4;
  // The first stage is converted in the loop, and not by code in front of it, which made 16-bit kernels of more than 64 elements spill 5 to 39
  // registers: 128 rows over 4 x 8 heads of 8192 bf16 keys of 128 elements 57 -> 54 us, 1024 rows of 256 elements 451 -> 413, int8 393 -> 383.
  // (fp16 and bf16 rows of 256 elements still spill 15, bf16 of 128 and e4m3 of 256 two.)
  // With 64 elements, where nothing spills, 1 to 10 % are lost.
  constexpr bool kInLoop = W >= 2;
  constexpr int kEarly = W == 1 || (W == 2 && F::codes) ? F::DT : F::DT / 2;                     // value operands that fit next to the weights
  static_assert(kTiles * (kApart ? 2 : 1) == WAVES * kMine, "every wave has its share of a stage");
  __shared__ u32x4 operands[2 * kStage];
  __shared__ __attribute__((aligned(16))) float scales[2][2][kKeys];     // of keys, of values
  __shared__ float most[2][kTiles];                                      // the largest scale of a tile's values
  __shared__ int flags[2][kTiles];                                       // a tile's page is there, and (bit 1) one of its values was not finite
  __shared__ float rest[WAVES][RT][16];                                  // powers of two that rows' scores are still to be multiplied by
  __shared__ int scan[WAVES + 2];
  const int wg = range_of(args, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Lane<F> at(threadIdx.x & 63);
  const int my_tile = kApart ? wave % kTiles : wave * kMine;
  const bool my_keys = !kApart || wave < kTiles, my_values = !kApart || wave >= kTiles;
  Deal<64 * WAVES, true> deal;
  if (!deal.start(arguments(), wg, scan)) return;
  do {
    const int b = deal.b, n = deal.n, context = deal.context;
    const int row0 = (deal.tile * WAVES + wave) * 16 * RT;
    const bool idle = row0 >= arguments().rows;                                    // (it converts all the same)
    const bool late = WAVES == 8 && wave >= 4;
    Keys<F> k[kMine];
    Values<F> v[kMine];
    const Source src(arguments(), b, deal.h, n);
    Place place[kMine], ahead[kMine];                                    // of the rows loaded last, and of the next ones
    const int pos0 = deal.blk * kBlock;
    const int steps = (deal.stop() - deal.blk) * (kBlock / 32), stages = steps / kSteps;
    const auto look = [&](int stage) {
#pragma unroll
      for (int t = 0; t < kMine; ++t) ahead[t] = Place(src, pos0 + stage * kKeys + (my_tile + t) * 16);
    };
    const auto fetch = [&](int stage) {
      const int D = arguments().D;
      const Lane<F> here = at.again();
#pragma unroll
      for (int t = 0; t < kMine; ++t) {
        place[t] = ahead[t];
        if (my_keys) k[t].template load<false>(src, D, place[t], here);
        if (my_values) v[t].load(src, D, place[t], here);
      }
      look(stage + 1);
    };
    look(0);
    fetch(0);
    Queries<F, RT> q;
    float by = arguments().scale2;
    q.load(arguments(), b, deal.h, row0, at);
    __syncthreads();                                                     // (the piece before has been used)
    bool apart = false;
    if (F::codes && arguments().bf16) {
      // One power of two for all rows of the workgroup, which the keys' scales undo; rows that it would leave under 2^-16 of the largest have
      // their own, and their scores are multiplied by the rest.
      int up[RT], least = kNoPower;
#pragma unroll
      for (int r = 0; r < RT; ++r) least = min(least, up[r] = q.power(r));
      least = least_of_row(least);
      if (at.lane == 0) scan[wave] = least;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) least = min(least, scan[w]);
      least = __builtin_amdgcn_readfirstlane(least);
      least = least == kNoPower ? 0 : least;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int mine = up[r] - least > 16 && up[r] != kNoPower ? up[r] : least;
        q.scale(r, mine);
        apart = apart || mine != least;
        if (at.g == 0) rest[wave][r][at.col] = __builtin_amdgcn_ldexpf(1.0f, least - mine);
      }
      apart = __any(apart);
      by = __builtin_amdgcn_ldexpf(by, -least);
    }
    q.arrive();
    State<F, RT> st;
    st.clear();
    const auto convert = [&](int stage) {
      u32x4* const to = operands + (stage & 1) * kStage + at.lane;
      float* const sc = scales[stage & 1][0];
      int flag[kMine];
#pragma unroll
      for (int t = 0; t < kMine; ++t) {
        const int pos = pos0 + stage * kKeys + (my_tile + t) * 16;
        flag[t] = place[t].there(src) ? 1 : 0;
        if (my_values && (!flag[t] || pos + 16 > min(context, n))) {
          v[t].drop(there_of(pos, n, flag[t], flag[t], at.g));
          if constexpr (!F::finite) flag[t] |= pos + 16 > context && __any(v[t].clean()) ? 2 : 0;
        }
        if (my_keys) {
#pragma unroll
          for (int c = 0; c < F::KS; ++c) to[((my_tile + t) * F::KS + c) * 64] = k[t].operand(c);
          if constexpr (!F::codes) {
            // What lies behind the rows becomes zeros here: addresses of their own cost rows of 256 elements 10 more spilled registers (256 rows over 4 x 8
            // heads of 8192 fp16 keys 118 -> 158 us).
            const int D = arguments().D;
            if (__builtin_expect(D % 64 != 0, 0)) {
              const Lane<F> here = at.again();
              uint32_t zero = 0;
              asm volatile("" : "+v"(zero));       // (formed here, not kept)
#pragma unroll
              for (int c = F::KS - 2; c < F::KS; ++c)
                if (here.behind(c, D)) to[((my_tile + t) * F::KS + c) * 64] = u32x4{zero, zero, zero, zero};
            }
          }
          if (F::codes && at.col == 0) *reinterpret_cast<f32x4*>(sc + (my_tile + t) * 16 + 4 * at.g) = k[t].scale * by;
        }
        if (my_values) {
          if constexpr (F::codes) {
            if (at.col == 0) *reinterpret_cast<f32x4*>(sc + kKeys + (my_tile + t) * 16 + 4 * at.g) = v[t].scale;
            const f32x4 x = v[t].scale;
            const float m = across(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))), true);
            if (at.lane == 0) most[stage & 1][my_tile + t] = fmaxf(m, 0.0f);   // (a NaN does not count)
          }
          if (at.lane == 0) flags[stage & 1][my_tile + t] = flag[t];
          if constexpr (kMine == 1) {
#pragma unroll
            for (int d = 0; d < F::DT; ++d)
              reinterpret_cast<u32x2*>(to + kValues + ((my_tile / 2) * F::DT + d) * 64)[my_tile & 1] = v[0].operand(d);
          } else if (t & 1) {
#pragma unroll
            for (int d = 0; d < F::DT; ++d)
              to[kValues + ((my_tile + t) / 2 * F::DT + d) * 64] = joined_operand(v[t - 1].operand(d), v[t].operand(d));
          }
        }
      }
    };
    // What a step reads from LDS is read ahead: keys, scales and flags under the products of the step before, values under the weights.
    // (Left to itself the scheduler reads each operand in front of its use, to save registers, and waits for it.)
    f32x4 s[RT][2], k_scale[2], v_scale[2];
    u32x4 kf[2][F::KS];
    float most_v = 1.0f;
    int flag[2];
    const auto read_keys = [&](int i, int t) {
      const u32x4* const from = operands + ((i / kSteps) & 1) * kStage + ((i % kSteps) * 2 + t) * F::KS * 64 + at.lane;
#pragma unroll
      for (int c = 0; c < F::KS; ++c) kf[t][c] = from[c * 64];
    };
    const auto read_scales = [&](int i) {
      const int buffer = (i / kSteps) & 1, j = i % kSteps;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (F::codes) {
          const float* const sc = scales[buffer][0] + j * 32 + 16 * t + 4 * at.g;
          k_scale[t] = *reinterpret_cast<const f32x4*>(sc);
          v_scale[t] = *reinterpret_cast<const f32x4*>(sc + kKeys);
        } else {
          k_scale[t] = f32x4{by, by, by, by};
          v_scale[t] = f32x4{1, 1, 1, 1};
        }
        flag[t] = flags[buffer][2 * j + t];
      }
      if constexpr (F::codes) most_v = fmaxf(most[buffer][2 * j], most[buffer][2 * j + 1]);
    };
    const auto products_of = [&](int t) {                                // of the keys read last with the queries
#pragma unroll
      for (int c = 0; c < F::KS; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][t] = mma<F::bf16>(kf[t][c], q.w[r][c], c ? s[r][t] : f32x4{0, 0, 0, 0});
    };
    if constexpr (!kInLoop) {
      convert(0);
      if (stages > 1) fetch(1);
      __syncthreads();
      if (!idle) {
        read_keys(0, 0);
        read_keys(0, 1);
        read_scales(0);
        products_of(0);
        products_of(1);
      }
    }
    // (in the loop: the step before the first one does this, with values and weights of 0)
    for (int i = kInLoop ? -1 : 0; i < steps; ++i) {
      const int stage = i < 0 ? -1 : i / kSteps, j = i < 0 ? kSteps - 1 : i % kSteps, pos = pos0 + i * 32;
      const bool run = !idle && pos < n, work = run && (!kInLoop || i >= 0);
      u32x4 vf[F::DT], p[RT];
      uint32_t seen[RT];
      bool not_finite = false;
      if (work) {
        const u32x4* const from = operands + (stage & 1) * kStage + kValues + j * F::DT * 64 + at.lane;
#pragma unroll
        for (int d = 0; d < kEarly; ++d) vf[d] = from[d * 64];
        const int f0 = __builtin_amdgcn_readfirstlane(flag[0]), f1 = __builtin_amdgcn_readfirstlane(flag[1]);
        const bool masked = pos + 32 > min(context, n) || !(f0 & f1 & 1);
        not_finite = !F::finite && ((f0 | f1) & 2) != 0;
#pragma unroll
        for (int r = 0; r < RT; ++r) seen[r] = 0xff;
        if (masked) {
          const uint32_t there = there_of(pos, n, f0 & 1, f1 & 1, at.g);
#pragma unroll
          for (int r = 0; r < RT; ++r) seen[r] = seen_by(arguments(), b, row0 + 16 * r + at.col, pos, context, there, at.g);
        }
        if (F::codes && __builtin_expect(apart, 0)) {
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float by_row = rest[wave][r][at.col];
#pragma unroll
            for (int t = 0; t < 2; ++t) s[r][t] = s[r][t] * by_row;
          }
        }
        weigh<F, RT>(k_scale, v_scale, most_v, s, masked, seen, st, p);
      } else if (kInLoop) {
#pragma unroll
        for (int d = 0; d < F::DT; ++d) vf[d] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < RT; ++r) p[r] = u32x4{0, 0, 0, 0}, seen[r] = 0;
      }
      if (((kInLoop && i < 0) || j == (late ? kSteps / 2 : 0)) && stage + 1 < stages) {
        convert(stage + 1);
        if (stage + 2 < stages) fetch(stage + 2);
      }
      const auto read_values = [&](int from_d) {
        const u32x4* const from = operands + (stage & 1) * kStage + kValues + j * F::DT * 64 + at.lane;
#pragma unroll
        for (int d = 0; d < F::DT / 2; ++d) vf[from_d + d] = from[(from_d + d) * 64];
      };
      // (behind the last step: what is read is not used)
      const int next = min(i + 1, steps - 1);
      if constexpr (kLean) {
        if (work) {
          add_values<F, RT, 0, F::DT / 2>(vf, p, st);
          read_values(F::DT / 2);
          add_values<F, RT, F::DT / 2, F::DT>(vf, p, st);
        }
        if (j == kSteps - 1) __syncthreads();
        if (run) {
          read_scales(next);
          read_keys(next, 0);
          read_keys(next, 1);
        }
      } else {
        if (kEarly < F::DT && work) read_values(F::DT / 2);                // (before the barrier: the stage's place is written behind it)
        if (j == kSteps - 1) __syncthreads();
        if (run) {
          __builtin_amdgcn_s_setprio(1);
          if (kEarly == F::DT) read_keys(next, 0);
          __builtin_amdgcn_sched_barrier(0);
          add_values<F, RT, 0, F::DT / 2>(vf, p, st);
          __builtin_amdgcn_sched_barrier(0);
          read_keys(next, kEarly == F::DT ? 1 : 0);
          read_scales(next);
          __builtin_amdgcn_sched_barrier(0);
          add_values<F, RT, F::DT / 2, F::DT>(vf, p, st);
          __builtin_amdgcn_sched_barrier(0);
          if (kEarly < F::DT) read_keys(next, 1);
        }
      }
      if (run) {
        if constexpr (!F::finite) {
          if (__builtin_expect(not_finite, 0)) add_not_finite<F, RT>(src, arguments().D, pos, p, seen, at, st);
        }
        products_of(0);
        products_of(1);
        __builtin_amdgcn_s_setprio(0);
      }
    }
    const Args& a = arguments();
    const bool final = deal.blk == 0 && deal.stop() == deal.nb;
    float* const slot = a.part + (int64_t)(2 * wg + (deal.blk == 0 ? 1 : 0)) * (16 * RT * WAVES) * (a.D + 4);
    if (deal.blk == 0 && threadIdx.x == 0) deal.tell(a, wg);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float l = across(st.l[r], false);
      const int row = row0 + 16 * r + at.col;
      if (row >= a.rows) continue;
      if (final) {
        const Output out(a, b, deal.h, row, l);
        const float inverse = 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[F::DT];
#pragma unroll
          for (int d = 0; d < F::DT; ++d) x[d] = st.o[r][d][i];
          emit<F>(a, out, Lane<F>::elements_of(a.D, 4 * at.g + i), x, inverse);
        }
        if (a.lse && at.g == 0) a.lse[out.row] = out.none ? -INFINITY : st.m[r] + __builtin_amdgcn_logf(l);
      } else {
        float* const to = slot + (int64_t)((wave * RT + r) * 16 + at.col) * (a.D + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[F::DT];
#pragma unroll
          for (int d = 0; d < F::DT; ++d) x[d] = st.o[r][d][i];
          emit_part<F>(to, Lane<F>::elements_of(a.D, 4 * at.g + i), x);
        }
        if (at.g == 0) to[0] = st.m[r], to[1] = l;
      }
    }
  } while (deal.next(arguments()));
}

#if FCR_HAS(0)
// Joins the parts of items that were cut, in the order of their keys.  Units are four elements of a row; a unit has `shares` threads, a
// power of two that take the parts in turn and meet in LDS: an item of few rows may have a part in every workgroup of the first kernel.
__global__ void __launch_bounds__(256) tree_join_kernel(Args a, int tile_rows, int shares, Div groups, Div pieces) {
  __shared__ f32x4 sums[256];
  __shared__ float stats[256][2];
  const int item = (int)groups.of(blockIdx.x);
  const int32_t* const told = a.first + kFirst + 2 * (int64_t)item;
  const int per = constant_at(a.first), from = constant_at(told), others = constant_at(told + 1);
  if (others <= 0) return;
  // workgroups behind the first (no more than there are, should lengths have changed under the call)
  const int more = min(followers(others, per), a.wgs - 1 - from);
  const int bh = (int)a.per_head.of((uint32_t)item), tile = item - bh * a.row_tiles;
  const int rows = min(tile_rows, a.rows - tile * tile_rows);
  const int units = 256 / shares, mine = (int)threadIdx.x / units;
  for (uint32_t group = blockIdx.x - (uint32_t)item * groups.d; group * units < (uint32_t)rows * pieces.d; group += groups.d) {
    const int unit = (int)group * units + ((int)threadIdx.x & (units - 1));
    const int r = (int)pieces.of((uint32_t)unit), d = 4 * (unit - r * (int)pieces.d);
    const bool live = r < rows;
    const int64_t stride = a.D + 4, part = (int64_t)tile_rows * stride;
    // the first part is in its workgroup's second slot, the others are in their workgroups' first ones
    const float* const parts = a.part + 2 * part * from + (live ? r : 0) * stride;
    float m = kNone, l = 0.0f;
    f32x4 x = {0, 0, 0, 0};
    const auto take = [&](float pm, float pl, f32x4 y) {
      const float top = fmaxf(m, pm);
      const float old = __builtin_amdgcn_exp2f(m - top), its = __builtin_amdgcn_exp2f(pm - top);
      l = l * old + pl * its;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = x[j] * old + y[j] * its;
      m = top;
    };
    if (live) {
      for (int w = mine; w <= more; w += shares) {
        const float* const p = parts + (w == 0 ? part : 2 * part * w);
        take(p[0], p[1], *reinterpret_cast<const f32x4*>(p + 4 + d));
      }
    }
    if (shares > 1) {
      __syncthreads();     // (of the units before)
      sums[threadIdx.x] = x;
      stats[threadIdx.x][0] = m, stats[threadIdx.x][1] = l;
      __syncthreads();
      if (mine == 0 && live) {
        for (int i = 1; i < shares && i <= more; ++i) {
          const int other = threadIdx.x + units * i;
          take(stats[other][0], stats[other][1], sums[other]);
        }
      }
    }
    if (mine != 0 || !live) continue;
    const int b = (int)a.heads.of((uint32_t)bh), h = bh - b * a.H;
    const Output out(a, b, h, tile * tile_rows + r, l);
    const float inverse = 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = out.none ? 0.0f : x[j] * inverse;
    *reinterpret_cast<u32x2*>(a.out + (out.row * a.D + d) * 2) = a.bf16 ? u32x2{pack2<FCR_DTYPE_BF16>(x[0], x[1]), pack2<FCR_DTYPE_BF16>(x[2], x[3])}
                                                                       : u32x2{pack2<FCR_DTYPE_F16>(x[0], x[1]), pack2<FCR_DTYPE_F16>(x[2], x[3])};
    if (a.lse && d == 0) a.lse[out.row] = out.none ? -INFINITY : m + __builtin_amdgcn_logf(l);
  }
}
#endif

template <int CD, int W>
bool launch_w(const Args& a, int form, hipStream_t s) {
  const dim3 grid((unsigned)a.wgs);
  if (form == 1) {
    hipLaunchKernelGGL((tree_attention_kernel<CD, W>), grid, dim3(256), 0, s, a);
  } else if (form == 8) {
    hipLaunchKernelGGL((tall_attention_kernel<CD, W, 8>), grid, dim3(512), 0, s, a);
  } else {
    if constexpr (W > 2) return false;
    else hipLaunchKernelGGL((tall_attention_kernel<CD, W, 4>), grid, dim3(256), 0, s, a);
  }
  return true;
}
template <int CD>
bool launch(const Args& a, int w, int form, hipStream_t s) {
  switch (w) {
    case 1: return launch_w<CD, 1>(a, form, s);
    case 2: return launch_w<CD, 2>(a, form, s);
    case 3: return launch_w<CD, 3>(a, form, s);
    default: return launch_w<CD, 4>(a, form, s);
  }
}
}  // namespace

#if FCR_HAS(1)
bool fcr_tree::attention_f16(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_F16>(a, w, form, s); }
#endif
#if FCR_HAS(2)
bool fcr_tree::attention_bf16(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_BF16>(a, w, form, s); }
#endif
#if FCR_HAS(3)
bool fcr_tree::attention_int8(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_INT8>(a, w, form, s); }
#endif
#if FCR_HAS(4)
bool fcr_tree::attention_e4m3(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_E4M3>(a, w, form, s); }
#endif

#if FCR_HAS(0)
namespace {
using fcr_detail::fail;
using fcr_detail::launched;

struct Plan {
  int form;                  // see form_of
  int tile_rows, row_tiles, wgs;
  int64_t items, first_bytes, bytes;
};
// What depends on sizes alone.  false: too large.
bool plan_of(bool codes, int B, int H, int G, int T, int D, int64_t capacity, Plan& p) {
  const int64_t rows = (int64_t)T * G;
  const int w = (D + 63) / 64;
  p.form = form_of(rows, w, codes);
  p.tile_rows = rows_of_tile(p.form, w);
  const int64_t tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  p.items = (int64_t)B * H * tiles;
  const int64_t blocks = p.items * ((capacity + kBlock - 1) / kBlock);
  if (rows > (1 << 24) || p.items > (1 << 22) || blocks > (1 << 30)) return false;
  p.row_tiles = (int)tiles;
  // As many as the CUs hold at once: one of eight waves, or of four that take more than 256 registers (8 x 8 heads of 1000 bf16 keys of 256
  // elements 21 us, 28 with twice as many, one behind the other); two of the others.
  int64_t wgs = (p.form == 8 || (!codes && w > 2) ? 1 : 2) * (int64_t)fcr_detail::chip_cus_of_current_device();
  if (blocks < wgs) wgs = blocks;
  p.wgs = (int)((wgs + 7) / 8 * 8);
  p.first_bytes = (kFirst * 4 + p.items * 8 + 15) / 16 * 16;
  p.bytes = p.first_bytes + 2ll * p.wgs * p.tile_rows * (D + 4) * 4;
  return true;
}
}  // namespace

extern "C" {

size_t fcr_tree_attention_bytes(int B, int H, int G, int T, int D, int64_t positions) {
  Plan p[2];             // for either kind of cache
  if (B < 1 || H < 1 || G < 1 || T < 1 || D < 16 || D > 256 || positions < 1 || positions > (1 << 30) || (int64_t)B * H > (1 << 24)) return 0;
  return plan_of(true, B, H, G, T, D, positions, p[0]) && plan_of(false, B, H, G, T, D, positions, p[1]) ? (size_t)std::max(p[0].bytes, p[1].bytes) : 0;
}

int fcr_tree_attention(const void* q, const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages,
                       const int32_t* context, const int64_t context_strides[2], const uint8_t* mask, int64_t mask_stride,
                       const int32_t* tree_lengths, void* out, float* lse, void* ws, size_t ws_bytes, int dtype, int B, int G, int T,
                       const int64_t q_strides[4], float scale, void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc) return rc;
  if ((rc = check_table(table, table_stride, table_pages, cache->page_size, B))) return rc;
  if (!q || !q_strides || !context || !context_strides || !out || !ws) return fail(FCR_E_NULL, "null pointer argument");
  if (dtype != FCR_DTYPE_F16 && dtype != FCR_DTYPE_BF16) return fail(FCR_E_DTYPE, "queries must be FCR_DTYPE_F16 or FCR_DTYPE_BF16");
  if (!has_codes(cache->dtype) && cache->dtype != dtype) return fail(FCR_E_DTYPE, "queries must have the type of a cache of 16-bit elements");
  const int H = cache->H, D = cache->D;
  const int64_t capacity = (int64_t)table_pages * cache->page_size;
  Plan plan;
  if (mask && T > 46340) return fail(FCR_E_SHAPE, "a mask of more than 2^31 bytes");
  if (G < 1 || T < 1 || T > (1 << 24) || G > (1 << 24) || (int64_t)B * H > (1 << 24) || (int64_t)H * G > (1 << 24) || 
      !plan_of(has_codes(cache->dtype), B, H, G, T, D, capacity, plan))
    return fail(FCR_E_SHAPE, "G and T must be >= 1; B, H, G, T and the table are too large for one call otherwise");
  if (!isfinite(scale)) return fail(FCR_E_SCALE, "scale must be finite");
  bool ok = q_strides[3] == 1 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  const int sizes[3] = {B, H * G, T};
  for (int j = 0; j < 3; ++j) ok = ok && (sizes[j] == 1 || (q_strides[j] >= 0 && q_strides[j] % 8 == 0 && q_strides[j] < (1ll << 40)));
  if (!ok) return fail(FCR_E_STRIDE, "q: unit stride of the last dimension, 16-byte aligned rows");
  if (context_strides[0] < 0 || context_strides[1] < 0 || mask_stride < 0) return fail(FCR_E_STRIDE, "strides must be >= 0");
  if ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || (reinterpret_cast<uintptr_t>(ws) & 15) != 0)
    return fail(FCR_E_STRIDE, "out and the workspace must be 16-byte aligned");
  if (ws_bytes < (size_t)plan.bytes) return fail(FCR_E_SCRATCH, "the workspace is smaller than fcr_tree_attention_bytes");
  Args a;
  a.q = static_cast<const char*>(q);
  a.qb = B > 1 ? 2 * q_strides[0] : 0, a.qh = H * G > 1 ? 2 * q_strides[1] : 0, a.qt = T > 1 ? 2 * q_strides[2] : 0;
  a.c = pages_of(*cache, table, table_stride, table_pages);
  a.context = Lengths{context, context_strides[0], context_strides[1]};
  a.tree_lengths = tree_lengths;
  a.mask = mask;
  a.mask_b = mask_stride;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.first = static_cast<int32_t*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + plan.first_bytes);
  a.B = B, a.H = H, a.T = T, a.D = D, a.rows = T * G, a.row_tiles = plan.row_tiles, a.bf16 = dtype == FCR_DTYPE_BF16;
  a.G.set((uint32_t)G), a.per_head.set((uint32_t)plan.row_tiles), a.heads.set((uint32_t)H), a.all.set((uint32_t)plan.wgs);
  a.positions = (int)capacity;
  a.scale2 = scale * 1.44269504088896340736f;
  a.wgs = plan.wgs;
  const int w = (D + 63) / 64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  bool there;
  switch (cache->dtype) {
    case FCR_DTYPE_F16: there = attention_f16(a, w, plan.form, s); break;
    case FCR_DTYPE_BF16: there = attention_bf16(a, w, plan.form, s); break;
    case FCR_DTYPE_INT8: there = attention_int8(a, w, plan.form, s); break;
    default: there = attention_e4m3(a, w, plan.form, s); break;
  }
  if (!there) return fail(FCR_E_SHAPE, "no kernel for these sizes");
  if ((rc = launched("tree_attention_kernel"))) return rc;
  Div groups, pieces;
  const int rows = std::min(plan.tile_rows, a.rows), shares = plan.wgs >= 16 * plan.items ? 8 : 1, units = 256 / shares;
  const int64_t most = (1 << 22) / plan.items;
  pieces.set((uint32_t)D / 4);
  groups.set((uint32_t)std::max<int64_t>(1, std::min<int64_t>(most, (rows * (D / 4) + units - 1) / units)));
  hipLaunchKernelGGL(tree_join_kernel, dim3((unsigned)(plan.items * groups.d)), dim3(256), 0, s, a, plan.tile_rows, shares, groups, pieces);
  return launched("tree_join_kernel");
}

}  // extern "C"
#endif
