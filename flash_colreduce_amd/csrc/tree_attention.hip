// Attention of drafted tokens over a paged cache of keys and values, quantised or not.
//
// T tokens of a sequence have been drafted (a single one in plain decoding, a chain, or a tree whose nodes share their prefixes) and their
// keys and values written behind the sequence's `context` rows.  A query row is a (token, query head of the key head) pair; it
// sees every key of the context, and of the drafted tokens those that the tree's mask names:
//   s_j = scale log2(e) <q, c_j> ks_j,   p_j = 2^(s_j - m),   o = sum_j p_j vs_j v_j / sum_j p_j,   lse2 = m + log2 sum_j p_j.
//
// The work is bound by reading the cache, so the G query heads of a key head and the drafted tokens are the 16 columns of the matrix
// instructions (RT column tiles per wave), and every key and value is read once per 16 RT query rows, from global memory into registers
// without a stop in LDS:
//   S^T = K Q^T   a lane owns one query (lane & 15) and keys 4 g + i of a 16-key tile (g = lane / 16, register i);
//   O^T = V^T P^T keeps that query in the lane.  The 8 keys that a lane feeds to one instruction are keys 4 g + i of two tiles, which is
//                 what the lane holds of P: the probabilities never leave their lane.  V^T is formed from 8 rows of V
//                 with byte permutes that convert codes at the same time.
// Softmax statistics are one scalar per lane and in 32 bits.
//
// Codes are multiplied in fp16, where each of them is exact: bf16 queries are scaled by a power of two per row to fit (elements under
// 2^-28 of the row's largest lose bits), the keys' scales multiply the scores, the values' scales the probabilities, in 32 bits, before these
// are rounded to 11 bits.  For that rounding each row has an exponent of its own (State::e), so that weights p_j vs_j fit fp16 whatever
// the scales are.  16-bit caches are multiplied in their own type.
//
// Distribution: the (batch, head, row tile) items are cut into blocks of 128 keys (a wave takes 32 of each), laid end to end, and every
// workgroup takes the same number of blocks, found from the lengths on the device.  Parts of an item that was cut are joined by a second
// kernel, in the order of the keys.

#include <math.h>

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
  int32_t* first;              // [items]: where an item begins, in blocks
  float* part;                 // [2 workgroups][rows of a tile][D + 2]
  int B, H, T, D, rows, row_tiles, bf16;
  Div G;
  float scale2;
  int wgs, least;              // workgroups of the launch; blocks that one takes at least
};
void attention_f16(const Args& a, int w, int rt, hipStream_t s);
void attention_bf16(const Args& a, int w, int rt, hipStream_t s);
void attention_int8(const Args& a, int w, int rt, hipStream_t s);
void attention_e4m3(const Args& a, int w, int rt, hipStream_t s);
}  // namespace fcr_tree

namespace {
using namespace fcr_tree;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32 * kWaves;          // keys of a block
constexpr float kNone = -3.0e38f;            // reference of a row that has seen no key
constexpr float kLazy = 4.0f;                // scores may pass the reference by this much before it is raised

__device__ __forceinline__ int blocks_of(int n) { return n <= 0 ? 1 : (n + kBlock - 1) / kBlock; }

// Keys of a sequence: those of the context, then those of the drafted tokens.
__device__ __forceinline__ void keys_of(const Args& a, int b, int h, int& context, int& n) {
  const int tree = a.tree_lengths ? min(max(a.tree_lengths[b], 0), a.T) : a.T;
  context = max(a.context.of(b, h), 0);
  n = (int)min((int64_t)context + tree, a.c.capacity);
}

__device__ __forceinline__ float across(float x, bool largest) {   // over the four lanes that share a query
  float y = __shfl_xor(x, 16);
  x = largest ? fmaxf(x, y) : x + y;
  y = __shfl_xor(x, 32);
  return largest ? fmaxf(x, y) : x + y;
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

// Four codes as four fp16, in their order.
template <int CD>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CD == FCR_DTYPE_INT8) {
    w ^= 0x80808080u;
    lo = centred(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
    hi = centred(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
  } else {
    lo = halves_of_e4m3<false>(w);
    hi = halves_of_e4m3<true>(w);
  }
}

// W: D / 64, rounded up.  RT: 16-row tiles of queries per wave.
template <int CD, int W, int RT>
struct Form {
  static constexpr bool codes = CD == FCR_DTYPE_INT8 || CD == FCR_DTYPE_E4M3;
  static constexpr bool bf16 = CD == FCR_DTYPE_BF16;
  static constexpr int KS = 2 * W;                // k-steps of 32 elements
  static constexpr int DT = 4 * W;                // 16-element tiles of the output; a lane's elements are consecutive
  static constexpr int KL = codes ? W : 2 * W;    // 16-byte loads of a key
  static constexpr int VW = codes ? W : 2 * W;    // words that a lane has of a value row
};

template <class F>
struct Keys {
  u32x4 w[2][F::KL];
  f32x4 scale[2];
};
template <class F>
struct Values {
  uint32_t w[8][F::VW];
  f32x4 scale[2];
};

// Where the two 16-key tiles of a wave's 32 keys lie: page (< 0: not there) and first row in it.
struct Place {
  int page[2];
  int row[2];
};

__device__ __forceinline__ Place place_of(const Args& a, int b, int pos, int n) {
  Place p;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    p.page[t] = -1;
    p.row[t] = 0;
    if (pos + 16 * t < n) {
      uint32_t row;
      p.page[t] = page_of(a.c, b, (uint32_t)(pos + 16 * t), row);
      p.row[t] = (int)row;
    }
  }
  return p;
}

template <int N>
__device__ __forceinline__ void load_words(const char* at, uint32_t (&w)[N]) {
  // (a lane's part of a row is 4 N bytes: aligned to 16 where N is a multiple of 4, to 8 where it is even)
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(at)[i];
      w[4 * i] = v[0], w[4 * i + 1] = v[1], w[4 * i + 2] = v[2], w[4 * i + 3] = v[3];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u32x2 v = reinterpret_cast<const u32x2*>(at)[i];
      w[2 * i] = v[0], w[2 * i + 1] = v[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(at)[i];
  }
}

// koff: bytes of the lane's key row (lane & 15), kchunk: its 16-byte pieces; a row's last piece stands for those behind it.
template <class F>
__device__ __forceinline__ void load_keys(const Args& a, int h, const Place& p, uint32_t koff, const uint32_t (&kchunk)[F::KL], int g,
                                          Keys<F>& k) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (p.page[t] >= 0) {
      const char* base = a.c.side[0].rows + p.page[t] * a.c.side[0].page + h * a.c.side[0].head + p.row[t] * a.c.side[0].row;
#pragma unroll
      for (int i = 0; i < F::KL; ++i) k.w[t][i] = *reinterpret_cast<const u32x4*>(base + (koff + kchunk[i]));
      if constexpr (F::codes)
        k.scale[t] = *reinterpret_cast<const f32x4*>(a.c.side[0].scale + p.page[t] * a.c.side[0].s_page + h * a.c.side[0].s_head +
                                                     p.row[t] + 4 * g);
    } else {
#pragma unroll
      for (int i = 0; i < F::KL; ++i) k.w[t][i] = u32x4{0, 0, 0, 0};
      k.scale[t] = f32x4{0, 0, 0, 0};
    }
  }
}

// voff: bytes of row 4 g and of the lane's elements.
template <class F>
__device__ __forceinline__ void load_values(const Args& a, int h, const Place& p, uint32_t voff, int g, Values<F>& v) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (p.page[t] >= 0) {
      const char* base = a.c.side[1].rows + p.page[t] * a.c.side[1].page + h * a.c.side[1].head + p.row[t] * a.c.side[1].row;
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words(base + (voff + (uint32_t)(i * a.c.side[1].row)), v.w[4 * t + i]);
      if constexpr (F::codes)
        v.scale[t] = *reinterpret_cast<const f32x4*>(a.c.side[1].scale + p.page[t] * a.c.side[1].s_page + h * a.c.side[1].s_head +
                                                     p.row[t] + 4 * g);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < F::VW; ++j) v.w[4 * t + i][j] = 0;
      v.scale[t] = f32x4{0, 0, 0, 0};
    }
  }
}

// The operand of element d (of the lane's DT) from the 8 rows: V[key][d] for the lane's 8 keys.
template <int CD, class F>
__device__ __forceinline__ u32x4 value_operand(const uint32_t (&v)[8][F::VW], int d) {
  u32x4 f;
  if constexpr (CD == FCR_DTYPE_INT8) {
    const uint32_t pick = 0x0c040c00u + 0x00010001u * (d & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)   // (of codes + 128)
      f[j] = centred(__builtin_amdgcn_perm(v[2 * j + 1][d / 4], v[2 * j][d / 4], pick) | 0x64006400u);
  } else if constexpr (CD == FCR_DTYPE_E4M3) {
    const uint32_t pick = (d & 2) ? 0x07030602u : 0x05010400u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = __builtin_amdgcn_perm(v[2 * j + 1][d / 4], v[2 * j][d / 4], pick);
      f[j] = (d & 1) ? halves_of_e4m3<true>(w) : halves_of_e4m3<false>(w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f[j] = __builtin_amdgcn_perm(v[2 * j + 1][d / 2], v[2 * j][d / 2], (d & 1) ? 0x07060302u : 0x05040100u);
  }
  return f;
}

// Whether a word holds a 16-bit element that is not finite.
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// What a lane knows of the query of each of its column tiles.
template <class F, int RT>
struct State {
  f32x4 o[RT][F::DT];
  float m[RT];        // reference exponent, a whole number (raised, not followed: see kLazy); kNone before the first key
  float l[RT];        // this lane's part of sum 2^(s - m)
  float e[RT];        // o holds sum 2^(s - m) vs v * 2^e
};

// The weights of 32 keys from their scores.  `masked`: seen holds the keys that a row sees, bit 4 t + i; else every key is seen.
template <class F, int RT>
__device__ __forceinline__ void weights(const f32x4 (&k_scale)[2], const f32x4 (&v_scale)[2], const f32x4 (&s)[RT][2], const float (&qf)[RT],
                                        bool masked, const uint32_t (&seen)[RT], State<F, RT>& st, u32x4 (&p)[RT]) {
  float most_v = 0.0f;
  if constexpr (F::codes) {
#pragma unroll
    for (int e = 0; e < 8; ++e) most_v = fmaxf(most_v, fabsf(v_scale[e / 4][e % 4]));
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float x[8], by[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      by[e] = F::codes ? qf[r] * k_scale[e / 4][e % 4] : qf[r];
      x[e] = __builtin_fmaf(s[r][e / 4][e % 4], by[e], -st.m[r]);
    }
    if (masked) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (seen[r] >> e) & 1u ? x[e] : -INFINITY;
    }
    float most = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) most = fmaxf(most, x[e]);
    if (__any(most > kLazy)) {
      // raise the reference of rows whose scores passed it
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[r][e / 4][e % 4] * by[e];
        if (masked) x[e] = (seen[r] >> e) & 1u ? x[e] : -INFINITY;
        most = e ? fmaxf(most, x[e]) : x[e];
      }
      most = across(most, true);
      const float m = most > st.m[r] ? ceilf(most) : st.m[r];
      float shrink = __builtin_amdgcn_exp2f(st.m[r] - m);
      st.l[r] *= shrink;
      if constexpr (F::codes) {
        // the weights' exponent rises instead of the sums shrinking, as far as fp32 can express 2^e
        const float e = st.e[r] + (m - st.m[r]);
        st.e[r] = fminf(e, 120.0f);
        shrink = __builtin_amdgcn_exp2f(st.e[r] - e);
      }
#pragma unroll
      for (int d = 0; d < F::DT; ++d) st.o[r][d] *= shrink;
      st.m[r] = m;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] -= m;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(x[e]);
      st.l[r] += x[e];
    }
    if constexpr (F::codes) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= v_scale[e / 4][e % 4];
      if (masked) {   // (a hidden value's scale may be a NaN)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (seen[r] >> e) & 1u ? x[e] : 0.0f;
      }
      float f = __builtin_amdgcn_exp2f(st.e[r]);
      if (__any(most_v * f > 0x1p11f)) {
        // probabilities are 2^kLazy at most: only here can a weight pass fp16
        float w = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) w = fmaxf(w, fabsf(x[e]));
        w = across(w, true);
        if (w * f > 0x1p15f) {
          const float to = fminf(st.e[r], (float)(126 - (int)(__builtin_bit_cast(uint32_t, w) >> 23)));   // w 2^to in [1/2, 1)
          const float by = __builtin_amdgcn_exp2f(to - st.e[r]);
#pragma unroll
          for (int d = 0; d < F::DT; ++d) st.o[r][d] *= by;
          st.e[r] = to;
          f = __builtin_amdgcn_exp2f(to);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) p[r][j] = F::bf16 ? pack2<FCR_DTYPE_BF16>(x[2 * j], x[2 * j + 1]) : pack2<FCR_DTYPE_F16>(x[2 * j], x[2 * j + 1]);
  }
}

// O^T += V^T P^T where a value that is not finite may stand at a key that some rows do not see: 0 * inf would reach them.  One key
// at a time, and only rows that see it take the result.
template <int CD, class F, int RT>
__device__ __forceinline__ void add_values_one_by_one(const Values<F>& v, const u32x4 (&p)[RT], const uint32_t (&seen)[RT], int lane, State<F, RT>& st) {
  for (int key = 0; key < 32; ++key) {
    const int e = key & 7, g = key >> 3;
    const bool mine = (lane >> 4) == g;
    uint32_t row[8][F::VW];
#pragma unroll
    for (int j = 0; j < F::VW; ++j) {
      uint32_t w = v.w[0][j];
#pragma unroll
      for (int i = 1; i < 8; ++i) w = e == i ? v.w[i][j] : w;
      w = mine ? w : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) row[i][j] = i == 0 ? w : 0;   // (the key takes the place of the lane's first)
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      uint32_t w = p[r][0];
#pragma unroll
      for (int j = 1; j < 4; ++j) w = (e >> 1) == j ? p[r][j] : w;
      w = mine ? ((e & 1) ? w >> 16 : w & 0xffffu) : 0;
      const bool see = (__shfl((int)seen[r], 16 * g + (lane & 15)) >> e) & 1;
#pragma unroll
      for (int d = 0; d < F::DT; ++d) {
        const f32x4 with = mma<F::bf16>(value_operand<CD, F>(row, d), u32x4{w, 0, 0, 0}, st.o[r][d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[r][d][i] = see ? with[i] : st.o[r][d][i];
      }
    }
  }
}

template <int CD, int W, int RT>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(Args a) {
  using F = Form<CD, W, RT>;
  __shared__ float joined[4 * F::DT * 4 * 64];          // [wave][register][tile][lane]
  __shared__ float stats[kWaves][RT][16][3];            // m, l, e
  __shared__ int scan[kWaves + 2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  // workgroups are dealt to 8 dies in turn: consecutive ranges of blocks, which share keys, go to one die
  const int wg = (blockIdx.x & 7) * (a.wgs >> 3) + (blockIdx.x >> 3);

  // Which blocks are this workgroup's: lengths are known on the device only.  Lengths of sequences: an entry is H heads.
  const bool by_head = a.context.sh != 0;
  const int entries = by_head ? a.B * a.H : a.B;
  const int weight = by_head ? a.row_tiles : a.H * a.row_tiles;
  const auto entry_blocks = [&](int e) {
    int context, n;
    keys_of(a, by_head ? e / a.H : e, by_head ? e % a.H : 0, context, n);
    return blocks_of(n) * weight;
  };
  int total = 0;
  for (int e = tid; e < entries; e += kThreads) total += entry_blocks(e);
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  if (lane == 0) scan[wave] = total;
  __syncthreads();
  total = scan[0] + scan[1] + scan[2] + scan[3];
  const int per = max((total + a.wgs - 1) / a.wgs, a.least);
  int at = wg * per;                                    // (wgs * per is total + wgs at most: checked by the host to fit)
  const int end = min(at + per, total);
  if (at >= end) return;
  int entry = 0, begun = 0;                             // the entry that holds `at`, and its first block
  for (int base = 0, before = 0;; base += kThreads) {
    const int e = base + tid;
    const int mine = e < entries ? entry_blocks(e) : 0;
    int sum = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(sum, o);
      if (lane >= o) sum += x;
    }
    __syncthreads();
    if (lane == 63) scan[wave] = sum;
    if (tid == 0) scan[kWaves] = -1;
    __syncthreads();
    int start = before + sum - mine;
    for (int i = 0; i < wave; ++i) start += scan[i];
    if (mine > 0 && at >= start && at < start + mine) {
      scan[kWaves] = e;
      scan[kWaves + 1] = start;
    }
    before += scan[0] + scan[1] + scan[2] + scan[3];
    __syncthreads();
    if (scan[kWaves] >= 0) {
      entry = scan[kWaves], begun = scan[kWaves + 1];
      break;
    }
    if (base + kThreads >= entries) return;             // (only if lengths change under the call)
  }
  entry = __builtin_amdgcn_readfirstlane(entry);
  begun = __builtin_amdgcn_readfirstlane(begun);

  // the lane's places in rows of keys and of values
  const int e_bytes = F::codes ? 1 : 2;
  const uint32_t row_bytes = (uint32_t)(a.D * e_bytes);
  const uint32_t koff = (uint32_t)(col * a.c.side[0].row);
  uint32_t kchunk[F::KL];
#pragma unroll
  for (int i = 0; i < F::KL; ++i) kchunk[i] = min(64u * i + 16u * g, row_bytes - 16u);
  const int dfirst = min(col * F::DT, a.D - F::DT);     // (behind the row's end: elements that another lane has as well)
  const uint32_t voff = (uint32_t)(4 * g * a.c.side[1].row) + (uint32_t)(dfirst * e_bytes);

  int b = by_head ? entry / a.H : entry, h = by_head ? entry % a.H : 0;
  int context, n;
  keys_of(a, b, h, context, n);
  int nb = blocks_of(n);
  int in = at - begun;                                  // blocks from the entry's begin
  if (!by_head) {
    h = in / (nb * a.row_tiles);
    in -= h * nb * a.row_tiles;
  }
  int tile = in / nb;
  int blk = in - tile * nb;

  while (at < end) {
    context = __builtin_amdgcn_readfirstlane(context);
    n = __builtin_amdgcn_readfirstlane(n);
    const int item = (b * a.H + h) * a.row_tiles + tile;
    const int stop = min(nb, blk + (end - at));         // blocks [blk, stop) of this item

    // queries: column col of tile r is row 16 r + col of the workgroup's, token t, head gq of the key head
    u32x4 q[RT][F::KS];
    float qf[RT];
    int token[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = (tile * RT + r) * 16 + col;
      const bool live = row < a.rows;
      const uint32_t t = a.G.of((uint32_t)(live ? row : 0)), gq = (uint32_t)(live ? row : 0) - t * a.G.d;
      token[r] = (int)t;
      const char* at_q = a.q + b * a.qb + (int64_t)(h * (int)a.G.d + (int)gq) * a.qh + t * a.qt;
      qf[r] = a.scale2;
      uint32_t most = 0;
#pragma unroll
      for (int s = 0; s < F::KS; ++s) {
        // the elements that the lane's part of a key stands for in k-step s
        const int d = F::codes ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
        q[r][s] = live && d < a.D ? *reinterpret_cast<const u32x4*>(at_q + 2 * d) : u32x4{0, 0, 0, 0};
        if constexpr (F::codes) {
#pragma unroll
          for (int j = 0; j < 4; ++j) most = max(most, max(q[r][s][j] & 0x7fffu, (q[r][s][j] >> 16) & 0x7fffu));
        }
      }
      if constexpr (F::codes) {
        if (a.bf16) {
          most = max(most, (uint32_t)__shfl_xor((int)most, 16));
          most = max(most, (uint32_t)__shfl_xor((int)most, 32));
          // largest element to [2^14, 2^15); exponents in steps of two halves, each in range
          const int up = most == 0 || most >= 0x7f80u ? 0 : min(14 - ((int)(most >> 7) - 127), 140);
          const float by1 = __builtin_bit_cast(float, (uint32_t)(127 + up / 2) << 23), by2 = __builtin_bit_cast(float, (uint32_t)(127 + up - up / 2) << 23);
          const float undo1 = __builtin_bit_cast(float, (uint32_t)(127 - up / 2) << 23), undo2 = __builtin_bit_cast(float, (uint32_t)(127 - (up - up / 2)) << 23);
          qf[r] = a.scale2 * undo1 * undo2;
#pragma unroll
          for (int s = 0; s < F::KS; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              q[r][s][j] = pack2<FCR_DTYPE_F16>(bf16_of(q[r][s][j], 0) * by1 * by2, bf16_of(q[r][s][j], 1) * by1 * by2);
        }
      }
    }

    State<F, RT> st;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      st.m[r] = kNone, st.l[r] = 0.0f, st.e[r] = F::codes ? 120.0f : 0.0f;
#pragma unroll
      for (int d = 0; d < F::DT; ++d) st.o[r][d] = f32x4{0, 0, 0, 0};
    }

    Keys<F> k;
    Values<F> v;
    Place here = place_of(a, b, blk * kBlock + wave * 32, n);
    load_keys<F>(a, h, here, koff, kchunk, g, k);
    load_values<F>(a, h, here, voff, g, v);
    for (int i = blk; i < stop; ++i) {
      const int pos = i * kBlock + wave * 32;
      const Place next = i + 1 < stop ? place_of(a, b, pos + kBlock, n) : Place{{-1, -1}, {0, 0}};
      if (pos >= n) break;                              // (a wave's later blocks lie behind this one)
      f32x4 s[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][0] = s[r][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < F::KL; ++c) {
          if constexpr (F::codes) {
            u32x4 f[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t lo, hi;
              widen<CD>(k.w[t][c][j], lo, hi);
              f[j / 2][2 * (j & 1)] = lo, f[j / 2][2 * (j & 1) + 1] = hi;
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              s[r][t] = mma<false>(f[0], q[r][2 * c], s[r][t]);
              s[r][t] = mma<false>(f[1], q[r][2 * c + 1], s[r][t]);
            }
          } else {
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][t] = mma<F::bf16>(k.w[t][c], q[r][c], s[r][t]);
          }
        }
      const f32x4 k_scale[2] = {k.scale[0], k.scale[1]};
      if (i + 1 < stop) load_keys<F>(a, h, next, koff, kchunk, g, k);

      u32x4 p[RT];
      uint32_t seen[RT] = {};
      const bool masked = pos + 32 > min(context, n) || here.page[0] < 0 || here.page[1] < 0;
      bool one_by_one = false;
      if (masked) {
        uint32_t there = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool is = pos + 16 * (e / 4) + 4 * g + e % 4 < n && here.page[e / 4] >= 0;
          there |= is ? 1u << e : 0u;
          if (!is) {
#pragma unroll
            for (int j = 0; j < F::VW; ++j) v.w[e][j] = 0;
            v.scale[e / 4][e % 4] = 0.0f;
          }
        }
        if constexpr (!F::codes) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int j = 0; j < F::VW; ++j) one_by_one = one_by_one || not_finite<F::bf16>(v.w[e][j]);
          one_by_one = __any(one_by_one) && pos + 32 > context;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int u = pos + 16 * (e / 4) + 4 * g + e % 4 - context;   // which drafted token
            bool is = (there >> e) & 1u;
            if (is && u >= 0) is = a.mask ? a.mask[b * a.mask_b + (int64_t)token[r] * a.T + u] != 0 : u <= token[r];
            seen[r] |= is ? 1u << e : 0u;
          }
        }
      }
      weights<F, RT>(k_scale, v.scale, s, qf, masked, seen, st, p);
      if constexpr (CD == FCR_DTYPE_INT8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int j = 0; j < F::VW; ++j) v.w[e][j] ^= 0x80808080u;   // codes + 128, see value_operand
      }
      if (one_by_one) {
        add_values_one_by_one<CD, F, RT>(v, p, seen, lane, st);
      } else {
#pragma unroll
        for (int d = 0; d < F::DT; ++d) {
          const u32x4 f = value_operand<CD, F>(v.w, d);
#pragma unroll
          for (int r = 0; r < RT; ++r) st.o[r][d] = mma<F::bf16>(f, p[r], st.o[r][d]);
        }
      }
      if (i + 1 < stop) load_values<F>(a, h, next, voff, g, v);
      here = next;
    }

    // join the four waves
    const bool final = blk == 0 && stop == nb;
    float* const slot = a.part + (int64_t)(2 * wg + (blk == 0 ? 1 : 0)) * (16 * RT) * (a.D + 2);
    if (blk == 0 && tid == 0 && a.first) a.first[item] = at;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float l = across(st.l[r], false);
      if (g == 0) {
        stats[wave][r][col][0] = st.m[r];
        stats[wave][r][col][1] = l;
        stats[wave][r][col][2] = st.e[r];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float m = stats[0][r][col][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) m = fmaxf(m, stats[w][r][col][0]);
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) l += stats[w][r][col][1] * __builtin_amdgcn_exp2f(stats[w][r][col][0] - m);
      const float by = __builtin_amdgcn_exp2f(st.m[r] - m - st.e[r]);
      // (a wave that has seen nothing has sums of zero; its exponent may not be expressible)
      const bool none = st.m[r] == kNone;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < F::DT; ++d) joined[((wave * 4 + i) * F::DT + d) * 64 + lane] = none ? 0.0f : st.o[r][d][i] * by;
      __syncthreads();
      // wave w writes register w of every tile: query col, elements from dfirst of lane 4 g + w on
      const int row = (tile * RT + r) * 16 + col;
      const int d0 = min((4 * g + wave) * F::DT, a.D - F::DT);
      float x[F::DT];
#pragma unroll
      for (int d = 0; d < F::DT; ++d) {
        x[d] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x[d] += joined[((w * 4 + wave) * F::DT + d) * 64 + lane];
      }
      if (row < a.rows) {
        if (final) {
          const bool none = (a.tree_lengths && token[r] >= a.tree_lengths[b]) || l == 0.0f;
          const float inverse = 1.0f / l;
          const int64_t to = ((int64_t)b * a.H * a.G.d + (int64_t)h * a.G.d + (row - token[r] * (int)a.G.d)) * a.T + token[r];
#pragma unroll
          for (int d = 0; d < F::DT; ++d) x[d] = none ? 0.0f : x[d] * inverse;
          uint32_t* const o = reinterpret_cast<uint32_t*>(a.out + (to * a.D + d0) * 2);
#pragma unroll
          for (int d = 0; d < F::DT / 2; ++d) o[d] = a.bf16 ? pack2<FCR_DTYPE_BF16>(x[2 * d], x[2 * d + 1]) : pack2<FCR_DTYPE_F16>(x[2 * d], x[2 * d + 1]);
          if (a.lse && wave == 0 && g == 0) a.lse[to] = none ? -INFINITY : m + __builtin_amdgcn_logf(l);
        } else {
          float* const o = slot + (16 * r + col) * (a.D + 2);
#pragma unroll
          for (int d = 0; d < F::DT; ++d) o[2 + d0 + d] = x[d];
          if (wave == 0 && g == 0) o[0] = m, o[1] = l;
        }
      }
      __syncthreads();
    }

    at += stop - blk;
    blk = 0;
    if (++tile == a.row_tiles) {
      tile = 0;
      if (++h == a.H) h = 0, ++b;
      if (at < end) {
        keys_of(a, b, h, context, n);
        nb = blocks_of(n);
      }
    }
  }
}

#if FCR_HAS(0)
// Joins the parts of items that were cut: a thread per two elements of a row.
__global__ void __launch_bounds__(256) tree_join_kernel(Args a, int tile_rows) {
  const int item = blockIdx.x;
  const int tile = item % a.row_tiles, bh = item / a.row_tiles;
  const int b = bh / a.H, h = bh - b * a.H;
  // how many blocks a workgroup took, as the first kernel found it
  __shared__ int scan[4];
  const bool by_head = a.context.sh != 0;
  const int entries = by_head ? a.B * a.H : a.B;
  const int weight = by_head ? a.row_tiles : a.H * a.row_tiles;
  int total = 0;
  for (int e = threadIdx.x; e < entries; e += 256) {
    int context, n;
    keys_of(a, by_head ? e / a.H : e, by_head ? e % a.H : 0, context, n);
    total += blocks_of(n) * weight;
  }
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  if ((threadIdx.x & 63) == 0) scan[threadIdx.x >> 6] = total;
  __syncthreads();
  total = scan[0] + scan[1] + scan[2] + scan[3];
  const int per = max((total + a.wgs - 1) / a.wgs, a.least);
  int context, n;
  keys_of(a, b, h, context, n);
  const int begin = a.first[item];
  const int from = begin / per, to = (begin + blocks_of(n) - 1) / per;
  if (from == to) return;
  const int pairs = a.D / 2;
  const int rows = min(tile_rows, a.rows - tile * tile_rows);
  const int64_t stride = a.D + 2;
  for (int i = threadIdx.x; i < rows * pairs; i += 256) {
    const int r = i / pairs, d = 2 * (i - r * pairs);
    float m = kNone;
    for (int w = from; w <= to; ++w) m = fmaxf(m, a.part[((2 * (int64_t)w + (w == from ? 1 : 0)) * tile_rows + r) * stride]);
    float l = 0.0f, x0 = 0.0f, x1 = 0.0f;
    for (int w = from; w <= to; ++w) {
      const float* o = a.part + ((2 * (int64_t)w + (w == from ? 1 : 0)) * tile_rows + r) * stride;
      const float by = __builtin_amdgcn_exp2f(o[0] - m);
      l += o[1] * by;
      x0 += o[2 + d] * by;
      x1 += o[3 + d] * by;
    }
    const int row = tile * tile_rows + r;
    const int t = (int)a.G.of((uint32_t)row), gq = row - t * (int)a.G.d;
    const bool drafted = !a.tree_lengths || t < a.tree_lengths[b];
    const bool none = !drafted || l == 0.0f;
    const float inverse = none ? 0.0f : 1.0f / l;
    const int64_t at = (((int64_t)b * a.H + h) * a.G.d + gq) * a.T + t;
    x0 = none ? 0.0f : x0 * inverse, x1 = none ? 0.0f : x1 * inverse;
    *reinterpret_cast<uint32_t*>(a.out + (at * a.D + d) * 2) = a.bf16 ? pack2<FCR_DTYPE_BF16>(x0, x1) : pack2<FCR_DTYPE_F16>(x0, x1);
    if (a.lse && d == 0) a.lse[at] = none ? -INFINITY : m + __builtin_amdgcn_logf(l);
  }
}
#endif

template <int CD, int W>
void launch_w(const Args& a, int rt, hipStream_t s) {
  const dim3 grid((unsigned)a.wgs);
  switch (rt) {
    case 1: hipLaunchKernelGGL((tree_attention_kernel<CD, W, 1>), grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL((tree_attention_kernel<CD, W, 2>), grid, dim3(kThreads), 0, s, a); break;
  }
}
template <int CD>
void launch(const Args& a, int w, int rt, hipStream_t s) {
  switch (w) {
    case 1: launch_w<CD, 1>(a, rt, s); break;
    case 2: launch_w<CD, 2>(a, rt, s); break;
    case 3: launch_w<CD, 3>(a, rt, s); break;
    default: launch_w<CD, 4>(a, rt, s); break;
  }
}
}  // namespace

#if FCR_HAS(1)
void fcr_tree::attention_f16(const Args& a, int w, int rt, hipStream_t s) { launch<FCR_DTYPE_F16>(a, w, rt, s); }
#endif
#if FCR_HAS(2)
void fcr_tree::attention_bf16(const Args& a, int w, int rt, hipStream_t s) { launch<FCR_DTYPE_BF16>(a, w, rt, s); }
#endif
#if FCR_HAS(3)
void fcr_tree::attention_int8(const Args& a, int w, int rt, hipStream_t s) { launch<FCR_DTYPE_INT8>(a, w, rt, s); }
#endif
#if FCR_HAS(4)
void fcr_tree::attention_e4m3(const Args& a, int w, int rt, hipStream_t s) { launch<FCR_DTYPE_E4M3>(a, w, rt, s); }
#endif

#if FCR_HAS(0)
namespace {
using fcr_detail::fail;
using fcr_detail::launched;

struct Plan {
  int rt, row_tiles, wgs, least;
  int64_t items, first_bytes, bytes;
};
// What depends on sizes alone.  false: too large.
bool plan_of(int B, int H, int G, int T, int D, int64_t capacity, Plan& p) {
  const int64_t rows = (int64_t)T * G;
  p.rt = rows <= 16 ? 1 : 2;
  const int64_t tiles = (rows + 16 * p.rt - 1) / (16 * p.rt);
  p.items = (int64_t)B * H * tiles;
  const int64_t blocks = p.items * ((capacity + kBlock - 1) / kBlock);
  if (rows > (1 << 24) || p.items > (1 << 24) || blocks > (1 << 30)) return false;
  p.row_tiles = (int)tiles;
  int64_t wgs = 2 * (int64_t)fcr_detail::chip_cus_of_current_device();
  if (blocks < wgs) wgs = blocks;
  p.wgs = (int)((wgs + 7) / 8 * 8);
  p.least = 1;
  p.first_bytes = (p.items * 4 + 15) / 16 * 16;
  p.bytes = p.first_bytes + 2ll * p.wgs * 16 * p.rt * (D + 2) * 4;
  return true;
}
}  // namespace

extern "C" {

size_t fcr_tree_attention_bytes(int B, int H, int G, int T, int D, int64_t positions) {
  Plan p;
  if (B < 1 || H < 1 || G < 1 || T < 1 || D < 16 || D > 256 || positions < 1 || positions > (1 << 30) || (int64_t)B * H > (1 << 24)) return 0;
  return plan_of(B, H, G, T, D, positions, p) ? (size_t)p.bytes : 0;
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
  if (G < 1 || T < 1 || T > (1 << 24) || G > (1 << 24) || (int64_t)B * H > (1 << 24) || (int64_t)H * G > (1 << 24) || !plan_of(B, H, G, T, D, capacity, plan))
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
  a.G.set((uint32_t)G);
  a.scale2 = scale * 1.44269504088896340736f;
  a.wgs = plan.wgs, a.least = plan.least;
  const int w = (D + 63) / 64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (cache->dtype) {
    case FCR_DTYPE_F16: attention_f16(a, w, plan.rt, s); break;
    case FCR_DTYPE_BF16: attention_bf16(a, w, plan.rt, s); break;
    case FCR_DTYPE_INT8: attention_int8(a, w, plan.rt, s); break;
    default: attention_e4m3(a, w, plan.rt, s); break;
  }
  if ((rc = launched("tree_attention_kernel"))) return rc;
  hipLaunchKernelGGL(tree_join_kernel, dim3((unsigned)plan.items), dim3(256), 0, s, a, 16 * plan.rt);
  return launched("tree_join_kernel");
}

}  // extern "C"
#endif
