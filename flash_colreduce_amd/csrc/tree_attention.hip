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
// few_attention_kernel (few rows): bound by reading the cache.  Each wave takes 32 keys of a block of 128, from global memory into
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
// was cut are joined by attention_join_kernel, in the order of the keys.

#include "attention.h"

namespace {
template <int CD, int W>
bool launch_w(const Args& a, int form, hipStream_t s) {
  const dim3 grid((unsigned)a.wgs);
  if (form == 1) {
    hipLaunchKernelGGL((few_attention_kernel<Tree, CD, W>), grid, dim3(256), 0, s, a);
  } else if (form == 8) {
    hipLaunchKernelGGL((tall_attention_kernel<CD, W, 8>), grid, dim3(512), 0, s, a);
  } else {
    if constexpr (W > 2) return false;
    else hipLaunchKernelGGL((tall_attention_kernel<CD, W, 4>), grid, dim3(256), 0, s, a);
  }
  return true;
}
// form: see form_of.  false: there is no such kernel
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

namespace fcr_tree {
bool tree_f16(const Args& a, int w, int form, hipStream_t s);
bool tree_bf16(const Args& a, int w, int form, hipStream_t s);
bool tree_int8(const Args& a, int w, int form, hipStream_t s);
bool tree_e4m3(const Args& a, int w, int form, hipStream_t s);
}  // namespace fcr_tree

#if FCR_HAS(1)
bool fcr_tree::tree_f16(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_F16>(a, w, form, s); }
#endif
#if FCR_HAS(2)
bool fcr_tree::tree_bf16(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_BF16>(a, w, form, s); }
#endif
#if FCR_HAS(3)
bool fcr_tree::tree_int8(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_INT8>(a, w, form, s); }
#endif
#if FCR_HAS(4)
bool fcr_tree::tree_e4m3(const Args& a, int w, int form, hipStream_t s) { return launch<FCR_DTYPE_E4M3>(a, w, form, s); }
#endif

#if FCR_HAS(0)
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
  Plan plan;
  Args a = {};
  if (mask && T > 46340) return fail(FCR_E_SHAPE, "a mask of more than 2^31 bytes");
  if ((rc = check_queries(a, plan, q, *cache, table, table_stride, table_pages, context, context_strides, out, lse, ws, ws_bytes, dtype, B, G, T, q_strides, scale,
                          [&](Plan& p) { return plan_of(has_codes(cache->dtype), B, cache->H, G, T, cache->D, (int64_t)table_pages * cache->page_size, p); })))
    return rc;
  if (mask_stride < 0) return fail(FCR_E_STRIDE, "strides must be >= 0");
  a.tree_lengths = tree_lengths;
  a.mask = mask;
  a.mask_b = mask_stride;
  a.scale2 = scale * 1.44269504088896340736f;
  const int w = (cache->D + 63) / 64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  bool there;
  switch (cache->dtype) {
    case FCR_DTYPE_F16: there = fcr_tree::tree_f16(a, w, plan.form, s); break;
    case FCR_DTYPE_BF16: there = fcr_tree::tree_bf16(a, w, plan.form, s); break;
    case FCR_DTYPE_INT8: there = fcr_tree::tree_int8(a, w, plan.form, s); break;
    default: there = fcr_tree::tree_e4m3(a, w, plan.form, s); break;
  }
  if (!there) return fail(FCR_E_SHAPE, "no kernel for these sizes");
  if ((rc = launched("tree attention"))) return rc;
  return join(a, plan, s);
}

}  // extern "C"
#endif
