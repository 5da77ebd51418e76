// Attention of chunks of new tokens over a paged cache of keys and values, quantised or not.
//
// T new tokens of a sequence (a prompt or a part of one, or a single token) stand behind its `context` rows, their keys and values written already.  Token t
// has position i = context + t and sees key j where j <= i and j > i - window, or where j < prefix, of those below context + count.  Its scores are
//   s = scale <q, k_j>,   s = cap tanh(s / cap) with a cap,   s -= slope_h |i - j| with slopes;   o = sum_j 2^(s_j log2(e) - m) v_j / sum_j 2^(s_j log2(e) - m).
//
// The kernels are those of attention.h.  What is different is which keys a tile of rows sees (Sight), two ranges at most, so that blocks that none of its tokens
// sees are neither dealt nor read, a wave leaves out the steps that its own rows do not see, and masks are formed on the borders only; how blocks
// are dealt, since tiles of one sequence have different numbers of them (ChunkDeal); and Bend, behind the products.

#include "attention.h"

namespace {

// What rows [r0, r1) of a (sequence, head) see.
__device__ __forceinline__ Sight view_of(const Args& a, int b, int h, int r0, int r1) {
  return Sight(a.context.of(b, h), a.tree_lengths ? constant_at(a.tree_lengths + b) : a.T, a.prefix ? constant_at(a.prefix + b) : 0, a.window, a.T, a.positions,
               (int)a.G.of((uint32_t)r0), (int)a.G.of((uint32_t)(min(r1, a.rows) - 1)));
}
// Blocks of all items laid end to end, `per` of them for every workgroup, found from the lengths on the device.  A thread adds up the blocks of some consecutive
// (entry, tile) pairs, an entry being a sequence, or one of its heads where these differ in length; all heads of a sequence have the same number S of blocks.  A place
// among the blocks is then found in two steps: its entry, by the place over the number of heads, and the tile, by what is left of the place over S.
template <int THREADS, bool TALL, int ROWS>
struct ChunkDeal {
  int at, end, b, h, tile, blk, nb;
  Sight seen;
  __device__ __forceinline__ bool start(const Args& a, int wg, int* scan) {   // scan: THREADS / 64 + 4 words of LDS
    constexpr int waves = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool by_head = a.context.sh != 0;
    const int entries = by_head ? a.B * a.H : a.B, times = by_head ? 1 : a.H, pairs = entries * a.row_tiles;
    const int each = (pairs + THREADS - 1) / THREADS, p0 = min(tid * each, pairs), p1 = min(p0 + each, pairs);
    const auto blocks_of_pair = [&](int p) {
      const int e = (int)a.per_head.of((uint32_t)p), t = p - e * a.row_tiles;
      int eb = e, eh = 0;
      if (by_head) eb = (int)a.heads.of((uint32_t)e), eh = e - eb * a.H;
      return view_of(a, eb, eh, t * ROWS, t * ROWS + ROWS).blocks();
    };
    int mine = 0;
    for (int p = p0; p < p1; ++p) mine += blocks_of_pair(p);
    const int upto = sum_up_to(mine);
    if (lane == 63) scan[wave] = upto;
    __syncthreads();
    int sum = 0, before = upto - mine;
#pragma unroll
    for (int i = 0; i < waves; ++i) {
      before += i < wave ? scan[i] : 0;
      sum += scan[i];
    }
    const int total = __builtin_amdgcn_readfirstlane(sum) * times, per = (int)a.all.of((uint32_t)(total + a.wgs - 1));
    if (wg == 0 && tid == 0) a.first[0] = per;
    at = wg * per;                                      // (wgs * per is total + wgs at most: checked by the host to fit)
    end = min(at + per, total);
    if (at >= end) return false;
    // the pair that has block x of its entries, and the blocks in front of it
    int* const found = scan + waves;
    const auto find = [&](int x) {
      if (x >= before && x < before + mine) {
        int p = p0, s = before;
        for (int blocks = blocks_of_pair(p); x >= s + blocks; blocks = blocks_of_pair(p)) s += blocks, ++p;
        found[0] = p, found[1] = s;
      }
      __syncthreads();
    };
    find(by_head ? at : (int)a.heads.of((uint32_t)at));
    // (everything found goes through locals to one place: stores on several ways would be joined into one to an address that is chosen, and the deal
    // would stay in memory, where nothing is known to be uniform)
    int pair = __builtin_amdgcn_readfirstlane(found[0]), in_front = __builtin_amdgcn_readfirstlane(found[1]);
    const int entry = (int)a.per_head.of((uint32_t)pair), q0 = entry * a.row_tiles;
    int place = at - times * in_front, head = 0;
    if (a.row_tiles == 1) {
      const int blocks = __builtin_amdgcn_readfirstlane(blocks_of_pair(pair));
      if (!by_head) head = (int)((uint32_t)place / (uint32_t)blocks), place -= head * blocks;
    } else {
      // blocks in front of the entry's pairs and behind them
      const int q1 = q0 + a.row_tiles;
      const auto mark = [&](int q, int to) {
        if (p0 <= q && q < p1) {
          int s = before;
          for (int p = p0; p < q; ++p) s += blocks_of_pair(p);
          found[to] = s;
        } else if (q == pairs && tid == 0) {
          found[to] = sum;
        }
      };
      mark(q0, 2);
      mark(q1, 3);
      __syncthreads();
      const int from = __builtin_amdgcn_readfirstlane(found[2]), blocks = __builtin_amdgcn_readfirstlane(found[3]) - from;
      place = at - times * from;
      if (!by_head) head = (int)((uint32_t)place / (uint32_t)blocks), place -= head * blocks;
      find(from + place);
      pair = __builtin_amdgcn_readfirstlane(found[0]), in_front = __builtin_amdgcn_readfirstlane(found[1]);
      place = from + place - in_front;
    }
    b = by_head ? (int)a.heads.of((uint32_t)entry) : entry;
    h = __builtin_amdgcn_readfirstlane(by_head ? entry - b * a.H : head);
    tile = pair - q0;
    blk = __builtin_amdgcn_readfirstlane(place);
    look(a);
    return true;
  }
  __device__ __forceinline__ void look(const Args& a) {
    seen = view_of(a, b, h, tile * ROWS, tile * ROWS + ROWS);
    nb = seen.blocks();
  }
  __device__ __forceinline__ const Sight& view() const { return seen; }
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
    }
    look(a);
    return true;
  }
};

template <bool BENT>
struct Chunk {
  static constexpr bool bent = BENT, rising = false;
  static constexpr int kScan = 4;
  template <int THREADS, bool TALL, int ROWS>
  using Deal = ChunkDeal<THREADS, TALL, ROWS>;
  static __device__ __forceinline__ bool idle(const Args& a, int b, int row0) {
    return row0 >= a.rows || (a.tree_lengths && (int)a.G.of((uint32_t)row0) >= constant_at(a.tree_lengths + b));
  }
  static __device__ __forceinline__ Sight of_rows(const Args& a, const Sight&, int b, int h, int row0, int rows) {
    return view_of(a, b, h, min(row0, a.rows - 1), row0 + rows);
  }
  static __device__ __forceinline__ uint32_t seen_by(const Args& a, const Sight& v, int, int row, int pos, uint32_t there, int g) {
    asm volatile("" : "+v"(row), "+v"(g));       // (formed here, not kept)
    const int token = row < a.rows ? (int)a.G.of((uint32_t)row) : 0;
    const int back = v.context + token - pos - 4 * g, first = v.prefix - pos - 4 * g;     // of the lane's first key: how far behind the token, in front of the prefix's end
    uint32_t seen = 0;
  #pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 16 * (e / 4) + e % 4;
      seen |= (uint32_t)(back - k) < (uint32_t)a.window || k < first ? 1u << e : 0u;
    }
    return seen & there;
  }
};
}  // namespace

namespace fcr_tree {
bool chunk_f16(const Args& a, int w, int form, hipStream_t s);
bool chunk_bf16(const Args& a, int w, int form, hipStream_t s);
bool chunk_int8(const Args& a, int w, int form, hipStream_t s);
bool chunk_e4m3(const Args& a, int w, int form, hipStream_t s);
}  // namespace fcr_tree

namespace {
template <int CD>
bool launch_chunk(const Args& a, int w, int form, hipStream_t s) {
  return a.cap2 != 0.0f || a.slopes ? launch<Chunk<true>, CD>(a, w, form, s) : launch<Chunk<false>, CD>(a, w, form, s);
}
}  // namespace

#if FCR_HAS(1)
bool fcr_tree::chunk_f16(const Args& a, int w, int form, hipStream_t s) { return launch_chunk<FCR_DTYPE_F16>(a, w, form, s); }
#endif
#if FCR_HAS(2)
bool fcr_tree::chunk_bf16(const Args& a, int w, int form, hipStream_t s) { return launch_chunk<FCR_DTYPE_BF16>(a, w, form, s); }
#endif
#if FCR_HAS(3)
bool fcr_tree::chunk_int8(const Args& a, int w, int form, hipStream_t s) { return launch_chunk<FCR_DTYPE_INT8>(a, w, form, s); }
#endif
#if FCR_HAS(4)
bool fcr_tree::chunk_e4m3(const Args& a, int w, int form, hipStream_t s) { return launch_chunk<FCR_DTYPE_E4M3>(a, w, form, s); }
#endif

#if FCR_HAS(0)
extern "C" {

size_t fcr_chunk_attention_bytes(int B, int H, int G, int T, int D, int64_t positions) {
  Plan p[2];             // for either kind of cache
  if (B < 1 || H < 1 || G < 1 || T < 1 || D < 16 || D > 256 || positions < 1 || positions > (1 << 30) || (int64_t)B * H > (1 << 24)) return 0;
  return plan_of(true, B, H, G, T, D, positions, p[0]) && plan_of(false, B, H, G, T, D, positions, p[1]) ? (size_t)std::max(p[0].bytes, p[1].bytes) : 0;
}

int fcr_chunk_attention(const void* q, const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages,
                        const int32_t* context, const int64_t context_strides[2], const int32_t* counts, const int32_t* prefix, const float* slopes,
                        void* out, float* lse, void* ws, size_t ws_bytes, int dtype, int B, int G, int T, const int64_t q_strides[4], float scale,
                        float cap, int window, void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc) return rc;
  Plan plan;
  Args a = {};
  if (window < 0) return fail(FCR_E_SHAPE, "window must be >= 0");
  if ((rc = check_queries(a, plan, q, *cache, table, table_stride, table_pages, context, context_strides, out, lse, ws, ws_bytes, dtype, B, G, T, q_strides, scale)))
    return rc;
  if (!isfinite(cap) || cap < 0.0f) return fail(FCR_E_SCALE, "cap must be finite and >= 0");
  a.tree_lengths = counts;
  a.prefix = prefix;
  a.slopes = slopes;
  a.window = window ? window : INT32_MAX;
  constexpr float log2e = 1.44269504088896340736f;
  a.cap2 = cap * log2e;
  a.scale2 = cap != 0.0f ? scale * (2.0f * log2e) / cap : scale * log2e;
  if (!isfinite(a.scale2) || !isfinite(a.cap2)) return fail(FCR_E_SCALE, "scale over cap must be finite");
  const int w = (cache->D + 63) / 64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  bool there;
  switch (cache->dtype) {
    case FCR_DTYPE_F16: there = fcr_tree::chunk_f16(a, w, plan.form, s); break;
    case FCR_DTYPE_BF16: there = fcr_tree::chunk_bf16(a, w, plan.form, s); break;
    case FCR_DTYPE_INT8: there = fcr_tree::chunk_int8(a, w, plan.form, s); break;
    default: there = fcr_tree::chunk_e4m3(a, w, plan.form, s); break;
  }
  if (!there) return fail(FCR_E_SHAPE, "no kernel for these sizes");
  if ((rc = launched("chunk attention"))) return rc;
  return join(a, plan, s);
}

}  // extern "C"
#endif
