// Attention of chunks of new tokens over a paged cache of keys and values, quantised or not.
//
// T new tokens of a sequence (a prompt or a part of one, or a single token) stand behind its `context` rows, their keys and values written already.  Token t
// has position i = context + t and sees key j where j <= i and j > i - window, or where j < prefix, of those below context + count.  Its scores are
//   s = scale <q, k_j>,   s = cap tanh(s / cap) with a cap,   s -= slope_h |i - j| with slopes;   o = sum_j 2^(s_j log2(e) - m) v_j / sum_j 2^(s_j log2(e) - m).
//
// The kernels are those of attention.h.  What is different is which keys a tile of rows sees (Sight), two ranges at most, so that blocks that none of its tokens
// sees are neither dealt nor read, a wave leaves out the steps that its own rows do not see, and masks are formed on the borders only; how blocks
// are dealt, since tiles of one sequence have different numbers of them (ChunkDeal); and Bend, behind the products.
//
// few_attention_kernel: one token of 48 sequences over 8 heads of up to 4096 e4m3 keys of 128 elements, 4 queries each, capped: 70 us, 4.4 TB/s; two chunks of 17 tokens,
// 4 heads of 2 queries, behind up to 300 fp16 keys of 64 elements with slopes: 7.6 us, one launch and a chain of loads: lengths, table, keys.
// chunk_attention_kernel, bound by vector and matrix instructions of two waves to a SIMD that run next to each other for a fifth of the time: a prompt of 8192 tokens, 8 heads of
// 8 queries, fp16, 128 elements: 1163 us, 946 TFLOP/s; 4 chunks of 512 behind 8192 keys, 8 heads of 4: 295 us, 955 TFLOP/s; two biased bf16 prompts of up to 4096 tokens,
// 16 heads: 132 to 204 us by the drawn lengths; two of 2048 behind up to 16384 keys of 96 fp16 elements that see 1024 and a prefix of 64: 77 us.

#include "attention.h"

namespace {

// What rows [r0, r1) of a (sequence, head) see.
__device__ __forceinline__ Sight view_of(const Args& a, int b, int h, int r0, int r1) {
  return Sight(a.context.of(b, h), a.tree_lengths ? constant_at(a.tree_lengths + b) : a.T, a.prefix ? constant_at(a.prefix + b) : 0, a.window, a.T, a.positions,
               (int)a.G.of((uint32_t)r0), (int)a.G.of((uint32_t)(min(r1, a.rows) - 1)));
}
// Blocks of all items laid end to end, each item behind some places for what runs once (once_of), `per` places for every workgroup, found from the lengths on the device; or
// items taken whole.  A thread adds up the blocks of some consecutive
// (entry, tile) pairs, an entry being a sequence, or one of its heads where these differ in length; all heads of a sequence have the same number S of places.  A place
// is then found in two steps: its entry, by the place over the number of heads, and the tile, by what is left of the place over S.
template <int THREADS, int ROWS>
struct ChunkDeal {
  int at, end, b, h, tile, blk, nb, once;
  Sight seen;
  // `at` and `end` are places; the piece is of blocks [blk, stop()) of the item's nb.
  // What is found goes through locals to one place: stores on several ways would be joined into one to an address that is chosen, and the deal would stay in
  // memory, where nothing is known to be uniform.
  struct Found {
    int at, end, b, h, tile, blk;     // blk: the place in the item; end below 0: it is taken whole
    int once;
    bool any;
  };
  // An item for this workgroup of a launch of one for each: the last tiles, which see the most keys, first, and tiles of one head on one die (workgroups are
  // dealt to 8 dies in turn) where the number of heads is a multiple of 8.
  static __device__ __forceinline__ Found one(const Args& a) {
    const int rank = (int)a.all_heads.of(blockIdx.x), bh = blockIdx.x - rank * a.all_heads.d, b = (int)a.heads.of((uint32_t)bh);
    return Found{0, -1, b, bh - b * a.H, a.row_tiles - 1 - rank, 0, 0, rank < a.row_tiles};
  }
  __device__ __forceinline__ bool start(const Args& a, int wg, int* scan) {   // scan: THREADS / 64 + 4 words of LDS and, where a.whole is 1, THREADS / 64 more
    const Found f = a.whole == 2 ? one(a) : dealt(a, wg, scan);
    if (!f.any) return false;
    b = __builtin_amdgcn_readfirstlane(f.b), h = __builtin_amdgcn_readfirstlane(f.h), tile = __builtin_amdgcn_readfirstlane(f.tile);
    blk = __builtin_amdgcn_readfirstlane(f.blk), at = __builtin_amdgcn_readfirstlane(f.at), once = __builtin_amdgcn_readfirstlane(f.once);
    look(a);
    const int last = __builtin_amdgcn_readfirstlane(f.end);
    end = last < 0 ? nb : last;
    const int skipped = max(once - blk, 0);
    at += skipped, blk += skipped - once;
    return at < end;                                    // (else the next workgroup has the first part of this item)
  }
  static __device__ __forceinline__ Found dealt(const Args& a, int wg, int* scan) {
    constexpr int waves = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool by_head = a.context.sh != 0;
    const int entries = by_head ? a.B * a.H : a.B, times = by_head ? 1 : a.H, pairs = entries * a.row_tiles;
    const int each = (pairs + THREADS - 1) / THREADS, p0 = min(tid * each, pairs), p1 = min(p0 + each, pairs);
    int once = 0;
    const auto weight_of_pair = [&](int p) {
      const int e = (int)a.per_head.of((uint32_t)p), t = p - e * a.row_tiles;
      int eb = e, eh = 0;
      if (by_head) eb = (int)a.heads.of((uint32_t)e), eh = e - eb * a.H;
      return view_of(a, eb, eh, t * ROWS, t * ROWS + ROWS).blocks() + once;
    };
    int mine = 0, most = 0;
    for (int p = p0; p < p1; ++p) {
      const int blocks = weight_of_pair(p);
      mine += blocks, most = max(most, blocks);
    }
    int before, sum;                                    // in front of this thread's, and all
    const auto add_up = [&](int x) {
      const int upto = sum_up_to(x);
      if (lane == 63) scan[wave] = upto;
      __syncthreads();
      sum = 0, before = upto - x;
#pragma unroll
      for (int i = 0; i < waves; ++i) {
        before += i < wave ? scan[i] : 0;
        sum += scan[i];
      }
    };
    if (a.whole) {
      for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o));
      if (lane == 63) scan[waves + 4 + wave] = most;
    }
    add_up(mine);
    int total = __builtin_amdgcn_readfirstlane(sum) * times, per = (int)a.all.of((uint32_t)(total + a.wgs - 1));
    const int more = once_of(per, ROWS != 16), weights = total + more * pairs * times, each_weight = (int)a.all.of((uint32_t)(weights + a.wgs - 1));
    if (wg == 0 && tid == 0) a.first[0] = each_weight;
    if (a.whole) {
#pragma unroll
      for (int i = 0; i < waves; ++i) most = max(most, scan[waves + 4 + i]);
      if (items_are_whole(__builtin_amdgcn_readfirstlane(most) + more, each_weight, pairs * times, a.wgs, ROWS != 16)) return one(a);
      if (blockIdx.x >= (unsigned)a.wgs) return Found{0, 0, 0, 0, 0, 0, 0, false};
    }
    if (ROWS == 16 && a.row_tiles == 1 && pieces_are_tried(entries, THREADS, per, 1, false)) {
      // Pieces of one item each, as in tree_attention.
      const int blocks = mine;
      const int longest = most_of(per, most_allowed(per, 1, false), [&](int p) {
        mine = tid < entries ? pieces_of(blocks, p) : 0;
        __syncthreads();
        add_up(mine);
        return __builtin_amdgcn_readfirstlane(sum) * times <= a.wgs;
      });
      if (longest) {
        if (wg == 0 && tid == 0) a.first[0] = longest;
        if (wg >= __builtin_amdgcn_readfirstlane(sum) * times) return Found{0, 0, 0, 0, 0, 0, 0, false};
        int* const found = scan + waves;
        const int x = by_head ? wg : (int)a.heads.of((uint32_t)wg);
        if (x >= before && x < before + mine) found[0] = tid, found[1] = before, found[2] = blocks;
        __syncthreads();
        const int entry = __builtin_amdgcn_readfirstlane(found[0]), nb = __builtin_amdgcn_readfirstlane(found[2]), pieces = pieces_of(nb, longest);
        int piece = wg - times * __builtin_amdgcn_readfirstlane(found[1]), head = 0;
        if (!by_head) head = (int)((uint32_t)piece / (uint32_t)pieces), piece -= head * pieces;
        const int length = piece_length(nb, pieces), b = by_head ? (int)a.heads.of((uint32_t)entry) : entry;
        return Found{0, least_of(length, nb - piece * length), b, by_head ? entry - b * a.H : head, 0, piece * length, 0, true};
      }
      mine = blocks;
      __syncthreads();
      add_up(mine);
    }
    once = more, per = each_weight, total = weights;
    before += once * p0, mine += once * (p1 - p0), sum += once * pairs;
    const int at = wg * per, end = min(at + per, total);   // (wgs * per is total + wgs at most: checked by the host to fit)
    if (at >= end) return Found{0, 0, 0, 0, 0, 0, 0, false};
    // the pair that has place x of its entries, and the places in front of it
    int* const found = scan + waves;
    const auto find = [&](int x) {
      if (x >= before && x < before + mine) {
        int p = p0, s = before;
        for (int weight = weight_of_pair(p); x >= s + weight; weight = weight_of_pair(p)) s += weight, ++p;
        found[0] = p, found[1] = s;
      }
      __syncthreads();
    };
    find(by_head ? at : (int)a.heads.of((uint32_t)at));
    int pair = __builtin_amdgcn_readfirstlane(found[0]), in_front = __builtin_amdgcn_readfirstlane(found[1]);
    const int entry = (int)a.per_head.of((uint32_t)pair), q0 = entry * a.row_tiles;
    int place = at - times * in_front, head = 0;
    if (a.row_tiles == 1) {
      const int weight = __builtin_amdgcn_readfirstlane(weight_of_pair(pair));
      if (!by_head) head = (int)((uint32_t)place / (uint32_t)weight), place -= head * weight;
    } else {
      // places in front of the entry's pairs and behind them
      const int q1 = q0 + a.row_tiles;
      const auto mark = [&](int q, int to) {
        if (p0 <= q && q < p1) {
          int s = before;
          for (int p = p0; p < q; ++p) s += weight_of_pair(p);
          found[to] = s;
        } else if (q == pairs && tid == 0) {
          found[to] = sum;
        }
      };
      mark(q0, 2);
      mark(q1, 3);
      __syncthreads();
      const int from = __builtin_amdgcn_readfirstlane(found[2]), weight = __builtin_amdgcn_readfirstlane(found[3]) - from;
      place = at - times * from;
      if (!by_head) head = (int)((uint32_t)place / (uint32_t)weight), place -= head * weight;
      find(from + place);
      pair = __builtin_amdgcn_readfirstlane(found[0]), in_front = __builtin_amdgcn_readfirstlane(found[1]);
      place = from + place - in_front;
    }
    const int b = by_head ? (int)a.heads.of((uint32_t)entry) : entry;
    return Found{at, end, b, by_head ? entry - b * a.H : head, pair - q0, place, once, true};
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
    at += stop() - blk + once;
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

template <int BENT>
struct Chunk {
  static constexpr int bent = BENT;
  static constexpr bool rising = false;
  static constexpr int kScan = 8;
  template <int THREADS>
  using Deal = ChunkDeal<THREADS, 16>;
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
// Many rows: the scheme of tall_attention_kernel (attention.h), two stages of keys in LDS, converted by all waves; a wave has 16 RT rows, of which it leaves out the
// steps that none sees.  What a step costs beside its products and weights is kept small, since it is the vector and scalar instructions of two waves that a SIMD
// spends its time on: a step is a slot of a ring in LDS at one address, what the wave sees of it follows from one number that falls by 32 (Steps), and what is used once per
// stage is formed there from the arguments.
template <int BENT, int CD, int W, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) chunk_attention_kernel(Args args) {
  using F = Form<CD, W>;
  constexpr int RT = tall_tiles(W), kKeys = tall_keys(W, WAVES), kSteps = kKeys / 32, kTiles = kKeys / 16, kStepsLog2 = kSteps == 4 ? 2 : 1;
  constexpr int kMine = kTiles > WAVES ? kTiles / WAVES : 1;             // 16-key tiles that a wave converts
  constexpr bool kApart = kTiles < WAVES;                                // a wave converts a tile's keys or its values
  constexpr int kValues = 2 * F::KS * 64, kStep = kValues + F::DT * 64;  // where a step's values begin, and the next step, in 16 bytes
  constexpr int kRing = 2 * kSteps;                                      // steps in LDS
  // Rows of 256 elements leave no registers for both halves of a step's values, or for keys next to them.
  constexpr bool kLean = W == 4;
  // Stages that all rows see run through straight-line code in which the products of values of a step stand between the vector instructions of the next step's weights.  4 x 8
  // heads of 4 queries, 512 tokens behind 8192 keys, us without and with it: 64 elements, int8 306, 272, fp16 282, 235; 128 elements of 16 bits 3 to 6 % less with it, but codes of
  // 128 8 to 12 % more: what converts them takes the registers that hold operands ahead, as rows of more elements do.
  constexpr bool kPiped = W == 1 || (W == 2 && !F::codes);
  constexpr int kEarly = W == 1 || (W == 2 && F::codes) ? F::DT : F::DT / 2;                     // value operands that fit next to the weights
  static_assert(kTiles * (kApart ? 2 : 1) == WAVES * kMine, "every wave has its share of a stage");
  __shared__ u32x4 operands[kRing * kStep];
  __shared__ __attribute__((aligned(16))) float scales[kRing][2][32];    // of keys, of values
  __shared__ float most[kRing][2];                                       // the largest scale of a tile's values
  __shared__ __attribute__((aligned(16))) int2 flags[kRing];             // a tile's page is there, and (bit 1) one of its values was not finite
  __shared__ float rest[WAVES][RT][16];                                  // powers of two that rows' scores are still to be multiplied by
  __shared__ int scan[2 * WAVES + 4];
  const int wg = range_of(args, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Lane<F> at(threadIdx.x & 63);
  const int my_tile = kApart ? wave % kTiles : wave * kMine;
  const bool my_keys = !kApart || wave < kTiles, my_values = !kApart || wave >= kTiles;
  ChunkDeal<64 * WAVES, 16 * RT * WAVES> deal;
  if (!deal.start(arguments(), wg, scan)) return;
  do {
    const int b = deal.b, h = deal.h, D = arguments().D;
    const Sight view = deal.view();
    const int n = view.n;
    const int row0 = (deal.tile * WAVES + wave) * 16 * RT;
    const bool late = WAVES == 8 && wave >= 4;
    // (a wave without rows converts all the same)
    const Steps sees(view_of(arguments(), b, h, min(row0, arguments().rows - 1), row0 + 16 * RT), view, row0 < arguments().rows);
    Keys<F> k[kMine];
    Values<F> v[kMine];
    // (formed from the arguments where it is used: it would take 25 scalar registers of all loops)
    const auto source = [&]() { return Source(arguments(), b, h, n); };
    Place place[kMine], ahead[kMine];                                    // of the rows loaded last, and of the next ones
    const int steps = (deal.stop() - deal.blk) * (kBlock / 32), stages = steps / kSteps;
    const int x0 = (deal.nb - deal.blk) * kBlock - 32;                   // of the first step: the last keys are taken first
    const auto x_of = [&](int stage, int t) { return x0 - 32 * (stage * kSteps + (my_tile + t) / 2) + 16 * ((my_tile + t) & 1); };
    const auto look = [&](const Source& src, int stage) {
#pragma unroll
      for (int t = 0; t < kMine; ++t) ahead[t] = Place(src, view.key(x_of(stage, t)));
    };
    const auto fetch = [&](int stage) {
      const Source src = source();
      const Lane<F> here = at.again();
#pragma unroll
      for (int t = 0; t < kMine; ++t) {
        place[t] = ahead[t];
        if (my_keys) k[t].template load<false>(src, D, place[t], here);
        if (my_values) v[t].load(src, D, place[t], here);
      }
      look(src, stage + 1);
    };
    Queries<F, RT> q;
    float by = arguments().scale2;
    q.load(arguments(), b, h, row0, at);
    look(source(), 0);
    fetch(0);
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
    Bend<RT, BENT> bend;
    if constexpr (BENT) bend.load(arguments(), h, row0, view.context, at.col);
    State<F, RT> st;
    st.clear();
    const auto convert = [&](int stage) {
      const int pages = arguments().c.pages;
#pragma unroll
      for (int t = 0; t < kMine; ++t) {
        const int x = x_of(stage, t), slot = (stage * kSteps + (my_tile + t) / 2) & (kRing - 1), half = (my_tile + t) & 1;
        u32x4* const to = operands + slot * kStep + at.lane;
        float* const sc = scales[slot][0] + 16 * half;
        const int pos = view.key(x);
        int flag = (uint32_t)place[t].page < (uint32_t)pages ? 1 : 0;
        if (my_values && (!flag || !view.whole(pos, 16))) {
          v[t].drop(there_of(pos, n, flag, flag, at.g));
          if constexpr (!F::finite) flag |= __any(v[t].clean()) ? 2 : 0;
        }
        if (my_keys) {
#pragma unroll
          for (int c = 0; c < F::KS; ++c) to[(half * F::KS + c) * 64] = k[t].operand(c);
          if constexpr (!F::codes) {
            // What lies behind the rows becomes zeros here (see tall_attention_kernel).
            if (__builtin_expect(D % 64 != 0, 0)) {
              const Lane<F> here = at.again();
              uint32_t zero = 0;
              asm volatile("" : "+v"(zero));       // (formed here, not kept)
#pragma unroll
              for (int c = F::KS - 2; c < F::KS; ++c)
                if (here.behind(c, D)) to[(half * F::KS + c) * 64] = u32x4{zero, zero, zero, zero};
            }
          }
          if (F::codes && at.col == 0) *reinterpret_cast<f32x4*>(sc + 4 * at.g) = k[t].scale * by;
        }
        if (my_values) {
          if constexpr (F::codes) {
            if (at.col == 0) *reinterpret_cast<f32x4*>(sc + 32 + 4 * at.g) = v[t].scale;
            const f32x4 x = v[t].scale;
            const float m = across(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))), true);
            if (at.lane == 0) most[slot][half] = fmaxf(m, 0.0f);   // (a NaN does not count)
          }
          if (at.lane == 0) reinterpret_cast<int*>(flags + slot)[half] = flag;
          if constexpr (kMine == 1) {
#pragma unroll
            for (int d = 0; d < F::DT; ++d) reinterpret_cast<u32x2*>(to + kValues + d * 64)[half] = v[0].operand(d);
          } else if (t & 1) {
#pragma unroll
            for (int d = 0; d < F::DT; ++d) to[kValues + d * 64] = joined_operand(v[t - 1].operand(d), v[t].operand(d));
          }
        }
      }
    };
    // What a step reads from LDS is read ahead: keys, scales and flags under the products of the step before, values under the weights.
    // (Left to itself the scheduler reads each operand in front of its use, to save registers, and waits for it.)
    f32x4 s[RT][2], k_scale[2], v_scale[2];
    u32x4 kf[2][F::KS];
    float most_v = 1.0f;
    int2 flag;
    const auto slot_of = [&](int i) { return operands + (i & (kRing - 1)) * kStep + at.lane; };
    const auto read_keys = [&](int i, int t) {
      const u32x4* const from = slot_of(i) + t * F::KS * 64;
#pragma unroll
      for (int c = 0; c < F::KS; ++c) kf[t][c] = from[c * 64];
    };
    const auto read_scales = [&](int i) {
      const int slot = i & (kRing - 1);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (F::codes) {
          const float* const sc = scales[slot][0] + 16 * t + 4 * at.g;
          k_scale[t] = *reinterpret_cast<const f32x4*>(sc);
          v_scale[t] = *reinterpret_cast<const f32x4*>(sc + 32);
        } else {
          k_scale[t] = f32x4{by, by, by, by};
          v_scale[t] = f32x4{1, 1, 1, 1};
        }
      }
      flag = flags[slot];
      if constexpr (F::codes) most_v = fmaxf(most[slot][0], most[slot][1]);
    };
    const auto products_of = [&](int t) {                                // of the keys read last with the queries
#pragma unroll
      for (int c = 0; c < F::KS; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][t] = mma<F::bf16>(kf[t][c], q.w[r][c], c ? s[r][t] : f32x4{0, 0, 0, 0});
    };
    // What rows see of the step at x, forms weights of its products s, and adds what is not finite of its values.
    const auto weigh_step = [&](int i, int x, u32x4 (&p)[RT]) {
      read_scales(i);
      const int f0 = __builtin_amdgcn_readfirstlane(flag.x), f1 = __builtin_amdgcn_readfirstlane(flag.y);
      const bool masked = !sees.whole(x) || ((f0 ^ 1) | (f1 ^ 1)) != 0;
      uint32_t seen[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) seen[r] = 0xff;
      if (__builtin_expect(masked, 0)) {
        const Lane<F> here = at.again();
        const int pos = view.key(x);
        const uint32_t there = there_of(pos, n, f0 & 1, f1 & 1, here.g);
        const Sight rows = view_of(arguments(), b, h, row0, row0 + 16 * RT);
#pragma unroll
        for (int r = 0; r < RT; ++r) seen[r] = Chunk<BENT>::seen_by(arguments(), rows, b, row0 + 16 * r + here.col, pos, there, here.g);
      }
      if (F::codes && __builtin_expect(apart, 0)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float by_row = rest[wave][r][at.col];
#pragma unroll
          for (int t = 0; t < 2; ++t) s[r][t] = s[r][t] * by_row;
        }
      }
      if constexpr (BENT) bend.of(k_scale, view.key(x), at.g, s);
      weigh<F, RT>(k_scale, v_scale, most_v, s, masked, seen, st, p);
      if constexpr (!F::finite) {
        if (__builtin_expect(((f0 | f1) & 2) != 0, 0)) add_not_finite<F, RT>(source(), D, view.key(x), p, seen, at, st);
      }
    };
    if constexpr (kPiped) {
      // Arrays are declared where they are read from LDS, without a condition: one that might hold an earlier turn's values would take its registers everywhere.
      const bool none = (sees.high | sees.prefix) == 0;
      u32x4 p[RT];
      const auto read_values = [&](int i, u32x4 (&vf)[F::DT]) {
        const u32x4* const from = slot_of(i) + kValues;
#pragma unroll
        for (int d = 0; d < F::DT; ++d) vf[d] = from[d * 64];
      };
      const auto keys = [&](int i, int t, u32x4 (&kf)[F::KS]) {
        const u32x4* const from = slot_of(i) + t * F::KS * 64;
#pragma unroll
        for (int c = 0; c < F::KS; ++c) kf[c] = from[c * 64];
      };
      const auto products = [&](const u32x4 (&kf)[2][F::KS]) {
#pragma unroll
        for (int c = 0; c < F::KS; ++c)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][t] = mma<F::bf16>(kf[t][c], q.w[r][c], c ? s[r][t] : f32x4{0, 0, 0, 0});
      };
      const auto next_stage = [&](int stage) {
        if (stage + 1 >= stages) return;
        convert(stage + 1);
        if (stage + 2 < stages) fetch(stage + 2);
      };
#pragma unroll
      for (int r = 0; r < RT; ++r) p[r] = u32x4{0, 0, 0, 0};
      bool live = false, fast = false;                   // p are weights; all rows see all of the stage
      for (int stage = -1; stage < stages; ++stage) {
        const int i0 = stage * kSteps;
        int x = x0 - 32 * i0;
        if (stage >= 0) {
          if (!late) next_stage(stage);
          if (__builtin_expect(fast, 1)) {
            u32x4 kf[2][F::KS], vf[F::DT];
            keys(i0 + 1, 0, kf[0]);
            keys(i0 + 1, 1, kf[1]);
            read_scales(i0 + 1);
            read_values(i0, vf);
#pragma unroll
            for (int j = 0; j < kSteps - 1; ++j) {
              float sum[RT];
              u32x4 following[RT];
              products(kf);
              __builtin_amdgcn_sched_barrier(0);
              if constexpr (BENT) bend.of(k_scale, view.key(x - 32 * (j + 1)), at.g, s);
              // A part of the products of values for each row tile: they run under the vector instructions of its weights.  Keys come as values go.
              bool up = false;
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const bool up_r = weights_of_row<false, F>(k_scale, v_scale, most_v, s[r], 0xff, st.m[r], st.l[r], sum[r], following[r]);
                up = up || up_r;
#pragma unroll
                for (int d = r * F::DT / RT; d < (r + 1) * F::DT / RT; ++d)
#pragma unroll
                  for (int i = 0; i < RT; ++i) st.o[i][d] = mma<F::bf16>(vf[d], p[i], st.o[i][d]);
#pragma unroll
                for (int k = 0; k < F::DT; ++k) {
                  __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                  __builtin_amdgcn_sched_group_barrier(0x2, 5, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (j + 2 < kSteps) keys(i0 + j + 2, r, kf[r]);
                __builtin_amdgcn_sched_barrier(0);
              }
              if (__builtin_expect(__any(up), 0)) {
                uint32_t seen[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) seen[r] = 0xff;
                raise<F, RT>(k_scale, v_scale, s, seen, st);
                weights<true, F, RT>(k_scale, v_scale, most_v, s, seen, st, sum, following);
              }
#pragma unroll
              for (int r = 0; r < RT; ++r) st.l[r] = sum[r], p[r] = following[r];
              if (j + 2 < kSteps) {
                read_scales(i0 + j + 2);
                read_values(i0 + j + 1, vf);
              }
            }
          } else if (!none) {
#pragma unroll 1
            for (int j = 0; j < kSteps - 1; ++j) {
              if (live) {
                u32x4 vf[F::DT];
                read_values(i0 + j, vf);
                add_values<F, RT, 0, F::DT>(vf, p, st);
              }
              live = sees.some(x - 32 * (j + 1));
              if (live) {
                u32x4 kf[2][F::KS];
                keys(i0 + j + 1, 0, kf[0]);
                keys(i0 + j + 1, 1, kf[1]);
                products(kf);
                weigh_step(i0 + j + 1, x - 32 * (j + 1), p);
              }
            }
          }
        }
        if (late || stage < 0) next_stage(stage);
        u32x4 vf[F::DT], kf[2][F::KS];
        read_values(i0 + kSteps - 1, vf);                   // (behind the barrier their place is written)
        __syncthreads();
        if (none) continue;
        keys(i0 + kSteps, 0, kf[0]);
        keys(i0 + kSteps, 1, kf[1]);
        if (live) add_values<F, RT, 0, F::DT>(vf, p, st);
        if (stage + 1 == stages) break;
        x -= 32 * kSteps;
        live = sees.some(x), fast = false;
        if (!live) continue;
        products(kf);
        const u32x4* const f = reinterpret_cast<const u32x4*>(flags + ((i0 + kSteps) & (kRing - 1)));
        u32x4 odd = f[0] ^ 1;
#pragma unroll
        for (int k = 1; k < kSteps / 2; ++k) odd |= f[k] ^ 1;
        weigh_step(i0 + kSteps, x, p);
        fast = sees.whole(x, x - 32 * (kSteps - 1)) && !apart && __builtin_amdgcn_readfirstlane((int)(odd[0] | odd[1] | odd[2] | odd[3])) == 0;
      }
    } else {
      // (in the loop: the step before the first one does this, with values and weights of 0)
      int x = x0 + 32;
      bool next = sees.some(x);
      for (int i = -1; i < steps; ++i, x -= 32) {
        const int stage = i >> kStepsLog2, j = i & (kSteps - 1);
        const bool work = next && i >= 0;
        next = i + 1 < steps && sees.some(x - 32);
        const bool run = work || next;                     // (rows that see nothing of this step may need the products of the next one)
        u32x4 vf[F::DT], p[RT];
        if (work) {
          const u32x4* const from = slot_of(i) + kValues;
#pragma unroll
          for (int d = 0; d < kEarly; ++d) vf[d] = from[d * 64];
          weigh_step(i, x, p);
        } else {
#pragma unroll
          for (int d = 0; d < F::DT; ++d) vf[d] = u32x4{0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < RT; ++r) p[r] = u32x4{0, 0, 0, 0};
        }
        if ((i < 0 || j == (late ? kSteps / 2 : 0)) && stage + 1 < stages) {
          convert(stage + 1);
          if (stage + 2 < stages) fetch(stage + 2);
        }
        const auto read_values = [&](int from_d) {
          const u32x4* const from = slot_of(i) + kValues;
#pragma unroll
          for (int d = 0; d < F::DT / 2; ++d) vf[from_d + d] = from[(from_d + d) * 64];
        };
        if constexpr (kLean) {
          if (work) {
            add_values<F, RT, 0, F::DT / 2>(vf, p, st);
            read_values(F::DT / 2);
            add_values<F, RT, F::DT / 2, F::DT>(vf, p, st);
          }
          if (j == kSteps - 1) __syncthreads();
          if (run) {
            read_keys(i + 1, 0);
            read_keys(i + 1, 1);
          }
        } else {
          if (kEarly < F::DT && work) read_values(F::DT / 2);                // (before the barrier: the stage's place is written behind it)
          if (j == kSteps - 1) __syncthreads();
          if (run) {
            __builtin_amdgcn_s_setprio(1);
            if (kEarly == F::DT) read_keys(i + 1, 0);
            __builtin_amdgcn_sched_barrier(0);
            add_values<F, RT, 0, F::DT / 2>(vf, p, st);
            __builtin_amdgcn_sched_barrier(0);
            read_keys(i + 1, kEarly == F::DT ? 1 : 0);
            __builtin_amdgcn_sched_barrier(0);
            add_values<F, RT, F::DT / 2, F::DT>(vf, p, st);
            __builtin_amdgcn_sched_barrier(0);
            if (kEarly < F::DT) read_keys(i + 1, 1);
          }
        }
        if (run) {
          products_of(0);
          products_of(1);
          __builtin_amdgcn_s_setprio(0);
        }
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
        const Output out(a, b, h, row, l);
        const float inverse = 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[F::DT];
#pragma unroll
          for (int d = 0; d < F::DT; ++d) x[d] = st.o[r][d][i];
          emit<F>(a, out, Lane<F>::elements_of(a.D, 4 * at.g + i), x, inverse);
        }
        if (a.lse && at.g == 0) a.lse[out.row] = out.none ? -INFINITY : st.m[r] + __builtin_amdgcn_logf(l) + (BENT ? left_off(a) : 0.0f);
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

// form: see form_of.  false: there is no such kernel
template <int BENT, int CD, int W>
bool launch_chunk(const Args& a, int form, hipStream_t s) {
  const dim3 grid((unsigned)(a.whole ? std::max(a.wgs, a.B * a.H * a.row_tiles) : a.wgs));
  if (form == 1) {
    hipLaunchKernelGGL((few_attention_kernel<Chunk<BENT>, CD, W>), grid, dim3(256), 0, s, a);
  } else if (form == 8) {
    hipLaunchKernelGGL((chunk_attention_kernel<BENT, CD, W, 8>), grid, dim3(512), 0, s, a);
  } else {
    if constexpr (W > 2) return false;
    else hipLaunchKernelGGL((chunk_attention_kernel<BENT, CD, W, 4>), grid, dim3(256), 0, s, a);
  }
  return true;
}
template <int BENT, int CD>
bool launch_chunk(const Args& a, int w, int form, hipStream_t s) {
  switch (w) {
    case 1: return launch_chunk<BENT, CD, 1>(a, form, s);
    case 2: return launch_chunk<BENT, CD, 2>(a, form, s);
    case 3: return launch_chunk<BENT, CD, 3>(a, form, s);
    default: return launch_chunk<BENT, CD, 4>(a, form, s);
  }
}
template <int CD>
bool launch_chunk(const Args& a, int w, int form, hipStream_t s) {
  return a.slopes ? launch_chunk<2, CD>(a, w, form, s) : a.cap2 != 0.0f ? launch_chunk<1, CD>(a, w, form, s) : launch_chunk<0, CD>(a, w, form, s);
}
}  // namespace

namespace fcr_tree {
bool chunk_f16(const Args& a, int w, int form, hipStream_t s);
bool chunk_bf16(const Args& a, int w, int form, hipStream_t s);
bool chunk_int8(const Args& a, int w, int form, hipStream_t s);
bool chunk_e4m3(const Args& a, int w, int form, hipStream_t s);
}  // namespace fcr_tree

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
namespace {
// Workgroups of few_attention_kernel in a launch for each CU, where not as many as tree_attention takes: rows of 64 elements leave registers for three and more.  One token
// of 16 sequences over 8 heads of 8192 e4m3 keys of 64 elements, 4 queries each: 39 us with two, 37 with three, 41 with four; of 128 elements 8 x 8 heads of 16384 keys 55 and
// 57 with three.
int few_per_cu(int D) { return D <= 64 ? 3 : 0; }
int64_t most_blocks(const Plan& p, int64_t positions, int window, int G) { return most_blocks_of(positions, window, p.tile_rows, G); }
bool few_rows(const Plan& p, int64_t longest) { return takes_few_rows(p.items, p.held, longest); }
bool half_tiles(const Plan& p, int64_t longest, int D, int64_t positions, int T) { return takes_half_tiles(p.items, p.held, longest, D, positions, T); }
bool chunk_plan(bool codes, int B, int H, int G, int T, int D, int64_t positions, int window, Plan& p) {
  if (plan_of(codes, B, H, G, T, D, positions, p, few_per_cu(D), 1) && few_rows(p, most_blocks(p, positions, window, G))) return true;
  if (D <= 128 && (int64_t)T * G > 128 && plan_of(codes, B, H, G, T, D, positions, p, 0, 4) && half_tiles(p, most_blocks(p, positions, window, G), D, positions, T)) return true;
  return plan_of(codes, B, H, G, T, D, positions, p, few_per_cu(D));
}
// Of any of them, whatever the window is.
int64_t chunk_bytes(bool codes, int B, int H, int G, int T, int D, int64_t positions) {
  Plan p;
  if (!plan_of(codes, B, H, G, T, D, positions, p, few_per_cu(D))) return 0;
  int64_t bytes = p.bytes;
  if (plan_of(codes, B, H, G, T, D, positions, p, few_per_cu(D), 1) && few_rows(p, 1)) bytes = std::max(bytes, p.bytes);
  if (D <= 128 && (int64_t)T * G > 128 && plan_of(codes, B, H, G, T, D, positions, p, 0, 4) && half_tiles(p, 1, D, positions, T)) bytes = std::max(bytes, p.bytes);
  return bytes;
}
}  // namespace

extern "C" {

size_t fcr_chunk_attention_bytes(int B, int H, int G, int T, int D, int64_t positions) {
  if (B < 1 || H < 1 || G < 1 || T < 1 || D < 16 || D > 256 || positions < 1 || positions > (1 << 30) || (int64_t)B * H > (1 << 24)) return 0;
  const int64_t codes = chunk_bytes(true, B, H, G, T, D, positions), others = chunk_bytes(false, B, H, G, T, D, positions);   // for either kind of cache
  return codes && others ? (size_t)std::max(codes, others) : 0;
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
  const int64_t positions = (int64_t)table_pages * cache->page_size;
  if ((rc = check_queries(a, plan, q, *cache, table, table_stride, table_pages, context, context_strides, out, lse, ws, ws_bytes, dtype, B, G, T, q_strides, scale,
                          [&](Plan& p) { return chunk_plan(has_codes(cache->dtype), B, cache->H, G, T, cache->D, positions, prefix ? 0 : window, p); })))
    return rc;
  if (!isfinite(cap) || cap < 0.0f) return fail(FCR_E_SCALE, "cap must be finite and >= 0");
  a.tree_lengths = counts;
  a.prefix = prefix;
  a.slopes = slopes;
  a.window = window ? window : INT32_MAX;
  constexpr float log2e = 1.44269504088896340736f;
  a.cap2 = cap * log2e;
  a.scale2 = cap != 0.0f && a.cap2 <= kWideCap ? scale * (2.0f * log2e) / cap : scale * log2e;
  if (!isfinite(a.cap2)) return fail(FCR_E_SCALE, "cap in base 2 (1.4427 cap) must be finite");
  if (!isfinite(a.scale2)) return fail(FCR_E_SCALE, "scale over cap must be finite");
  a.whole = whole_items_of(plan.items, plan.held, most_blocks(plan, positions, prefix ? 0 : window, G), plan.form != 1);
  a.all_heads.set((uint32_t)(B * cache->H));
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
  if ((rc = launched("chunk attention")) || a.whole == 2) return rc;
  return join(a, plan, s);
}

}  // extern "C"
#endif
