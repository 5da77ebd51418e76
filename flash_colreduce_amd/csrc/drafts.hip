// What follows a step of drafted tokens: which of them stand and what comes next, their rows moved to where they belong, and the pages of
// sequences that have grown or shrunk.
//
// verify_drafts.  Row 0 of a sequence's target is the distribution behind its context, row i + 1 the one behind token i.  Whether a token is taken, if the
// one that it continues is, depends on its own row, number and siblings alone, so all of them are looked at side by side; those on the path are the ones whose
// every predecessor is taken (pointers that double: log2 T steps).  The path ends at one row.  The next token is the first v there with
//   sum_{w <= v} r(w) > sample sum r,
// r = (p - q)+ where drafted tokens come with what they were drawn from, p without the row's own drafted tokens where not.  Bound by reading that row: its
// sums are formed in 64 bits, where the order of additions moves a border between tokens by 1e-15 of the sum and not by 1e-7 (200000 borders: a sum in 32 bits would
// often end up on the other side of one).  First kernel: sums of pieces of the row, many workgroups, each of which finds the row by itself (a few
// gathers); second one: the piece, then the element.
// One sequence, 4 tokens of 32000 fp32 probabilities with what they were drawn from: 10 us, two launches and a chain of loads (tokens, their probabilities, sums, the piece); 64 of 7
// tokens of 131072: 24 us, 67 MB, 2.8 TB/s of them; 16 trees of 63 of 100003 bf16 ones: 14.5 us, 10 of them the first launch: tokens, their probabilities, siblings and the path, one behind the other.
// cache_accept and cache_reserve are bound by one launch and a chain of loads: 16 rows of 8 heads of 128 bf16 elements 5.2 us, 63 int8 rows of 32 heads and 64 sequences
// 5.8; a page here and there for 48 sequences, and back, 9.5 us together (two launches); pages for 256 prompts and back 40 us, 33000 entries of a table each way through
// one workgroup, 0.45 us for 1024, so that their order on the stack is that of the sequences without a second launch.

#include "paged.h"

namespace {
using namespace fcr_paged;
using fcr_detail::fail;
using fcr_detail::launched;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 8;                       // elements that a thread takes at once
constexpr int kPiece = kThreads * kEach;       // least number of elements of a piece
constexpr int kMostDrafted = 1024;

struct VerifyArgs {
  const char *target, *draft;        // draft null: tokens come without what they were drawn from
  int64_t target_b, target_r, draft_b, draft_r;   // bytes
  const void* tokens;                // [B, T] of 4 or 8 bytes
  const int32_t* parents;            // [T] per sequence or shared, null: a chain
  int64_t parents_b;
  const int32_t* counts;             // [B] or null
  const float *uniform, *sample;     // [B, T], [B]
  int32_t *accepted, *path;          // [B], [B, T]
  void* token;                       // [B]
  int32_t* row;                      // [B]: where a path ends
  double* sums;                      // [B][pieces][2]: of r, of p
  int B, T, V, wide, piece;          // wide: 8-byte tokens
  Div pieces;
};

__device__ __forceinline__ int64_t token_at(const VerifyArgs& a, int64_t i) {
  return a.wide ? static_cast<const int64_t*>(a.tokens)[i] : static_cast<const int32_t*>(a.tokens)[i];
}
// A weight: what is no number above zero is none.
__device__ __forceinline__ double weight(float x) { return x > 0.0f ? (double)x : 0.0; }

template <int DT>
__device__ __forceinline__ float number(const char* row, int64_t v) {
  if constexpr (DT == FCR_DTYPE_F32) return reinterpret_cast<const float*>(row)[v];
  else return element<DT>(reinterpret_cast<const uint16_t*>(row)[v], 0);
}
// kEach of them from v on (v < V); those behind the end are zeros.
template <int DT>
__device__ __forceinline__ void numbers(const char* row, int v, int V, float (&x)[kEach]) {
  constexpr int e = DT == FCR_DTYPE_F32 ? 4 : 2, words = kEach * e / 16;
  if (v + kEach <= V) {
    u32x4 w[words];
    __builtin_memcpy(w, row + (int64_t)v * e, sizeof(w));   // (rows of odd lengths: any alignment)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      x[i] = DT == FCR_DTYPE_F32 ? __builtin_bit_cast(float, (uint32_t)w[i / 4][i % 4]) : element<DT == FCR_DTYPE_F32 ? FCR_DTYPE_F16 : DT>(w[i / 8][i / 2 % 4], i & 1);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      x[i] = number<DT>(row, min(v + i, V - 1));
      x[i] = v + i < V ? x[i] : 0.0f;
    }
  }
}

// Where a sequence's path ends, and what is hidden there.
struct Rest {
  const char *p, *q;      // rows of V; q null: nothing is taken off
  const int* hidden;      // tokens that have no weight any more (in LDS)
  int n;
  // r and p of kEach tokens from v on.
  template <int DT>
  __device__ __forceinline__ void weights(int v, int V, double (&r)[kEach], double (&p_of)[kEach]) const {
    float x[kEach], y[kEach];
    numbers<DT>(p, v, V, x);
    if (q) {
      numbers<DT>(q, v, V, y);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) y[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      p_of[i] = weight(x[i]);
      const double d = p_of[i] - weight(y[i]);
      r[i] = d > 0.0 ? d : 0.0;
    }
    for (int j = 0; j < n; ++j) {
      const int at = hidden[j] - v;
#pragma unroll
      for (int i = 0; i < kEach; ++i) r[i] = at == i ? 0.0 : r[i];
    }
  }
};

// The sum over the workgroup's threads in front of this one, and over all.  part: kWaves words of LDS, free again behind the next barrier.
__device__ __forceinline__ double sum_in_front(double x, double* part, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(sum, o);
    if (lane >= o) sum += y;
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  // (what the lane in front has: the sum up to here less x may be off by a rounding)
  double before = __shfl_up(sum, 1);
  if (lane == 0) before = 0.0;
  all = 0.0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) before += part[i];
    all += part[i];
  }
  return before;
}

// Tokens of a sequence that the row where its path ends has as children, between tokens v0 and v1: into `list`, their number to *n.
__device__ __forceinline__ void hide(const VerifyArgs& a, int b, int count, int row, int v0, int v1, int* list, int* n) {
  if (a.draft) return;
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int parent = a.parents ? a.parents[b * a.parents_b + i] : i - 1;
    if (parent < -1 || parent >= i || parent + 1 != row) continue;
    const int64_t x = token_at(a, (int64_t)b * a.T + i);
    if (x >= v0 && x < v1) list[atomicAdd(n, 1)] = (int)x;       // (in LDS; the list has no order that matters)
  }
}

__device__ __forceinline__ Rest rest_of(const VerifyArgs& a, int b, int count, int row, const int* list, int n) {
  Rest r;
  r.p = a.target + b * a.target_b + row * a.target_r;
  r.q = a.draft && row < count ? a.draft + b * a.draft_b + row * a.draft_r : nullptr;
  r.hidden = list, r.n = n;
  return r;
}

__device__ __forceinline__ int count_of(const VerifyArgs& a, int b) { return a.counts ? min(max(a.counts[b], 0), a.T) : a.T; }

template <int DT>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  __shared__ __attribute__((aligned(16))) double p_of[kMostDrafted];
  __shared__ float uniform_of[kMostDrafted], q_of[kMostDrafted];
  __shared__ __attribute__((aligned(16))) int token_of[kMostDrafted], parent_of[kMostDrafted];     // -1: none of V; kMostDrafted: not there
  __shared__ int up[2][kMostDrafted];                                 // bit 31: not taken; else the predecessor + 1
  __shared__ uint64_t path[kMostDrafted / 64];
  __shared__ int hidden;
  __shared__ double part[2][kWaves];
  const int b = (int)a.pieces.of(blockIdx.x), piece = (int)(blockIdx.x - b * a.pieces.d);
  const int tid = threadIdx.x, count = count_of(a, b);
  const char* const target = a.target + b * a.target_b;
  if (tid == 0) hidden = 0;
  for (int i = tid; i < count; i += kThreads) {
    const int64_t x = token_at(a, (int64_t)b * a.T + i);
    const int parent = a.parents ? a.parents[b * a.parents_b + i] : i - 1;
    const bool there = parent >= -1 && parent < i, known = x >= 0 && x < a.V;
    parent_of[i] = there ? parent : kMostDrafted;
    token_of[i] = known ? (int)x : -1;
    p_of[i] = there && known ? weight(number<DT>(target + (parent + 1) * a.target_r, x)) : 0.0;
    uniform_of[i] = a.uniform[(int64_t)b * a.T + i];
    q_of[i] = a.draft && known ? number<DT>(a.draft + b * a.draft_b + i * a.draft_r, x) : 0.0f;
  }
  __syncthreads();
  if (a.parents && !a.draft) {
    // a token that a sibling in front has already has nothing left
    uint32_t again = 0;
#pragma unroll 1
    for (int i = tid, k = 0; i < count; i += kThreads, ++k) {
      const int parent = parent_of[i], token = token_of[i];
      bool found = false;
#pragma unroll 2
      for (int j = 0; j < i; j += 4) {
        const int4 p = *reinterpret_cast<const int4*>(parent_of + j), x = *reinterpret_cast<const int4*>(token_of + j);
        found |= ((p.x == parent) & (x.x == token)) | ((p.y == parent) & (x.y == token) & (j + 1 < i)) | ((p.z == parent) & (x.z == token) & (j + 2 < i)) |
                 ((p.w == parent) & (x.w == token) & (j + 3 < i));
      }
      again |= (found ? 1u : 0u) << k;
    }
    __syncthreads();
    for (int i = tid; again; i += kThreads, again >>= 1)
      if (again & 1) p_of[i] = 0.0;
    __syncthreads();
  }
  for (int i = tid; i < count; i += kThreads) {
    const int parent = parent_of[i];
    bool taken = parent != kMostDrafted && token_of[i] >= 0;
    if (taken) {
      const double u = uniform_of[parent + 1];
      if (a.draft) {
        taken = u * weight(q_of[i]) < p_of[i];
      } else {
        double low = 0.0;
        if (a.parents) {
#pragma unroll 2
          for (int j = 0; j < i; j += 4) {
            const int4 p = *reinterpret_cast<const int4*>(parent_of + j);
            const double2 w0 = *reinterpret_cast<const double2*>(p_of + j), w1 = *reinterpret_cast<const double2*>(p_of + j + 2);
            low += p.x == parent ? w0.x : 0.0;
            low += (p.y == parent) & (j + 1 < i) ? w0.y : 0.0;
            low += (p.z == parent) & (j + 2 < i) ? w1.x : 0.0;
            low += (p.w == parent) & (j + 3 < i) ? w1.y : 0.0;
          }
        }
        taken = low <= u && u < low + p_of[i];
      }
    }
    up[0][i] = taken ? parent + 1 : INT32_MIN;
  }
  __syncthreads();
  int now = 0;
  for (int step = 1; step < count; step <<= 1, now ^= 1) {
    for (int i = tid; i < count; i += kThreads) {
      const int x = up[now][i];
      up[now ^ 1][i] = x > 0 ? up[now][x - 1] : x;
    }
    __syncthreads();
  }
  // the path, in the order of its tokens, 64 of them to a word
  for (int i = tid; i < ((count + 63) & ~63); i += kThreads) {
    const uint64_t on = __ballot(i < count && up[now][i] >= 0);
    if ((tid & 63) == 0) path[i >> 6] = on;
  }
  __syncthreads();
  int row = 0, taken = 0;
  for (int g = 0; g < (count + 63) / 64; ++g) {
    const uint64_t on = path[g];
    if (on) row = 64 * g + 64 - __clzll(on);
    taken += __popcll(on);
  }
  if (piece == 0) {
    for (int i = tid; i < count; i += kThreads) {
      int before = 0;
      for (int g = 0; g < i >> 6; ++g) before += __popcll(path[g]);
      const uint64_t on = path[i >> 6];
      before += __popcll(on & ((1ull << (i & 63)) - 1));
      if (on >> (i & 63) & 1) a.path[(int64_t)b * a.T + before] = i;
    }
    for (int i = taken + tid; i < a.T; i += kThreads) a.path[(int64_t)b * a.T + i] = -1;
    if (tid == 0) a.accepted[b] = taken, a.row[b] = row;
  }
  const int v0 = piece * a.piece, v1 = min(v0 + a.piece, a.V);
  int* const list = parent_of;                   // (read last before several barriers)
  hide(a, b, count, row, v0, v1, list, &hidden);
  __syncthreads();
  const Rest rest = rest_of(a, b, count, row, list, hidden);
  double sum_r = 0.0, sum_p = 0.0;
  for (int v = v0 + tid * kEach; v < v1; v += kPiece) {
    double r[kEach], p[kEach];
    rest.weights<DT>(v, a.V, r, p);
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum_r += r[i], sum_p += p[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum_r += __shfl_xor(sum_r, o), sum_p += __shfl_xor(sum_p, o);
  if ((tid & 63) == 0) part[0][tid >> 6] = sum_r, part[1][tid >> 6] = sum_p;
  __syncthreads();
  if (tid < 2) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += part[tid][i];
    a.sums[2 * (int64_t)blockIdx.x + tid] = sum;
  }
}

// The first thread of the workgroup with `is`, or the last one: its `at`; `none` where there is no such thread.  words: kWaves of LDS; a barrier is in front of the
// result, and one must be behind it before the words are used again.
__device__ __forceinline__ int one_of(bool is, int at, bool first, int none, int* words) {
  const uint64_t lanes = __ballot(is);
  const int lane = first ? __ffsll((unsigned long long)lanes) - 1 : 63 - __clzll(lanes);
  const int found = __shfl(at, lanes ? lane : 0);
  if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = lanes ? found : none;
  __syncthreads();
  int x = none;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int w = words[first ? kWaves - 1 - i : i];
    x = w == none ? x : w;
  }
  return x;
}

// The piece that holds the sample's place, then the element.  A thread takes consecutive pieces, or elements.  Sums that meet a border from two sides in another order
// may disagree by a rounding: the last weight above zero stands where none is found.
template <int DT>
__global__ void __launch_bounds__(kThreads) next_token_kernel(VerifyArgs a) {
  __shared__ int list[kMostDrafted];
  __shared__ double part[3][kWaves];
  __shared__ double before_piece;
  __shared__ int hidden, words[4][kWaves];
  const int b = blockIdx.x, tid = threadIdx.x, count = count_of(a, b), row = a.row[b];
  const int pieces = (int)a.pieces.d, each = (pieces + kThreads - 1) / kThreads;
  const double* const sums = a.sums + 2 * (int64_t)b * pieces;
  const int first = min(tid * each, pieces), end = min(first + each, pieces);
  if (tid == 0) hidden = 0;
  double mine[2] = {0.0, 0.0}, all[2], before[2];
  for (int i = first; i < end; ++i) mine[0] += sums[2 * i], mine[1] += sums[2 * i + 1];
#pragma unroll
  for (int k = 0; k < 2; ++k) before[k] = sum_in_front(mine[k], part[k], all[k]);
  const int of = all[0] > 0.0 ? 0 : 1;            // nothing is left: the row as it is
  const double place = (double)a.sample[b] * all[of];
  int chosen = -1, last = -1;
  double upto = of ? before[1] : before[0], before_mine = 0.0;
  for (int i = first; i < end; ++i) {
    const double s = sums[2 * i + of];
    if (s > 0.0 && chosen < 0) {
      last = i, before_mine = upto;
      if (upto + s > place) chosen = i;
    }
    upto += s;
  }
  int piece = one_of(chosen >= 0, chosen, true, -1, words[0]);
  const int last_piece = one_of(last >= 0, last, false, -1, words[1]);
  piece = piece < 0 ? last_piece : piece;
  const auto give = [&](int x) {
    if (tid == 0) {
      if (a.wide) static_cast<int64_t*>(a.token)[b] = x;
      else static_cast<int32_t*>(a.token)[b] = x;
    }
  };
  if (piece < 0 || !(all[of] < INFINITY)) {       // no weight at all
    give(-1);
    return;
  }
  if (last == piece) before_piece = before_mine;   // (one thread's)
  const int v0 = piece * a.piece, v1 = min(v0 + a.piece, a.V);
  hide(a, b, count, row, v0, v1, list, &hidden);
  __syncthreads();
  const Rest rest = rest_of(a, b, count, row, list, hidden);
  // (a piece is a multiple of kPiece; in turns of kPiece, so that neighbours read what lies together)
  double from = before_piece;
  int token = -1;
  for (int t0 = v0; t0 < v1; t0 += kPiece) {
    const int v = t0 + tid * kEach;
    double r[kEach], p[kEach], sum = 0.0, turn;
#pragma unroll
    for (int i = 0; i < kEach; ++i) r[i] = p[i] = 0.0;
    if (v < v1) rest.weights<DT>(v, a.V, r, p);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      r[i] = of ? p[i] : r[i];
      sum += r[i];
    }
    double at = from + sum_in_front(sum, part[2], turn);
    chosen = last = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      at += r[i];
      if (r[i] > 0.0) {
        last = v + i;
        if (chosen < 0 && at > place) chosen = v + i;
      }
    }
    const int there = one_of(chosen >= 0, chosen, true, -1, words[2]), behind = one_of(last >= 0, last, false, -1, words[3]);
    from += turn;
    if (there >= 0) {
      token = there;
      break;
    }
    token = behind >= 0 ? behind : token;
    __syncthreads();
  }
  give(token);
}

// Accepted rows ------------------------------------------------------------------------------------------------------

struct AcceptArgs {
  Pages c;
  Lengths context;
  const int32_t *path, *accepted;    // [B, T], [B]
  int32_t* out;                      // [B] or [B, H]
  int T, by_head;
  Div H, pieces;                     // by heads, by 16-byte pieces of a row
};

// A workgroup has the keys or the values of one (sequence, head).  Rows move towards the front and in their order, path[i] >= i: those of one turn are
// read before any of them is written, and no later turn reads what an earlier one has written.
__global__ void __launch_bounds__(kThreads) cache_accept_kernel(AcceptArgs a) {
  const int which = blockIdx.y;
  const Side side = a.c.side[which];
  const int b = (int)a.H.of(blockIdx.x), h = (int)(blockIdx.x - b * a.H.d), tid = threadIdx.x;
  const int context = max(a.context.of(b, h), 0), n = min(max(a.accepted[b], 0), a.T);
  if (which == 0 && tid == 0 && (h == 0 || a.by_head)) a.out[a.by_head ? blockIdx.x : b] = context + n;
  const int each = (int)blockDim.x / (int)a.pieces.d, mine = (int)a.pieces.of(tid), piece = tid - mine * (int)a.pieces.d;
  for (int i0 = 0; i0 < n; i0 += each) {
    const int i = i0 + mine;
    bool move = mine < each && i < n;
    char* to = nullptr;
    u32x4 x = {0, 0, 0, 0};
    float scale = 0.0f;
    int64_t to_scale = 0;
    if (move) {
      const int step = a.path[(int64_t)b * a.T + i];
      const int64_t at = (int64_t)context + step, pos = (int64_t)context + i;
      move = step > i && at < a.c.capacity;
      if (move) {
        uint32_t row, to_row;
        const int page = page_of(a.c, b, (uint32_t)at, row), to_page = page_of(a.c, b, (uint32_t)pos, to_row);
        move = page >= 0 && to_page >= 0;
        if (move) {
          x = *reinterpret_cast<const u32x4*>(side.rows + page * side.page + h * side.head + row * side.row + piece * 16);
          to = side.rows + to_page * side.page + h * side.head + to_row * side.row + piece * 16;
          if (side.scale && piece == 0) scale = side.scale[page * side.s_page + h * side.s_head + row];
          to_scale = to_page * side.s_page + h * side.s_head + to_row;
        }
      }
    }
    __syncthreads();
    if (move) {
      *reinterpret_cast<u32x4*>(to) = x;
      if (side.scale && piece == 0) side.scale[to_scale] = scale;
    }
  }
}

// Pages --------------------------------------------------------------------------------------------------------------

struct ReserveArgs {
  int32_t *table, *held, *free, *available;
  int64_t table_stride;
  Lengths lengths;
  uint8_t* granted;
  int B, H, table_pages, pages;      // H: lengths of a sequence
  Div page_size;
};

template <int THREADS>
__device__ __forceinline__ int sum_upto(int x, int* part) {   // over the workgroup; part: a word of LDS for each wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) part[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += part[i];
  return x;
}

// One workgroup.  First the pages of sequences that need fewer go on the stack, then those that need more take theirs.  Sequences are added up
// a thread each, in turns of as many as there are threads; then every thread moves entries, of any sequence: the k-th of a turn belongs to the last sequence that
// begins at or before k.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) cache_reserve_kernel(ReserveArgs a) {
  __shared__ int start[THREADS], entry[THREADS], part[THREADS / 64], total, refused;
  const int tid = threadIdx.x;
  int there = min(max(*a.available, 0), a.pages);
  const auto sequence_of = [&](int k, int low, int high) {   // the last one of [low, high) with start <= k
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (start[mid] <= k) low = mid;
      else high = mid;
    }
    return low;
  };
  constexpr int kMoves = 16;                     // of a thread at once, at most, so that its loads overlap
  if (tid == 0) refused = 0;
  int need = 0, held = 0;
#pragma unroll 1
  for (int grow = 0; grow < 2; ++grow) {
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
      const int b = b0 + tid, n = min(THREADS, a.B - b0);
      int moves = 0;
      if (b < a.B && (!grow || a.B > THREADS)) {
        int length = 0;
        for (int h = 0; h < a.H; ++h) length = max(length, a.lengths.at[b * a.lengths.sb + h * a.lengths.sh]);
        need = (int)a.page_size.of((uint32_t)length);
        need += need * (int)a.page_size.d < length ? 1 : 0;
        held = min(max(a.held[b], 0), a.table_pages);
      }
      if (b < a.B && need <= a.table_pages) moves = max(grow ? need - held : held - need, 0);
      if (tid == 0) total = 0;
      const int upto = sum_upto<THREADS>(moves, part);
      // (of those that grow upto never falls: from the first one that does not fit on)
      const bool fits = grow ? !refused && upto <= there : upto <= a.pages - there;
      start[tid] = upto - moves;
      entry[tid] = grow ? held : need;
      if (fits && moves) atomicMax(&total, upto);
      if (b < a.B) {
        if (moves && fits) a.held[b] = held = need;
        if (grow) a.granted[b] = need <= a.table_pages && (moves == 0 || fits);
      }
      __syncthreads();
      if (grow && !fits && moves) refused = 1;
      const int all = total, moved = min((all + THREADS - 1) / THREADS, kMoves);
#pragma unroll 1
      for (int k0 = (tid & ~63) * moved; k0 < all; k0 += moved * THREADS) {
        const int lane = tid & 63;
        int s = sequence_of(min(k0 + lane, all - 1), 0, n), next = s + 1 < n ? start[s + 1] : INT32_MAX;
        int32_t *place[kMoves], x[kMoves];
#pragma unroll
        for (int j = 0; j < kMoves; ++j) {
          const int k = k0 + j * 64 + lane;
          place[j] = nullptr;
          if (j >= moved || k >= all) continue;
          while (k >= next) ++s, next = s + 1 < n ? start[s + 1] : INT32_MAX;   // (a turn of 64 moves stays in a long sequence)
          place[j] = a.table + (b0 + s) * a.table_stride + entry[s] + (k - start[s]);
          x[j] = grow ? a.free[there - 1 - k] : *place[j];
        }
#pragma unroll
        for (int j = 0; j < kMoves; ++j) {
          if (!place[j]) continue;
          if (grow) {
            *place[j] = x[j];
          } else {
            a.free[there + k0 + j * 64 + lane] = x[j];
            *place[j] = -1;
          }
        }
      }
      there += grow ? -all : all;
      __syncthreads();
    }
  }
  if (tid == 0) *a.available = there;
}

template <int DT>
void launch_verify(const VerifyArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((verify_kernel<DT>), dim3((unsigned)(a.B * (int64_t)a.pieces.d)), dim3(kThreads), 0, s, a);
}
template <int DT>
void launch_next(const VerifyArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((next_token_kernel<DT>), dim3((unsigned)a.B), dim3(kThreads), 0, s, a);
}

// Pieces of a row of V: as short as keeps a launch near what the CUs hold at once.
int piece_of(int B, int V) {
  const int64_t wgs = 8ll * fcr_detail::chip_cus_of_current_device();
  int piece = kPiece;
  while ((int64_t)B * ((V + piece - 1) / piece) > wgs && piece < V) piece *= 2;
  return piece;
}
size_t verify_bytes(int B, int V) {
  const int piece = piece_of(B, V);
  return ((size_t)B * 4 + 15) / 16 * 16 + (size_t)B * ((V + piece - 1) / piece) * 16;
}
bool verify_sizes(int B, int T, int V) {
  return B >= 1 && B <= (1 << 20) && T >= 0 && T <= kMostDrafted && V >= 1 && V <= (1 << 28);
}

}  // namespace

extern "C" {

size_t fcr_verify_drafts_bytes(int B, int T, int V) { return verify_sizes(B, T, V) ? verify_bytes(B, V) : 0; }

int fcr_verify_drafts(const void* target, const int64_t target_strides[2], const void* draft, const int64_t draft_strides[2], const void* tokens,
                      int token_bytes, const int32_t* parents, int64_t parents_stride, const int32_t* counts, const float* uniform,
                      const float* sample, int32_t* accepted, int32_t* path, void* token, void* ws, size_t ws_bytes, int dtype, int B,
                      int T, int V, void* stream) {
  if (!target || !target_strides || !sample || !accepted || !token || !ws || (draft && !draft_strides)) return fail(FCR_E_NULL, "null pointer argument");
  if (T != 0 && (!tokens || !uniform || !path)) return fail(FCR_E_NULL, "null pointer argument");
  if (dtype != FCR_DTYPE_F16 && dtype != FCR_DTYPE_BF16 && dtype != FCR_DTYPE_F32)
    return fail(FCR_E_DTYPE, "probabilities must be FCR_DTYPE_F16, FCR_DTYPE_BF16 or FCR_DTYPE_F32");
  if (token_bytes != 4 && token_bytes != 8) return fail(FCR_E_DTYPE, "tokens must have 4 or 8 bytes");
  if (!verify_sizes(B, T, V)) return fail(FCR_E_SHAPE, "B must be in [1, 2^20], T in [0, 1024], V in [1, 2^28]");
  if (draft && parents) return fail(FCR_E_SHAPE, "tokens that come with the probabilities that they were drawn from must be a chain");
  const int e = dtype == FCR_DTYPE_F32 ? 4 : 2;
  const auto off = [&](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; };
  bool ok = !off(target, e) && !off(draft, e) && !off(tokens, token_bytes) && !off(token, token_bytes) && !off(parents, 4) && !off(counts, 4) &&
            !off(uniform, 4) && !off(sample, 4) && !off(accepted, 4) && !off(path, 4) && parents_stride >= 0;
  for (int i = 0; i < 2; ++i) {
    ok = ok && target_strides[i] >= 0 && target_strides[i] < (1ll << 40);
    if (draft) ok = ok && draft_strides[i] >= 0 && draft_strides[i] < (1ll << 40);
  }
  if (!ok) return fail(FCR_E_STRIDE, "operands must be aligned to their elements, with strides that are >= 0");
  if (off(ws, 16)) return fail(FCR_E_STRIDE, "the workspace must be 16-byte aligned");
  if (ws_bytes < verify_bytes(B, V)) return fail(FCR_E_SCRATCH, "the workspace is smaller than fcr_verify_drafts_bytes");
  VerifyArgs a;
  a.target = static_cast<const char*>(target), a.target_b = target_strides[0] * e, a.target_r = target_strides[1] * e;
  a.draft = T ? static_cast<const char*>(draft) : nullptr, a.draft_b = draft ? draft_strides[0] * e : 0, a.draft_r = draft ? draft_strides[1] * e : 0;
  a.tokens = tokens, a.parents = parents, a.parents_b = parents_stride, a.counts = counts, a.uniform = uniform, a.sample = sample;
  a.accepted = accepted, a.path = path, a.token = token;
  a.row = static_cast<int32_t*>(ws);
  a.sums = reinterpret_cast<double*>(static_cast<char*>(ws) + ((size_t)B * 4 + 15) / 16 * 16);
  a.B = B, a.T = T, a.V = V, a.wide = token_bytes == 8;
  a.piece = piece_of(B, V);
  a.pieces.set((uint32_t)((V + a.piece - 1) / a.piece));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FCR_DTYPE_F16) launch_verify<FCR_DTYPE_F16>(a, s);
  else if (dtype == FCR_DTYPE_BF16) launch_verify<FCR_DTYPE_BF16>(a, s);
  else launch_verify<FCR_DTYPE_F32>(a, s);
  const int rc = launched("verify_kernel");
  if (rc) return rc;
  if (dtype == FCR_DTYPE_F16) launch_next<FCR_DTYPE_F16>(a, s);
  else if (dtype == FCR_DTYPE_BF16) launch_next<FCR_DTYPE_BF16>(a, s);
  else launch_next<FCR_DTYPE_F32>(a, s);
  return launched("next_token_kernel");
}

int fcr_cache_accept(const fcr_cache* cache, const int32_t* table, int64_t table_stride, int table_pages, const int32_t* context,
                     const int64_t context_strides[2], const int32_t* path, const int32_t* accepted, int32_t* out, int B, int T, void* stream) {
  int rc = check_cache(cache, "cache");
  if (rc) return rc;
  if ((rc = check_table(table, table_stride, table_pages, cache->page_size, B))) return rc;
  if (!context || !context_strides || !path || !accepted || !out) return fail(FCR_E_NULL, "null pointer argument");
  if (context_strides[0] < 0 || context_strides[1] < 0) return fail(FCR_E_STRIDE, "context: strides must be >= 0");
  if (T < 1 || T > (1 << 20) || (int64_t)B * cache->H > (1 << 22)) return fail(FCR_E_SHAPE, "T must be in [1, 2^20], B*H at most 2^22");
  if ((rc = check_written(*cache, "cache"))) return rc;
  AcceptArgs a;
  a.c = pages_of(*cache, table, table_stride, table_pages);
  a.context = Lengths{context, context_strides[0], context_strides[1]};
  a.path = path, a.accepted = accepted, a.out = out, a.T = T, a.by_head = context_strides[1] != 0;
  a.H.set((uint32_t)cache->H);
  a.pieces.set((uint32_t)(cache->D * element_bytes(cache->dtype) / 16));
  // Half the threads where there are more workgroups than the CUs hold at once: most of a tree's tokens do not stand, and so most threads have nothing to move.  8 of 63 rows of 32
  // int8 heads and 64 sequences 6.7 -> 5.1 us, 50 of them 11.6 -> 11.2; for 8 heads of one sequence all 63 bf16 rows of 256 elements 3.5 with 256 threads, 4.4 with 128.
  const int threads = 2ll * B * cache->H >= 8ll * fcr_detail::chip_cus_of_current_device() ? kThreads / 2 : kThreads;
  hipLaunchKernelGGL(cache_accept_kernel, dim3((unsigned)(B * cache->H), 2), dim3(threads), 0, static_cast<hipStream_t>(stream), a);
  return launched("cache_accept_kernel");
}

int fcr_cache_reserve(int32_t* table, int64_t table_stride, int table_pages, int32_t* held, int32_t* free_pages, int pages, int32_t* available,
                      const int32_t* lengths, const int64_t lengths_strides[2], int H, int page_size, uint8_t* granted, int B, void* stream) {
  if (!table || !held || !free_pages || !available || !lengths || !lengths_strides || !granted) return fail(FCR_E_NULL, "null pointer argument");
  if (B < 1 || B > (1 << 20) || H < 1 || pages < 1 || pages > (1 << 28) || table_pages < 1 || page_size < 1 || (int64_t)table_pages * page_size > (1 << 30) ||
      (int64_t)B * table_pages > (1 << 30))
    return fail(FCR_E_SHAPE, "B in [1, 2^20], pages in [1, 2^28], H, the table's pages and page_size >= 1, at most 2^30 entries of a table and positions of its row");
  if (table_stride < table_pages && B > 1) return fail(FCR_E_STRIDE, "rows of a table that is written must not overlap");
  if (lengths_strides[0] < 0 || lengths_strides[1] < 0) return fail(FCR_E_STRIDE, "lengths: strides must be >= 0");
  ReserveArgs a;
  a.table = table, a.held = held, a.free = free_pages, a.available = available;
  a.table_stride = table_stride;
  a.lengths = Lengths{lengths, lengths_strides[0], lengths_strides[1]};
  a.granted = granted;
  a.B = B, a.H = lengths_strides[1] ? H : 1, a.table_pages = table_pages, a.pages = pages;
  a.page_size.set((uint32_t)page_size);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (B <= 64) hipLaunchKernelGGL((cache_reserve_kernel<256>), dim3(1), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((cache_reserve_kernel<1024>), dim3(1), dim3(1024), 0, s, a);
  return launched("cache_reserve_kernel");
}

}  // extern "C"
