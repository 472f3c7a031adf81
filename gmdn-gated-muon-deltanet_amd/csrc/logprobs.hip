// Log probabilities of given tokens with entropy and top alternatives, and
// the logits' gradient (include/gmdn_lm.h).
//
// A row x of V logits, its token t:  M = max x,  s = sum e^(x - M),
// log p_j = x_j - M - log s,  lp = log p_t,
// H = -sum p_j log p_j = log s - (sum e^(x - M) (x - M)) / s,
// in one pass over the row: each thread keeps a running M, s and
// w = sum e^(x - M) (x - M), rescaled when its M grows; they are joined at the
// row's end.  Backward, with gl, gh, gt_i the cotangents of lp, H and the
// alternatives' log probabilities and G = gl + sum gt_i:
//   dx_j = gl [j = t] + sum_i gt_i [j = t_i] - G p_j - gh p_j (log p_j + H)
//
// The forward reads the logits once; nothing of their size is written.  It is
// near both bounds: 10.6 instruction slots a logit (the exponential takes four)
// keep the vector units busy in 91 % of its cycles, and 16384 x 32000 bf16 logits go by
// in 163 us, 6.4 TB/s (172 between backward passes; a kernel that only reads
// reaches 7.0).  The backward reads and writes once: 333 us, 6.3 TB/s (a copy 5.1).
#include "../../include/gmdn_lm.h"
#include "logsums.h"

namespace gmdn {
namespace {

constexpr int PIECES = 4;  // pieces a thread loads before it works on them

// The instruction by name: for fmaxf of loaded values the compiler first
// quiets each one, which costs as much again.  A NaN gives way to the others.
GMDN_DEV float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
GMDN_DEV float max8(const float (&x)[8], float m) {
  return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], m));
}
GMDN_DEV float min8(const float (&x)[8]) {
  float r, s;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(s) : "v"(x[3]), "v"(x[4]), "v"(x[5]));
  asm("v_min3_f32 %0, %0, %1, %2" : "+v"(r) : "v"(x[6]), "v"(x[7]));
  return fminf(r, s);
}
// The terms of a piece at the maximum that `a` has.
GMDN_DEV void terms8(Sums& a, const float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = x[j] - a.m, e = exp_of(u);
    a.s += e;
    a.w += e * fmaxf(u, FAR);
  }
}

// The first wave's sums from the waves', in each of its lanes.
template <int W>
GMDN_DEV Sums join_waves(const Sums* waves) {
  const Sums a = join_lanes<16>(lane_id() < W ? waves[lane_id()] : no_sums());
  auto first = [](float x) { return float_of(__builtin_amdgcn_readfirstlane(bits_of(x))); };
  return {first(a.m), first(a.s), first(a.w)};
}
// The sums of a row's NT threads, in its first wave: each wave its own, then
// the first wave all of them (the work is small beside that of 16 waves doing
// it side by side).  `waves` is LDS for a wave's each.
template <int NT>
GMDN_DEV Sums join(Sums a, Sums* waves) {
  a = join_lanes<(NT < 64 ? NT : 64)>(a);
  if constexpr (NT > 64) {
    if (lane_id() == 0) waves[wave_id()] = a;
    __syncthreads();
    if (wave_id() == 0) a = join_waves<NT / 64>(waves);
  }
  return a;
}

// The outputs of a call, and its tokens.
struct Out {
  const int64_t* tokens;
  int64_t ignore;
  float *lp, *entropy, *stats, *top_lp;
  int64_t* top_tokens;
  int V, top;
  Out from(int64_t row) const {
    return {tokens + row, ignore, lp + row, entropy + row, stats + 2 * row, top ? top_lp + row * top : nullptr,
            top ? top_tokens + row * top : nullptr, V, top};
  }
  template <typename T>
  GMDN_DEV void row(int64_t row, const Row& r, const T* x) const {
    const int64_t token = tokens[row];
    float l = 0.f;
    if (token != ignore) l = token >= 0 && token < V ? r.logprob((float)x[token]) : NAN;
    lp[row] = l;
    entropy[row] = r.entropy;
    stats[2 * row] = r.m;
    stats[2 * row + 1] = r.logs;
  }
  template <typename T>
  GMDN_DEV void alternative(int64_t row, int i, int token, const Row& r, const T* x) const {
    top_tokens[row * top + i] = token;
    top_lp[row * top + i] = r.logprob((float)x[token]);
  }
};

// Where a row's columns are shared by several workgroups: what each leaves
// for lp_join, its sums and its best logits.
struct Parts {
  Sums* sums;      // (rows, parts)
  uint64_t* best;  // (rows, parts, top)
  int parts, span; // workgroups of a row, columns of each
};

// The sums of columns first .. last - 1 of a row by NT threads.  Four pieces
// share one maximum and one rescaling (a piece at a time: 170 us, not 160).
template <typename T, int NT, bool FAR>
GMDN_DEV Sums sums_of(const T* x, int first, int last, int t) {
  Sums a = no_sums();
  int c0 = first + 8 * t;
  for (; c0 + 8 * NT * (PIECES - 1) + 8 <= last; c0 += 8 * NT * PIECES) {
    Raw8<T> raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i].template load<FAR>(x + c0 + 8 * NT * i, 8);
    float v[PIECES][8], m = a.m;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      raw[i].get(v[i]);
      m = max8(v[i], m);
    }
    rescale(a, m);  // once for all of them
#pragma unroll
    for (int i = 0; i < PIECES; ++i) terms8(a, v[i]);
  }
  for (; c0 < last; c0 += 8 * NT) {
    float v[8];
    load8(x + c0, last - c0, v, -INFINITY);
    rescale(a, max8(v, a.m));
    terms8(a, v);
  }
  return a;
}

// A row is TPR threads of the workgroup's 256 (SPLIT: 256 for a part of it): 16
// up to 512 logits (65536 x 257 float32: 14 us, a wave each 23, 256 threads each 53),
// a wave up to 4096 (16384 x 4096 bf16: 26 us, 256 threads 37; x 8000: 54 and 53).
constexpr int LP_THREADS = 256;
template <typename T, int TPR, bool SPLIT, bool FAR>
__global__ void __launch_bounds__(LP_THREADS)
lp_fwd(const T* __restrict__ logits, int64_t stride, int64_t rows, Out out, Parts parts) {
  __shared__ Sums waves[LP_THREADS / 64];
  const int64_t item = (int64_t)blockIdx.x * (LP_THREADS / TPR) + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  if (item >= rows * (SPLIT ? parts.parts : 1)) return;  // rows of no more than a wave only
  const int64_t row = SPLIT ? item / parts.parts : item;
  const int first = SPLIT ? (int)(item - row * parts.parts) * parts.span : 0;
  const int last = SPLIT && first + parts.span < out.V ? first + parts.span : out.V;
  const T* x = logits + row * stride;
  const Sums a = join<TPR>(sums_of<T, TPR, FAR>(x, first, last, t), waves);
  if (t != 0) return;
  if constexpr (SPLIT)
    parts.sums[item] = a;
  else
    out.row(row, row_of(a), x);
}

// ------------------------------------------------------------ top alternatives
// Order of logits: larger first, NaN before all, equal ones by index.  As one
// 64-bit key, larger is better; 0 is none, and no key is all ones.
GMDN_DEV uint64_t key_of(float x, int index) {
  uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 as 0
  b = x != x ? 0xfffffffeu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((uint64_t)b << 32) | (0xffffffffu - (uint32_t)index);
}
// The value of a key (none: -inf, which every logit reaches).
GMDN_DEV float value_of(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return b == 0 ? -INFINITY : __builtin_bit_cast(float, (b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
GMDN_DEV int index_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

GMDN_DEV uint64_t lane_key(uint64_t k, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}
GMDN_DEV uint64_t lanes_max64(uint64_t x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = ((uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), o, 64) << 32) |
                       (uint32_t)__shfl_xor((int)(uint32_t)x, o, 64);
    x = y > x ? y : x;
  }
  return x;
}

constexpr int TOP_MAX = 32;

// A workgroup's LDS: at most LIST candidates of a tile, from at most PIECES_
// pieces; less for a workgroup of one wave, so that a CU holds 28 of them.
template <int NT>
struct TopLds {
  static constexpr int LIST = NT > 64 ? 1024 : 256, PIECES_ = NT > 64 ? 256 : 64;
  float piece[PIECES_][8];
  int column[PIECES_];
  uint64_t groups[64];
  uint64_t list[LIST + TOP_MAX];
  uint64_t run[TOP_MAX];  // the best so far, in order
  uint64_t bound;
  uint64_t red64[16];
  Sums waves[16];
  int pieces, count, nan;
};

// The n keys of the list by rank into run: a key's rank is the number of
// better ones, counted over 64 lanes at a time; a wave ranks every W-th key.
template <int NT>
GMDN_DEV void rank_list(TopLds<NT>& lds, int n, int top) {
  const int lane = lane_id();
  const uint64_t a = lane < n ? lds.list[lane] : 0, b = 64 + lane < n ? lds.list[64 + lane] : 0;
  if (NT == 64 && n <= 64) {  // alone: each lane its own key, against each of the others
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) rank += lane_key(a, i) > a;
    if (lane < n && rank < top) lds.run[rank] = a;
    return;
  }
  for (int i = wave_id(); i < n; i += NT / 64) {
    const uint64_t k = i < 64 ? lane_key(a, i) : i < 128 ? lane_key(b, i - 64) : lds.list[i];
    int rank = __popcll(__ballot(a > k)) + __popcll(__ballot(b > k));
    for (int o = 128; o < n; o += 64) rank += __popcll(__ballot(o + lane < n && lds.list[o + lane] > k));
    if (rank < top && lane == 0) lds.run[rank] = k;
  }
}

// The top-th largest of a wave's 64 keys (0: fewer are there), bit by bit:
// first of their values, then, where several keys have that value, of their
// indexes.
GMDN_DEV uint64_t kth(uint64_t key, int top) {
  const uint32_t value = (uint32_t)(key >> 32), index = (uint32_t)key;
  uint32_t v = 0;
#pragma unroll
  for (int b = 31; b >= 0; --b)
    if (__popcll(__ballot(value >= (v | 1u << b))) >= top) v |= 1u << b;
  if (v == 0) return 0;
  const int need = top - __popcll(__ballot(value > v));
  const uint64_t ties = __ballot(value == v);
  if (__popcll(ties) == 1) return lane_key(key, __ffsll((long long)ties) - 1);
  uint32_t x = 0;
  for (int b = 31; b >= 0; --b)
    if (__popcll(__ballot(value == v && index >= (x | 1u << b))) >= need) x |= 1u << b;
  return (uint64_t)v << 32 | x;
}

// The best `top` of columns first .. last - 1 by one logit a round: for rows
// that the tiles below give up on.
template <typename T, int NT>
GMDN_DEV void slow_top(const T* x, int first, int last, int top, TopLds<NT>& lds) {
  uint64_t prev = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int c = first + threadIdx.x; c < last; c += NT) {
      const uint64_t key = key_of((float)x[c], c);
      if (key < prev && key > best) best = key;
    }
    best = lanes_max64(best);
    __syncthreads();
    if (lane_id() == 0) lds.red64[wave_id()] = best;
    __syncthreads();
    prev = lds.red64[0];
    for (int i = 1; i < NT / 64; ++i) prev = lds.red64[i] > prev ? lds.red64[i] : prev;
    if (threadIdx.x == 0) lds.run[k] = prev;
  }
  __syncthreads();
}

// Sums and the best `top` (into lds.run, `have` of them) of columns
// first .. last - 1, in tiles of NT x 4 pieces held in registers.  Of a tile,
// threads of the same lane number form 64 groups; the top-th best of the 64
// groups' best logits bounds the tile's top-th best from below, and few
// logits reach it (24 of random ones for 20 wanted: each group's pieces lie
// 512 apart, so that neighbours do not share a group).  A group's best is its
// largest value with the last index of the first piece that has it, which no
// better logit of that value exceeds: equal logits, masked ones above all,
// stay out of the list by their index.  In a row with fewer allowed
// tokens than are wanted the bound is the masks' value, and of the first wave's
// pieces of nothing else only those with the first `top` logits go on (4816 x 1220
// float32, five allowed of each, 32 wanted: 128 -> 24 us).  With 512 threads that is
// done for -inf alone: to know other values cost 5 to 10 % of every row.  Those that reach the bound join the best
// of the tiles before in the list, which is ranked.  A tile that gives more
// than LDS holds, or a NaN, is left to slow_top.  The sums are returned in the
// first wave.
template <typename T, int NT>
GMDN_DEV Sums top_of(const T* x, int first, int last, int top, TopLds<NT>& lds, int& have) {
  const int tid = threadIdx.x;
  Sums a = no_sums();
  have = 0;
  bool over = false;
  if (tid < 64) lds.groups[tid] = 0;
  if (tid == 0) lds.pieces = lds.count = lds.nan = 0;
  __syncthreads();
  for (int c0 = first; c0 < last; c0 += 8 * NT * PIECES) {
    Raw8<T> raw[PIECES];
    float most[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = c0 + 8 * (i * NT + tid);
      raw[i].load(x + c, last - c, -INFINITY);
    }
    // the thread's best: its value, and the first piece that has it
    float bv = -INFINITY;
    int bp = 0;
    [[maybe_unused]] uint64_t flat = 0;  // the wave's first pieces of one value
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float v[8];
      raw[i].get(v);
      most[i] = max8(v, -INFINITY);
      if (NT <= 256 && i == 0) flat = __ballot(min8(v) == most[0]);
      rescale(a, max3(a.m, most[i], most[i]));
      terms8(a, v);
      if (most[i] > bv) {
        bv = most[i];
        bp = i;
      }
      __builtin_amdgcn_sched_barrier(0);  // one piece's values at a time in registers
    }
    if (over) continue;
    if (c0 + 8 * tid < last)
      atomicMax((unsigned long long*)&lds.groups[lane_id()],
                (unsigned long long)key_of(bv, c0 + 8 * (bp * NT + tid) + 7));
    __syncthreads();
    // the groups' top-th best, or the best so far's: found by the first wave
    // where that is not many waves' wait, else shared
    if constexpr (NT <= 256) {
      if (wave_id() == 0) {
        const uint64_t k = kth(lds.groups[lane_id()], top);
        if (lane_id() == 0) lds.bound = have == top && lds.run[top - 1] > k ? lds.run[top - 1] : k;
      }
    } else {
      // a wave ranks its share of the groups against all 64; equal only where there is none
      const uint64_t mine = lds.groups[lane_id()];
      constexpr int SHARE = 64 / (NT / 64);
      for (int g = wave_id() * SHARE; g < (wave_id() + 1) * SHARE; ++g) {
        const uint64_t k = lane_key(mine, g);
        if (__popcll(__ballot(mine > k || (mine == k && lane_id() < g))) == top - 1 && lane_id() == 0)
          lds.bound = have == top && lds.run[top - 1] > k ? lds.run[top - 1] : k;
      }
    }
    __syncthreads();
    if (tid < 64) lds.groups[tid] = 0;
    // the pieces that hold candidates go to LDS, where each of their values is
    // a thread's: by value, and for the bound's own value by index
    const uint64_t least = lds.bound;
    const float lv = value_of(least);
    const int upto = least ? index_of(least) : 0x7fffffff;
    int upto0 = upto;  // in a thread's first piece
    if (tid < 64 && (NT <= 256 || lv == -INFINITY)) {
      uint64_t equal = __ballot(most[0] == lv && c0 + 8 * tid + 8 <= last);
      if constexpr (NT <= 256) equal &= flat;
      for (int k = 8; k < top; k += 8) equal &= equal - 1;
      const int enough = c0 + 8 * (__ffsll((long long)equal) - 1);
      if (equal && enough < upto) upto0 = enough;
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = c0 + 8 * (i * NT + tid);
      if ((most[i] > lv || (most[i] == lv && c <= (i == 0 ? upto0 : upto))) && c < last) {
        const int at = atomicAdd(&lds.pieces, 1);
        if (at < TopLds<NT>::PIECES_) {
          float v[8];
          raw[i].get(v);
          *reinterpret_cast<f32x4*>(&lds.piece[at][0]) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(&lds.piece[at][4]) = f32x4{v[4], v[5], v[6], v[7]};
          lds.column[at] = c;
        }
      }
    }
    __syncthreads();
    const int np = lds.pieces;
    for (int e = tid; e < 8 * np && np <= TopLds<NT>::PIECES_; e += NT) {
      const float v = lds.piece[e / 8][e % 8];
      const int c = lds.column[e / 8] + e % 8;
      if ((v > lv || (v == lv && c <= upto)) && c < last) {
        const int at = atomicAdd(&lds.count, 1);
        if (at < TopLds<NT>::LIST) lds.list[at] = key_of(v, c);
      }
    }
    __syncthreads();
    int n = lds.count;
    over = n > TopLds<NT>::LIST || np > TopLds<NT>::PIECES_;
    if (!over && tid < have) lds.list[n + tid] = lds.run[tid];
    __syncthreads();
    if (tid == 0) lds.pieces = lds.count = 0;
    if (!over) {
      n += have;
      rank_list<NT>(lds, n, top);
      have = n < top ? n : top;
    }
    __syncthreads();
  }
  a = join_lanes<64>(a);
  if (lane_id() == 0) {
    lds.waves[wave_id()] = a;
    if (a.s != a.s) lds.nan = 1;
  }
  __syncthreads();
  if (over || lds.nan) {
    have = top < last - first ? top : last - first;
    slow_top<T, NT>(x, first, last, have, lds);
  }
  return join_waves<NT / 64>(lds.waves);
}

template <typename T, int NT, bool SPLIT>
__global__ void __launch_bounds__(NT, NT > 64 ? 8 : 6)
lp_top(const T* __restrict__ logits, int64_t stride, Out out, Parts parts) {
  __shared__ TopLds<NT> lds;
  const int64_t item = blockIdx.x, row = SPLIT ? item / parts.parts : item;
  const int first = SPLIT ? (int)(item - row * parts.parts) * parts.span : 0;
  const int last = SPLIT && first + parts.span < out.V ? first + parts.span : out.V;
  const T* x = logits + row * stride;
  int have;
  const Sums a = top_of<T, NT>(x, first, last, out.top, lds, have);
  if (wave_id() > 0) return;
  const int i = threadIdx.x;
  if constexpr (SPLIT) {
    if (i == 0) parts.sums[item] = a;
    if (i < out.top) parts.best[item * out.top + i] = i < have ? lds.run[i] : 0;
  } else {
    const Row r = row_of(a);
    if (i == 0) out.row(row, r, x);
    if (i < out.top) out.alternative(row, i, index_of(lds.run[i]), r, x);
  }
}

// A row's outputs from its parts.
constexpr int MAX_PARTS = 32;
constexpr int JOIN_THREADS = 1024;
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS)
lp_join(const T* __restrict__ logits, int64_t stride, Out out, Parts parts) {
  static_assert(MAX_PARTS * TOP_MAX <= JOIN_THREADS && JOIN_THREADS <= TopLds<JOIN_THREADS>::LIST, "a key a thread");
  __shared__ TopLds<JOIN_THREADS> lds;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  int n = parts.parts * out.top;
  const int i = threadIdx.x;
  const uint64_t key = i < n ? parts.best[row * n + i] : 0;
  if (i < n) lds.list[i] = key;
  if (i == 0) lds.count = 0;
  Sums a = no_sums();
  if (i < parts.parts) a = parts.sums[row * parts.parts + i];
  a = join<JOIN_THREADS>(a, lds.waves);
  if (n > 128) {
    // ranking them all would be n^2 (1 x 262144, 20 alternatives: 21 us, so 11.5);
    // as in a tile, few reach the top-th best of 64 lanes' bests
    if (wave_id() == 0) {
      uint64_t best = 0;
      for (int k = lane_id(); k < n; k += 64) best = lds.list[k] > best ? lds.list[k] : best;
      best = kth(best, out.top);
      if (i == 0) lds.bound = best;
    }
    __syncthreads();
    if (i < n && key >= lds.bound) lds.list[atomicAdd(&lds.count, 1)] = key;
    __syncthreads();
    n = lds.count;
  }
  rank_list<JOIN_THREADS>(lds, n, out.top);
  __syncthreads();
  if (wave_id() > 0) return;
  const Row r = row_of(a);
  if (threadIdx.x == 0) out.row(row, r, x);
  if ((int)threadIdx.x < out.top) out.alternative(row, threadIdx.x, index_of(lds.run[threadIdx.x]), r, x);
}

// ------------------------------------------------------------------ backward
// TPR threads take `span` columns of a row; a workgroup NT / TPR rows.  The
// token's term goes to its column where that is computed.  TOP: the columns of
// token and alternatives are written again with their terms at the end.
// Rows of 1024 threads past 8192 logits (16384 x 32000 bf16: 337 us, of 256
// threads 403; x 8000: 112 and 90, x 9000 still 130 and 109), of a wave up to 4096
// (x 4096: 47 and 46), of 16 up to 512 (65536 x 257 float32: 28 us, of a wave 32,
// of 256 threads 54).  With alternatives' terms always of 256, also where that is
// far off: 16384 x 257 float32 with 20 takes 71 us, without them 8.7.
template <typename T, int NT, int TPR, bool TOP>
__global__ void __launch_bounds__(NT)
lp_bwd(const T* __restrict__ logits, int64_t stride, int64_t rows, const int64_t* __restrict__ tokens,
       const float* __restrict__ stats, const float* __restrict__ entropy, const int64_t* __restrict__ top_tokens,
       const float* __restrict__ dlp, const float* __restrict__ dent, const float* __restrict__ dtop,
       T* __restrict__ dx, int V, int top, int64_t ignore, int span, int parts) {
  const int64_t item = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  if (item >= rows * parts) return;  // rows of no more than a wave only
  const int64_t row = item / parts;
  const int first = (int)(item - row * parts) * span, last = first + span < V ? first + span : V;
  const T* x = logits + row * stride;
  T* out = dx + row * V;
  const int64_t token = tokens[row];
  const bool empty = stats[2 * row] == -INFINITY;
  const float m = empty ? 0.f : stats[2 * row], logs = stats[2 * row + 1], h = entropy[row];
  const float gh = dent ? dent[row] : 0.f;
  // of a token outside the vocabulary NaN; the entropy's and the alternatives' gradients
  // do not see the token
  const float gl = !dlp || token == ignore ? 0.f : token >= 0 && token < V ? dlp[row] : NAN;
  float all = gl;
  if constexpr (TOP)
    for (int i = 0; i < top; ++i) all += dtop[row * top + i];
  // the terms of p (0 throughout an empty row), p as the square of e^(l / 2):
  // the exponential flushes results below 2^-126, the product does not
  auto grad = [&](float z) {
    const float l = z - m - logs, e = __builtin_amdgcn_exp2f(l * (0.5f * LOG2E));
    return -e * (e * (all + gh * (fmaxf(l, FAR) + h)));
  };
  auto grad8 = [&](float (&v)[8], int c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = grad(v[j]);
    if constexpr (!TOP)
      if (token >= c && token < c + 8 && !empty)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (token == c + j) v[j] += gl;
  };
  int c0 = first + 8 * t;
  for (; c0 + 8 * TPR * (PIECES - 1) + 8 <= last; c0 += 8 * TPR * PIECES) {
    Raw8<T> raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i].load(x + c0 + 8 * TPR * i, 8);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float v[8];
      raw[i].get(v);
      grad8(v, c0 + 8 * TPR * i);
      stream8(out + c0 + 8 * TPR * i, 8, v);
    }
  }
  for (; c0 < last; c0 += 8 * TPR) {
    float v[8];
    load8(x + c0, last - c0, v);
    grad8(v, c0);
    store8(out + c0, last - c0, v);
  }
  if constexpr (TOP) {
    static_assert(NT == TPR, "all of a workgroup comes here");
    __syncthreads();
    if (t <= top && !empty) {
      auto which = [&](int i) { return i == 0 ? token : top_tokens[row * top + i - 1]; };
      const int64_t c = which(t);
      if (c >= first && c < last) {
        float g = 0.f;
        for (int i = 0; i <= top; ++i)
          if (which(i) == c) g += i == 0 ? gl : dtop[row * top + i - 1];
        out[c] = (T)(grad((float)x[c]) + g);
      }
    }
  }
}

int check_lp(int64_t rows, int64_t V, int64_t stride, int32_t top, int32_t dtype) {
  if (rows < 0 || V <= 0 || stride < 0 || top < 0 || top > V) return GMDN_ERR_ARG;
  if (!type_ok(dtype) || top > TOP_MAX || V > (1 << 30)) return GMDN_ERR_UNSUPPORTED;
  if (rows > ((int64_t)1 << 30)) return GMDN_ERR_ARG;
  return GMDN_OK;
}

// Workgroups of a row in the forward: more than one where rows alone leave the
// chip idle and a row is long enough to pay for the second launch that joins
// them (1 x 131072 float32: 7.8 us, one workgroup 11; with 20 alternatives 11 and
// 22.  8 x 32000 bf16, 20 alternatives: two parts 10.5 us, a whole row 8.1).
constexpr int64_t SPLIT_GRID = 512, SPLIT_SPAN = 16384;
constexpr int64_t SMALL_ROW = 512, ONE_WAVE = 4096;  // see lp_fwd
int parts_of(int64_t rows, int64_t V) {
  const int64_t room = SPLIT_GRID / rows, most = V <= 2 * SPLIT_SPAN ? 1 : (V + SPLIT_SPAN - 1) / SPLIT_SPAN;
  const int64_t n = room < most ? room : most;
  return n < 2 ? 1 : (int)(n < MAX_PARTS ? n : MAX_PARTS);
}
int span_of(int64_t V, int parts) { return (int)(((V + parts - 1) / parts + 7) / 8 * 8); }

// With alternatives (20 of bf16 rows here): a wave a row for many short rows (8192 x
// 2000: 22 us, 256 threads 44; 64 x 2000: 7.8 and 7.6), 256 threads while a row is
// one tile of theirs (2048 x 8000: 17 us, 512 threads 24; x 9000: 27 and 24), 512
// for many rows (16384 x 32000: 279 us, 1024 threads 365), 1024 for few (256 x
// 32000: 9.8 us, 512 threads 12.4; 8 x 32000: 8.1 and 11.3).  A part: 512 threads
// while it is one tile of theirs (16 x 131072, 5 alternatives: 10.2 us, 1024 threads
// 11.4), 1024 past that, where rows or parts are too many for more of them (100 x
// 100000 in 5 parts of 20000: 18.6 us, 512 threads 21.2; 1 x 1000000 in 32: 13.3
// and 16.6).
//
// A launch has fewer than 2^32 threads, so more rows than these go in several
// (1024 threads a row at most).
constexpr int64_t LAUNCH_ROWS = 1 << 21;
template <typename T>
void fwd_launch(const T* x, int64_t stride, int64_t rows, const Out& out, Parts p, hipStream_t st) {
  const dim3 grid((unsigned)(rows * p.parts)), block(LP_THREADS);
  const bool split = p.parts > 1;
  if (out.top > 0) {
    if (split && p.span <= 8 * 512 * PIECES)
      hipLaunchKernelGGL((lp_top<T, 512, true>), grid, dim3(512), 0, st, x, stride, out, p);
    else if (split)
      hipLaunchKernelGGL((lp_top<T, 1024, true>), grid, dim3(1024), 0, st, x, stride, out, p);
    else if (out.V <= 8 * 64 * PIECES && rows >= 1024)
      hipLaunchKernelGGL((lp_top<T, 64, false>), grid, dim3(64), 0, st, x, stride, out, p);
    else if (out.V <= 8 * 256 * PIECES)
      hipLaunchKernelGGL((lp_top<T, 256, false>), grid, dim3(256), 0, st, x, stride, out, p);
    else if (rows > 256)
      hipLaunchKernelGGL((lp_top<T, 512, false>), grid, dim3(512), 0, st, x, stride, out, p);
    else
      hipLaunchKernelGGL((lp_top<T, 1024, false>), grid, dim3(1024), 0, st, x, stride, out, p);
  } else if (split) {
    hipLaunchKernelGGL((lp_fwd<T, 256, true, false>), grid, block, 0, st, x, stride, rows, out, p);
  } else if (out.V <= SMALL_ROW) {
    hipLaunchKernelGGL((lp_fwd<T, 16, false, false>), dim3((unsigned)((rows + 15) / 16)), block, 0, st, x, stride, rows,
                       out, p);
  } else if (out.V <= ONE_WAVE) {
    hipLaunchKernelGGL((lp_fwd<T, 64, false, false>), dim3((unsigned)((rows + 3) / 4)), block, 0, st, x, stride, rows, out, p);
  } else if (sizeof(T) == 2 && rows * out.V * 2 >= FAR_BYTES) {
    hipLaunchKernelGGL((lp_fwd<T, 256, false, sizeof(T) == 2>), grid, block, 0, st, x, stride, rows, out, p);
  } else {
    hipLaunchKernelGGL((lp_fwd<T, 256, false, false>), grid, block, 0, st, x, stride, rows, out, p);
  }
  if (split) hipLaunchKernelGGL((lp_join<T>), dim3((unsigned)rows), dim3(JOIN_THREADS), 0, st, x, stride, out, p);
}

template <typename T>
void bwd_launch(const T* x, int64_t stride, int64_t rows, const int64_t* tokens, const float* stats,
                const float* entropy, const int64_t* top_tokens, const float* dlp, const float* dent,
                const float* dtop, T* dx, int64_t V, int32_t top, int64_t ignore, hipStream_t st) {
  const bool alternatives = dtop && top > 0;
  // a row's columns over several workgroups where rows do not fill the chip
  int64_t parts = 512 / rows, most = V / 8192;
  parts = parts < most ? parts : most;
  parts = parts < 1 ? 1 : parts;
  const int span = span_of(V, (int)parts);
  const int64_t items = rows * parts;
#define GMDN_LP_BWD(NT, TPR, TOP)                                                                                    \
  hipLaunchKernelGGL((lp_bwd<T, NT, TPR, TOP>), dim3((unsigned)((items + NT / TPR - 1) / (NT / TPR))), dim3(NT), 0, \
                     st, x, stride, rows, tokens, stats, entropy, top_tokens, dlp, dent, dtop, dx, (int)V, top,     \
                     ignore, span, (int)parts)
  if (alternatives)
    GMDN_LP_BWD(256, 256, true);
  else if (V <= SMALL_ROW)
    GMDN_LP_BWD(256, 16, false);
  else if (V <= ONE_WAVE)
    GMDN_LP_BWD(256, 64, false);
  else if (V <= 8 * 256 * PIECES)
    GMDN_LP_BWD(256, 256, false);
  else
    GMDN_LP_BWD(1024, 1024, false);
#undef GMDN_LP_BWD
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

size_t gmdn_logprobs_fwd_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) {
  if (check_lp(rows, vocab, 0, top, GMDN_DTYPE_F32) != GMDN_OK || rows == 0) return 0;
  const int64_t items = rows * parts_of(rows, vocab);
  return items == rows ? 0 : (size_t)(items * (16 + 8 * top));
}

int gmdn_logprobs_fwd(const void* logits, const int64_t* tokens, float* logprob, float* entropy, float* top_logprobs,
                      int64_t* top_tokens, float* stats, void* workspace, size_t workspace_bytes, int64_t rows,
                      int64_t vocab, int64_t stride, int32_t top, int64_t ignore_index, int32_t dtype, void* stream) {
  const int rc = check_lp(rows, vocab, stride, top, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!logits || !tokens || !logprob || !entropy || !stats || (top && (!top_logprobs || !top_tokens)))
    return GMDN_ERR_ARG;
  const size_t need = gmdn_logprobs_fwd_workspace_bytes(rows, vocab, top);
  if (need && (!workspace || workspace_bytes < need)) return GMDN_ERR_WORKSPACE;
  const Out out{tokens, ignore_index, logprob, entropy, stats, top_logprobs, top_tokens, (int)vocab, top};
  const int parts = parts_of(rows, vocab);
  // the keys first: 8-byte values at the workspace's start, the sums behind them
  uint64_t* best = static_cast<uint64_t*>(workspace);
  const Parts p{need ? reinterpret_cast<Sums*>(best + rows * parts * top) : nullptr, best, parts, span_of(vocab, parts)};
  for (int64_t r = 0; r < rows; r += LAUNCH_ROWS) {
    const int64_t n = rows - r < LAUNCH_ROWS ? rows - r : LAUNCH_ROWS;
    if (dtype == GMDN_DTYPE_BF16)
      fwd_launch((const bf16*)logits + r * stride, stride, n, out.from(r), p, (hipStream_t)stream);
    else
      fwd_launch((const float*)logits + r * stride, stride, n, out.from(r), p, (hipStream_t)stream);
  }
  return launched();
}

int gmdn_logprobs_bwd(const void* logits, const int64_t* tokens, const float* stats, const float* entropy,
                      const int64_t* top_tokens, const float* dlogprob, const float* dentropy, const float* dtop,
                      void* dlogits, int64_t rows, int64_t vocab, int64_t stride, int32_t top, int64_t ignore_index,
                      int32_t dtype, void* stream) {
  const int rc = check_lp(rows, vocab, stride, top, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!logits || !tokens || !stats || !entropy || !dlogits || (dtop && top && !top_tokens)) return GMDN_ERR_ARG;
  auto launch = [&](auto* x, auto* dx, int64_t r, int64_t n) {
    bwd_launch(x + r * stride, stride, n, tokens + r, stats + 2 * r, entropy + r,
               top_tokens ? top_tokens + r * top : nullptr, dlogprob ? dlogprob + r : nullptr,
               dentropy ? dentropy + r : nullptr, dtop ? dtop + r * top : nullptr, dx + r * vocab, vocab, top,
               ignore_index, (hipStream_t)stream);
  };
  for (int64_t r = 0; r < rows; r += LAUNCH_ROWS) {
    const int64_t n = rows - r < LAUNCH_ROWS ? rows - r : LAUNCH_ROWS;
    if (dtype == GMDN_DTYPE_BF16)
      launch((const bf16*)logits, (bf16*)dlogits, r, n);
    else
      launch((const float*)logits, (float*)dlogits, r, n);
  }
  return launched();
}

}  // extern "C"
