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
#include "../../include/gmdn_lm.h"
#include <float.h>
#include "rows8.h"

namespace gmdn {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
// Differences of logits are clamped here where they multiply a sum: e^-200
// is 0 in float32, and 0 times the clamped value is 0, not NaN.
constexpr float FAR = -200.f;

GMDN_DEV float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

struct Sums {
  float m, s, w;
};
GMDN_DEV Sums no_sums() { return {-FLT_MAX, 0.f, 0.f}; }

// Rescale to the maximum m >= a.m.  NaN stays in s; an infinite m makes its
// own terms NaN.
GMDN_DEV void rescale(Sums& a, float m) {
  const float u = fmaxf(a.m - m, FAR), k = exp_of(u);
  a.w = k * (a.w + u * a.s);
  a.s *= k;
  a.m = m;
}
GMDN_DEV float max8(const float (&x)[8]) {
  return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
}
GMDN_DEV void add8(Sums& a, const float (&x)[8], float most) {
  const float m = fmaxf(a.m, most);
  rescale(a, m);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = x[j] - m, e = exp_of(u);
    a.s += e;
    a.w += e * fmaxf(u, FAR);
  }
}
GMDN_DEV void add8(Sums& a, const float (&x)[8]) { add8(a, x, max8(x)); }

// The row's sums from its threads': the maximum of all, then s and w at it.
template <int NT>
GMDN_DEV Sums join(Sums a, float (*red)[16]) {
  constexpr int W = NT / 64;
  float m = lanes_max<64>(a.m);
  if (lane_id() == 0) red[0][wave_id()] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, red[0][i]);
  rescale(a, m);
  const float s = lanes_sum<64>(a.s), w = lanes_sum<64>(a.w);
  if (lane_id() == 0) {
    red[1][wave_id()] = s;
    red[2][wave_id()] = w;
  }
  __syncthreads();
  a.s = a.w = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    a.s += red[1][i];
    a.w += red[2][i];
  }
  return a;
}

// What a row's sums say.  No logit above -inf: s = 0, and the row's
// distribution is empty (stats -inf, 0).
struct Row {
  float m, logs, entropy;
  bool empty;
  GMDN_DEV float logprob(float x) const { return empty ? -INFINITY : x - m - logs; }
};
GMDN_DEV Row row_of(const Sums& a) {
  if (a.s == 0.f) return {-INFINITY, 0.f, 0.f, true};
  const float logs = logf(a.s), h = logs - a.w / a.s;
  return {a.m, logs, h < 0.f ? 0.f : h, false};
}

template <typename T>
GMDN_DEV void write_row(const Row& r, const T* x, int64_t token, int64_t ignore, int V, int64_t row, float* lp,
                        float* entropy, float* stats) {
  float l = 0.f;
  if (token != ignore) l = token >= 0 && token < V ? r.logprob((float)x[token]) : NAN;
  lp[row] = l;
  entropy[row] = r.entropy;
  stats[2 * row] = r.m;
  stats[2 * row + 1] = r.logs;
}

constexpr int PIECES = 4;  // pieces a thread loads before it works on them

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
lp_fwd(const T* __restrict__ logits, const int64_t* __restrict__ tokens, float* __restrict__ lp,
       float* __restrict__ entropy, float* __restrict__ stats, int V, int64_t stride, int64_t ignore) {
  __shared__ float red[3][16];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  Sums a = no_sums();
  int c0 = 8 * threadIdx.x;
  for (; c0 + 8 * NT * (PIECES - 1) + 8 <= V; c0 += 8 * NT * PIECES) {
    Raw8<T> raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i].load(x + c0 + 8 * NT * i, 8);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      float v[8];
      raw[i].get(v);
      add8(a, v);
    }
  }
  for (; c0 < V; c0 += 8 * NT) {
    float v[8];
    load8(x + c0, V - c0, v, -INFINITY);
    add8(a, v);
  }
  a = join<NT>(a, red);
  if (threadIdx.x == 0) write_row(row_of(a), x, tokens[row], ignore, V, row, lp, entropy, stats);
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

constexpr int TOP_MAX = 32;
constexpr int TOP_PIECES = 4;    // pieces a thread holds of a tile
constexpr int TOP_LIST = 1024;   // candidates of a tile

GMDN_DEV uint64_t lanes_max64(uint64_t x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = ((uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), o, 64) << 32) |
                       (uint32_t)__shfl_xor((int)(uint32_t)x, o, 64);
    x = y > x ? y : x;
  }
  return x;
}

// The row goes by in tiles of NT x 4 pieces held in registers.  Of a tile,
// threads of the same lane number form 64 groups; the top-th best of the 64
// groups' best logits bounds the tile's top-th best from below, and few
// logits reach it (24 of random ones for 20 wanted: each group's pieces lie
// 512 apart, so that neighbours do not share a group).  A group's best is its
// largest value with the last index of the first piece that has it, which no
// better logit of that value exceeds: equal logits, masked ones above all,
// stay out of the list by their index.  Those that reach the bound join the best
// of the tiles before in the list, and a logit's rank is the number of better
// ones in it.  A tile that gives more than the list holds, or a row with a
// NaN, is done over by `slow_top`.
template <typename T, int NT>
GMDN_DEV void slow_top(const T* x, int V, int top, uint64_t* run, uint64_t* red) {
  uint64_t prev = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int c = threadIdx.x; c < V; c += NT) {
      const uint64_t key = key_of((float)x[c], c);
      if (key < prev && key > best) best = key;
    }
    best = lanes_max64(best);
    __syncthreads();
    if (lane_id() == 0) red[wave_id()] = best;
    __syncthreads();
    prev = red[0];
    for (int i = 1; i < NT / 64; ++i) prev = red[i] > prev ? red[i] : prev;
    if (threadIdx.x == 0) run[k] = prev;
  }
  __syncthreads();
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
lp_top(const T* __restrict__ logits, const int64_t* __restrict__ tokens, float* __restrict__ lp,
       float* __restrict__ entropy, float* __restrict__ top_lp, int64_t* __restrict__ top_tokens,
       float* __restrict__ stats, int V, int64_t stride, int top, int64_t ignore) {
  constexpr int TILE = NT * TOP_PIECES * 8;
  __shared__ float red[3][16];
  __shared__ uint64_t red64[16];
  __shared__ uint64_t best[NT];
  __shared__ uint64_t list[TOP_LIST + TOP_MAX];
  __shared__ uint64_t run[2][TOP_MAX];
  __shared__ uint64_t bound;
  __shared__ int count;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  Sums a = no_sums();
  int have = 0, cur = 0;  // of the best so far, and which half of run holds them
  bool over = false;
  for (int c0 = 0; c0 < V; c0 += TILE) {
    float v[TOP_PIECES][8];
#pragma unroll
    for (int i = 0; i < TOP_PIECES; ++i) {
      const int c = c0 + 8 * (i * NT + tid);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = -INFINITY;
      if (c < V) load8(x + c, V - c, v[i], -INFINITY);
    }
    // the thread's best: its value, and the first piece that has it
    float bv = -INFINITY;
    int bp = 0;
#pragma unroll
    for (int i = 0; i < TOP_PIECES; ++i) {
      const float pm = max8(v[i]);
      add8(a, v[i], pm);
      if (pm > bv) {
        bv = pm;
        bp = i;
      }
    }
    if (over) continue;
    best[tid] = c0 + 8 * tid < V ? key_of(bv, c0 + 8 * (bp * NT + tid) + 7) : 0;
    if (tid == 0) count = 0;
    __syncthreads();
    if (wave_id() == 0) {
      uint64_t k = best[tid];
#pragma unroll
      for (int i = 1; i < NT / 64; ++i) {
        const uint64_t o = best[i * 64 + tid];
        k = o > k ? o : k;
      }
      int rank = 0;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, i);
        rank += o > k || (o == k && i < tid);  // equal only where there is none
      }
      if (rank == top - 1) bound = have == top && run[cur][top - 1] > k ? run[cur][top - 1] : k;
    }
    __syncthreads();
    // by value first: few logits come as far as their keys
    const uint64_t least = bound;
    const float lv = value_of(least);
#pragma unroll
    for (int i = 0; i < TOP_PIECES; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v[i][j] >= lv) {
          const int c = c0 + 8 * (i * NT + tid) + j;
          const uint64_t k = key_of(v[i][j], c);
          if (c < V && k >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < TOP_LIST) list[at] = k;
          }
        }
    __syncthreads();
    int n = count;
    over = n > TOP_LIST;
    if (!over) {
      if (tid < have) list[n + tid] = run[cur][tid];
      __syncthreads();
      n += have;
      for (int i = tid; i < n; i += NT) {
        const uint64_t k = list[i];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += list[o] > k;
        if (rank < top) run[cur ^ 1][rank] = k;
      }
      have = n < top ? n : top;
      cur ^= 1;
    }
    __syncthreads();
  }
  a = join<NT>(a, red);
  const Row r = row_of(a);
  if (over || a.s != a.s) slow_top<T, NT>(x, V, top, run[cur], red64);
  if (tid == 0) write_row(r, x, tokens[row], ignore, V, row, lp, entropy, stats);
  if (tid < top) {
    const int i = index_of(run[cur][tid]);
    top_tokens[row * top + tid] = i;
    top_lp[row * top + tid] = r.logprob((float)x[i]);
  }
}

// ------------------------------------------------------------------ backward
// A workgroup takes `span` columns of a row.  The columns of the token and
// the alternatives are written again with their terms once the others are.
constexpr int LPB_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(LPB_THREADS)
lp_bwd(const T* __restrict__ logits, const int64_t* __restrict__ tokens, const float* __restrict__ stats,
       const float* __restrict__ entropy, const int64_t* __restrict__ top_tokens, const float* __restrict__ dlp,
       const float* __restrict__ dent, const float* __restrict__ dtop, T* __restrict__ dx, int V, int64_t stride,
       int top, int64_t ignore, int span, int parts) {
  const int64_t row = blockIdx.x / parts;
  const int first = (int)(blockIdx.x % parts) * span, last = first + span < V ? first + span : V;
  const T* x = logits + row * stride;
  T* out = dx + row * V;
  const int64_t token = tokens[row];
  const bool empty = stats[2 * row] == -INFINITY;
  const float m = empty ? 0.f : stats[2 * row], logs = stats[2 * row + 1], h = entropy[row];
  const float gh = dent ? dent[row] : 0.f;
  float gl = dlp && token != ignore ? dlp[row] : 0.f;
  if (token != ignore && (token < 0 || token >= V)) gl = NAN;
  float all = gl;
  if (dtop)
    for (int i = 0; i < top; ++i) all += dtop[row * top + i];
  // the terms of p (0 throughout an empty row), p as the square of e^(l / 2):
  // the exponential flushes results below 2^-126, the product does not
  auto grad = [&](float z) {
    const float l = z - m - logs, e = __builtin_amdgcn_exp2f(l * (0.5f * LOG2E));
    return -e * (e * (all + gh * (fmaxf(l, FAR) + h)));
  };
  for (int c = first + 8 * threadIdx.x; c < last; c += 8 * LPB_THREADS) {
    float v[8];
    load8(x + c, last - c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = grad(v[j]);
    store8(out + c, last - c, v);
  }
  __syncthreads();
  const int n = dtop ? top : 0;
  if ((int)threadIdx.x <= n && !empty) {
    auto which = [&](int i) { return i == 0 ? token : top_tokens[row * top + i - 1]; };
    const int64_t c = which(threadIdx.x);
    if (c >= first && c < last) {
      float g = 0.f;
      for (int i = 0; i <= n; ++i)
        if (which(i) == c) g += i == 0 ? gl : dtop[row * top + i - 1];
      out[c] = (T)(grad((float)x[c]) + g);
    }
  }
}

int check_lp(int64_t rows, int64_t V, int64_t stride, int32_t top, int32_t dtype) {
  if (rows < 0 || V <= 0 || stride < 0 || top < 0 || top > V) return GMDN_ERR_ARG;
  if (!type_ok(dtype) || top > TOP_MAX || V > (1 << 30)) return GMDN_ERR_UNSUPPORTED;
  if (rows >= ((int64_t)1 << 31)) return GMDN_ERR_ARG;
  return GMDN_OK;
}

template <typename T>
void fwd_launch(const T* x, const int64_t* tokens, float* lp, float* entropy, float* top_lp, int64_t* top_tokens,
                float* stats, int64_t rows, int64_t V, int64_t stride, int32_t top, int64_t ignore, hipStream_t st) {
  const dim3 grid((unsigned)rows);
  if (top > 0) {
    if (V <= 8192)
      hipLaunchKernelGGL((lp_top<T, 256>), grid, dim3(256), 0, st, x, tokens, lp, entropy, top_lp, top_tokens, stats,
                         (int)V, stride, top, ignore);
    else
      hipLaunchKernelGGL((lp_top<T, 1024>), grid, dim3(1024), 0, st, x, tokens, lp, entropy, top_lp, top_tokens, stats,
                         (int)V, stride, top, ignore);
  } else {
    hipLaunchKernelGGL((lp_fwd<T, 256>), grid, dim3(256), 0, st, x, tokens, lp, entropy, stats, (int)V, stride, ignore);
  }
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

int gmdn_logprobs_fwd(const void* logits, const int64_t* tokens, float* logprob, float* entropy, float* top_logprobs,
                      int64_t* top_tokens, float* stats, int64_t rows, int64_t vocab, int64_t stride, int32_t top,
                      int64_t ignore_index, int32_t dtype, void* stream) {
  const int rc = check_lp(rows, vocab, stride, top, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!logits || !tokens || !logprob || !entropy || !stats || (top && (!top_logprobs || !top_tokens)))
    return GMDN_ERR_ARG;
  if (dtype == GMDN_DTYPE_BF16)
    fwd_launch((const bf16*)logits, tokens, logprob, entropy, top_logprobs, top_tokens, stats, rows, vocab, stride, top,
               ignore_index, (hipStream_t)stream);
  else
    fwd_launch((const float*)logits, tokens, logprob, entropy, top_logprobs, top_tokens, stats, rows, vocab, stride,
               top, ignore_index, (hipStream_t)stream);
  return launched();
}

int gmdn_logprobs_bwd(const void* logits, const int64_t* tokens, const float* stats, const float* entropy,
                      const int64_t* top_tokens, const float* dlogprob, const float* dentropy, const float* dtop,
                      void* dlogits, int64_t rows, int64_t vocab, int64_t stride, int32_t top, int64_t ignore_index,
                      int32_t dtype, void* stream) {
  const int rc = check_lp(rows, vocab, stride, top, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!logits || !tokens || !stats || !entropy || !dlogits || (dtop && !top_tokens)) return GMDN_ERR_ARG;
  const int64_t parts = 1, span = (vocab + 7) / 8 * 8;
  const dim3 grid((unsigned)(rows * parts)), block(LPB_THREADS);
  if (dtype == GMDN_DTYPE_BF16)
    hipLaunchKernelGGL(lp_bwd<bf16>, grid, block, 0, (hipStream_t)stream, (const bf16*)logits, tokens, stats, entropy,
                       top_tokens, dlogprob, dentropy, dtop, (bf16*)dlogits, (int)vocab, stride, top, ignore_index,
                       (int)span, (int)parts);
  else
    hipLaunchKernelGGL(lp_bwd<float>, grid, block, 0, (hipStream_t)stream, (const float*)logits, tokens, stats, entropy,
                       top_tokens, dlogprob, dentropy, dtop, (float*)dlogits, (int)vocab, stride, top, ignore_index,
                       (int)span, (int)parts);
  return launched();
}

}  // extern "C"
