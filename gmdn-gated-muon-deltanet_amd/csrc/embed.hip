// Token embedding and its gradient (include/gmdn_lm.h).
//
//   y_i = s W[t_i],     dW[v] = s sum over the i with t_i = v of dy_i
//
// Memory bound both ways where the table is large: 16384 tokens of 131072 x 4096 bf16 take
// 55 us forward (4.9 TB/s) and their sums 229 us (5.2 TB/s, nine tenths of it zeros of the
// table); for 32000 x 1024 the gradient is 25 us of sums beside 23 of the sort, on 16
// workgroups, and 5 of the join.  The forward copies rows.  The gradient is a sum by
// token in a fixed order, without atomics on values: the positions are sorted
// by token (a stable radix sort, so equal tokens keep their order), blocks of
// the sorted positions add the rows of dy they name, and a token whose run
// crosses blocks is joined from their partial sums, in order.  Rows of dW that
// no token names are zeroed beside the sums, in the same launch.
#include "../../include/gmdn_lm.h"
#include "rows8.h"

namespace gmdn {
namespace {

// ------------------------------------------------------------------ forward
constexpr int EM_THREADS = 256;

// A thread for each piece of eight values of y.
template <typename T>
__global__ void __launch_bounds__(EM_THREADS)
em_gather(const T* __restrict__ w, const int64_t* __restrict__ tokens, T* __restrict__ y, uint32_t pieces,
          uint32_t per_row, int d, int64_t vocab, int64_t ws, float scale) {
  const uint32_t i = blockIdx.x * EM_THREADS + threadIdx.x;
  if (i >= pieces) return;
  const int64_t row = i / per_row;
  const int c = 8 * (int)(i % per_row);
  const int64_t token = tokens[row];
  float v[8];
  if (token >= 0 && token < vocab) {
    load8(w + token * ws + c, d - c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __builtin_nanf("");
  }
  store8(y + row * d + c, d - c, v);
}

// ---------------------------------------------------- positions by token
// Least significant digit first, up to 9 bits a pass.  A workgroup moves one
// tile of consecutive positions; where they go follows from how often each
// digit comes in all tiles and in the earlier ones, counted by a launch before it
// (workgroups that count all tokens themselves instead save it, and lose: the whole
// gradient of 16384 tokens of 32000 x 1024 took 62 us so and takes 52, of 64 tokens 34 and 28,
// of 65536 161 and 109).  Tokens outside the vocabulary and the padding token get the key
// `vocab`, behind all others.
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WAVES = SORT_THREADS / 64;
constexpr int SORT_BITS = 9;
constexpr int SORT_BINS = 1 << SORT_BITS;
constexpr int SORT_TILES = 256;          // at most; a tile is a multiple of SORT_THREADS

struct SortInput {
  const int64_t* tokens;  // the first pass's, else null
  const uint32_t *keys, *at;
  int64_t n, vocab, padding;
  GMDN_DEV uint32_t key(int64_t i) const {
    if (!tokens) return keys[i];
    const int64_t t = tokens[i];
    return (uint32_t)(t >= 0 && t < vocab && t != padding ? t : vocab);
  }
  GMDN_DEV uint32_t position(int64_t i) const { return tokens ? (uint32_t)i : at[i]; }
};

// The lanes of the wave that hold the same digit (none for a lane that is not live).
GMDN_DEV uint64_t same_digit(uint32_t digit, bool live, int bits) {
  uint64_t m = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const bool set = (digit >> b) & 1;
    const uint64_t with = __ballot(set);
    m &= set ? with : ~with;
  }
  return live ? m : 0;
}

// counts[digit * tiles + tile]
__global__ void __launch_bounds__(SORT_THREADS)
em_count(SortInput in, uint32_t* __restrict__ counts, int64_t tile, int shift, int bits) {
  __shared__ uint32_t bins[SORT_BINS];
  const int t = threadIdx.x;
  if (t < SORT_BINS) bins[t] = 0;
  __syncthreads();
  const int64_t first = blockIdx.x * tile;
  for (int64_t i0 = first; i0 < first + tile && i0 < in.n; i0 += SORT_THREADS) {
    const int64_t i = i0 + t;
    const bool live = i < in.n;
    const uint32_t digit = live ? (in.key(i) >> shift) & ((1u << bits) - 1) : 0;
    const uint64_t peers = same_digit(digit, live, bits);
    if (live && (peers & ((1ull << lane_id()) - 1)) == 0) atomicAdd(&bins[digit], (uint32_t)__popcll(peers));
  }
  __syncthreads();
  if (t < SORT_BINS) counts[(int64_t)t * gridDim.x + blockIdx.x] = bins[t];
}

__global__ void __launch_bounds__(SORT_THREADS)
em_scatter(SortInput in, const uint32_t* __restrict__ counts, uint32_t* __restrict__ keys, uint32_t* __restrict__ at,
           int64_t tile, int shift, int bits) {
  __shared__ uint32_t waves[SORT_WAVES][SORT_BINS];
  __shared__ uint32_t sums[SORT_BINS / 64];
  const int t = threadIdx.x, w = wave_id();
  const uint64_t before = (1ull << lane_id()) - 1;
  const int64_t first = blockIdx.x * tile;
  // how often each digit comes, and where the smaller ones of a wave's 64 end
  uint32_t mine = 0, below = 0, run = 0;
  if (t < SORT_BINS) {
    for (unsigned i = 0; i < gridDim.x; ++i) {
      const uint32_t c = counts[(int64_t)t * gridDim.x + i];
      mine += c;
      below += i < blockIdx.x ? c : 0;
    }
    run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = (uint32_t)__shfl_up((int)run, o, 64);
      if (lane_id() >= o) run += u;
    }
    if (lane_id() == 63) sums[w] = run;
  }
  __syncthreads();
  // where each digit of this tile starts: the smaller digits, and its own in earlier tiles
  uint32_t base = 0;
  if (t < SORT_BINS) {
    for (int i = 0; i < w; ++i) base += sums[i];
    base += run - mine + below;
  }
  for (int64_t i0 = first; i0 < first + tile && i0 < in.n; i0 += SORT_THREADS) {
    for (int i = t; i < SORT_WAVES * SORT_BINS; i += SORT_THREADS) (&waves[0][0])[i] = 0;
    __syncthreads();
    const int64_t i = i0 + t;
    const bool live = i < in.n;
    const uint32_t key = live ? in.key(i) : 0, digit = (key >> shift) & ((1u << bits) - 1);
    const uint64_t peers = same_digit(digit, live, bits);
    const uint32_t rank = (uint32_t)__popcll(peers & before);
    if (live && rank == 0) waves[w][digit] = (uint32_t)__popcll(peers);
    __syncthreads();
    if (t < SORT_BINS) {
#pragma unroll
      for (int i = 0; i < SORT_WAVES; ++i) {
        const uint32_t c = waves[i][t];
        waves[i][t] = base;
        base += c;
      }
    }
    __syncthreads();
    if (live) {
      const uint32_t to = waves[w][digit] + rank;
      keys[to] = key;
      at[to] = in.position(i);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ sums
// Blocks of `block` sorted positions, TPR threads of 8 columns each; wider rows
// are shared by workgroups along the grid's y.  A run of equal tokens inside one
// block is a whole row of dW.  One that goes on into the next block leaves its
// sum in part (blocks, 2, d): slot 0 where it came from the block before, slot 1
// where it begins here.
struct Sorted {
  const uint32_t *keys, *at;
  int64_t n, vocab;
  // first position in [lo, hi) whose key is not below k (hi without one)
  GMDN_DEV int64_t lower(uint32_t k, int64_t lo, int64_t hi) const {
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < k)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo;
  }
  // The same over all positions by the two halves of a wave, each for its own k: 32
  // probes a step, three steps for 16384 positions where a bisection waits for memory
  // fourteen times.
  GMDN_DEV int64_t lower_half_wave(uint32_t k) const {
    const int i = lane_id() & 31, shift = lane_id() & 32;
    int64_t lo = 0, hi = n;
    while (__ballot(lo < hi) != 0) {
      const int64_t step = (hi - lo + 31) / 32, p = lo + i * step;
      const uint32_t below = (uint32_t)(__ballot(p < hi && keys[p] < k) >> shift);
      const int c = __popcll(below);  // probes below k: the first c
      const int64_t next = lo + c * step;
      lo = c ? next - step + 1 : lo;
      hi = next < hi ? next : hi;
    }
    return lo;
  }
};

constexpr int SUM_AHEAD = 8;   // rows of dy in flight
constexpr int ZERO_ROWS = 64;  // rows of dW that a zeroing workgroup looks after: a wave's lanes

template <typename T, int TPR>
__global__ void __launch_bounds__(EM_THREADS)
em_sums(Sorted s, const T* __restrict__ dy, T* __restrict__ dw, float* __restrict__ part, int64_t block,
        unsigned sum_groups, int d, int64_t ds, float scale) {
  constexpr int GROUPS = EM_THREADS / TPR;
  const int g = threadIdx.x / TPR, t = threadIdx.x % TPR;
  if (blockIdx.x >= sum_groups) {
    __shared__ int absent[ZERO_ROWS];
    const int64_t v0 = (int64_t)(blockIdx.x - sum_groups) * ZERO_ROWS;
    const int64_t v1 = v0 + ZERO_ROWS < s.vocab ? v0 + ZERO_ROWS : s.vocab;
    if (threadIdx.x < 64) {
      // Where the keys of these rows begin and end, and between them each lane's row by
      // bisection (looking at every key is no faster where the rows have few: 16384 tokens of
      // 32000 x 1024 take the same; of 65536 of 32000 x 256, nine in ten one token, the whole
      // gradient takes 172 us so and 155 by bisection).
      const int64_t p = s.lower_half_wave((uint32_t)(threadIdx.x < 32 ? v0 : v1));
      const int64_t lo = __shfl(p, 0, 64), hi = __shfl(p, 32, 64), v = v0 + threadIdx.x;
      const int64_t at = s.lower((uint32_t)v, lo, hi);
      absent[threadIdx.x] = v < v1 && !(at < hi && s.keys[at] == (uint32_t)v);
    }
    __syncthreads();
    const float zero[8] = {};
    const int c = 8 * (blockIdx.y * TPR + t);
    if (c < d)
      for (int r = g; r < ZERO_ROWS; r += GROUPS)
        if (absent[r]) store8(dw + (v0 + r) * d + c, d - c, zero);
    return;
  }
  const int64_t b = (int64_t)blockIdx.x * GROUPS + g;
  const int64_t p0 = b * block, p1 = p0 + block < s.n ? p0 + block : s.n;
  const int c = 8 * (blockIdx.y * TPR + t);
  if (p0 >= s.n || c >= d) return;
  uint32_t cur = s.keys[p0];
  bool from_before = p0 > 0 && s.keys[p0 - 1] == cur;
  float sum[8] = {};
  auto flush = [&](bool goes_on) {
    if (cur >= s.vocab) return;
    if (from_before || goes_on) {
      store8(part + (2 * b + (from_before ? 0 : 1)) * d + c, d - c, sum);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] *= scale;
      store8(dw + (int64_t)cur * d + c, d - c, sum);
    }
  };
  // the next rows' places are loaded beside these rows
  uint32_t key[SUM_AHEAD], next_key[SUM_AHEAD], next_at[SUM_AHEAD];
  auto places = [&](int64_t p) {
#pragma unroll
    for (int i = 0; i < SUM_AHEAD; ++i) {
      const int64_t q = p + i < p1 ? p + i : p1 - 1;
      next_key[i] = s.keys[q];
      next_at[i] = s.at[q];
    }
  };
  places(p0);
  for (int64_t p = p0; p < p1; p += SUM_AHEAD) {
    Raw8<T> raw[SUM_AHEAD];
#pragma unroll
    for (int i = 0; i < SUM_AHEAD; ++i) {
      raw[i].load(dy + (int64_t)next_at[i] * ds + c, d - c);
      key[i] = next_key[i];
    }
    places(p + SUM_AHEAD);
#pragma unroll
    for (int i = 0; i < SUM_AHEAD; ++i) {
      if (p + i >= p1) break;
      if (key[i] != cur) {
        flush(false);
        cur = key[i];
        from_before = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = 0.f;
      }
      float v[8];
      raw[i].get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += v[j];
    }
  }
  flush(p1 < s.n && s.keys[p1] == cur);
}

// The runs that cross blocks: the block where one begins adds its parts.
template <typename T, int TPR>
__global__ void __launch_bounds__(EM_THREADS)
em_join(Sorted s, const float* __restrict__ part, T* __restrict__ dw, int64_t block, int d, float scale) {
  constexpr int GROUPS = EM_THREADS / TPR;
  const int64_t b = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;
  const int64_t p0 = b * block, p1 = p0 + block;
  const int c = 8 * (blockIdx.y * TPR + threadIdx.x % TPR);
  if (p1 >= s.n) return;
  const uint32_t k = s.keys[p1];
  if (k >= s.vocab || s.keys[p1 - 1] != k || (p0 > 0 && s.keys[p0] == k && s.keys[p0 - 1] == k)) return;
  // The block where the run ends: the first whose successor begins with another
  // token.  Each lane of the group looks at one (a group's lanes are here together).
  constexpr int LANES = TPR < 64 ? TPR : 64;
  const int i = lane_id() % LANES, shift = lane_id() - i;
  int64_t last = b + 1;
  for (;; last += LANES) {
    const int64_t q = (last + i + 1) * block;
    const uint64_t ends = __ballot(q >= s.n || s.keys[q] != k) >> shift & (~0ull >> (64 - LANES));
    if (ends) {
      last += __builtin_ctzll(ends);
      break;
    }
  }
  if (c >= d) return;
  float sum[8];
  load8(part + (2 * b + 1) * d + c, d - c, sum);
  for (int64_t i = b + 1; i <= last; i += SUM_AHEAD) {
    Raw8<float> raw[SUM_AHEAD];
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j) raw[j].load(part + 2 * (i + j <= last ? i + j : last) * d + c, d - c);
#pragma unroll
    for (int j = 0; j < SUM_AHEAD; ++j) {
      if (i + j > last) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += raw[j].v[e];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] *= scale;
  store8(dw + (int64_t)k * d + c, d - c, sum);
}

template <int N>
struct Threads {
  static constexpr int TPR = N;
};
template <class F>
void with_threads(int64_t d, F&& f) {
  if (d <= 64) f(Threads<8>{});
  else if (d <= 128) f(Threads<16>{});
  else if (d <= 256) f(Threads<32>{});
  else if (d <= 512) f(Threads<64>{});
  else if (d <= 1024) f(Threads<128>{});
  else f(Threads<256>{});
}
template <class F>
void with_type(int32_t dtype, F&& f) {
  if (dtype == GMDN_DTYPE_BF16) f(bf16{});
  else f(float{});
}

// How a gradient's work is cut.  A block adds its positions one after another
// and a token's run of them is joined one after another, so the block grows with the
// square root of the positions.  That is for batches where one token fills much of them:
// 65536 of 32000 x 256, nine in ten a padding token, take 155 us in blocks of 128, 188 of 64,
// 298 of 32; 16384 x 1024, half of them, 75 in blocks of 64, 85 of 32.  Without such a token
// less is better by a little (16384: 62 in blocks of 64, 58 of 32; 65536: 109 of 128, 101 of
// 64), and below 32 nothing is won from a few thousand tokens on.
struct Plan {
  int64_t tile, tiles, block, blocks;
  int passes, bits;
  size_t keys, counts, part;  // bytes
  size_t bytes() const { return 4 * keys + counts + part; }
};
size_t up(size_t n) { return (n + 255) / 256 * 256; }
Plan plan_of(int64_t n, int64_t vocab, int64_t d) {
  Plan p{};
  const int64_t per = (n + SORT_TILES * (int64_t)SORT_THREADS - 1) / (SORT_TILES * (int64_t)SORT_THREADS);
  p.tile = (per > 0 ? per : 1) * SORT_THREADS;
  p.tiles = (n + p.tile - 1) / p.tile;
  int width = 1;
  while ((vocab >> width) != 0) ++width;
  p.passes = (width + SORT_BITS - 1) / SORT_BITS;
  p.bits = (width + p.passes - 1) / p.passes;
  p.block = 32;
  while (p.block * p.block * 8 < n) p.block *= 2;
  p.blocks = (n + p.block - 1) / p.block;
  p.keys = up((size_t)n * 4);
  p.counts = up((size_t)p.tiles * SORT_BINS * 4);
  p.part = up((size_t)p.blocks * 2 * d * 4);
  return p;
}

int check_sizes(int64_t rows, int64_t vocab, int64_t d) {
  if (rows < 0 || vocab <= 0 || d <= 0 || rows > INT32_MAX) return GMDN_ERR_ARG;
  return vocab > (1 << 27) || d > (1 << 20) ? GMDN_ERR_UNSUPPORTED : GMDN_OK;
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

int gmdn_embed_fwd(const void* weight, const int64_t* tokens, void* y, int64_t rows, int64_t vocab, int64_t d,
                   int64_t w_stride, float scale, int32_t dtype, void* stream) {
  const int rc = check_sizes(rows, vocab, d);
  if (rc != GMDN_OK) return rc;
  if (!type_ok(dtype)) return GMDN_ERR_UNSUPPORTED;
  if (w_stride < 0) return GMDN_ERR_ARG;
  if (rows == 0) return GMDN_OK;
  if (!weight || !tokens || !y) return GMDN_ERR_ARG;
  const int64_t per_row = (d + 7) / 8, pieces = rows * per_row, groups = (pieces + EM_THREADS - 1) / EM_THREADS;
  if (pieces > UINT32_MAX - EM_THREADS) return GMDN_ERR_UNSUPPORTED;
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((em_gather<T>), dim3((unsigned)groups), dim3(EM_THREADS), 0, (hipStream_t)stream,
                       (const T*)weight, tokens, (T*)y, (uint32_t)pieces, (uint32_t)per_row, (int)d, vocab, w_stride,
                       scale);
  });
  return launched();
}

size_t gmdn_embed_bwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t d) {
  if (rows <= 0 || check_sizes(rows, vocab, d) != GMDN_OK) return 0;
  return plan_of(rows, vocab, d).bytes();
}

int gmdn_embed_bwd(const void* dy, const int64_t* tokens, void* dweight, void* workspace, size_t workspace_bytes,
                   int64_t rows, int64_t vocab, int64_t d, int64_t dy_stride, float scale, int64_t padding_idx,
                   int32_t dtype, void* stream) {
  const int rc = check_sizes(rows, vocab, d);
  if (rc != GMDN_OK) return rc;
  if (!type_ok(dtype)) return GMDN_ERR_UNSUPPORTED;
  if (dy_stride < 0 || !dweight || (rows > 0 && (!dy || !tokens))) return GMDN_ERR_ARG;
  const Plan p = plan_of(rows, vocab, d);
  if (rows > 0 && (!workspace || workspace_bytes < p.bytes())) return GMDN_ERR_WORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  char* at = (char*)workspace;
  uint32_t* buf[4];
  for (auto& b : buf) {
    b = (uint32_t*)at;
    at += p.keys;
  }
  uint32_t* const counts = (uint32_t*)at;
  float* const part = (float*)(at + p.counts);
  SortInput in{tokens, nullptr, nullptr, rows, vocab, padding_idx};
  int to = 0;
  for (int pass = 0; pass < p.passes && rows > 0; ++pass, to ^= 1) {
    const int shift = pass * p.bits;
    hipLaunchKernelGGL(em_count, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, st, in, counts, p.tile, shift, p.bits);
    hipLaunchKernelGGL(em_scatter, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, st, in, counts, buf[2 * to],
                       buf[2 * to + 1], p.tile, shift, p.bits);
    in.tokens = nullptr;
    in.keys = buf[2 * to];
    in.at = buf[2 * to + 1];
  }
  const Sorted sorted{in.keys, in.at, rows, vocab};
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_threads(d, [&](auto n) {
      constexpr int TPR = decltype(n)::TPR;
      constexpr int GROUPS = EM_THREADS / TPR;
      const unsigned slices = (unsigned)((d + 8 * TPR - 1) / (8 * TPR));
      const unsigned sums = (unsigned)((p.blocks + GROUPS - 1) / GROUPS);
      const unsigned zeros = (unsigned)((vocab + ZERO_ROWS - 1) / ZERO_ROWS);
      hipLaunchKernelGGL((em_sums<T, TPR>), dim3(sums + zeros, slices), dim3(EM_THREADS), 0, st, sorted, (const T*)dy,
                         (T*)dweight, part, p.block, sums, (int)d, dy_stride, scale);
      if (p.blocks > 1)
        hipLaunchKernelGGL((em_join<T, TPR>), dim3(sums, slices), dim3(EM_THREADS), 0, st, sorted, part, (T*)dweight,
                           p.block, (int)d, scale);
    });
  });
  return launched();
}

}  // extern "C"
