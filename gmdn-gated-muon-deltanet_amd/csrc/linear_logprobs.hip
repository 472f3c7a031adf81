// Log probabilities of given tokens from hidden states and the head's weight,
// without the logits, and the gradients of both (include/gmdn_lm.h).
//
// With logits l = x W^T of a row x, its token t and the cotangents gl, gh of the
// two outputs:
//   lp = l_t - M - log s,  H = log s - w / s      (M, s, w: logsums.h)
//   d_v = gl ([v = t] - p_v) - gh p_v (log p_v + H),   p = softmax(l)
//   dx = d W,    dW = d^T x     (over all rows)
//
// Matrix bound: 2 T V D operations a product.  The forward forms tiles of the logits
// in registers and leaves of each row of a tile three sums; they are joined
// by row afterwards.  The backward forms the logits again, a piece of the
// vocabulary at a time, writes the piece's d in bfloat16 and takes both
// products from it: four products in all, and of d no more than PIECE_BYTES of
// memory, or 256 columns of all rows where those are more.
//
// 16384 x 32000 x 1024 bf16: the forward takes 974 us, 1.10 PFLOP/s, and the backward's three
// products 2.77 ms, 1.16; the matrix units are busy for 52% of the forward's clocks, 44% of the
// logits' again, 58% of dx's and 65% of dW's, and no LDS read has a bank conflict.  A tile of 256 reads and copies
// its operands in as many clocks of LDS as its products take, and a tile of logits of k =
// 1024 has only 16 stages beside its first copies and its epilogue.
//
// bfloat16 operands are multiplied as they are; d is rounded to bfloat16 as the
// gradient of bfloat16 logits would be.  float32 operands, and d beside them, are
// split into bfloat16 pieces, each the rounding of what the ones before it leave:
// in 'tf32' two (x = hi + lo up to 2^-18 |x|) multiplied as lo hi + hi lo + hi hi, what
// this library's other float32 products do; in 'ieee' three (up to 2^-27 |x|), with the six
// products above 2^-27, which leaves float32's rounding (1021 x 32003 x 1001, forward and
// backward: 866 us and 1486).
#include "../../include/gmdn_lm.h"
#include <type_traits>
#include "bf16mm.h"
#include "logsums.h"

namespace gmdn {
namespace {

constexpr int64_t PIECE_BYTES = 512 << 20;
constexpr int64_t PIECE_MOST = 1 << 20;   // columns: 256 rows of them within 32 bits of bytes
constexpr int UNIT = 256;                 // a piece's columns: a multiple
constexpr int KPAD = 64;                  // k in planes: a multiple, zeros behind the values
constexpr float HALF_LOG2E = 0.5f * LOG2E;

// ------------------------------------------------------------------ planes
// (rows, d) matrices as P planes (rows, kp) of bfloat16 pieces, zeros behind d: one
// matrix for each y of the grid.
template <typename T>
struct Whole {
  const T* x;
  int64_t stride, rows;
  bf16* out;
};
template <typename T, int P>
__global__ void __launch_bounds__(256)
ll_planes(Whole<T> a, Whole<T> b, int d, int kp) {
  const Whole<T>& m = blockIdx.y == 0 ? a : b;
  const uint32_t per = kp / 8, i = blockIdx.x * 256 + threadIdx.x;  // below 2^32 (check_ll)
  const int64_t r = i / per;
  if (r >= m.rows) return;
  const int c = 8 * (int)(i % per);
  float v[8];
  load8(m.x + r * m.stride + c, d - c, v);
  bf16* o = m.out + r * kp + c;
#pragma unroll
  for (int p = 0; p < P; ++p, o += m.rows * kp) {
    bf16x8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[j] = (bf16)v[j];
      v[j] -= (float)h[j];
    }
    *reinterpret_cast<bf16x8*>(o) = h;
  }
}

// ------------------------------------------------------------------ forward
// m: vocabulary, n: rows of x.  part (tiles of m, 3, rows): each tile's sums.
struct SumsArgs {
  const int64_t* tokens;
  float *at_token, *part;
  int64_t rows;
  int V;
};
GMDN_DEV void join_sums(Sums& a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  a.s += b.s;
  a.w += b.w;
}
template <class S, bool PERM>
struct SumsEpi {
  SumsArgs e;
  GMDN_DEV void operator()(f32x4 (&acc)[S::MT][S::NT], const MMTile& tile, int64_t m0, int64_t n0, int wm, int wn,
                           char* smem) const {
    const int l = lane_id(), G = l >> 4;
    Sums* const waves = reinterpret_cast<Sums*>(smem);  // (WM, TN)
    const int left = e.V - (int)m0;
    if (left < S::TM)  // the vocabulary ends in this tile
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (m_of<PERM>(wm * S::MT + i, G) + q >= left)
#pragma unroll
            for (int j = 0; j < S::NT; ++j) acc[i][j][q] = -INFINITY;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
      const int n = 16 * (wn * S::NT + j) + (l & 15);
      const int64_t row = n0 + n, token = row < e.rows ? e.tokens[row] : -1;
      if (token >= m0 && token < m0 + S::TM && token < e.V)
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (m_of<PERM>(wm * S::MT + i, G) + q == (int)(token - m0)) e.at_token[row] = acc[i][j][q];
      Sums a = no_sums();
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) a.m = fmaxf(a.m, acc[i][j][q]);
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float u = acc[i][j][q] - a.m, x = exp_of(u);
          a.s += x;
          a.w += x * fmaxf(u, FAR);
        }
      // the four lane groups, then the waves along m through LDS
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) join_sums(a, {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.w, o, 64)});
      if (G == 0) waves[wm * S::TN + n] = a;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < S::TN; n += S::THREADS) {
      Sums a = waves[n];
      for (int i = 1; i < S::WM; ++i) join_sums(a, waves[i * S::TN + n]);
      const int64_t row = n0 + n;
      if (row >= e.rows) continue;
      float* const p = e.part + (int64_t)tile.m * 3 * e.rows + row;
      p[0] = a.m;
      p[e.rows] = a.s;
      p[2 * e.rows] = a.w;
    }
  }
};

// A row's sums from its tiles': R rows a workgroup, 256 / R threads each.
template <int R>
__global__ void __launch_bounds__(256)
ll_join(const float* __restrict__ part, const float* __restrict__ at_token, const int64_t* __restrict__ tokens,
        float* __restrict__ lp, float* __restrict__ entropy, float* __restrict__ stats, int tiles, int64_t rows,
        int64_t V, int64_t ignore) {
  constexpr int PER = 256 / R;
  __shared__ Sums all[PER][R];
  const int r = threadIdx.x % R, part_of = threadIdx.x / R;
  const int64_t row = (int64_t)blockIdx.x * R + r;
  Sums a = no_sums();
  if (row < rows)
    for (int i = part_of; i < tiles; i += PER) {
      const float* const p = part + (int64_t)i * 3 * rows + row;
      join_sums(a, {p[0], p[rows], p[2 * rows]});
    }
  all[part_of][r] = a;
  for (int n = PER / 2; n > 0; n /= 2) {
    __syncthreads();
    if (part_of < n) {
      join_sums(a, all[part_of + n][r]);
      all[part_of][r] = a;
    }
  }
  if (part_of != 0 || row >= rows) return;
  const Row w = row_of(a);
  const int64_t token = tokens[row];
  lp[row] = token == ignore ? 0.f : token >= 0 && token < V ? w.logprob(at_token[row]) : NAN;
  entropy[row] = w.entropy;
  stats[2 * row] = w.m;
  stats[2 * row + 1] = w.logs;
}
// One row a workgroup while those are few: the tiles of a large vocabulary are read one
// after another by each thread (forward, 16 x 131072 x 64: 16.5 us, 16 rows a workgroup 47;
// 1024 x 32000 x 256: 33 and 32; 4096: 110 and 105).
constexpr int64_t JOIN_FEW = 1024;

// ------------------------------------------------------------------ backward
// d of a piece of the vocabulary: P planes (padded rows, columns) of bfloat16, zeros
// behind the vocabulary, to the end of its tile of it, and behind the rows.
struct GradArgs {
  const int64_t* tokens;
  const float *stats, *entropy, *dlp, *dent;
  bf16* d;
  int64_t rows, padded, columns, left, first, V, ignore;  // left: the piece's columns inside the vocabulary
};
template <class S, bool PERM, int P>
struct GradEpi {
  GradArgs e;
  GMDN_DEV void operator()(f32x4 (&acc)[S::MT][S::NT], const MMTile&, int64_t m0, int64_t n0, int wm, int wn,
                           char*) const {
    static_assert(PERM && S::MT % 2 == 0, "two tiles hold eight consecutive columns");
    const int l = lane_id(), G = l >> 4;
    const int left = (int)(e.left - m0);  // the tile's columns inside the vocabulary
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
      const int64_t row = n0 + 16 * (wn * S::NT + j) + (l & 15);
      if (row >= e.padded) continue;
      float m = 0.f, logs = 0.f, h = 0.f, gl = 0.f, gh = 0.f;
      int token = -1;  // from the tile's first column
      if (row < e.rows) {
        const int64_t t = e.tokens[row];
        // of a token outside the vocabulary NaN; the entropy's gradient does not see the token
        if (e.dlp && t != e.ignore) gl = t >= 0 && t < e.V ? e.dlp[row] : NAN;
        gh = e.dent ? e.dent[row] : 0.f;
        m = e.stats[2 * row];
        logs = e.stats[2 * row + 1];
        h = e.entropy[row];
        const int64_t from = t - e.first - m0;
        token = from >= 0 && from < S::TM ? (int)from : -1;
      }
      // a row without a gradient has zeros, whatever its logits are
      const bool none = (gl == 0.f && gh == 0.f) || m == -INFINITY;
      const uint32_t keep = none ? 0u : ~0u;
      bf16* const to = e.d + row * e.columns + m0;
      // p as the square of x = e^(log p / 2): the exponential flushes results below 2^-126
      auto columns = [&](auto&& term) {
#pragma unroll
        for (int i = 0; i < S::MT; i += 2) {
          const int c = m_of<PERM>(wm * S::MT + i, G);
          float g[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float u = acc[i + q / 4][j][q % 4] - m - logs;
            g[q] = term(u, __builtin_amdgcn_exp2f(u * HALF_LOG2E));
          }
          if (token >= 0)
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (c + q == token) g[q] += gl;
          if (left < S::TM)  // the vocabulary ends in this tile
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (c + q >= left) g[q] = 0.f;
          bf16* o = to + c;
#pragma unroll
          for (int p = 0; p < P; ++p, o += e.padded * e.columns) {
            const bf16x8 b = cat8(to_bf16x4(f32x4{g[0], g[1], g[2], g[3]}), to_bf16x4(f32x4{g[4], g[5], g[6], g[7]}));
            *reinterpret_cast<u32x4*>(o) = __builtin_bit_cast(u32x4, b) & keep;
            if (p + 1 < P)
#pragma unroll
              for (int q = 0; q < 8; ++q) g[q] -= (float)b[q];
          }
        }
      };
      if (e.dent)
        columns([&](float u, float x) { return -x * (x * (gl + gh * (fmaxf(u, FAR) + h))); });
      else
        columns([&](float, float x) { return -x * (x * gl); });
    }
  }
};

// C (n, m): to `out` in its type, or to float32 planes (splits, n, m); `add`: on
// what the plane holds.
template <typename T>
struct StoreArgs {
  float* plane;
  T* out;
  int64_t M, N;
  bool add;
};
template <class S, typename T>
struct StoreEpi {
  StoreArgs<T> e;
  GMDN_DEV void operator()(f32x4 (&acc)[S::MT][S::NT], const MMTile&, int64_t m0, int64_t n0, int wm, int wn,
                           char*) const {
    const int l = lane_id(), G = l >> 4;
    float* const plane = e.plane ? e.plane + (int64_t)blockIdx.y * e.M * e.N : nullptr;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
      const int64_t n = n0 + 16 * (wn * S::NT + j) + (l & 15);
      if (n >= e.N) continue;
#pragma unroll
      for (int i = 0; i < S::MT; ++i) {
        const int64_t m = m0 + m_of<false>(wm * S::MT + i, G);
        if (m >= e.M) continue;
        f32x4 v = acc[i][j];
        const int64_t at = n * e.M + m;
        const bool whole = m + 4 <= e.M;
        if (e.add) {
          if (whole) {
            v += *reinterpret_cast<const f32x4_any*>(plane + at);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (m + q < e.M) v[q] += plane[at + q];
          }
        }
        if (e.out)
          put(e.out + at, v, whole, e.M - m);
        else
          put(plane + at, v, whole, e.M - m);
      }
    }
  }
  static GMDN_DEV void put(float* o, const f32x4& v, bool whole, int64_t left) {
    if (whole) {
      *reinterpret_cast<f32x4_any*>(o) = v;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < left) o[q] = v[q];
    }
  }
  static GMDN_DEV void put(bf16* o, const f32x4& v, bool whole, int64_t left) {
    typedef bf16 bf16x4_any __attribute__((ext_vector_type(4), aligned(2)));
    const bf16x4 b = to_bf16x4(v);
    if (whole) {
      *reinterpret_cast<bf16x4_any*>(o) = b;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < left) o[q] = b[q];
    }
  }
};

// out = the sum of the planes, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
ll_sum_planes(const float* __restrict__ planes, T* __restrict__ out, int64_t n, int count) {
  const int64_t at = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (at >= n) return;
  const int left = n - at < 8 ? (int)(n - at) : 8;
  float s[8] = {};
  for (int p = 0; p < count; ++p) {
    float v[8];
    load8(planes + p * n + at, left, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += v[j];
  }
  store8(out + at, left, s);
}

// ------------------------------------------------------------------ the calls
// Tiles of 256, 128 and 64: 8 waves of 128 x 64, 4 of 64 x 64 and of 32 x 32.
using Tile256 = MMShape<256, 256, 64, 2, 2, 4>;
using Tile128 = MMShape<128, 128, 64, 2, 2, 2>;
using Tile64 = MMShape<64, 64, 64, 3, 2, 2>;

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return div_up(a, b) * b; }
size_t up(size_t n) { return (n + 255) / 256 * 256; }

// Whether the products read a matrix where it is: bfloat16 rows of whole stages at
// 16-byte addresses, 256 of which stay within 32 bits.
bool in_place(const void* p, int64_t stride, int64_t d, int32_t dtype) {
  return dtype == GMDN_DTYPE_BF16 && d % KPAD == 0 && stride % 8 == 0 && stride <= (1 << 22) && (uintptr_t)p % 16 == 0;
}

// How a product of tiles_m x tiles_n tiles over `steps` stages of k runs: which
// tile, and the stages of a split along k.
struct Product {
  int edge, per, splits;
};
// A product of few tiles is split until the chip is filled (dx of 8 x 32000 x 1024, backward:
// 32 us, whole 179), while a part keeps sixteen turns of the loop or more: joining the
// parts is a launch more (1024 x 8192 x 1024: 56 us, from four turns on 64; 16384 x 257 x 256,
// dW: 32 and 41; but 512 x 257 x 256 float32, dW: 22 and 19).
int splits_of(int64_t tiles, int64_t turns) {
  int64_t s = 256 / tiles;
  if (s > turns / 16) s = turns / 16;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
// The tile of the least cost: rounds over the 256 CUs, times a tile's work at the rate that its
// reads from LDS leave it, of two stages more than it has (its ramp and epilogue).  For a stage
// of 32 k the matrix units take 1024, 256 and 64 clocks, LDS at 128 bytes a clock 1024,
// 384 and 192: rates as 6 to 4 to 2.  It takes the fastest tile or one within 8% of it in
// all that was measured (forward in tiles of 64, 128 and 256: 8 x 32000 x 1024 bf16: 16, 19
// and 30 us; 1024 x 8192 x 1024: 35, 25 and 33; 16384 x 32000 x 1024: 1626, 1047 and 908).
Product product_of(int64_t M, int64_t N, int64_t steps, int pairs, bool split) {
  Product best{};
  double least = 0;
  const int edges[3] = {64, 128, 256}, clocks[3] = {6, 3, 2};
  for (int i = 0; i < 3; ++i) {
    const int64_t e = edges[i], tiles = div_up(M, e) * div_up(N, e);
    Product p{edges[i], (int)div_up(steps, split ? splits_of(tiles, steps * pairs) : 1), 1};
    p.splits = (int)div_up(steps, p.per);
    const double cost = (double)div_up(tiles * p.splits, 256) * (double)(e * e) * (p.per * pairs + 2) * clocks[i];
    if (i == 0 || cost < least) {
      best = p;
      least = cost;
    }
  }
  return best;
}
// f(tile's shape)
template <class F>
bool with_tile(const Product& p, F&& f) {
  return p.edge == 64 ? f(Tile64{}) : p.edge == 128 ? f(Tile128{}) : f(Tile256{});
}

struct Sizes {
  int64_t rows, V, d, kp;
  int P, pairs;                    // pieces of an operand, and products of two
  bool x_in, w_in;
  size_t x, w;                     // bytes of the operands' planes
  // forward
  Product logits;
  size_t at_token, part;
  // backward
  int64_t piece, pieces, padded;   // columns, pieces, rows of d
  Product again, for_x, for_w;     // a piece's logits, and the products for dx and dW
  size_t grad, x_acc, w_acc;
  size_t forward() const { return x + w + at_token + part; }
  size_t backward() const { return x + w + grad + x_acc + w_acc; }
};

Sizes sizes_of(const void* x, const void* w, int64_t rows, int64_t V, int64_t d, int64_t xs, int64_t ws, int32_t dtype) {
  Sizes z{};
  z.rows = rows;
  z.V = V;
  z.d = d;
  z.kp = round_up(d, KPAD);
  z.P = dtype == GMDN_DTYPE_F32_IEEE ? 3 : dtype == GMDN_DTYPE_F32 ? 2 : 1;
  z.pairs = z.P * (z.P + 1) / 2;
  z.x_in = in_place(x, xs, d, dtype);
  z.w_in = in_place(w, ws, d, dtype);
  z.x = z.x_in ? 0 : up((size_t)(z.P * rows * z.kp * 2));
  z.w = z.w_in ? 0 : up((size_t)(z.P * V * z.kp * 2));
  z.logits = product_of(V, rows, z.kp / KPAD, z.pairs, false);
  z.at_token = up((size_t)rows * 4);
  z.part = up((size_t)(div_up(V, z.logits.edge) * 3 * rows * 4));
  z.padded = round_up(rows, KPAD);
  int64_t most = PIECE_BYTES / (z.padded * 2 * z.P) / UNIT * UNIT;
  most = most < UNIT ? UNIT : most > PIECE_MOST ? PIECE_MOST : most;
  z.pieces = div_up(V, most);
  z.piece = round_up(div_up(V, z.pieces), UNIT);
  z.pieces = div_up(V, z.piece);
  z.grad = up((size_t)(z.P * z.padded * z.piece * 2));
  // every piece as the first: the last may be shorter
  const int64_t columns = z.piece < V ? z.piece : V;
  z.again = product_of(columns, rows, z.kp / KPAD, z.pairs, false);
  z.for_x = product_of(d, rows, div_up(columns, KPAD), z.pairs, true);
  z.for_w = product_of(d, columns, z.padded / KPAD, z.pairs, true);
  z.x_acc = z.for_x.splits > 1 || z.pieces > 1 ? up((size_t)(z.for_x.splits * rows * d * 4)) : 0;
  z.w_acc = z.for_w.splits > 1 ? up((size_t)(z.for_w.splits * columns * d * 4)) : 0;
  return z;
}

int check_ll(int64_t rows, int64_t V, int64_t d, int64_t xs, int64_t ws, int32_t dtype) {
  if (rows < 0 || V <= 0 || d <= 0 || xs < 0 || ws < 0 || rows > ((int64_t)1 << 30)) return GMDN_ERR_ARG;
  if ((!type_ok(dtype) && dtype != GMDN_DTYPE_F32_IEEE) || rows > (1 << 27) || V > (1 << 27) || d > (1 << 17)) return GMDN_ERR_UNSUPPORTED;
  // what a launch's grid holds: 2^32 threads (tiles below 256 are taken where one side has
  // few of them)
  const int64_t longer = rows > V ? rows : V, most = 1 << 22;
  const bool fits = div_up(V, 256) * div_up(rows, 256) <= most && div_up(d, 256) * div_up(longer, 256) <= most &&
                    longer * (round_up(d, KPAD) / 8) < ((int64_t)1 << 32) - 256;
  return fits ? GMDN_OK : GMDN_ERR_UNSUPPORTED;
}

// A product's arguments; the pairs of planes with the small terms first: lo hi, hi lo, hi hi
// of two, and of three (0 the largest) 2 0, 1 1, 0 2, 1 0, 0 1, 0 0.
template <class S>
MMArgs args_of(const MMOperand& a, const MMOperand& b, int64_t M, int64_t N, int64_t k, int pairs, int per) {
  static_assert(S::BK == KPAD, "a stage is what the operands are padded to");
  MMArgs r{};
  r.a = a;
  r.b = b;
  r.steps = (int)div_up(k, S::BK);
  r.per = per;
  r.tiles_m = (int)div_up(M, S::TM);
  r.tiles_n = (int)div_up(N, S::TN);
  r.pairs = pairs;
  r.pair_a = pairs == 1 ? 0 : pairs == 3 ? 0x001 : 0x001012;
  r.pair_b = pairs == 1 ? 0 : pairs == 3 ? 0x010 : 0x010210;
  return r;
}

struct Matrices {
  const bf16 *x, *w;
  int64_t xs, ws, xp, wp;  // row strides, plane strides
};
// The operands' planes: where they lie, or made at `at`, which moves on.
template <typename T, int P>
Matrices matrices_of(const void* x, const void* w, int64_t xs, int64_t ws, const Sizes& z, char*& at, hipStream_t st) {
  Matrices m{(const bf16*)x, (const bf16*)w, xs, ws, z.rows * z.kp, z.V * z.kp};
  Whole<T> list[2];
  int n = 0;
  if (!z.x_in) {
    list[n++] = {(const T*)x, xs, z.rows, (bf16*)at};
    m.x = (const bf16*)at;
    m.xs = z.kp;
    at += z.x;
  }
  if (!z.w_in) {
    list[n++] = {(const T*)w, ws, z.V, (bf16*)at};
    m.w = (const bf16*)at;
    m.ws = z.kp;
    at += z.w;
  }
  if (n) {
    const int64_t longest = n == 2 && list[1].rows > list[0].rows ? list[1].rows : list[0].rows;
    hipLaunchKernelGGL((ll_planes<T, P>), dim3((unsigned)div_up(longest * (z.kp / 8), 256), (unsigned)n), dim3(256),
                       0, st, list[0], list[n - 1], (int)z.d, (int)z.kp);
  }
  return m;
}

// Logits of `columns` of the vocabulary from v0 on.
template <class S, class Epi>
bool logits(const Matrices& m, const Sizes& z, int64_t v0, int64_t columns, const Epi& epi, hipStream_t st) {
  const MMArgs a = args_of<S>({m.w + v0 * m.ws, m.ws, m.wp, columns - 1, 0}, {m.x, m.xs, m.xp, z.rows - 1, 0}, columns,
                              z.rows, z.kp, z.pairs, (int)(z.kp / KPAD));
  return mm_launch<S, false, false, true>(a, epi, 1, st);
}

template <typename T>
void sum_planes(const float* planes, T* out, int64_t n, int count, hipStream_t st) {
  hipLaunchKernelGGL((ll_sum_planes<T>), dim3((unsigned)div_up(n, 8 * 256)), dim3(256), 0, st, planes, out, n, count);
}

template <typename T, int P>
bool backward(const Matrices& m, const Sizes& z, GradArgs e, float* x_acc, float* w_acc, T* dx, T* dw, hipStream_t st) {
  const int64_t plane = z.padded * z.piece;
  for (int64_t i = 0; i < z.pieces; ++i) {
    const int64_t v0 = i * z.piece, left = z.V - v0 < z.piece ? z.V - v0 : z.piece;
    const bool last = i + 1 == z.pieces;
    e.first = v0;
    e.left = left;
    bool ok = with_tile(z.again, [&](auto s) {
      using S = decltype(s);
      return logits<S>(m, z, v0, left, GradEpi<S, true, P>{e}, st);
    });
    if (dx && ok) {
      const int count = z.for_x.splits;
      const StoreArgs<T> to{x_acc, last && count == 1 ? dx : nullptr, z.d, z.rows, i > 0};
      ok = with_tile(z.for_x, [&](auto s) {
        using S = decltype(s);
        const MMArgs a = args_of<S>({m.w + v0 * m.ws, m.ws, m.wp, z.kp - 1, left - 1},
                                    {e.d, z.piece, plane, z.rows - 1, 0}, z.d, z.rows, left, z.pairs, z.for_x.per);
        return mm_launch<S, true, false, false>(a, StoreEpi<S, T>{to}, (int)div_up(a.steps, a.per), st);
      });
      if (ok && last && count > 1) sum_planes(x_acc, dx, z.rows * z.d, count, st);
    }
    if (dw && ok) {
      const int count = z.for_w.splits;
      const StoreArgs<T> to{w_acc, count == 1 ? dw + v0 * z.d : nullptr, z.d, left, false};
      ok = with_tile(z.for_w, [&](auto s) {
        using S = decltype(s);
        const MMArgs a = args_of<S>({m.x, m.xs, m.xp, z.kp - 1, z.rows - 1},
                                    {e.d, z.piece, plane, z.piece - 1, z.padded - 1}, z.d, left, z.padded, z.pairs,
                                    z.for_w.per);
        return mm_launch<S, true, true, false>(a, StoreEpi<S, T>{to}, count, st);
      });
      if (ok && count > 1) sum_planes(w_acc, dw + v0 * z.d, left * z.d, count, st);
    }
    if (!ok) return false;
  }
  return true;
}

template <typename T_, int P_>
struct Operands {
  using T = T_;
  static constexpr int P = P_;
};
// f(type and pieces of the operands)
template <class F>
void with_operands(int32_t dtype, F&& f) {
  if (dtype == GMDN_DTYPE_BF16) f(Operands<bf16, 1>{});
  else if (dtype == GMDN_DTYPE_F32) f(Operands<float, 2>{});
  else f(Operands<float, 3>{});
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

size_t gmdn_linear_logprobs_fwd_workspace_bytes(const void* x, const void* weight, int64_t rows, int64_t vocab,
                                                int64_t d, int64_t x_stride, int64_t w_stride, int32_t dtype) {
  if (rows == 0 || check_ll(rows, vocab, d, x_stride, w_stride, dtype) != GMDN_OK) return 0;
  return sizes_of(x, weight, rows, vocab, d, x_stride, w_stride, dtype).forward();
}

int gmdn_linear_logprobs_fwd(const void* x, const void* weight, const int64_t* tokens, float* logprob, float* entropy,
                             float* stats, void* workspace, size_t workspace_bytes, int64_t rows, int64_t vocab,
                             int64_t d, int64_t x_stride, int64_t w_stride, int64_t ignore_index, int32_t dtype,
                             void* stream) {
  const int rc = check_ll(rows, vocab, d, x_stride, w_stride, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!x || !weight || !tokens || !logprob || !entropy || !stats) return GMDN_ERR_ARG;
  const Sizes z = sizes_of(x, weight, rows, vocab, d, x_stride, w_stride, dtype);
  if (!workspace || workspace_bytes < z.forward()) return GMDN_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16) return GMDN_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  char* at = (char*)workspace;
  Matrices m;
  with_operands(dtype, [&](auto o) {
    using O = decltype(o);
    m = matrices_of<typename O::T, O::P>(x, weight, x_stride, w_stride, z, at, st);
  });
  const SumsArgs e{tokens, (float*)at, (float*)(at + z.at_token), rows, (int)vocab};
  const int tiles = (int)div_up(vocab, z.logits.edge);
  const bool ok = with_tile(z.logits, [&](auto s) {
    using S = decltype(s);
    return logits<S>(m, z, 0, vocab, SumsEpi<S, true>{e}, st);
  });
  if (!ok) return GMDN_ERR_LAUNCH;
  if (rows <= JOIN_FEW)
    hipLaunchKernelGGL((ll_join<1>), dim3((unsigned)rows), dim3(256), 0, st, e.part, e.at_token, tokens, logprob, entropy,
                       stats, tiles, rows, vocab, ignore_index);
  else
    hipLaunchKernelGGL((ll_join<16>), dim3((unsigned)div_up(rows, 16)), dim3(256), 0, st, e.part, e.at_token, tokens,
                       logprob, entropy, stats, tiles, rows, vocab, ignore_index);
  return launched();
}

size_t gmdn_linear_logprobs_bwd_workspace_bytes(const void* x, const void* weight, int64_t rows, int64_t vocab,
                                                int64_t d, int64_t x_stride, int64_t w_stride, int32_t dtype) {
  if (rows == 0 || check_ll(rows, vocab, d, x_stride, w_stride, dtype) != GMDN_OK) return 0;
  return sizes_of(x, weight, rows, vocab, d, x_stride, w_stride, dtype).backward();
}

int gmdn_linear_logprobs_bwd(const void* x, const void* weight, const int64_t* tokens, const float* stats,
                             const float* entropy, const float* dlogprob, const float* dentropy, void* dx,
                             void* dweight, void* workspace, size_t workspace_bytes, int64_t rows, int64_t vocab,
                             int64_t d, int64_t x_stride, int64_t w_stride, int64_t ignore_index, int32_t dtype,
                             void* stream) {
  const int rc = check_ll(rows, vocab, d, x_stride, w_stride, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!x || !weight || !tokens || !stats || !entropy || (!dx && !dweight)) return GMDN_ERR_ARG;
  const Sizes z = sizes_of(x, weight, rows, vocab, d, x_stride, w_stride, dtype);
  if (!workspace || workspace_bytes < z.backward()) return GMDN_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16) return GMDN_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  char* at = (char*)workspace;
  bool ok = false;
  with_operands(dtype, [&](auto o) {
    using T = typename decltype(o)::T;
    constexpr int P = decltype(o)::P;
    const Matrices m = matrices_of<T, P>(x, weight, x_stride, w_stride, z, at, st);
    const GradArgs e{tokens, stats, entropy, dlogprob, dentropy, (bf16*)at, rows, z.padded, z.piece, 0, 0, vocab,
                     ignore_index};
    float* const xa = (float*)(at + z.grad);
    float* const wa = (float*)(at + z.grad + z.x_acc);
    ok = backward<T, P>(m, z, e, xa, wa, (T*)dx, (T*)dweight, st);
  });
  return ok ? launched() : GMDN_ERR_LAUNCH;
}

}  // extern "C"
