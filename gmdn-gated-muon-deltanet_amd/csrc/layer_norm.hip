// Layer norm over the last dimension, forward and backward, and the same with
// the input kept as an 8-bit checkpoint (include/gmdn_lm.h).
//
// A row x of d values:  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps),
// xh = (x - m) r,  y = xh w + b.  With g = dy w:
//   dx = r (g - mean(g) - xh mean(g xh)),   dw = sum dy xh,  db = sum dy
// over the rows.
//
// Memory bound: 8 and 12 operations a value, against 4 to 10 bytes.  A row
// stays in its threads' registers between the sums and the output, so each
// matrix is read and written once; the deviation is a second sum over the
// centred registers (a sum of squares would cancel for rows far from zero).
// At 5.1 TB/s (what a 1 GiB copy reaches):
//   16384 x 1024, float32 in, bf16 out   forward 19 us (floor 20), backward 31 + 5 us (33)
//   8192 x 8192 bf16                     forward 48 us (53), backward 64 + 6 us (79)
// (in brackets the floor: the outputs stay in the cache in part).
#include "../../include/gmdn_lm.h"
#include <type_traits>
#include "rows8.h"

namespace gmdn {
namespace {

constexpr int LN_THREADS = 512;      // threads of a workgroup, or a row's if more
constexpr int LN_MAX_D = 16384;
// Workgroups of a launch at most; each takes rows in turn.  Forward: 1024 took
// 55 us where 512 take 48 at 8192 x 8192, and the same at 16384 x 1024.
// Backward: each writes 2 d partial sums, at 8192 x 8192 with 1024 of them a sixth
// of all bytes (94 + 17 us, with 256 65 + 6).
constexpr int LN_FWD_BLOCKS = 512;
constexpr int LN_BWD_BLOCKS = 256;

constexpr int ln_threads(int tpr) { return tpr > LN_THREADS ? tpr : LN_THREADS; }

// Sum over the TPR threads of a row: butterflies within a wave, then the
// row's waves through LDS.  `slot` alternates between two halves of red, so
// that one barrier a sum is enough.
template <int TPR>
GMDN_DEV float row_sum(float x, float (*red)[16], int& slot) {
  x = lanes_sum<(TPR < 64 ? TPR : 64)>(x);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int w = wave_id(), first = w / W * W;
    if (lane_id() == 0) red[slot][w] = x;
    __syncthreads();
    x = red[slot][first];
#pragma unroll
    for (int i = 1; i < W; ++i) x += red[slot][first + i];
    slot ^= 1;
  }
  return x;
}

// A thread's columns of weight and bias (1 and 0 without).
template <int TPR, int NV>
GMDN_DEV void load_weights(const void* w, const void* b, bool w16, int d, int t, float (&wv)[NV][8],
                           float (&bv)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (i * TPR + t);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wv[i][j] = 1.f;
      bv[i][j] = 0.f;
    }
    if (c < d && w) load8_weight(w, w16, c, d - c, wv[i]);
    if (c < d && b) load8_weight(b, w16, c, d - c, bv[i]);
  }
}

// Forward.  A row is TPR threads with NV pieces each, piece i of thread t at
// i TPR + t; a workgroup takes its threads / TPR rows at a time.
template <typename TX, typename TY, int TPR, int NV, bool PACK>
__global__ void __launch_bounds__(ln_threads(TPR))
ln_fwd(const TX* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, bool w16,
       TY* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int8_t* __restrict__ q,
       float* __restrict__ scale, int64_t rows, int d, int64_t xs, float eps) {
  constexpr int RPB = ln_threads(TPR) / TPR;
  __shared__ float red[2][16];
  const int lr = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int slot = 0;
  float wv[NV][8], bv[NV][8];
  load_weights<TPR, NV>(w, b, w16, d, t, wv, bv);
  // the next row's pieces are loaded before this row's sums (rows of several
  // waves wait at two barriers: 62 -> 55 us at 8192 x 8192)
  Raw8<TX> raw[NV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      raw[i].load(x + r * xs + c, r < rows ? d - c : 0);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + lr;
  fetch(r);
  for (; r - lr < rows; r += step) {
    const bool live = r < rows;
    float v[NV][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i].get(v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
    fetch(r + step);
    const float m = row_sum<TPR>(s, red, slot) / (float)d;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = c + j < d ? v[i][j] - m : 0.f;
        ss += u * u;
      }
    }
    const float rs = 1.f / sqrtf(row_sum<TPR>(ss, red, slot) / (float)d + eps);
    if constexpr (PACK) {
      constexpr int GL = TPR < GROUP8_PIECES ? TPR : GROUP8_PIECES;  // lanes of a group
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + t);
        const Scale8 sc = scale8(lanes_max<GL>(amax_bits(v[i])));
        if (live && c < d) {
          store_q8(q + r * d + c, d - c, quant8(v[i], sc.inverse));
          if (t % GL == 0) scale[r * groups8(d) + c / GROUP8] = sc.scale;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - m) * rs * wv[i][j] + bv[i][j];
      if (live && c < d) stream8(y + r * d + c, d - c, v[i]);
    }
    if (live && t == 0) {
      mean[r] = m;
      rstd[r] = rs;
    }
  }
}

// Where the backward's input comes from: x itself, or its checkpoint.
template <typename TX>
struct FromX {
  const TX* x;
  int64_t stride;
  struct Raw : Raw8<TX> {
    template <bool FAR = false>
    GMDN_DEV void load(const FromX& src, int64_t r, int c, int n, int) {
      Raw8<TX>::template load<FAR>(src.x + r * src.stride + c, n);
    }
  };
};
struct From8 {
  const int8_t* q;
  const float* scale;
  struct Raw {
    u32x2_any v;
    float s;
    template <bool FAR = false>
    GMDN_DEV void load(const From8& src, int64_t r, int c, int n, int d) {
      v = load_q8(src.q + r * d + c, n);
      s = n > 0 ? src.scale[r * groups8(d) + c / GROUP8] : 0.f;
    }
    GMDN_DEV void get(float (&x)[8]) const { dequant8(v, s, x); }
  };
};

// dx, and per workgroup the sums of dy xh and dy over its rows: part is
// (workgroups, 2, d).  A thread's columns are the same in every row, so the
// sums stay in its registers; the rows a workgroup takes side by side are
// added in LDS at the end, in a fixed order.  No atomics: they would add in
// another order on every run.  A workgroup alone (see bwd_blocks) has the whole sums
// and writes them to dweight and dbias, which are null otherwise.  `large`: the matrix is FAR_BYTES or more; rows of
// several waves are then loaded past the caches (8192 x 8192: 80 -> 78 us; from
// 8 bits at 16384 x 4096: 66 -> 58).
template <typename Src, typename TX, typename TY, int TPR, int NV>
__global__ void __launch_bounds__(ln_threads(TPR))
ln_bwd(Src src, const TY* __restrict__ dy, int64_t ds, const void* __restrict__ w, bool w16,
       const float* __restrict__ mean, const float* __restrict__ rstd, TX* __restrict__ dx,
       float* __restrict__ part, void* __restrict__ dweight, void* __restrict__ dbias, int64_t rows, int d,
       bool large) {
  constexpr int RPB = ln_threads(TPR) / TPR;
  // a row's loads before the last row's work (8192 x 8192: 103 -> 88 us), where
  // the registers hold them: 1024 threads have 128 each, and spilled
  constexpr bool AHEAD = TPR < 1024;
  __shared__ float red[2][16];
  const int lr = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int slot = 0;
  float wv[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (i * TPR + t);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wv[i][j] = 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
    if (c < d && w) load8_weight(w, w16, c, d - c, wv[i]);
  }
  typename Src::Raw xr[NV];
  Raw8<TY> gr[NV];
  float mr, rr;
  auto pieces = [&](int64_t r, auto far) {
    const bool live = r < rows;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      xr[i].template load<decltype(far)::value>(src, r, c, live ? d - c : 0, d);
      gr[i].template load<decltype(far)::value>(dy + r * ds + c, live ? d - c : 0);
    }
  };
  auto fetch = [&](int64_t r) {
    const bool live = r < rows;
    mr = live ? mean[r] : 0.f;
    rr = live ? rstd[r] : 0.f;
    if (TPR > 64 && sizeof(TY) == 2 && large) {
      apart();
      pieces(r, std::true_type{});
      apart();
    } else {
      pieces(r, std::false_type{});
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + lr;
  if constexpr (AHEAD) fetch(r);
  for (; r - lr < rows; r += step) {
    if constexpr (!AHEAD) fetch(r);
    const bool live = r < rows;
    float v[NV][8], g[NV][8];
    const float m = mr, rs = rr;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i].get(v[i]);
      gr[i].get(g[i]);
    }
    if constexpr (AHEAD) fetch(r + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - m) * rs;  // xh
      if (c + 8 > d) {  // past the row's end g is 0, but -m rs may be infinite
        int end = d;
        asm volatile("" : "+s"(end));  // compared here: sixteen masks kept over the loop spill
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j >= end) v[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] += g[i][j] * v[i][j];
        db[i][j] += g[i][j];
        g[i][j] *= wv[i][j];
        s0 += g[i][j];
        s1 += g[i][j] * v[i][j];
      }
    }
    const float mg = row_sum<TPR>(s0, red, slot) / (float)d;
    const float mx = row_sum<TPR>(s1, red, slot) / (float)d;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) g[i][j] = rs * (g[i][j] - mg - v[i][j] * mx);
    if (sizeof(TX) == 4 && !large) {
      apart();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + t);
        if (live && c < d) stream8_f32(dx + r * d + c, d - c, g[i]);
      }
      apart();
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + t);
        if (live && c < d) stream8(dx + r * d + c, d - c, g[i]);
      }
    }
  }
  if (!w) return;
  const bool narrow = dweight && w16;
  float* first = dweight ? reinterpret_cast<float*>(dweight) : part + (int64_t)blockIdx.x * 2 * d;
  float* second = dweight ? reinterpret_cast<float*>(dbias) : first + d;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      if (c >= d) continue;
      if (narrow) {
        store8(reinterpret_cast<bf16*>(dweight) + c, d - c, dw[i]);
        store8(reinterpret_cast<bf16*>(dbias) + c, d - c, db[i]);
      } else {
        store8(first + c, d - c, dw[i]);
        store8(second + c, d - c, db[i]);
      }
    }
  } else {
    __shared__ float sums[RPB][TPR * NV * 8];
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[lr][8 * (i * TPR + t) + j] = which ? db[i][j] : dw[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < d; c += ln_threads(TPR)) {
        float s = sums[0][c];
#pragma unroll
        for (int i = 1; i < RPB; ++i) s += sums[i][c];
        if (narrow)
          reinterpret_cast<bf16*>(which ? dbias : dweight)[c] = (bf16)s;
        else
          (which ? second : first)[c] = s;
      }
    }
  }
}

// dweight and dbias from the workgroups' sums: a workgroup takes 32 columns
// of (2, d) -- 8 lanes of 4 -- and 128 lane groups every 128th partial row, four
// of them in flight; joined in a wave, then over the waves in LDS.  The order
// is fixed: the same bits on every run.  Bound by latency: 4 to 5 us for 256 rows of
// 2 x 1024 (12 us when a thread added 128 rows one after the other).
constexpr int LN_COLS = 32;
constexpr int LN_SUM_THREADS = 1024;
__global__ void __launch_bounds__(LN_SUM_THREADS)
ln_sums(const float* __restrict__ part, void* __restrict__ dw, void* __restrict__ db, bool w16, int d, int nblk) {
  constexpr int SPLIT = LN_SUM_THREADS / 8;
  __shared__ f32x4 red[LN_SUM_THREADS / 64][8];
  const int64_t width = 2 * (int64_t)d;
  const int quad = threadIdx.x % 8, sp = threadIdx.x / 8;
  const int64_t c = (int64_t)blockIdx.x * LN_COLS + 4 * quad;
  f32x4 a[4] = {zero4(), zero4(), zero4(), zero4()};
  for (int i0 = sp; i0 < nblk; i0 += 4 * SPLIT)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * SPLIT;
      if (i >= nblk) continue;
      const float* p = part + i * width + c;
      if (c + 4 <= width) {
        a[k] += *reinterpret_cast<const f32x4_any*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < width) a[k][j] += p[j];
      }
    }
  f32x4 s = (a[0] + a[1]) + (a[2] + a[3]);
#pragma unroll
  for (int o = 8; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += __shfl_xor(s[j], o, 64);
  if (lane_id() < 8) red[wave_id()][quad] = s;
  __syncthreads();
  if (threadIdx.x < 8) {
    s = red[0][quad];
#pragma unroll
    for (int i = 1; i < LN_SUM_THREADS / 64; ++i) s += red[i][quad];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j >= width) continue;
      void* out = c + j < d ? dw : db;
      const int64_t at = c + j < d ? c + j : c + j - d;
      if (w16)
        reinterpret_cast<bf16*>(out)[at] = (bf16)s[j];
      else
        reinterpret_cast<float*>(out)[at] = s[j];
    }
  }
}

// y again from the checkpoint and the saved statistics: 9.4 us at 16384 x 1024,
// 32 us at 8192 x 8192 (6.3 TB/s; a thread for each piece, which loads its
// weights each time, took 55).
template <typename TY, int TPR, int NV>
__global__ void __launch_bounds__(ln_threads(TPR))
ln_rebuild(From8 src, const void* __restrict__ w, const void* __restrict__ b, bool w16,
           const float* __restrict__ mean, const float* __restrict__ rstd, TY* __restrict__ y, int64_t rows, int d) {
  constexpr int RPB = ln_threads(TPR) / TPR;
  const int lr = threadIdx.x / TPR, t = threadIdx.x % TPR;
  float wv[NV][8], bv[NV][8];
  load_weights<TPR, NV>(w, b, w16, d, t, wv, bv);
  From8::Raw raw[NV];
  float mr, rr;
  auto fetch = [&](int64_t r) {
    const bool live = r < rows;
    mr = live ? mean[r] : 0.f;
    rr = live ? rstd[r] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      raw[i].load(src, r, c, live ? d - c : 0, d);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + lr;
  fetch(r);
  for (; r < rows; r += step) {
    float v[NV][8];
    const float m = mr, rs = rr;
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i].get(v[i]);
    fetch(r + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - m) * rs * wv[i][j] + bv[i][j];
      if (c < d) stream8(y + r * d + c, d - c, v[i]);
    }
  }
}

template <int TPR_, int NV_>
struct Shape {
  static constexpr int TPR = TPR_, NV = NV_;
};
// f(Shape) with the threads and pieces of a row of d values: one piece a
// thread while the row fits a wave, then two (more would not leave the backward's
// sums in registers).
template <class F>
void with_shape(int64_t d, F&& f) {
  if (d <= 64) f(Shape<8, 1>{});
  else if (d <= 128) f(Shape<16, 1>{});
  else if (d <= 256) f(Shape<32, 1>{});
  else if (d <= 512) f(Shape<64, 1>{});
  else if (d <= 1024) f(Shape<64, 2>{});
  else if (d <= 2048) f(Shape<128, 2>{});
  else if (d <= 4096) f(Shape<256, 2>{});
  else if (d <= 8192) f(Shape<512, 2>{});
  else f(Shape<1024, 2>{});
}

int64_t ln_blocks(int64_t rows, int64_t d, int64_t most) {
  int64_t n = 0;
  with_shape(d, [&](auto s) {
    using S = decltype(s);
    constexpr int RPB = ln_threads(S::TPR) / S::TPR;
    n = (rows + RPB - 1) / RPB;
  });
  return n < most ? n : most;
}

// The backward's workgroups.  One alone does without the partial sums' launch:
// 5.5 us instead of 8.5 for 128 x 128 bf16, and 4 us of the caller's.  Past its
// first few rows it loses that again (32 x 1024: 8.3 us, with partial sums
// 8.6; 64 x 1024: 12.7 and 8.7).  Narrow rows take less each (152 x 112, five
// turns: 7.9 and 8.7; 512 x 128, sixteen: 13.4 and 9.1).
int64_t bwd_blocks(int64_t rows, int64_t d) {
  const int64_t alone = d <= 256 ? 8 : 4;
  return ln_blocks(rows, d, alone + 1) <= alone ? 1 : ln_blocks(rows, d, LN_BWD_BLOCKS);
}

// The built pairs of types: (bf16, bf16), (float32, float32) and a float32
// input beside a bf16 output.
bool pair_ok(int32_t xt, int32_t yt) {
  return type_ok(xt) && type_ok(yt) && !(xt == GMDN_DTYPE_BF16 && yt == GMDN_DTYPE_F32);
}
template <class F>
void with_types(int32_t xt, int32_t yt, F&& f) {
  if (xt == GMDN_DTYPE_BF16) f(bf16{}, bf16{});
  else if (yt == GMDN_DTYPE_F32) f(float{}, float{});
  else f(float{}, bf16{});
}

int check_dims(int64_t rows, int64_t d) {
  if (rows < 0 || d <= 0 || rows > ((int64_t)1 << 40)) return GMDN_ERR_ARG;
  return d > LN_MAX_D ? GMDN_ERR_UNSUPPORTED : GMDN_OK;
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

int gmdn_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                        int8_t* q, float* scale, int64_t rows, int64_t d, int64_t x_stride, float eps,
                        int32_t x_type, int32_t y_type, int32_t w_type, void* stream) {
  const int rc = check_dims(rows, d);
  if (rc != GMDN_OK) return rc;
  if (!pair_ok(x_type, y_type) || !type_ok(w_type)) return GMDN_ERR_UNSUPPORTED;
  if (!(eps >= 0.f) || x_stride < 0 || (bias && !weight) || !q != !scale) return GMDN_ERR_ARG;
  if (rows == 0) return GMDN_OK;
  if (!x || !y || !mean || !rstd) return GMDN_ERR_ARG;
  const dim3 grid((unsigned)ln_blocks(rows, d, LN_FWD_BLOCKS));
  const bool w16 = w_type == GMDN_DTYPE_BF16;
  with_types(x_type, y_type, [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    with_shape(d, [&](auto s) {
      using S = decltype(s);
      const dim3 block(ln_threads(S::TPR));
      if (q)
        hipLaunchKernelGGL((ln_fwd<TX, TY, S::TPR, S::NV, true>), grid, block, 0, (hipStream_t)stream, (const TX*)x,
                           weight, bias, w16, (TY*)y, mean, rstd, q, scale, rows, (int)d, x_stride, eps);
      else
        hipLaunchKernelGGL((ln_fwd<TX, TY, S::TPR, S::NV, false>), grid, block, 0, (hipStream_t)stream, (const TX*)x,
                           weight, bias, w16, (TY*)y, mean, rstd, q, scale, rows, (int)d, x_stride, eps);
    });
  });
  return launched();
}

size_t gmdn_layer_norm_bwd_workspace_floats(int64_t rows, int64_t d) {
  if (rows <= 0 || check_dims(rows, d) != GMDN_OK) return 0;
  const int64_t nb = bwd_blocks(rows, d);
  return nb == 1 ? 0 : (size_t)(nb * 2 * d);
}

int gmdn_layer_norm_bwd(const void* dy, const void* x, const int8_t* q, const float* scale, const void* weight,
                        const float* mean, const float* rstd, void* dx, void* dweight, void* dbias, float* workspace,
                        size_t workspace_floats, int64_t rows, int64_t d, int64_t dy_stride, int64_t x_stride,
                        int32_t x_type, int32_t y_type, int32_t w_type, void* stream) {
  const int rc = check_dims(rows, d);
  if (rc != GMDN_OK) return rc;
  if (!pair_ok(x_type, y_type) || !type_ok(w_type)) return GMDN_ERR_UNSUPPORTED;
  if (dy_stride < 0 || x_stride < 0 || !q != !scale) return GMDN_ERR_ARG;
  if (weight && (!dweight || !dbias)) return GMDN_ERR_ARG;
  const bool w16 = w_type == GMDN_DTYPE_BF16;
  const hipStream_t st = (hipStream_t)stream;
  int64_t nb = 0;
  if (rows > 0) {
    if (!dy || (!x && !q) || (x && q) || !mean || !rstd || !dx) return GMDN_ERR_ARG;
    nb = bwd_blocks(rows, d);
    if (weight && nb > 1 && (!workspace || workspace_floats < (size_t)(nb * 2 * d))) return GMDN_ERR_WORKSPACE;
    void *const dw = nb == 1 ? dweight : nullptr, *const db = nb == 1 ? dbias : nullptr;
    const bool large = rows * d * (x_type == GMDN_DTYPE_F32 ? 4 : 2) >= FAR_BYTES;
    with_types(x_type, y_type, [&](auto tx, auto ty) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      with_shape(d, [&](auto s) {
        using S = decltype(s);
        const dim3 grid((unsigned)nb), block(ln_threads(S::TPR));
        if (q)
          hipLaunchKernelGGL((ln_bwd<From8, TX, TY, S::TPR, S::NV>), grid, block, 0, st, From8{q, scale},
                             (const TY*)dy, dy_stride, weight, w16, mean, rstd, (TX*)dx, workspace, dw, db, rows,
                             (int)d, large);
        else
          hipLaunchKernelGGL((ln_bwd<FromX<TX>, TX, TY, S::TPR, S::NV>), grid, block, 0, st,
                             FromX<TX>{(const TX*)x, x_stride}, (const TY*)dy, dy_stride, weight, w16, mean, rstd,
                             (TX*)dx, workspace, dw, db, rows,
                             (int)d, large);
      });
    });
    if (hipGetLastError() != hipSuccess) return GMDN_ERR_LAUNCH;
  }
  if (!weight || nb == 1) return GMDN_OK;
  hipLaunchKernelGGL(ln_sums, dim3((unsigned)((2 * d + LN_COLS - 1) / LN_COLS)), dim3(LN_SUM_THREADS), 0, st, workspace,
                     dweight, dbias, w16, (int)d, (int)nb);
  return launched();
}

int gmdn_layer_norm8_rebuild(const int8_t* q, const float* scale, const void* weight, const void* bias,
                             const float* mean, const float* rstd, void* y, int64_t rows, int64_t d, int32_t y_type,
                             int32_t w_type, void* stream) {
  const int rc = check_dims(rows, d);
  if (rc != GMDN_OK) return rc;
  if (!type_ok(y_type) || !type_ok(w_type)) return GMDN_ERR_UNSUPPORTED;
  if (bias && !weight) return GMDN_ERR_ARG;
  if (rows == 0) return GMDN_OK;
  if (!q || !scale || !mean || !rstd || !y) return GMDN_ERR_ARG;
  const dim3 grid((unsigned)ln_blocks(rows, d, LN_FWD_BLOCKS));
  const bool w16 = w_type == GMDN_DTYPE_BF16;
  with_shape(d, [&](auto s) {
    using S = decltype(s);
    const dim3 block(ln_threads(S::TPR));
    if (y_type == GMDN_DTYPE_BF16)
      hipLaunchKernelGGL((ln_rebuild<bf16, S::TPR, S::NV>), grid, block, 0, (hipStream_t)stream, From8{q, scale}, weight,
                         bias, w16, mean, rstd, (bf16*)y, rows, (int)d);
    else
      hipLaunchKernelGGL((ln_rebuild<float, S::TPR, S::NV>), grid, block, 0, (hipStream_t)stream, From8{q, scale}, weight,
                         bias, w16, mean, rstd, (float*)y, rows, (int)d);
  });
  return launched();
}

}  // extern "C"
