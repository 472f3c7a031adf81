// A branch's way back into the residual stream with the norms on both sides of
// it, forward and backward (include/gmdn_lm.h).
//
// Rows of d values: x the stream, y a branch's output.  With rms(v) =
// 1 / sqrt(mean v^2 + eps), sigma the logistic function:
//   n = y rho p,  rho = rms(y)        (n = y without a post norm p)
//   r = x + s sigma(g) n              (the scale s (d), the gate g (rows, d))
//   z = r tau w,  tau = rms(r)
// Backward from dr, dz, with rh = r tau, yh = y rho, u = sigma(g):
//   dx = dr + tau (w dz - rh mean(w dz rh))
//   dn = dx s u,    dy = rho (p dn - yh mean(p dn yh))   (dy = dn without p)
//   dg = dx s n u (1 - u)
//   dw = sum dz rh,  dp = sum dn yh,  ds = sum dx u n     over the rows
//
// The backward forms r again from x and y, unrounded; with a float32 stream and nothing
// but the sum it reads the kept r instead.
//
// Memory bound: about 60 operations a value against 16 to 26 bytes.  16384 x 1024, a
// float32 stream and bf16 branches: 36 us forward and 44 backward, 5.6 and 6.0 TB/s; 8192 x
// 8192 bf16 with everything 118 and 205, 5.7 and 5.2 TB/s.  As in the
// layer norm a row stays in its threads' registers between the sums and the
// outputs, so each matrix is read and written once, and the weights' sums stay
// there from row to row, joined over workgroups in a fixed order.
#include "../../include/gmdn_lm.h"
#include <type_traits>
#include "rows8.h"

namespace gmdn {
namespace {

constexpr int RN_THREADS = 512;    // threads of a workgroup, or a row's if more
constexpr int RN_MAX_D = 8192;
// Workgroups of a launch, at most; each goes on to further rows.  Forward two a CU (8192 x 8192
// bf16 with everything, 256 of 1024 threads: 121 us, 128 of them 199; more: the same or
// slower), backward one, whose partial sums are fewest (16384 x 1024, float32 and bf16: 50 us,
// two a CU 55, four 63, one for two CUs 70).
constexpr int RN_FWD_BLOCKS = 512;
constexpr int RN_BWD_BLOCKS = 256;
constexpr float LOG2E = 1.44269504088896340736f;

constexpr int rn_threads(int tpr) { return tpr > RN_THREADS ? tpr : RN_THREADS; }

// What a call has beside x, y and the norm.
enum Parts { ADD, SCALED, GATED };  // nothing; a post norm or a scale; a gate (and they)

// Whether the backward keeps its vectors in LDS.
constexpr bool rn_in_lds(int tpr, Parts p) { return p != ADD && tpr == 1024; }

// Sum over the TPR threads of a row: within a wave, then the row's waves through
// LDS.  `slot` alternates between two halves of red, so that one barrier a
// sum is enough.
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

// A vector's values at a thread's columns, 1 without one (and past the row's end).
GMDN_DEV void load_ones(const void* w, bool w16, int d, int c, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 1.f;
  if (c < d && w) load8_weight(w, w16, c, d - c, v);
}

// by the hardware's exponential and reciprocal, one unit in the last place each
GMDN_DEV float sigmoid(float g) { return hw_rcp(1.f + __builtin_amdgcn_exp2f(-g * LOG2E)); }

// The vectors of a call: the norm's weight, the post norm's, the scale.
struct Vectors {
  const void *w, *p, *s;
  bool w16;
};
template <typename TY>
struct Branch {
  const TY *y, *g;
  int64_t ys, gs;
};

template <typename TX, typename TY, int TPR, int NV, Parts P>
__global__ void __launch_bounds__(rn_threads(TPR))
rn_fwd(const TX* __restrict__ x, int64_t xs, Branch<TY> in, Vectors vec, TX* __restrict__ r_out, TY* __restrict__ z,
       float* __restrict__ rstd, float* __restrict__ post_rstd, int64_t rows, int d, float eps) {
  constexpr int RPB = rn_threads(TPR) / TPR;
  constexpr int NP = P == ADD ? 1 : NV, NG = P == GATED ? NV : 1;
  __shared__ float red[2][16];
  const int lr = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int slot = 0;
  float wv[NV][8], ps[NP][8];  // ps: the post norm's weight times the scale
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (i * TPR + t);
    load_ones(vec.w, vec.w16, d, c, wv[i]);
    if constexpr (P != ADD) {
      float sv[8];
      load_ones(vec.p, vec.w16, d, c, ps[i]);
      load_ones(vec.s, vec.w16, d, c, sv);
#pragma unroll
      for (int j = 0; j < 8; ++j) ps[i][j] *= sv[j];
    }
  }
  // the next row's pieces are loaded before this row's sums
  Raw8<TX> xr[NV];
  Raw8<TY> yr[NV], gr[NG];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t), left = r < rows ? d - c : 0;
      xr[i].load(x + r * xs + c, left);
      yr[i].load(in.y + r * in.ys + c, left);
      if constexpr (P == GATED) gr[i].load(in.g + r * in.gs + c, left);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + lr;
  fetch(r);
  for (; r - lr < rows; r += step) {
    const bool live = r < rows;
    float v[NV][8], n[NV][8], u[NG][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i].get(v[i]);
      yr[i].get(n[i]);
      if constexpr (P == GATED) gr[i].get(u[i]);
    }
    fetch(r + step);
    if constexpr (P != ADD) {
      float rho = 1.f;
      if (vec.p) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += n[i][j] * n[i][j];
        rho = 1.f / sqrtf(row_sum<TPR>(ss, red, slot) / (float)d + eps);
        if (live && t == 0) post_rstd[r] = rho;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          n[i][j] *= rho * ps[i][j];
          if constexpr (P == GATED) n[i][j] *= sigmoid(u[i][j]);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] += n[i][j];
        ss += c + j < d ? v[i][j] * v[i][j] : 0.f;
      }
      if (live && c < d) stream8(r_out + r * d + c, d - c, v[i]);
    }
    const float tau = 1.f / sqrtf(row_sum<TPR>(ss, red, slot) / (float)d + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= tau * wv[i][j];
      if (live && c < d) stream8(z + r * d + c, d - c, v[i]);
    }
    if (live && t == 0) rstd[r] = tau;
  }
}

// Whether the backward reads r: where it was kept in full and nothing else wants y.  It
// forms r again from x and the branch otherwise: a bfloat16 r would put its rounding,
// 2^-9 of a value, into the vectors' float32 gradients (2e-3 of their norm; from x and y
// 1e-7).  A branch with parts is read for them anyway, and x costs what r would; a
// bfloat16 stream that only adds reads y, and keeps it, for this alone.
template <typename TX>
constexpr bool rn_from_r(Parts p) { return p == ADD && sizeof(TX) == 4; }

// A backward call's matrices: stream is r or x.  dr, dz and dy may be null: zeros, and
// not wanted.
template <typename TX, typename TY>
struct Grads {
  const TX *dr, *stream;
  const TY* dz;
  int64_t drs, ss, dzs;
  TX* dx;
  TY *dy, *dg;
};

// dx, dy, dg, and per workgroup the sums of dz rh, dn yh and dx u n over its rows:
// part is (workgroups, 1 or 3, d).  A thread's columns are the same in every
// row, so the sums stay in its registers; the rows a workgroup takes side by
// side are added in LDS at the end, in a fixed order.
template <typename TX, typename TY, int TPR, int NV, Parts P>
__global__ void __launch_bounds__(rn_threads(TPR))
rn_bwd(Grads<TX, TY> gr, Branch<TY> in, Vectors vec, const float* __restrict__ rstd,
       const float* __restrict__ post_rstd, float* __restrict__ part, int64_t rows, int d) {
  constexpr int RPB = rn_threads(TPR) / TPR;
  constexpr int NP = P == ADD ? 1 : NV, NG = P == GATED ? NV : 1, SUMS = P == ADD ? 1 : 3;
  constexpr bool FROM_R = rn_from_r<TX>(P);
  constexpr int NY = FROM_R ? 1 : NV;
  __shared__ float red[2][16];
  const int lr = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int slot = 0;
  // The vectors at the thread's columns: in registers, or where 1024 threads have
  // too few of them (128 each) in LDS, each thread its own.
  constexpr bool IN_LDS = rn_in_lds(TPR, P);
  extern __shared__ __align__(16) char rn_smem[];
  float* const lds = reinterpret_cast<float*>(rn_smem);
  float wv[NV][8], pv[NP][8], sv[NP][8];
  float dw[NV][8] = {}, dp[NP][8] = {}, ds[NP][8] = {};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (i * TPR + t);
    load_ones(vec.w, vec.w16, d, c, wv[i]);
    if constexpr (P != ADD) {
      load_ones(vec.p, vec.w16, d, c, pv[i]);
      load_ones(vec.s, vec.w16, d, c, sv[i]);
    }
    if constexpr (IN_LDS) {
      store8(lds + c, 8, wv[i]);
      store8(lds + 8 * TPR + c, 8, pv[i]);
      store8(lds + 16 * TPR + c, 8, sv[i]);
    }
  }
  Raw8<TX> ar[NV], xr[NV];  // dr, r or x
  Raw8<TY> zr[NV], yr[NY], cr[NG];  // dz, y, gate
  float tau1, rho1;
  auto fetch = [&](int64_t r) {
    const bool live = r < rows;
    tau1 = live ? rstd[r] : 0.f;
    rho1 = P == ADD ? 1.f : !vec.p ? 1.f : live ? post_rstd[r] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t), left = live ? d - c : 0;
      xr[i].load(gr.stream + r * gr.ss + c, left);
      ar[i].load(gr.dr + r * gr.drs + c, gr.dr ? left : 0);
      zr[i].load(gr.dz + r * gr.dzs + c, gr.dz ? left : 0);
      if constexpr (!FROM_R) yr[i].load(in.y + r * in.ys + c, left);
      if constexpr (P == GATED && !IN_LDS) cr[i].load(in.g + r * in.gs + c, left);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + lr;
  // a row's loads before the last row's work, where the registers hold them
  constexpr bool AHEAD = !(IN_LDS && sizeof(TX) == 4);
  if constexpr (AHEAD) fetch(r);
  for (; r - lr < rows; r += step) {
    if constexpr (!AHEAD) fetch(r);
    const bool live = r < rows;
    const float tau = tau1, rho = rho1;
    if constexpr (P == GATED && IN_LDS) cr[0].load(in.g + r * in.gs + 8 * t, live ? d - 8 * t : 0);
    if constexpr (IN_LDS) load8(lds + 8 * t, 8, wv[0]);
    float h[NV][8], g[NV][8], a[NV][8], y[NY][8], u[NG][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i].get(h[i]);
      zr[i].get(g[i]);
      ar[i].get(a[i]);
      if constexpr (!FROM_R) yr[i].get(y[i]);
      if constexpr (P == GATED) cr[i].get(u[i]);
    }
    if constexpr (AHEAD) fetch(r + step);
    // the vectors of the thread's piece again, where they are in LDS
    auto vectors = [&](int i, int j) {
      if constexpr (IN_LDS) {
        pv[i][j] = lds[8 * TPR + 8 * t + j];
        sv[i][j] = lds[16 * TPR + 8 * t + j];
      }
    };
    float s0 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (P != ADD) {
          vectors(i, j);
          y[i][j] *= rho;  // yh
          float n = y[i][j] * pv[i][j] * sv[i][j];
          if constexpr (P == GATED) {
            u[i][j] = sigmoid(u[i][j]);
            n *= u[i][j];
          }
          h[i][j] += n;
        } else if constexpr (!FROM_R) {
          h[i][j] += y[i][j];
        }
        h[i][j] *= tau;  // rh
        dw[i][j] += g[i][j] * h[i][j];
        g[i][j] *= wv[i][j];
        s0 += g[i][j] * h[i][j];
      }
    const float m0 = row_sum<TPR>(s0, red, slot) / (float)d;
    float s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + t);
      const bool at = live && c < d;
#pragma unroll
      for (int j = 0; j < 8; ++j) a[i][j] += tau * (g[i][j] - h[i][j] * m0);  // dx
      if (at) stream8(gr.dx + r * d + c, d - c, a[i]);
      if constexpr (P == ADD) {
        if (at && gr.dy) stream8(gr.dy + r * d + c, d - c, a[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          vectors(i, j);
          const float n = y[i][j] * pv[i][j];
          if constexpr (P == GATED) {
            const float q = u[i][j];
            u[i][j] = a[i][j] * sv[i][j] * n * q * (1.f - q);  // dg
            a[i][j] *= q;
          }
          ds[i][j] += a[i][j] * n;
          a[i][j] *= sv[i][j];  // dn
          dp[i][j] += a[i][j] * y[i][j];
          a[i][j] *= pv[i][j];
          s1 += a[i][j] * y[i][j];
        }
        if constexpr (P == GATED) {
          if (at) stream8(gr.dg + r * d + c, d - c, u[i]);
        }
      }
    }
    if constexpr (P != ADD) {
      if (vec.p) {
        const float m1 = row_sum<TPR>(s1, red, slot) / (float)d;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) a[i][j] = rho * (a[i][j] - y[i][j] * m1);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + t);
        if (live && c < d) stream8(gr.dy + r * d + c, d - c, a[i]);
      }
    }
  }
  if (!part) return;
  float* const out = part + (int64_t)blockIdx.x * SUMS * d;
  auto sum_of = [&](int which, int i, int j) {
    if constexpr (P == ADD)
      return dw[i][j];
    else
      return which == 0 ? dw[i][j] : which == 1 ? dp[i][j] : ds[i][j];
  };
  if constexpr (RPB == 1) {
#pragma unroll
    for (int which = 0; which < SUMS; ++which)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + t);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = sum_of(which, i, j);
        if (c < d) store8(out + which * d + c, d - c, v);
      }
  } else {
    __shared__ float sums[RPB][TPR * NV * 8];
#pragma unroll
    for (int which = 0; which < SUMS; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[lr][8 * (i * TPR + t) + j] = sum_of(which, i, j);
      __syncthreads();
      for (int c = threadIdx.x; c < d; c += rn_threads(TPR)) {
        float s = sums[0][c];
#pragma unroll
        for (int i = 1; i < RPB; ++i) s += sums[i][c];
        out[which * d + c] = s;
      }
    }
  }
}

// The vectors' gradients from the workgroups' sums: a workgroup takes 32 columns
// of (sums, d) -- 8 lanes of 4 -- and its lane groups every 128th partial row, four in
// flight; joined in a wave, then over the waves in LDS, in a fixed order.
constexpr int RN_COLS = 32;
constexpr int RN_SUM_THREADS = 1024;
struct VectorGrads {
  void* out[3];  // of the norm's weight, the post norm's, the scale; null where not wanted
};
__global__ void __launch_bounds__(RN_SUM_THREADS)
rn_sums(const float* __restrict__ part, VectorGrads g, bool w16, int d, int64_t width, int nblk) {
  constexpr int SPLIT = RN_SUM_THREADS / 8;
  __shared__ f32x4 red[RN_SUM_THREADS / 64][8];
  const int quad = threadIdx.x % 8, sp = threadIdx.x / 8;
  const int64_t c = (int64_t)blockIdx.x * RN_COLS + 4 * quad;
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
    for (int i = 1; i < RN_SUM_THREADS / 64; ++i) s += red[i][quad];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j >= width) continue;
      const int which = (int)((c + j) / d);
      void* const out = which == 0 ? g.out[0] : which == 1 ? g.out[1] : g.out[2];
      const int64_t at = c + j - (int64_t)which * d;
      if (!out) continue;
      if (w16)
        reinterpret_cast<bf16*>(out)[at] = (bf16)s[j];
      else
        reinterpret_cast<float*>(out)[at] = s[j];
    }
  }
}

template <int TPR_, int NV_>
struct Shape {
  static constexpr int TPR = TPR_, NV = NV_;
};
// f(Shape) with the threads and pieces of a row of d values: where the vectors and their sums
// are many (a post norm, a gate, a scale) one piece a thread, else two once the row
// fills a wave.
template <Parts P, class F>
void with_shape(int64_t d, F&& f) {
  if (d <= 64) f(Shape<8, 1>{});
  else if (d <= 128) f(Shape<16, 1>{});
  else if (d <= 256) f(Shape<32, 1>{});
  else if (d <= 512) f(Shape<64, 1>{});
  else if (d <= 1024) f(std::conditional_t<P == ADD, Shape<64, 2>, Shape<128, 1>>{});
  else if (d <= 2048) f(std::conditional_t<P == ADD, Shape<128, 2>, Shape<256, 1>>{});
  else if (d <= 4096) f(std::conditional_t<P == ADD, Shape<256, 2>, Shape<512, 1>>{});
  else f(std::conditional_t<P == ADD, Shape<512, 2>, Shape<1024, 1>>{});
}
template <Parts P_>
struct With {
  static constexpr Parts P = P_;
};
template <class F>
void with_parts(const void* post, const void* gate, const void* scale, F&& f) {
  if (gate) f(With<GATED>{});
  else if (post || scale) f(With<SCALED>{});
  else f(With<ADD>{});
}
template <Parts P>
int64_t rn_blocks(int64_t rows, int64_t d, int64_t most) {
  int64_t n = 0;
  with_shape<P>(d, [&](auto s) {
    using S = decltype(s);
    constexpr int RPB = rn_threads(S::TPR) / S::TPR;
    n = (rows + RPB - 1) / RPB;
  });
  return n < most ? n : most;
}

// The built pairs of types: (bf16, bf16), (float32, float32) and a float32
// stream beside bf16 branches.
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
  return d > RN_MAX_D ? GMDN_ERR_UNSUPPORTED : GMDN_OK;
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

int gmdn_residual_norm_fwd(const void* x, const void* y, const void* weight, const void* post_weight, const void* gate,
                           const void* scale, void* r, void* z, float* rstd, float* post_rstd, int64_t rows, int64_t d,
                           int64_t x_stride, int64_t y_stride, int64_t gate_stride, float eps, int32_t x_type,
                           int32_t y_type, int32_t w_type, void* stream) {
  const int rc = check_dims(rows, d);
  if (rc != GMDN_OK) return rc;
  if (!pair_ok(x_type, y_type) || !type_ok(w_type)) return GMDN_ERR_UNSUPPORTED;
  if (!(eps >= 0.f) || x_stride < 0 || y_stride < 0 || gate_stride < 0) return GMDN_ERR_ARG;
  if (rows == 0) return GMDN_OK;
  if (!x || !y || !r || !z || !rstd || (post_weight && !post_rstd)) return GMDN_ERR_ARG;
  const Vectors vec{weight, post_weight, scale, w_type == GMDN_DTYPE_BF16};
  with_types(x_type, y_type, [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    const Branch<TY> in{(const TY*)y, (const TY*)gate, y_stride, gate_stride};
    with_parts(post_weight, gate, scale, [&](auto w) {
      constexpr Parts P = decltype(w)::P;
      with_shape<P>(d, [&](auto s) {
        using S = decltype(s);
        // one workgroup of 1024 threads is what a CU holds of this kernel
        const dim3 grid((unsigned)rn_blocks<P>(rows, d, S::TPR == 1024 ? RN_FWD_BLOCKS / 2 : RN_FWD_BLOCKS));
        hipLaunchKernelGGL((rn_fwd<TX, TY, S::TPR, S::NV, P>), grid, dim3(rn_threads(S::TPR)), 0, (hipStream_t)stream,
                           (const TX*)x, x_stride, in, vec, (TX*)r, (TY*)z, rstd, post_rstd, rows, (int)d, eps);
      });
    });
  });
  return launched();
}

size_t gmdn_residual_norm_bwd_workspace_floats(int64_t rows, int64_t d) {
  if (rows <= 0 || check_dims(rows, d) != GMDN_OK) return 0;
  const int64_t add = rn_blocks<ADD>(rows, d, RN_BWD_BLOCKS) * d, full = rn_blocks<GATED>(rows, d, RN_BWD_BLOCKS) * 3 * d;
  return (size_t)(add > full ? add : full);
}

int gmdn_residual_norm_bwd(const void* dr, const void* dz, const void* r_or_x, const void* y, const void* weight,
                           const void* post_weight, const void* gate, const void* scale, const float* rstd,
                           const float* post_rstd, void* dx, void* dy, void* dgate, void* dweight, void* dpost_weight,
                           void* dscale, float* workspace, size_t workspace_floats, int64_t rows, int64_t d,
                           int64_t dr_stride, int64_t dz_stride, int64_t r_or_x_stride, int64_t y_stride,
                           int64_t gate_stride, int32_t x_type, int32_t y_type, int32_t w_type, void* stream) {
  const int rc = check_dims(rows, d);
  if (rc != GMDN_OK) return rc;
  if (!pair_ok(x_type, y_type) || !type_ok(w_type)) return GMDN_ERR_UNSUPPORTED;
  if (dr_stride < 0 || dz_stride < 0 || r_or_x_stride < 0 || y_stride < 0 || gate_stride < 0) return GMDN_ERR_ARG;
  const bool plain = !post_weight && !gate && !scale;
  const bool wants = dweight || dpost_weight || dscale;
  if ((dweight && !weight) || (dpost_weight && !post_weight) || (dscale && !scale)) return GMDN_ERR_ARG;
  if (rows > 0) {
    const bool from_r = plain && x_type == GMDN_DTYPE_F32;
    if (!r_or_x || !rstd || !dx || (!from_r && !y) || (!plain && !dy) || (gate && !dgate) || (post_weight && !post_rstd))
      return GMDN_ERR_ARG;
    if (plain && !dy && x_type != y_type) return GMDN_ERR_ARG;
  }
  const int64_t nb = rows <= 0 ? 0 : plain ? rn_blocks<ADD>(rows, d, RN_BWD_BLOCKS) : rn_blocks<GATED>(rows, d, RN_BWD_BLOCKS);
  const int sums = plain ? 1 : 3;
  if (nb && wants && (!workspace || workspace_floats < (size_t)(nb * sums * d))) return GMDN_ERR_WORKSPACE;
  const Vectors vec{weight, post_weight, scale, w_type == GMDN_DTYPE_BF16};
  const hipStream_t st = (hipStream_t)stream;
  bool ok = false;
  if (nb) {
    with_types(x_type, y_type, [&](auto tx, auto ty) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      const Branch<TY> in{(const TY*)y, (const TY*)gate, y_stride, gate_stride};
      const Grads<TX, TY> g{(const TX*)dr, (const TX*)r_or_x, (const TY*)dz, dr_stride, r_or_x_stride, dz_stride,
                            (TX*)dx, (TY*)dy, (TY*)dgate};
      with_parts(post_weight, gate, scale, [&](auto w) {
        constexpr Parts P = decltype(w)::P;
        with_shape<P>(d, [&](auto s) {
          using S = decltype(s);
          auto* const kern = rn_bwd<TX, TY, S::TPR, S::NV, P>;
          const int lds = rn_in_lds(S::TPR, P) ? 3 * 8 * S::TPR * (int)sizeof(float) : 0;
          if (lds && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
            return;
          hipLaunchKernelGGL(kern, dim3((unsigned)nb), dim3(rn_threads(S::TPR)), lds, st, g, in, vec, rstd, post_rstd,
                             wants ? workspace : nullptr, rows, (int)d);
          ok = true;
        });
      });
    });
    if (hipGetLastError() != hipSuccess || !ok) return GMDN_ERR_LAUNCH;
  }
  if (!wants) return GMDN_OK;
  const int64_t width = sums * d;
  hipLaunchKernelGGL(rn_sums, dim3((unsigned)((width + RN_COLS - 1) / RN_COLS)), dim3(RN_SUM_THREADS), 0, st, workspace,
                     VectorGrads{{dweight, dpost_weight, dscale}}, w_type == GMDN_DTYPE_BF16, (int)d, width, (int)nb);
  return launched();
}

}  // extern "C"
