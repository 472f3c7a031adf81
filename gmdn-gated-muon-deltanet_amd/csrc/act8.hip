// 8-bit activation checkpoints (rows8.h has the format): packing and reading
// back, and GELU that keeps its input packed (include/gmdn_lm.h).
//
// All four kernels stream: a group of 128 values is 16 lanes of one piece
// each, its amax a butterfly over them; nothing is shared between groups.
#include "../../include/gmdn_lm.h"
#include "rows8.h"

namespace gmdn {
namespace {

constexpr int A8_THREADS = 256;
constexpr int A8_GROUPS = A8_THREADS / GROUP8_PIECES;  // groups of a workgroup

// The group, and the piece in it, of this thread: row, first column, values
// of the piece (0: past the row's end), and the group's index in `scale`.
struct Place {
  int64_t row, unit;
  int c, n;
};
GMDN_DEV Place place(int64_t unit, int64_t d) {
  const int64_t g = groups8(d);
  Place p;
  p.unit = unit;
  p.row = unit / g;
  const int64_t c = (unit - p.row * g) * GROUP8 + 8 * (threadIdx.x % GROUP8_PIECES);
  p.c = (int)c;
  p.n = c < d ? (int)(d - c < 8 ? d - c : 8) : 0;
  return p;
}

// GELU with the normal distribution function Phi, and its derivative
// Phi(h) + h phi(h).  With u = |h|, t = 1 / (1 + 0.27 u) and E = e^(-u^2 / 4):
//   Phi(-u) = E E t R(t),
// R the polynomial of degree 8 whose largest relative error on 0 <= u <= 14.5
// is least (Remez exchange on 0.5 erfc(u / sqrt 2) e^(u^2 / 2) / t; 2.4e-8,
// and E E is 0 in float32 beyond).  Relative accuracy holds into the lower
// tail (18 u of float32 up to |h| = 3, then h^2 / 2 u from rounding the
// exponent), where 1 + erf would cancel, and one exponential serves Phi and
// phi.  E stands for half the exponent: the instruction flushes results below
// 2^-126, which the product E E reaches without.
GMDN_DEV float lower_tail(float h, float& half) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.27f, fabsf(h), 1.f));
  float r = 0x1.da7fa0p-6f;
  r = __builtin_fmaf(r, t, -0x1.030b00p-3f);
  r = __builtin_fmaf(r, t, 0x1.5bb8ccp-3f);
  r = __builtin_fmaf(r, t, -0x1.1b7ca4p-4f);
  r = __builtin_fmaf(r, t, 0x1.b9a74ap-4f);
  r = __builtin_fmaf(r, t, 0x1.271d86p-4f);
  r = __builtin_fmaf(r, t, 0x1.a10426p-4f);
  r = __builtin_fmaf(r, t, 0x1.b87ee0p-4f);
  r = __builtin_fmaf(r, t, 0x1.b9394cp-4f);
  half = __builtin_amdgcn_exp2f(h * h * -0.36067376022224085f);  // log2(e) / 4
  return r * t * half * half;
}
GMDN_DEV float gelu(float h) {
  float half;
  const float low = lower_tail(h, half);
  return h * (h < 0.f ? low : 1.f - low);
}
GMDN_DEV void gelu(float h, float& a, float& slope) {
  float half;
  const float low = lower_tail(h, half), cdf = h < 0.f ? low : 1.f - low;
  a = h * cdf;
  slope = __builtin_fmaf(h * (0.39894228040143268f * half), half, cdf);
}

template <typename T, bool GELU>
__global__ void __launch_bounds__(A8_THREADS)
pack(const T* __restrict__ x, T* __restrict__ a, int8_t* __restrict__ q, float* __restrict__ scale, int64_t units,
     int64_t d, int64_t xs) {
  for (int64_t u0 = (int64_t)blockIdx.x * A8_GROUPS; u0 < units; u0 += (int64_t)gridDim.x * A8_GROUPS) {
    const int64_t u = u0 + threadIdx.x / GROUP8_PIECES;
    if (u >= units) continue;  // whole groups of 16 lanes
    const Place p = place(u, d);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (p.n) load8(x + p.row * xs + p.c, p.n, v);
    const Scale8 sc = scale8(lanes_max<GROUP8_PIECES>(amax_bits(v)));
    if (threadIdx.x % GROUP8_PIECES == 0) scale[u] = sc.scale;
    if (!p.n) continue;
    const int64_t at = p.row * d + p.c;
    store_q8(q + at, p.n, quant8(v, sc.inverse));
    if constexpr (GELU) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = gelu(v[j]);
      store8(a + at, p.n, y);
    }
  }
}

// UNPACK: x from the checkpoint.  Otherwise GELU's backward: dh, and the
// output again where `a` is given.
template <typename T, bool UNPACK>
__global__ void __launch_bounds__(A8_THREADS)
unpack(const int8_t* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ da, int64_t das,
       T* __restrict__ dh, T* __restrict__ a, int64_t units, int64_t d) {
  for (int64_t u0 = (int64_t)blockIdx.x * A8_GROUPS; u0 < units; u0 += (int64_t)gridDim.x * A8_GROUPS) {
    const int64_t u = u0 + threadIdx.x / GROUP8_PIECES;
    if (u >= units) continue;
    const Place p = place(u, d);
    if (!p.n) continue;
    const int64_t at = p.row * d + p.c;
    float v[8];
    dequant8(load_q8(q + at, p.n), scale[u], v);
    if constexpr (UNPACK) {
      store8(a + at, p.n, v);
    } else {
      float g[8], y[8];
      load8(da + p.row * das + p.c, p.n, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float slope;
        gelu(v[j], y[j], slope);
        g[j] *= slope;
      }
      store8(dh + at, p.n, g);
      if (a) store8(a + at, p.n, y);
    }
  }
}

int check8(int64_t rows, int64_t d, int64_t stride, int32_t dtype) {
  if (rows < 0 || d <= 0 || stride < 0) return GMDN_ERR_ARG;
  if (!type_ok(dtype)) return GMDN_ERR_UNSUPPORTED;
  if (d >= ((int64_t)1 << 31) || rows > ((int64_t)1 << 40)) return GMDN_ERR_ARG;
  return GMDN_OK;
}
dim3 grid8(int64_t units) {
  const int64_t n = (units + A8_GROUPS - 1) / A8_GROUPS;
  return dim3((unsigned)(n < ((int64_t)1 << 30) ? n : (int64_t)1 << 30));
}

template <bool GELU>
int pack_call(const void* x, void* a, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t xs, int32_t dtype,
              void* stream) {
  const int rc = check8(rows, d, xs, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!x || !q || !scale || (GELU && !a)) return GMDN_ERR_ARG;
  const int64_t units = rows * groups8(d);
  if (dtype == GMDN_DTYPE_BF16)
    hipLaunchKernelGGL((pack<bf16, GELU>), grid8(units), dim3(A8_THREADS), 0, (hipStream_t)stream, (const bf16*)x,
                       (bf16*)a, q, scale, units, d, xs);
  else
    hipLaunchKernelGGL((pack<float, GELU>), grid8(units), dim3(A8_THREADS), 0, (hipStream_t)stream, (const float*)x,
                       (float*)a, q, scale, units, d, xs);
  return launched();
}
template <bool UNPACK>
int unpack_call(const int8_t* q, const float* scale, const void* da, int64_t das, void* dh, void* a, int64_t rows,
                int64_t d, int32_t dtype, void* stream) {
  const int rc = check8(rows, d, das, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!q || !scale || (UNPACK ? !a : !da || !dh)) return GMDN_ERR_ARG;
  const int64_t units = rows * groups8(d);
  if (dtype == GMDN_DTYPE_BF16)
    hipLaunchKernelGGL((unpack<bf16, UNPACK>), grid8(units), dim3(A8_THREADS), 0, (hipStream_t)stream, q, scale,
                       (const bf16*)da, das, (bf16*)dh, (bf16*)a, units, d);
  else
    hipLaunchKernelGGL((unpack<float, UNPACK>), grid8(units), dim3(A8_THREADS), 0, (hipStream_t)stream, q, scale,
                       (const float*)da, das, (float*)dh, (float*)a, units, d);
  return launched();
}

}  // namespace
}  // namespace gmdn

using namespace gmdn;

extern "C" {

int64_t gmdn_act8_groups(int64_t d) { return d > 0 ? groups8(d) : 0; }

int gmdn_act8_pack(const void* x, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t x_stride, int32_t dtype,
                   void* stream) {
  return pack_call<false>(x, nullptr, q, scale, rows, d, x_stride, dtype, stream);
}

int gmdn_act8_unpack(const int8_t* q, const float* scale, void* x, int64_t rows, int64_t d, int32_t dtype,
                     void* stream) {
  return unpack_call<true>(q, scale, nullptr, 0, nullptr, x, rows, d, dtype, stream);
}

int gmdn_gelu8_fwd(const void* h, void* a, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t h_stride,
                   int32_t dtype, void* stream) {
  return pack_call<true>(h, a, q, scale, rows, d, h_stride, dtype, stream);
}

int gmdn_gelu8_bwd(const void* da, const int8_t* q, const float* scale, void* dh, void* a, int64_t rows, int64_t d,
                   int64_t da_stride, int32_t dtype, void* stream) {
  return unpack_call<false>(q, scale, da, da_stride, dh, a, rows, d, dtype, stream);
}

}  // extern "C"
