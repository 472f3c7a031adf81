// 8-bit activation checkpoints (rows8.h has the format): packing and reading
// back, and GELU that keeps its input packed (include/gmdn_lm.h).
//
// All four kernels stream: a group of 128 values is 16 lanes of one piece
// each, its amax a butterfly over them; nothing is shared between groups.
// Memory bound (GELU's forward nearly by its vector instructions too: they are
// active in 98 % of its cycles; fewer of them gained nothing).  At 16384 x 4096 bf16:
// pack 35 us (5.8 TB/s), unpack 29 us (6.9), GELU 61 us (5.5), its backward with
// the output again 76 us (6.2); a 1 GiB copy reaches 5.1 TB/s.
#include "../../include/gmdn_lm.h"
#include "rows8.h"

namespace gmdn {
namespace {

// Threads, and pieces a thread has in flight, A8_THREADS apart.  GELU's backward at
// 16384 x 4096: 256 x 2 76 us, 256 x 4 79, 1024 x 4 90; at 256 x 512 4, 6 and 12 us.
constexpr int A8_THREADS = 256;
constexpr int A8_PIECES = 2;
constexpr int A8_SPAN = A8_THREADS * A8_PIECES;
constexpr int64_t A8_GRID = 1 << 20;

// A piece's place.  Groups are 16 pieces; where rows are whole groups and lie
// one after the other (`flat`), groups are numbered through the matrix.
struct Place {
  int64_t row, unit;  // the group's index in `scale`
  int c, n;           // first column, values (0: past the row's or the matrix's end)
};
struct Shape {
  int64_t units, d, groups;
  bool flat;
};
GMDN_DEV Place place(int64_t piece, const Shape& s) {
  Place p;
  p.unit = piece / GROUP8_PIECES;
  const int lane = (int)(piece % GROUP8_PIECES);
  if (s.flat) {  // as one row
    p.row = 0;
    p.c = 0;
    p.n = p.unit < s.units ? 8 : 0;
    return p;
  }
  p.row = p.unit < ((int64_t)1 << 32) ? (uint32_t)p.unit / (uint32_t)s.groups : p.unit / s.groups;
  const int64_t c = (p.unit - p.row * s.groups) * GROUP8 + 8 * lane;
  p.c = (int)c;
  p.n = p.unit < s.units && c < s.d ? (int)(s.d - c < 8 ? s.d - c : 8) : 0;
  return p;
}
// Offsets of a piece in a matrix of row stride `stride`, and in a contiguous one.
GMDN_DEV int64_t offset(const Place& p, int64_t piece, const Shape& s, int64_t stride) {
  return s.flat ? piece * 8 : p.row * stride + p.c;
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

// The checkpoint of x; GELU: and a = GELU(x), or that alone (q null).
template <typename T, bool GELU, bool FAR>
__global__ void __launch_bounds__(A8_THREADS)
pack(const T* __restrict__ x, T* __restrict__ a, int8_t* __restrict__ q, float* __restrict__ scale, Shape s,
     int64_t xs) {
  for (int64_t b0 = (int64_t)blockIdx.x * A8_SPAN; b0 < s.units * GROUP8_PIECES; b0 += (int64_t)gridDim.x * A8_SPAN) {
    Raw8<T> raw[A8_PIECES];
#pragma unroll
    for (int i = 0; i < A8_PIECES; ++i) {
      const int64_t piece = b0 + i * A8_THREADS + threadIdx.x;
      const Place p = place(piece, s);
      const T* from = x + offset(p, piece, s, xs);
      raw[i].template load<FAR>(from, p.n);
    }
#pragma unroll
    for (int i = 0; i < A8_PIECES; ++i) {
      const int64_t piece = b0 + i * A8_THREADS + threadIdx.x;
      const Place p = place(piece, s);
      float v[8];
      raw[i].get(v);
      const int64_t at = offset(p, piece, s, s.d);
      if (!GELU || q) {
        const Scale8 sc = scale8(lanes_max<GROUP8_PIECES>(amax_bits(v)));
        if (p.n && piece % GROUP8_PIECES == 0) scale[p.unit] = sc.scale;
        if (p.n) store_q8(q + at, p.n, quant8(v, sc.inverse));
      }
      if (!p.n) continue;
      if constexpr (GELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = gelu(v[j]);
        stream8(a + at, p.n, v);
      }
    }
  }
}

// UNPACK: x from the checkpoint.  Otherwise GELU's backward: dh, and the
// output again where `a` is given.
template <typename T, bool UNPACK, bool FAR>
__global__ void __launch_bounds__(A8_THREADS)
unpack(const int8_t* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ da, int64_t das,
       T* __restrict__ dh, T* __restrict__ a, Shape s) {
  for (int64_t b0 = (int64_t)blockIdx.x * A8_SPAN; b0 < s.units * GROUP8_PIECES; b0 += (int64_t)gridDim.x * A8_SPAN) {
    Raw8<T> raw[A8_PIECES];
    u32x2_any kept[A8_PIECES];
    float sc[A8_PIECES];
#pragma unroll
    for (int i = 0; i < A8_PIECES; ++i) {
      const int64_t piece = b0 + i * A8_THREADS + threadIdx.x;
      const Place p = place(piece, s);
      kept[i] = load_q8(q + offset(p, piece, s, s.d), p.n);
      sc[i] = p.n ? scale[p.unit] : 0.f;
      if constexpr (!UNPACK) {
        const T* from = da + offset(p, piece, s, das);
        raw[i].template load<FAR>(from, p.n);
      }
    }
#pragma unroll
    for (int i = 0; i < A8_PIECES; ++i) {
      const int64_t piece = b0 + i * A8_THREADS + threadIdx.x;
      const Place p = place(piece, s);
      if (!p.n) continue;
      const int64_t at = offset(p, piece, s, s.d);
      float v[8];
      dequant8(kept[i], sc[i], v);
      if constexpr (!UNPACK) {
        float g[8];
        raw[i].get(g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float y, slope;
          gelu(v[j], y, slope);
          g[j] *= slope;
          v[j] = y;
        }
        stream8(dh + at, p.n, g);
      }
      if (UNPACK || a) stream8(a + at, p.n, v);
    }
  }
}

int check8(int64_t rows, int64_t d, int64_t stride, int32_t dtype) {
  if (rows < 0 || d <= 0 || stride < 0) return GMDN_ERR_ARG;
  if (!type_ok(dtype)) return GMDN_ERR_UNSUPPORTED;
  if (d >= ((int64_t)1 << 31) || rows > ((int64_t)1 << 48) / d) return GMDN_ERR_ARG;
  return GMDN_OK;
}
Shape shape_of(int64_t rows, int64_t d, int64_t stride) {
  const int64_t g = groups8(d);
  return {rows * g, d, g, d % GROUP8 == 0 && (stride == d || rows == 1)};
}
dim3 grid8(const Shape& s) {
  const int64_t n = (s.units * GROUP8_PIECES + A8_SPAN - 1) / A8_SPAN;
  return dim3((unsigned)(n < A8_GRID ? n : A8_GRID));
}

template <bool GELU>
int pack_call(const void* x, void* a, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t xs, int32_t dtype,
              void* stream) {
  const int rc = check8(rows, d, xs, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!x || !q != !scale || (GELU ? !a : !q)) return GMDN_ERR_ARG;
  const Shape s = shape_of(rows, d, xs);
  if (dtype == GMDN_DTYPE_BF16 && rows * d * 2 >= FAR_BYTES)
    hipLaunchKernelGGL((pack<bf16, GELU, true>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, (const bf16*)x,
                       (bf16*)a, q, scale, s, xs);
  else if (dtype == GMDN_DTYPE_BF16)
    hipLaunchKernelGGL((pack<bf16, GELU, false>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, (const bf16*)x,
                       (bf16*)a, q, scale, s, xs);
  else
    hipLaunchKernelGGL((pack<float, GELU, false>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, (const float*)x,
                       (float*)a, q, scale, s, xs);
  return launched();
}
template <bool UNPACK>
int unpack_call(const int8_t* q, const float* scale, const void* da, int64_t das, void* dh, void* a, int64_t rows,
                int64_t d, int32_t dtype, void* stream) {
  const int rc = check8(rows, d, das, dtype);
  if (rc != GMDN_OK || rows == 0) return rc;
  if (!q || !scale || (UNPACK ? !a : !da || !dh)) return GMDN_ERR_ARG;
  const Shape s = shape_of(rows, d, das);
  if (!UNPACK && dtype == GMDN_DTYPE_BF16 && rows * d * 2 >= FAR_BYTES)
    hipLaunchKernelGGL((unpack<bf16, UNPACK, !UNPACK>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, q, scale,
                       (const bf16*)da, das, (bf16*)dh, (bf16*)a, s);
  else if (dtype == GMDN_DTYPE_BF16)
    hipLaunchKernelGGL((unpack<bf16, UNPACK, false>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, q, scale,
                       (const bf16*)da, das, (bf16*)dh, (bf16*)a, s);
  else
    hipLaunchKernelGGL((unpack<float, UNPACK, false>), grid8(s), dim3(A8_THREADS), 0, (hipStream_t)stream, q, scale,
                       (const float*)da, das, (float*)dh, (float*)a, s);
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
  return unpack_call<true>(q, scale, nullptr, d, nullptr, x, rows, d, dtype, stream);
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
