// Rows of values in pieces of eight, for the kernels that stream (rows, d)
// matrices: loads and stores of a piece at any alignment, sums and maxima
// over the threads of a row, and the 8-bit checkpoint format.
//
// A piece is 8 consecutive values of a row (16 bytes of bf16, 32 of float32).
// Rows of odd widths start at any element, so the vector types below promise
// element alignment only; gfx950 loads and stores them by one instruction all
// the same (packing 16384 x 4095 bf16 takes 44 us, 16384 x 4096 35 us: the
// pieces cross cache lines).  Only the short last piece of a row is read and
// written by elements.
#pragma once
#include "../../include/gmdn_scan.h"
#include "tile.h"

namespace gmdn {

typedef bf16 bf16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Piece of n >= 1 values at p; values from n on are `pad`.
GMDN_DEV void load8(const bf16* p, int n, float (&x)[8], float pad = 0.f) {
  if (n >= 8) {
    const bf16x8_any v = *reinterpret_cast<const bf16x8_any*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? (float)p[j] : pad;
  }
}
GMDN_DEV void load8(const float* p, int n, float (&x)[8], float pad = 0.f) {
  if (n >= 8) {
    const f32x4_any a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? p[j] : pad;
  }
}
GMDN_DEV void store8(bf16* p, int n, const float (&x)[8]) {
  const bf16x8 v = cat8(to_bf16x4(f32x4{x[0], x[1], x[2], x[3]}), to_bf16x4(f32x4{x[4], x[5], x[6], x[7]}));
  if (n >= 8) {
    *reinterpret_cast<bf16x8_any*>(p) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = v[j];
  }
}
GMDN_DEV void store8(float* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    *reinterpret_cast<f32x4_any*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4_any*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = x[j];
  }
}
// The same past the caches (nontemporal) for outputs that a kernel does not
// read again.  bf16 only: a wave's pieces fill whole lines in one instruction.  The
// two halves of float32 pieces do not, and went slower so (a layer norm's dx
// at 16384 x 2048: 89 us, with plain stores 80; bf16 at 16384 x 1024: 35 and 39).
GMDN_DEV void stream8(bf16* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    const bf16x8_any v = cat8(to_bf16x4(f32x4{x[0], x[1], x[2], x[3]}), to_bf16x4(f32x4{x[4], x[5], x[6], x[7]}));
    __builtin_nontemporal_store(v, reinterpret_cast<bf16x8_any*>(p));
  } else {
    store8(p, n, x);
  }
}
GMDN_DEV void stream8(float* p, int n, const float (&x)[8]) { store8(p, n, x); }
// float32 past the caches all the same: faster while the whole matrix would fit
// them (a norm's dx at 16384 x 1024: 37 us, plain 39; 16384 x 2048 above).
GMDN_DEV void stream8_f32(float* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    f32x4_any* q = reinterpret_cast<f32x4_any*>(p);
    __builtin_nontemporal_store(f32x4_any{x[0], x[1], x[2], x[3]}, q);
    __builtin_nontemporal_store(f32x4_any{x[4], x[5], x[6], x[7]}, q + 1);
  } else {
    store8(p, n, x);
  }
}
GMDN_DEV void stream8_f32(bf16* p, int n, const float (&x)[8]) { stream8(p, n, x); }
// At both ends of one side of a branch whose sides differ in their caching
// only: the compiler would join them into one, without the difference.
GMDN_DEV void apart() { asm volatile(""); }

// A piece as it lies in memory, for loads that are to be in flight over other
// work; values from n on are `pad` (0 or an infinity).  FAR: whole bf16 pieces are
// loaded past the caches (nontemporal), for matrices of at least FAR_BYTES:
// what the last kernel left in the 256 MB cache is then little of them, and
// the outputs keep it.  GELU's backward at 16384 x 4096 takes 76 us so and 83 us
// without; at 16384 x 1024, 24 and 21.
constexpr int64_t FAR_BYTES = 96 << 20;
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16> {
  u32x4 v;
  template <bool FAR = false>
  GMDN_DEV void load(const bf16* p, int n, float pad = 0.f) {
    const u32x4_any* q = reinterpret_cast<const u32x4_any*>(p);
    if (n >= 8) {
      if constexpr (FAR)
        v = __builtin_nontemporal_load(q);
      else
        v = *q;
    } else {
      const uint32_t bits = __builtin_bit_cast(uint32_t, pad) >> 16;
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = (2 * j < n ? h[2 * j] : bits) | (2 * j + 1 < n ? (uint32_t)h[2 * j + 1] : bits) << 16;
    }
  }
  GMDN_DEV void get(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __builtin_bit_cast(float, v[j] << 16);
      x[2 * j + 1] = __builtin_bit_cast(float, v[j] & 0xffff0000u);
    }
  }
};
template <>
struct Raw8<float> {
  float v[8];
  template <bool FAR = false>
  GMDN_DEV void load(const float* p, int n, float pad = 0.f) {
    load8(p, n, v, pad);
  }
  GMDN_DEV void get(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v[j];
  }
};
// Values of a weight vector held in float32 or bf16 (is_bf16).
GMDN_DEV void load8_weight(const void* w, bool is_bf16, int at, int n, float (&x)[8]) {
  if (is_bf16)
    load8(reinterpret_cast<const bf16*>(w) + at, n, x);
  else
    load8(reinterpret_cast<const float*>(w) + at, n, x);
}

// ------------------------------------------------- the 8-bit checkpoint
// Groups of 128 consecutive values of a row (the last one may be short).
// With amax the group's largest magnitude:
//   scale = amax * STEP8     q = rint(x * (127 / amax))     x' = q * scale
// in float32, each operation rounded by itself (no contraction), so that any
// float32 evaluation gives the same bytes.  STEP8 is the float32 below
// 1 / 127: 127 * scale does not exceed amax, so that x' is finite wherever x
// is, up to the type's largest value.  A group whose amax is below 2^-100
// is kept as zeros; one that holds an infinity or a NaN reads back as NaN
// (scale NaN).  |x' - x| <= amax / 254 up to rounding.
constexpr int GROUP8 = 128;
constexpr int GROUP8_PIECES = GROUP8 / 8;
constexpr float STEP8 = 0x1.020406p-7f;
constexpr uint32_t TINY8 = 0x0d800000u;  // bits of 2^-100
constexpr uint32_t INF_BITS = 0x7f800000u;

inline __host__ __device__ int64_t groups8(int64_t d) { return (d + GROUP8 - 1) / GROUP8; }

// Largest magnitude of a piece, as bits: their order is that of the values,
// with infinity and then NaN at the end.
GMDN_DEV uint32_t amax_bits(const float (&x)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu;
    a = b > a ? b : a;
  }
  return a;
}

struct Scale8 {
  float inverse, scale;
};
GMDN_DEV Scale8 scale8(uint32_t amax) {
#pragma clang fp contract(off)
  if (amax < TINY8) return {0.f, 0.f};
  if (amax >= INF_BITS) return {0.f, __builtin_nanf("")};
  const float a = __builtin_bit_cast(float, amax);
  return {127.f / a, a * STEP8};
}
// The bytes of a piece.  x * inverse is rounded to float32, then to an
// integer by adding 1.5 * 2^23 (round to nearest even), whose low byte is
// the integer's; inverse 0 (a group without a scale) gives 0 for every x, as
// the product may be NaN there.
GMDN_DEV u32x2_any quant8(const float (&x)[8], float inverse) {
#pragma clang fp contract(off)
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = x[j] * inverse;
    b[j] = __builtin_bit_cast(uint32_t, t + 12582912.f);
  }
  u32x2_any r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000c0cu);
    r[h] = inverse == 0.f ? 0u : lo | hi;
  }
  return r;
}
GMDN_DEV void store_q8(int8_t* p, int n, u32x2_any v) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_any*>(p) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (int8_t)(v[j / 4] >> (8 * (j % 4)));
  }
}
GMDN_DEV void dequant8(u32x2_any v, float scale, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)(v[j / 4] >> (8 * (j % 4))) * scale;
}
GMDN_DEV u32x2_any load_q8(const int8_t* p, int n) {
  if (n >= 8) return *reinterpret_cast<const u32x2_any*>(p);
  u32x2_any v = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) v[j / 4] |= (uint32_t)(uint8_t)p[j] << (8 * (j % 4));
  return v;
}

// ------------------------------------------------- over the threads of a row
// Over aligned groups of N lanes (N a power of two up to 64), the result in
// each of them: within 16 lanes by DPP (the quad's neighbours, then mirrors of 8 and
// 16: once a quad agrees, a mirror pairs it with another), the rows of 16 of a
// wave through scalar registers.  A butterfly of LDS permutes instead costs its
// latency at every step: in a workgroup of 16 waves the three reductions of a
// row of logits took 6400 cycles so.
template <int CTRL>
GMDN_DEV uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
template <int N, class F>
GMDN_DEV uint32_t lanes_fold(uint32_t x, F&& f) {
  if constexpr (N > 1) x = f(x, dpp<0xb1>(x));   // quad_perm 1 0 3 2
  if constexpr (N > 2) x = f(x, dpp<0x4e>(x));   // quad_perm 2 3 0 1
  if constexpr (N > 4) x = f(x, dpp<0x141>(x));  // row_half_mirror
  if constexpr (N > 8) x = f(x, dpp<0x140>(x));  // row_mirror
  if constexpr (N == 32) x = f(x, (uint32_t)__shfl_xor((int)x, 16, 64));
  if constexpr (N == 64) {
    const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16),
                   c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    x = f(f(a, b), f(c, d));
  }
  return x;
}
GMDN_DEV uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
GMDN_DEV float float_of(uint32_t x) { return __builtin_bit_cast(float, x); }
template <int N>
GMDN_DEV float lanes_sum(float x) {
  return float_of(lanes_fold<N>(bits_of(x), [](uint32_t a, uint32_t b) { return bits_of(float_of(a) + float_of(b)); }));
}
template <int N>
GMDN_DEV uint32_t lanes_max(uint32_t x) {
  return lanes_fold<N>(x, [](uint32_t a, uint32_t b) { return b > a ? b : a; });
}
template <int N>
GMDN_DEV float lanes_max(float x) {
  return float_of(lanes_fold<N>(bits_of(x), [](uint32_t a, uint32_t b) { return bits_of(fmaxf(float_of(a), float_of(b))); }));
}

// Element type codes of the C-ABI.
inline bool type_ok(int32_t t) { return t == GMDN_DTYPE_BF16 || t == GMDN_DTYPE_F32; }
inline int launched() { return hipGetLastError() == hipSuccess ? GMDN_OK : GMDN_ERR_LAUNCH; }

}  // namespace gmdn
