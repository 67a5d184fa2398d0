// 8-bit floating-point codes with scales: the conversion shared by the norm with 8-bit output and by block_quantize.
//
//   scale = max(amax * (1 / top), 2^-126)   amax: largest magnitude of the block, top: largest finite value of the format
//   code  = round(x * (1 / scale))          to nearest even, beyond top: top
//
// in 32 bits, each quotient and product rounded: the scale is next to amax / top or the same (1.0e-7 apart at most), and a
// value next to the middle of two codes may get either.  The lower bound keeps 1 / scale finite, so that a block of zeros gets codes of zero.  A NaN in the block
// makes the scale and every code NaN; an infinity makes the scale infinite, its own code NaN and the others zero, so
// that no product with the block is finite.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include "solid_core_gpu.h"
#include "layout.h"

namespace sd {

constexpr int B8_BLOCK = 128;                            // elements along dimension 0 that share a scale
constexpr int B8_E4M3 = SOLID_GPU_E4M3, B8_E5M2 = SOLID_GPU_E5M2;

// A caller's codes and scales: what every entry point asks of them.  Those of a matrix without elements may have no address.
static inline int check_blocks(const solid_gpu_blocks *b, const char *op, const char *what, bool empty)
{
   if (b == nullptr || (!empty && (b->codes == nullptr || b->scales == nullptr))) SD_ERROR("%s: missing codes or scales of %s", op, what);
   if (b->format != SOLID_GPU_E4M3 && b->format != SOLID_GPU_E5M2) SD_ERROR("%s: unknown 8-bit format %d of %s", op, b->format, what);
   if (b->block != 1 && b->block != B8_BLOCK) SD_ERROR("%s: a scale of %s belongs to 1 or 128 rows, not to %d", op, what, b->block);
   if ((uintptr_t)b->scales % 4 != 0 || b->scale_stride0 % 4 != 0 || b->scale_stride1 % 4 != 0)
      SD_ERROR("%s: the scales of %s must be aligned to their element size", op, what);
   return 0;
}

// Magnitudes are compared as bit patterns: for non-negative floats the order of the patterns is the order of the
// values, and NaN lies above infinity, so that it survives the maximum (fmaxf would drop it).
__device__ __forceinline__ uint32_t b8_magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ float b8_scale(uint32_t amax, int format)
{
   const float s = __uint_as_float(amax) * (format == B8_E4M3 ? 1.0f / 448.0f : 1.0f / 57344.0f);
   return __uint_as_float(max(__float_as_uint(s), 0x00800000u));
}

// Two values to two codes, x in the low byte
__device__ __forceinline__ uint32_t b8_pair(float x, float y, int format)
{
   uint16_t r;
   if (format == B8_E4M3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
   else                   asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
   return r;
}

__device__ __forceinline__ uint32_t b8_four(const float *x, float inv, int format)
{
   return b8_pair(x[0] * inv, x[1] * inv, format) | (b8_pair(x[2] * inv, x[3] * inv, format) << 16);
}

// Element types as these operators compute with them.  Halves are rounded to nearest even and keep their subnormals:
// gradients live there.  (The copy family rounds as the reference's CPU code does, which is neither.)
template <class T> struct Real { using acc = float; };
template <> struct Real<double> { using acc = double; };
__device__ __forceinline__ float  to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float  to_acc(float v)  { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ void from_acc(__half &d, float v)  { d = __float2half_rn(v); }
__device__ __forceinline__ void from_acc(float &d, float v)   { d = v; }
__device__ __forceinline__ void from_acc(double &d, double v) { d = v; }

// Eight elements of a row as one or more 16-byte accesses
template <class T> struct alignas(16) Eight { T e[8]; };

template <class T> __device__ __forceinline__ Eight<T> load_eight(const void *p)
{
   Eight<T> c;
#pragma unroll
   for (int i = 0; i < (int)sizeof(Eight<T>) / 16; i++) reinterpret_cast<uint4 *>(&c)[i] = reinterpret_cast<const uint4 *>(p)[i];
   return c;
}
template <class T> __device__ __forceinline__ void store_eight(void *p, const Eight<T> &c)
{
#pragma unroll
   for (int i = 0; i < (int)sizeof(Eight<T>) / 16; i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(&c)[i];
}

} // namespace sd
