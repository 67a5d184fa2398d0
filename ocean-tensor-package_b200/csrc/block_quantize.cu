// solid_gpu_block_quantize: the codes and scales of a matrix, a scale for 128 elements of dimension 0 by 1 or 128 rows.
//
// Bound by memory: a block of 256 threads loads a tile (128 x 64, 128 x 128) once into registers, finds the largest magnitudes,
// and writes the codes.  The tile is read along whichever dimension of the source is contiguous, eight elements a
// thread; where that is the rows' dimension (the codes of a transposed matrix) the codes turn in shared memory, one
// byte each, so that both sides of the copy move whole lines.
//
// Measured in a captured graph with inputs that rotate over more than the L2 cache: floats to e4m3 with square blocks, 8192 x
// 4096, 32.1 us (5.2 TB/s, 80 % of the copy rate); halves of 4096 x 4096 with a scale for each row along 20.3 us, across
// 19.4 us (38 and 40 %: a tile's load, two barriers and store are a chain that five blocks an SM overlap only in part; with
// 128 x 128 tiles and three blocks 30 % slower), with square blocks 25.9 and 23.4 us (30 and 33 %); floats 17.4 to
// 19.4 us (73 to 66 %), doubles 32.4 to 38.7 us (71 to 60 %); halves off 16-byte boundaries 31.5 us along, 24.8 across.
#include "block8.cuh"

namespace sd {

struct QuantArgs {
   int64_t n, rows;
   const char *x; int64_t s0, s1;
   char *codes; int64_t ld;
   float *scale; int64_t ss0, ss1;
   int format;
};

constexpr int QT = 128;                                   // tile edge along dimension 0

// Values of one thread: runs of eight.  Doubles are taken in 32 bits, as the scales are.
template <class T> struct Held { using type = T; };
template <> struct Held<double> { using type = float; };

// RB: rows that share a scale.  Where each row has its own a tile takes 64 rows, so that more and smaller blocks are on an
// SM and one's loads run beside another's stores; 128 by 128 it has to be for a common scale.
template <class T, int RB> struct QuantShape {
   static constexpr int rows = RB == 1 ? 64 : QT;
   static constexpr int runs = rows / 16;                 // of a thread
   static constexpr int resident = RB == 1 ? (sizeof(T) == 2 ? 5 : 4) : sizeof(T) == 2 ? 3 : 2;
};

// ACROSS: the source is contiguous along the rows' dimension.  VEC: runs of eight start on 16-byte boundaries.
template <class T, bool ACROSS, bool VEC, int RB>
__global__ void __launch_bounds__(256, QuantShape<T, RB>::resident) quantize_tiles(const __grid_constant__ QuantArgs a)
{
   using H = typename Held<T>::type;
   constexpr int QR = QuantShape<T, RB>::rows, P = QuantShape<T, RB>::runs;
   constexpr int TX = ACROSS ? QR / 8 : QT / 8;           // threads side by side along the contiguous dimension
   __shared__ uint32_t most[QT];
   __shared__ alignas(16) float inverse[QT];
   __shared__ alignas(16) unsigned char turned[ACROSS ? QR * QT : 16];
   const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, lane = threadIdx.x & 31;
   const int64_t ntiles = (a.n + QT - 1) / QT, rtiles = (a.rows + QR - 1) / QR;
   // neighbouring blocks take neighbouring tiles of the contiguous dimension
   const int64_t tile_n = ACROSS ? blockIdx.x / rtiles : blockIdx.x % ntiles;
   const int64_t tile_r = ACROSS ? blockIdx.x % rtiles : blockIdx.x / ntiles;
   const int64_t i0 = tile_n * QT, r0 = tile_r * QR;
   // run p of a thread lies at `other(p)` of the dimension that is not contiguous; element j of it at `along(j)` of the
   // contiguous one.  Scalar accesses interleave the lanes.
   auto along = [&](int j) { return VEC ? tx * 8 + j : tx + TX * j; };
   auto other = [&](int p) { return ACROSS ? ty * P + p : p * 16 + ty; };
   const int64_t along_left = ACROSS ? a.rows - r0 : a.n - i0, other_left = ACROSS ? a.n - i0 : a.rows - r0;
   const int64_t along_step = ACROSS ? a.s1 : a.s0, other_step = ACROSS ? a.s0 : a.s1;
   const char *base = a.x + i0 * a.s0 + r0 * a.s1;
   H v[P][8];
#pragma unroll
   for (int p = 0; p < P; p++) {
      const char *q = base + other(p) * other_step;
      const bool in = other(p) < other_left;
      if (VEC && in && tx * 8 + 8 <= along_left) {
         const Eight<T> c = load_eight<T>(q + tx * 8 * (int)sizeof(T));
#pragma unroll
         for (int j = 0; j < 8; j++) v[p][j] = (H)c.e[j];
      } else {
#pragma unroll
         for (int j = 0; j < 8; j++) v[p][j] = in && along(j) < along_left ? (H)*reinterpret_cast<const T *>(q + along(j) * along_step) : (H)0.0f;
      }
   }
   auto value = [&](int p, int j) { return to_acc(v[p][j]); };
   auto store_scale = [&](int64_t row_block, float s) { a.scale[row_block * a.ss0 + tile_n * a.ss1] = s; };

   float inv[8];                                          // of the thread's runs, ACROSS of its elements
   if (RB == QT || ACROSS) {                              // maxima meet in shared memory
      if (threadIdx.x < QT) most[threadIdx.x] = 0;
      __syncthreads();
   }
   if (RB == QT) {
      uint32_t m = 0;
#pragma unroll
      for (int p = 0; p < P; p++)
#pragma unroll
         for (int j = 0; j < 8; j++) m = max(m, b8_magnitude(value(p, j)));
      m = __reduce_max_sync(0xFFFFFFFFu, m);
      if (lane == 0) atomicMax(&most[0], m);              // a maximum of whole numbers: any order gives the same
      __syncthreads();
      const float s = b8_scale(most[0], a.format);
      if (threadIdx.x == 0) store_scale(tile_r, s);
#pragma unroll
      for (int k = 0; k < 8; k++) inv[k] = 1.0f / s;
   } else if (ACROSS) {                                   // a row is one j of 256 / TX threads
#pragma unroll
      for (int j = 0; j < 8; j++) {
         uint32_t m = 0;
#pragma unroll
         for (int p = 0; p < P; p++) m = max(m, b8_magnitude(value(p, j)));
#pragma unroll
         for (int d = 16; d >= TX; d >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
         if (lane < TX) atomicMax(&most[along(j)], m);
      }
      __syncthreads();
      if (threadIdx.x < QR) {
         const float s = b8_scale(most[threadIdx.x], a.format);
         inverse[threadIdx.x] = 1.0f / s;
         if (threadIdx.x < along_left) store_scale(r0 + threadIdx.x, s);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j++) inv[j] = inverse[along(j)];
   } else {                                               // a row is one p of 16 lanes
#pragma unroll
      for (int p = 0; p < P; p++) {
         uint32_t m = 0;
#pragma unroll
         for (int j = 0; j < 8; j++) m = max(m, b8_magnitude(value(p, j)));
#pragma unroll
         for (int d = 8; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
         const float s = b8_scale(m, a.format);
         inv[p] = 1.0f / s;
         if (tx == 0 && other(p) < other_left) store_scale(r0 + other(p), s);
      }
   }

   if (!ACROSS) {
      const bool whole_out = VEC && (reinterpret_cast<uintptr_t>(a.codes) | (uintptr_t)a.ld) % 8 == 0;
#pragma unroll
      for (int p = 0; p < P; p++) {
         if (other(p) >= other_left) continue;
         char *q = a.codes + i0 + (r0 + other(p)) * a.ld;
         float f[8];
#pragma unroll
         for (int j = 0; j < 8; j++) f[j] = value(p, j);
         if (whole_out && tx * 8 + 8 <= along_left)
            *reinterpret_cast<uint2 *>(q + tx * 8) = make_uint2(b8_four(f, inv[p], a.format), b8_four(f + 4, inv[p], a.format));
         else {
#pragma unroll
            for (int j = 0; j < 8; j++) if (along(j) < along_left) q[along(j)] = (char)b8_pair(f[j] * inv[p], 0.0f, a.format);
         }
      }
   } else {
      // Row `along(j)` gets this thread's P codes at element ty * P.  A row's places of P bytes are permuted by the row,
      // so that the lanes of a warp write to different banks; 16 bytes stay together in steps of P.
      auto turn = [](int row) { return VEC ? row >> 3 : row % TX; };
#pragma unroll
      for (int j = 0; j < 8; j++) {
         float f[P];
#pragma unroll
         for (int p = 0; p < P; p++) f[p] = value(p, j);
         const int row = along(j);
         unsigned char *d = turned + row * QT + (P == 8 ? (ty ^ turn(row)) * 8 : (ty ^ (turn(row) * 4)) * 4);
         if constexpr (P == 8) *reinterpret_cast<uint2 *>(d) = make_uint2(b8_four(f, inv[j], a.format), b8_four(f + 4, inv[j], a.format));
         else *reinterpret_cast<uint32_t *>(d) = b8_four(f, inv[j], a.format);
      }
      __syncthreads();
      const bool whole_out = (reinterpret_cast<uintptr_t>(a.codes) | (uintptr_t)a.ld) % 16 == 0;
      const int part = threadIdx.x & 7;
#pragma unroll
      for (int q = 0; q < QR / 32; q++) {
         const int row = (threadIdx.x >> 3) + 32 * q;
         if (row >= along_left) continue;
         uint4 w;
         if constexpr (P == 8) {
            const uint2 lo = *reinterpret_cast<const uint2 *>(turned + row * QT + ((2 * part) ^ turn(row)) * 8);
            const uint2 hi = *reinterpret_cast<const uint2 *>(turned + row * QT + ((2 * part + 1) ^ turn(row)) * 8);
            w = make_uint4(lo.x, lo.y, hi.x, hi.y);
         } else w = *reinterpret_cast<const uint4 *>(turned + row * QT + (part ^ turn(row)) * 16);
         const int64_t left = other_left - part * 16;
         char *d = a.codes + i0 + part * 16 + (r0 + row) * a.ld;
         if (whole_out && left >= 16) *reinterpret_cast<uint4 *>(d) = w;
         else {
            const uint32_t word[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
            for (int k = 0; k < 16; k++) if (k < left) d[k] = (char)(word[k >> 2] >> (8 * (k & 3)));
         }
      }
   }
}

template <class T, bool ACROSS, bool VEC>
static void quantize_launch(const QuantArgs &a, int block, unsigned int grid, cudaStream_t stream)
{
   if (block == 1) quantize_tiles<T, ACROSS, VEC, 1><<<grid, 256, 0, stream>>>(a);
   else            quantize_tiles<T, ACROSS, VEC, QT><<<grid, 256, 0, stream>>>(a);
}

template <class T> static int quantize_typed(const QuantArgs &a, int block, cudaStream_t stream)
{
   const int64_t es = (int64_t)sizeof(T);
   const int64_t edge = block == 1 ? QuantShape<T, 1>::rows : QT;
   const int64_t ntiles = (a.n + QT - 1) / QT, rtiles = (a.rows + edge - 1) / edge, tiles = ntiles * rtiles;
   if (ntiles > 0x7FFFFFFF / rtiles) SD_ERROR("block_quantize: matrix too large");
   auto magnitude = [](int64_t v) { return v < 0 ? -v : v; };
   const bool across = magnitude(a.s1) < magnitude(a.s0) && a.rows > 1;
   const int64_t step = across ? a.s1 : a.s0, other = across ? a.s0 : a.s1;
   const int64_t others = across ? a.n : a.rows;
   const bool vec = step == es && (uintptr_t)a.x % 16 == 0 && (others == 1 || other % 16 == 0);
   if (across) { if (vec) quantize_launch<T, true, true>(a, block, (unsigned)tiles, stream);
                 else     quantize_launch<T, true, false>(a, block, (unsigned)tiles, stream); }
   else        { if (vec) quantize_launch<T, false, true>(a, block, (unsigned)tiles, stream);
                 else     quantize_launch<T, false, false>(a, block, (unsigned)tiles, stream); }
   SD_LAUNCH_CHECK();
   return 0;
}

} // namespace sd

extern "C" int solid_gpu_block_quantize(int dtype, size_t n, size_t rows, const solid_gpu_matrix *x, const solid_gpu_blocks *y,
                                        cudaStream_t stream)
{
   if (dtype != SD_HALF && dtype != SD_FLOAT && dtype != SD_DOUBLE) SD_ERROR("block_quantize: the type must be half, float or double");
   if (n > ((size_t)1 << 40) || rows > ((size_t)1 << 40)) SD_ERROR("block_quantize: matrix too large");
   const bool empty = n == 0 || rows == 0;
   if (x == nullptr || (x->ptr == nullptr && !empty)) SD_ERROR("block_quantize: missing matrix x");
   const ptrdiff_t es = solid_gpu_type_size[dtype];
   if ((uintptr_t)x->ptr % es != 0 || x->stride0 % es != 0 || x->stride1 % es != 0)
      SD_ERROR("block_quantize: matrix x must be aligned to its element size");
   if (sd::check_blocks(y, "block_quantize", "y", empty) != 0) return -1;
   if (empty) return 0;
   sd::QuantArgs a = { (int64_t)n, (int64_t)rows, (const char *)x->ptr, (int64_t)x->stride0, (int64_t)x->stride1,
                       (char *)y->codes, (int64_t)y->ld, y->scales, (int64_t)y->scale_stride0 / 4, (int64_t)y->scale_stride1 / 4, y->format };
   if (dtype == SD_HALF)  return sd::quantize_typed<__half>(a, y->block, stream);
   if (dtype == SD_FLOAT) return sd::quantize_typed<float>(a, y->block, stream);
   return sd::quantize_typed<double>(a, y->block, stream);
}
