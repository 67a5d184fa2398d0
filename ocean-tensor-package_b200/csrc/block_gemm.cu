// solid_gpu_block_gemm: product of two matrices of 8-bit floating-point codes with a scale for each 128 of the depth,
//
//   c[m, n] = sum over blocks kb of  sa[m, kb] sb[n, kb]  sum over k in kb of  a[k, m] b[k, n]
//
// The inner sum runs on the tensor cores into tensor memory (products of two codes are exact, sums have 32 bits); after
// each block of 128 the epilogue's warps read it, apply both scales and add it to sums in registers.  While they do,
// the tensor core works on the next block into the other half of tensor memory.
//
// The rows of a tile lie on tensor memory's lanes, a thread of the epilogue each, so that their scale is one register; its
// columns have one number a block where 128 of them share a scale, and a vector in shared memory where each has its own.
// Many tokens: tokens on the lanes, weights (128 x 128 scales) on the columns, tiles of 256 x 256 for a pair of blocks or
// of 128 x 128 for one.  Few tokens: weights on the lanes, the tokens on 16 to 128 columns, and where the tiles do not
// fill the GPU a cluster of blocks shares a tile, each with a part of the depth, and adds the parts up through
// distributed shared memory in the order of the blocks.
//
// Measured in a captured graph of a few calls (K = 8192, 8192 rows of weights, half results): 8192 tokens 487 us (2.26
// PFLOP/s, 1.38 times the rate of the 16-bit library product, 69 % of twice that rate; in a long row of calls, at the power
// limit, 583 to 598 us, 1.84 to 1.89 PFLOP/s, 56 to 58 %), 1024 tokens 71 us, 128 tokens 29 us, 64 tokens 20.5 us, 16 tokens
// 17.3 us (59 % of the copy rate); 4096 x 4096 by one token 8.3 us.  The tensor cores take 512 cycles for a block of a pair,
// 555 with the loads alone; the epilogue's chain (tensor memory's latency, scales, sums) makes it about 880.  With a scale
// for every column (weight gradients, 4096 x 2000 x 5000: 76 us) the columns' vector costs another multiplication a sum
// and a shared-memory read, 1300 cycles.  The look at the scales' range is 1 to 1.5 % of the large products.  Where it finds
// scales for which the order of multiplication matters a depth block takes longer: half of 8192 tokens zeros, float
// results, 523 us (480 without the look; half results, where it does not matter, 459 and 451); weight gradient with half of
// its depth zeros 89 us (76).
// Tried and slower: 16 epilogue warps of 64 columns (619 us), scales fetched four blocks at a time (558 us), one block a
// tile of 128 x 256 (556 us: its 48 KB a block exceed the 64 bytes a cycle that an SM takes in).
//
// Operands whose codes are not on 16-byte boundaries take a plain kernel (shared-memory tiles, 32-bit arithmetic; 13 TFLOP/s
// at 2048 x 2048 x 2048).
#include <type_traits>
#include <cuda.h>
#include "block8.cuh"
#include "tcgen05.cuh"

namespace sd {

struct Side {                                             // one operand as a kernel sees it
   const uint8_t *codes; int64_t ld;
   const float *scale; int64_t s0, s1;                    // scale of (row block, depth block), strides in floats
   int64_t rows; int shift, format;                       // shift: 0 or 7, rows that share a scale as a power of two
};
struct GemmArgs {
   Side p, q;                                             // p on the lanes, q on the columns
   int64_t K;
   char *c; int64_t cp, cq;                               // element (row of p, row of q) at c + p * cp + q * cq
   int half_out;
};

__device__ __forceinline__ float scale_at(const Side &s, int64_t row, int64_t kb)
{
   return row < s.rows ? __ldg(s.scale + (row >> s.shift) * s.s0 + kb * s.s1) : 0.0f;
}
// Scales p and q meet a sum x of 128 products of codes (zero, or 2^-32 to 2^39) as two factors, x * first * second: one and
// their product, where that is an ordinary number or one of them is zero; else the larger one and the smaller.  x times the
// larger leaves the range of 32 bits only where the result does, while a product out of range would make NaN of a sum of
// zero, or lose bits of an ordinary result.  A half keeps its bits under any product but zero: x times one below 2^-126 is
// below 2^-87, and wrong by 2^-110 at most.
constexpr uint32_t LEAST_NORMAL = 0x00800000u, LEAST = 1u;         // as bits
__device__ __forceinline__ bool out_of_range(float v, uint32_t least = LEAST_NORMAL) { return ((__float_as_uint(v) & 0x7FFFFFFFu) - least) >= 0x7F800000u - least; }
__device__ __forceinline__ bool in_turn(float p, float q) { return out_of_range(p * q) && p != 0.0f && q != 0.0f; }
__device__ __forceinline__ float first_factor(float p, float q)  { return !in_turn(p, q) ? 1.0f : fabsf(p) > fabsf(q) ? p : q; }
__device__ __forceinline__ float second_factor(float p, float q) { return !in_turn(p, q) ? p * q : fabsf(p) > fabsf(q) ? q : p; }
// A row's scale that meets the sum before the column's: what lies outside 2^-90 to 2^88 gives a part of its exponent away,
// so that x times the rest keeps its bits and stays finite; the column's scale takes that, and where it leaves the range
// so does the result.  A small one may stay whole where no column's scale is above one: what x times it loses among the
// subnormals is then at most half the smallest one in the result too.  A batch's padding (zeros, scales of 2^-126) is that case.
__device__ __forceinline__ bool far_scale(float p) { return (__float_as_uint(p) & 0x7FFFFFFFu) - (37u << 23) > (178u << 23); }      // by the exponent's bits
__device__ __forceinline__ float away(float p) { return fabsf(p) > 0x1p88f ? 0x1p40f : fabsf(p) < 0x1p-90f ? 0x1p-50f : 1.0f; }
__device__ __forceinline__ float near_part(float p) { return fabsf(p) > 0x1p88f ? p * 0x1p-40f : fabsf(p) < 0x1p-90f ? p * 0x1p50f : p; }
__device__ __forceinline__ uint32_t take_away(float q, float part)
{
   const float w = q * part;
   return __float_as_uint(fabsf(w) == INFINITY && fabsf(q) < INFINITY ? copysignf(0x1.fffffep127f, q) : w);
}
__device__ __forceinline__ void store_c(const GemmArgs &a, int64_t p, int64_t q, float v)
{
   char *d = a.c + p * a.cp + q * a.cq;
   if (a.half_out) *reinterpret_cast<__half *>(d) = __float2half_rn(v);
   else            *reinterpret_cast<float *>(d) = v;
}
__device__ __forceinline__ float decode(uint8_t code, int format)
{
   uint32_t h;
   if (format == B8_E4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
   else                   asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
   return __half2float(__ushort_as_half((uint16_t)h));
}

// ---------------------------------------------------------------------------
// any alignment: 64 x 64 tiles, four by four sums a thread
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) gemm_plain(const __grid_constant__ GemmArgs a)
{
   __shared__ float sp[32][65], sq[32][65];
   const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
   const int64_t ptiles = (a.p.rows + 63) / 64;
   const int64_t p0 = blockIdx.x % ptiles * 64, q0 = blockIdx.x / ptiles * 64;
   float acc[4][4] = {};
   for (int64_t kb = 0; kb * B8_BLOCK < a.K; kb++) {
      float sum[4][4] = {};
      for (int k0 = 0; k0 < B8_BLOCK; k0 += 32) {
         __syncthreads();
#pragma unroll
         for (int e = 0; e < 8; e++) {
            const int r = (threadIdx.x >> 5) + 8 * e, k = threadIdx.x & 31;
            const int64_t kk = kb * B8_BLOCK + k0 + k;
            sp[k][r] = p0 + r < a.p.rows && kk < a.K ? decode(a.p.codes[(p0 + r) * a.p.ld + kk], a.p.format) : 0.0f;
            sq[k][r] = q0 + r < a.q.rows && kk < a.K ? decode(a.q.codes[(q0 + r) * a.q.ld + kk], a.q.format) : 0.0f;
         }
         __syncthreads();
#pragma unroll 4
         for (int k = 0; k < 32; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
               for (int j = 0; j < 4; j++) sum[i][j] = fmaf(sp[k][tx + 16 * i], sq[k][ty + 16 * j], sum[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
         const float s = scale_at(a.p, p0 + tx + 16 * i, kb);
#pragma unroll
         for (int j = 0; j < 4; j++) {
            const float t = scale_at(a.q, q0 + ty + 16 * j, kb);
            acc[i][j] = fmaf(sum[i][j] * first_factor(s, t), second_factor(s, t), acc[i][j]);
         }
      }
   }
#pragma unroll
   for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++)
         if (p0 + tx + 16 * i < a.p.rows && q0 + ty + 16 * j < a.q.rows) store_c(a, p0 + tx + 16 * i, q0 + ty + 16 * j, acc[i][j]);
}

// ---------------------------------------------------------------------------
// tensor cores
// ---------------------------------------------------------------------------
constexpr int BM = 128;
constexpr int TILE_P = BM * B8_BLOCK;                     // bytes of a stage's 128 rows

constexpr int MAX_SPLITS = 8;                             // blocks of a cluster that share a tile: its portable size
constexpr int AHEAD = 8;                                  // places for depth blocks' scales

// PAIR: two blocks share a tile of 256 rows, each holds half of either operand's rows; the columns' half travels once
// instead of twice, and the 64 bytes a cycle that a block can take in no longer bound the products.
template <int BN, bool PAIR> struct Shape {
   static constexpr int groups = BN > 128 ? 2 : 1;        // epilogue warpgroups, 128 columns at most each
   static constexpr int columns = BN / groups;
   static constexpr int run = columns >= 64 ? 32 : columns / 2;     // columns of one read of tensor memory
   // and a warp that loads, a warp that multiplies; with two groups a third whole one, so that registers can be moved:
   // 384 x 168 = 128 x 40 + 256 x 232
   static constexpr int threads = groups == 2 ? 384 : groups * 128 + 64;
   static constexpr int rows_q = PAIR ? BN / 2 : BN;      // of q in this block's shared memory
   static constexpr int stage = TILE_P + rows_q * B8_BLOCK;
   static constexpr int resident = BN >= 128 ? 1 : 2;     // blocks an SM: one whose ring fills shared memory, or two
   static constexpr int stages = PAIR || BN != 64 ? 5 : 4;
   static constexpr int tmem = 2 * BN < 32 ? 32 : 2 * BN;
   static constexpr int scales = 2 * AHEAD * groups * 128 * 4;      // a row's and a column's for each epilogue thread
   static constexpr int out = BN >= 128 ? groups * 4 * 4096 : 0;    // 32 rows of 128 bytes for each epilogue warp
   static constexpr int smem = 1024 + stages * stage + scales + out;
};

// A warp's 32 rows of results, a thread each, to memory where a row's results lie side by side: 128 bytes of every row
// at a time through shared memory, so that a store writes whole lines.  Places of 16 bytes are permuted by the row.
template <int CW, bool HALF>
__device__ __forceinline__ void store_rows(const GemmArgs &a, const float (&acc)[CW], char *buf, int64_t p0, int64_t q0, int lane)
{
   constexpr int PER = HALF ? 64 : 32, UNIT = PER / 8;    // results in 128 bytes, in 16
#pragma unroll
   for (int c = 0; c < CW; c += PER) {
      if (PER > CW) break;
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 8; u++) {
         uint4 w;
         if (HALF) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
               const __half2 h = __floats2half2_rn(acc[c + 8 * u + 2 * k], acc[c + 8 * u + 2 * k + 1]);
               x[k] = *reinterpret_cast<const uint32_t *>(&h);
            }
            w = make_uint4(x[0], x[1], x[2], x[3]);
         } else w = make_uint4(__float_as_uint(acc[c + 4 * u]), __float_as_uint(acc[c + 4 * u + 1]), __float_as_uint(acc[c + 4 * u + 2]), __float_as_uint(acc[c + 4 * u + 3]));
         *reinterpret_cast<uint4 *>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = w;
      }
      __syncwarp();
#pragma unroll
      for (int r = 0; r < 8; r++) {
         const int row = 4 * r + (lane >> 3), u = lane & 7;
         const uint4 w = *reinterpret_cast<const uint4 *>(buf + row * 128 + ((u ^ (row & 7)) << 4));
         const int64_t p = p0 + row, q = q0 + c + u * UNIT;
         char *d = a.c + p * a.cp + q * (HALF ? 2 : 4);
         if (p < a.p.rows) {
            if (q + UNIT <= a.q.rows) *reinterpret_cast<uint4 *>(d) = w;
            else {
               const uint32_t x[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
               for (int k = 0; k < UNIT; k++) {
                  if (q + k >= a.q.rows) continue;
                  if (HALF) reinterpret_cast<uint16_t *>(d)[k] = (uint16_t)(x[k >> 1] >> (16 * (k & 1)));
                  else      reinterpret_cast<uint32_t *>(d)[k] = x[k];
               }
            }
         }
      }
   }
}

// COLVEC: a scale for every row of q (a vector over the columns); otherwise for 128 rows (one number).
// SPLIT: a cluster shares the tile, block r takes the r-th part of the depth.
template <int BN, bool PAIR, bool COLVEC, bool SPLIT>
__global__ void __launch_bounds__(Shape<BN, PAIR>::threads, Shape<BN, PAIR>::resident)
gemm_tiles(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ GemmArgs a,
           int splits, int kblocks, int ptiles, int qtiles)
{
   using S = Shape<BN, PAIR>;
   constexpr int ST = S::stages, CW = S::columns;
   extern __shared__ char raw[];
   __shared__ alignas(8) uint64_t bars[2 * ST + 4];
   __shared__ uint32_t tmem_base;
   __shared__ int failed;
   char *ring = raw + ((1024 - (tc::smem_u32(raw) & 1023)) & 1023);
   float *scales = (float *)(ring + ST * S::stage);       // [AHEAD][groups * 128] of rows, the same of columns
   char *out = ring + ST * S::stage + S::scales;
   const uint32_t ring_u = tc::smem_u32(ring);
   const uint32_t full = tc::smem_u32(bars), empty = full + 8 * ST, tfull = full + 16 * ST, tempty = tfull + 16;
   const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
   constexpr int EPI = S::groups * 4;                     // epilogue warps come first: warp w reads lanes 32 (w % 4)
   const int rank = PAIR || SPLIT ? (int)tc::cluster_rank() : 0;
   const bool leader = !PAIR || rank == 0;

   if (threadIdx.x == 0) {
      for (int s = 0; s < ST; s++) { tc::bar_init(full + 8 * s, 1); tc::bar_init(empty + 8 * s, 1); }
      for (int b = 0; b < 2; b++) { tc::bar_init(tfull + 8 * b, 1); tc::bar_init(tempty + 8 * b, PAIR ? 2 * EPI : EPI); }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      failed = 0;
   }
   if (warp == EPI) tc::alloc<PAIR>(tc::smem_u32(&tmem_base), S::tmem);
   tc::fence_before();
   __syncthreads();
   if (PAIR) tc::cluster_sync();
   tc::fence_after();
   const uint32_t tmem = *(volatile uint32_t *)&tmem_base;

   // ptiles counts tiles of 128 rows, or of 256 for pairs
   const int ntiles = ptiles * qtiles;
   const int first = SPLIT ? (int)blockIdx.x / splits : PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x;
   const int step = SPLIT ? ntiles : PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
   const int kb0 = SPLIT ? (int)((long long)kblocks * rank / splits) : 0;
   const int kb1 = SPLIT ? (int)((long long)kblocks * (rank + 1) / splits) : kblocks;
   constexpr int ROWS = PAIR ? 2 * BM : BM;
   const int prow = PAIR ? rank * BM : 0, qrow = PAIR ? rank * S::rows_q : 0;
   // Tiles in panels of `ROWS` times 16 or 8 rows, so that blocks at work share both operands in the L2 cache
   auto place = [&](int tile, int &tp, int &tq) {
      constexpr int PANEL = PAIR ? 8 : 16;
      const int panel = tile / (PANEL * qtiles), rest = tile - panel * PANEL * qtiles;
      const int height = min(PANEL, ptiles - panel * PANEL);
      tp = panel * PANEL + rest % height; tq = rest / height;
   };

   if (warp >= EPI) {
      if (S::groups == 2) tc::registers_down<40>();
      // s and turn: place in the ring, and how often it came round; b and round the same for tensor memory
      if (warp == EPI) {                                  // ---- loads
         const uint32_t full_at = PAIR ? tc::at_rank(full, 0) : full;
         int it = 0, s = 0; uint32_t turn = 0; bool ok = true;
         for (int tile = first; tile < ntiles && ok; tile += step) {
            int tp, tq; place(tile, tp, tq);
            for (int kb = kb0; kb < kb1; kb++, it++) {
               if (it >= ST && !tc::bar_wait_warp(empty + 8 * s, turn ^ 1)) { ok = false; break; }
               if (tc::elect()) {
                  const uint32_t dst = ring_u + s * S::stage;
                  if (leader) tc::bar_expect(full + 8 * s, PAIR ? 2 * S::stage : S::stage);
                  tc::load_box<PAIR>(dst, &map_p, full_at + 8 * s, kb * B8_BLOCK, tp * ROWS + prow);
                  tc::load_box<PAIR>(dst + TILE_P, &map_q, full_at + 8 * s, kb * B8_BLOCK, tq * BN + qrow);
               }
               if (++s == ST) { s = 0; turn ^= 1; }
            }
         }
         if (!ok) {                                       // the copies under way end before shared memory is given back
            *(volatile int *)&failed = 1;
            if (leader) for (int k = max(0, it - ST); k < it; k++) tc::bar_wait(full + 8 * (k % ST), (k / ST) & 1);
         }
      } else if (warp == EPI + 1 && leader) {             // ---- products
         const uint32_t idesc = (1u << 4) | ((uint32_t)a.p.format << 7) | ((uint32_t)a.q.format << 10) | ((uint32_t)(BN / 8) << 17) | ((uint32_t)(ROWS / 16) << 24);
         const uint64_t desc_p = tc::tile_descriptor(ring_u), desc_q = tc::tile_descriptor(ring_u + TILE_P);
         int it = 0, s = 0; uint32_t turn = 0, b = 0, round = 0; bool ok = true;
         for (int tile = first; tile < ntiles && ok; tile += step)
            for (int kb = kb0; kb < kb1; kb++, it++) {
               if (it >= 2 && !tc::bar_wait_warp(tempty + 8 * b, round ^ 1)) { ok = false; break; }
               if (!tc::bar_wait_warp(full + 8 * s, turn)) { ok = false; break; }
               tc::fence_after();
               if (tc::elect()) {
                  const uint64_t dp = desc_p + (uint32_t)(s * S::stage / 16), dq = desc_q + (uint32_t)(s * S::stage / 16);
#pragma unroll
                  for (int k = 0; k < 4; k++) tc::mma_f8<PAIR>(tmem + b * BN, dp + 2 * k, dq + 2 * k, idesc, k > 0);
                  tc::commit<PAIR>(empty + 8 * s);
                  tc::commit<PAIR>(tfull + 8 * b);
               }
               if (++s == ST) { s = 0; turn ^= 1; }
               b ^= 1; if (b == 0) round ^= 1;
            }
         if (!ok) {
            *(volatile int *)&failed = 1;
            if (it > 0) tc::bar_wait(tfull + 8 * ((it - 1) & 1), ((it - 1) / 2) & 1);
         }
      }
   } else {                                               // ---- scales and sums
      if (S::groups == 2) tc::registers_up<232>();
      const int group = warp >> 2, row = (warp & 3) * 32 + lane, col0 = group * CW;
      const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + col0;
      const uint32_t tempty_at = PAIR ? tc::at_rank(tempty, 0) : tempty;
      const uint32_t my_slot = tc::smem_u32(scales + threadIdx.x);
      constexpr int SLOT = S::groups * 128;               // floats of a depth block's rows or columns
      int it = 0; bool ok = true;
      for (int tile = first; tile < ntiles; tile += step) {
         int tp, tq; place(tile, tp, tq);
         const int64_t p = (int64_t)tp * ROWS + prow + row, q0 = (int64_t)tq * BN + col0;
         // Scales come AHEAD blocks early, straight to shared memory: the row's own, and one column's (of all columns
         // where each has its own: the threads of the group fetch them for each other)
         const int64_t my_col = COLVEC ? q0 + row : q0;
         const bool in_p = p < a.p.rows, in_q = my_col < a.q.rows && (!COLVEC || row < CW);
         const float *next_p = a.p.scale + (in_p ? (p >> a.p.shift) * a.p.s0 + kb0 * a.p.s1 : 0);
         const float *next_q = a.q.scale + (in_q ? (my_col >> a.q.shift) * a.q.s0 + kb0 * a.q.s1 : 0);
         int fetched = kb0;
         auto fetch = [&] {
            if (fetched < kb1) {
               const uint32_t slot = my_slot + (fetched % AHEAD) * SLOT * 4;
               tc::copy4(slot, next_p, in_p);
               tc::copy4(slot + AHEAD * SLOT * 4, next_q, in_q);
               if (in_p) next_p += a.p.s1;
               if (in_q) next_q += a.q.s1;
               fetched++;
            }
            tc::copies_commit();
         };
#pragma unroll
         for (int d = 0; d < AHEAD - 1; d++) fetch();
         uint64_t sum[CW / 2];                            // pairs of neighbouring columns
         auto row_scale = [&](int kb) { return scales[kb % AHEAD * SLOT + threadIdx.x]; };
         auto col_scale = [&](int kb) { return scales[(AHEAD + kb % AHEAD) * SLOT + threadIdx.x]; };
         auto group_sync = [&] {
            if (group == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
            else            asm volatile("bar.sync 2, 128;" ::: "memory");
         };
         auto wait_sums = [&](int i) {
            if (ok) ok = tc::bar_wait(tfull + 8 * (i & 1), (i / 2) & 1);
            __syncwarp();
            tc::fence_after();
         };
#pragma unroll
         for (int j = 0; j < CW / 2; j++) sum[j] = 0;
         // The scales of a depth block: s for the whole warp's sums, unless it is `apart`, which is when a lane has scales for
         // which the order of the multiplications matters.  Only rows and columns of the matrices count; others have zeros.
         float s;
         bool apart;
         const bool inside = in_p && (COLVEC || in_q);
         auto take_scales = [&](int kb) {
            const float sp = row_scale(kb);
            s = COLVEC ? sp : sp * col_scale(kb);
            apart = __any_sync(0xFFFFFFFFu, inside && (COLVEC ? far_scale(sp) : out_of_range(s)));
         };
         auto next_scales = [&](int kb) {
            tc::copies_wait<AHEAD - 3>();                 // the next block's scales, of every thread of the group
            if (COLVEC) group_sync();                     // which is also past the place that is filled again
            fetch();
            take_scales(kb + 1 < kb1 ? kb + 1 : kb);
         };
         auto all_read = [&](int b) {                     // the next products may overwrite it
            tc::fence_before();
            __syncwarp();
            if (lane == 0) { if (PAIR) tc::bar_arrive_at(tempty_at + 8 * b); else tc::bar_arrive(tempty + 8 * b); }
         };
         tc::copies_wait<AHEAD - 2>();
         if (COLVEC) group_sync();
         take_scales(kb0);
         for (int kb = kb0; kb < kb1; ) {
            if (BN >= 128 && apart) {                     // small scales, a padded batch's: they may be no matter
               if (COLVEC) {
                  const float *cs = scales + (AHEAD + kb % AHEAD) * SLOT + group * 128;
                  bool large = false;
                  for (int c = lane; c < CW; c += 32) large |= fabsf(cs[c]) > 1.0f;
                  large = __any_sync(0xFFFFFFFFu, large);
                  apart = __any_sync(0xFFFFFFFFu, inside && far_scale(s) && (large || fabsf(s) > 1.0f));
               } else if (a.half_out) apart = __any_sync(0xFFFFFFFFu, inside && out_of_range(s, LEAST));
            }
            if (apart) {                                  // one block by itself, with two factors for each sum
               const float sp = row_scale(kb), sq = col_scale(kb);
               const float *cs = scales + (AHEAD + kb % AHEAD) * SLOT + group * 128;
               const float one = COLVEC ? near_part(sp) : first_factor(sp, sq), two = COLVEC ? away(sp) : second_factor(sp, sq);
               wait_sums(it);
               next_scales(kb);
#pragma unroll
               for (int c = 0; c < CW; c += 8) {
                  uint32_t x[8];
                  tc::ld(from + (it & 1) * BN + c, x);
                  tc::ld_wait(x);
                  if (c + 8 == CW) all_read(it & 1);
#pragma unroll
                  for (int j = 0; j < 8; j += 2) {
                     const uint64_t f = COLVEC ? tc::pair(take_away(cs[c + j], two), take_away(cs[c + j + 1], two)) : tc::pair(__float_as_uint(two), __float_as_uint(two));
                     const uint64_t y = tc::mul2(tc::pair(x[j], x[j + 1]), tc::pair(__float_as_uint(one), __float_as_uint(one)));
                     sum[(c + j) / 2] = tc::fma2(y, f, sum[(c + j) / 2]);
                  }
               }
               kb++; it++;
               continue;
            }
            // Everything that the next block needs is under way before the present block's sums are done: its scales are
            // read, its first columns are on their way from tensor memory.
            constexpr int RUN = S::run, RUNS = CW / RUN;  // an even number: a block's first run is in v[0]
            uint32_t v[2][RUN];
            bool more;
            wait_sums(it);
            tc::ld(from + (it & 1) * BN, v[0]);
            do {
               const int b = it & 1;
               const float *cs = scales + (AHEAD + kb % AHEAD) * SLOT + group * 128;
               const uint64_t s2 = tc::pair(__float_as_uint(s), __float_as_uint(s));
#pragma unroll
               for (int c = 0; c < RUNS; c++) {
                  tc::ld_wait(v[c & 1]);
                  if (c + 1 < RUNS) tc::ld(from + b * BN + RUN * (c + 1), v[(c + 1) & 1]);
                  else {
                     all_read(b);
                     more = kb + 1 < kb1 && !apart;
                     if (more) { wait_sums(it + 1); tc::ld(from + (b ^ 1) * BN, v[0]); }
                  }
                  if (c == 0) next_scales(kb);
#pragma unroll
                  for (int j = 0; j < RUN; j += 4) {
                     uint64_t x = tc::pair(v[c & 1][j], v[c & 1][j + 1]), y = tc::pair(v[c & 1][j + 2], v[c & 1][j + 3]);
                     const int k = (RUN * c + j) / 2;
                     if (COLVEC) {
                        const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(cs + RUN * c + j);
                        x = tc::mul2(x, s2); y = tc::mul2(y, s2);
                        sum[k] = tc::fma2(x, w.x, sum[k]);
                        sum[k + 1] = tc::fma2(y, w.y, sum[k + 1]);
                     } else {
                        sum[k] = tc::fma2(x, s2, sum[k]);
                        sum[k + 1] = tc::fma2(y, s2, sum[k + 1]);
                     }
                  }
               }
               kb++; it++;
            } while (more);
         }
         float acc[CW];
#pragma unroll
         for (int j = 0; j < CW / 2; j++) { acc[2 * j] = tc::lo_of(sum[j]); acc[2 * j + 1] = tc::hi_of(sum[j]); }
         if (!ok) {                                       // a wait ran out: no result is better than a wrong one
            failed = 1;
#pragma unroll
            for (int j = 0; j < CW; j++) acc[j] = __int_as_float(0x7FFFFFFF);
         }
         tc::copies_wait<0>();
         if (COLVEC) group_sync();                        // every thread is past the scales before the next tile's
         if (SPLIT) {
            // this block's part to shared memory, over the ring: all its copies have been consumed
            float *part = (float *)ring;
#pragma unroll
            for (int j = 0; j < CW; j++) part[(col0 + j) * BM + row] = acc[j];
            continue;
         }
         const int es = a.half_out ? 2 : 4;
         const int64_t p0 = p - lane;
         if (BN >= 128 && a.cq == es && (reinterpret_cast<uintptr_t>(a.c) | (uintptr_t)a.cp) % 16 == 0) {
            if (a.half_out) store_rows<CW, true>(a, acc, out + warp * 4096, p0, q0, lane);
            else            store_rows<CW, false>(a, acc, out + warp * 4096, p0, q0, lane);
         } else if (p < a.p.rows) {                       // lanes side by side, or any strides
#pragma unroll
            for (int j = 0; j < CW; j++) if (q0 + j < a.q.rows) store_c(a, p, q0 + j, acc[j]);
         }
      }
   }
   __syncwarp();
   __syncthreads();
   if (SPLIT) {                                           // the blocks' parts, added in the order of the blocks
      if (failed) for (int e = threadIdx.x; e < BN * BM; e += S::threads) ((float *)ring)[e] = __int_as_float(0x7FFFFFFF);
      tc::cluster_sync();
      int tp, tq; place(first, tp, tq);
      const uint32_t part = tc::smem_u32(ring);
      const int cols = min(BN, (int)(a.q.rows - (int64_t)tq * BN));
      // four rows of a column at a time, all blocks' parts under way before the first is added
      for (int e = rank * S::threads + threadIdx.x; e < cols * (BM / 4); e += splits * S::threads) {
         float4 x[MAX_SPLITS];
#pragma unroll
         for (int r = 0; r < MAX_SPLITS; r++) if (r < splits) x[r] = tc::peer_load(part + 16 * e, r);
         float v[4] = { x[0].x, x[0].y, x[0].z, x[0].w };
#pragma unroll
         for (int r = 1; r < MAX_SPLITS; r++) if (r < splits) { v[0] += x[r].x; v[1] += x[r].y; v[2] += x[r].z; v[3] += x[r].w; }
         const int64_t p = (int64_t)tp * BM + (e & (BM / 4 - 1)) * 4, q = (int64_t)tq * BN + e / (BM / 4);
#pragma unroll
         for (int k = 0; k < 4; k++) if (p + k < a.p.rows) store_c(a, p + k, q, v[k]);
      }
   }
   if (PAIR || SPLIT) tc::cluster_sync();                 // no block leaves while another reads it or signals to it
   if (warp == EPI) tc::dealloc<PAIR>(tmem, S::tmem);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder()
{
   static EncodeTiled f = [] {
      void *p = nullptr; cudaDriverEntryPointQueryResult found;
      if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
          found != cudaDriverEntryPointSuccess) { cudaGetLastError(); p = nullptr; }
      return (EncodeTiled)p;
   }();
   return f;
}

static int map_of(CUtensorMap *map, const Side &s, int64_t K, int box_rows)
{
   EncodeTiled f = encoder();
   if (f == nullptr) SD_ERROR("block_gemm: the driver has no tensor maps");
   const cuuint64_t dims[2] = { (cuuint64_t)K, (cuuint64_t)s.rows };
   const cuuint64_t strides[1] = { (cuuint64_t)(s.rows == 1 ? (K + 15) / 16 * 16 : s.ld) };
   const cuuint32_t box[2] = { B8_BLOCK, (cuuint32_t)box_rows }, ones[2] = { 1, 1 };
   if (f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)s.codes, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      SD_ERROR("block_gemm: the driver refused a tensor map");
   return 0;
}

template <int BN, bool PAIR, bool COLVEC, bool SPLIT>
static int launch_tiles(const GemmArgs &a, int splits, int sms, cudaStream_t stream)
{
   using S = Shape<BN, PAIR>;
   CUtensorMap map_p, map_q;
   if (map_of(&map_p, a.p, a.K, BM) != 0 || map_of(&map_q, a.q, a.K, S::rows_q) != 0) return -1;
   auto *kernel = gemm_tiles<BN, PAIR, COLVEC, SPLIT>;
   SD_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem));
   if (S::groups == 2) {                                  // moved registers have to be there: a block that waits for more waits for good
      static const int registers = [&] { cudaFuncAttributes at; return cudaFuncGetAttributes(&at, kernel) == cudaSuccess ? at.numRegs : 0; }();
      if (registers * 384 < 128 * 40 + 256 * 232) SD_ERROR("block_gemm: built with %d registers a thread, 168 are needed", registers);
   }
   constexpr int ROWS = PAIR ? 2 * BM : BM;
   const int64_t ptiles = (a.p.rows + ROWS - 1) / ROWS, qtiles = (a.q.rows + BN - 1) / BN;
   const int kblocks = (int)((a.K + B8_BLOCK - 1) / B8_BLOCK);
   const int cluster = SPLIT ? splits : PAIR ? 2 : 1;
   cudaLaunchConfig_t cfg = {};
   const int64_t room = (int64_t)sms * S::resident;
   cfg.gridDim = dim3((unsigned)(SPLIT ? ptiles * qtiles * splits : std::min(ptiles * qtiles * cluster, room / cluster * cluster)));
   cfg.blockDim = dim3(S::threads);
   cfg.dynamicSmemBytes = S::smem;
   cfg.stream = stream;
   cudaLaunchAttribute attr[1];
   attr[0].id = cudaLaunchAttributeClusterDimension;
   attr[0].val.clusterDim.x = (unsigned)cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
   if (cluster > 1) { cfg.attrs = attr; cfg.numAttrs = 1; }
   SD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_p, map_q, a, splits, kblocks, (int)ptiles, (int)qtiles));
   return 0;
}

template <int BN> static int launch_width(const GemmArgs &a, int splits, int sms, cudaStream_t stream)
{
   const bool vec = a.q.shift == 0;
   if (splits > 1) return vec ? launch_tiles<BN, false, true, true>(a, splits, sms, stream) : launch_tiles<BN, false, false, true>(a, splits, sms, stream);
   return vec ? launch_tiles<BN, false, true, false>(a, 1, sms, stream) : launch_tiles<BN, false, false, false>(a, 1, sms, stream);
}

static bool on_boundaries(const Side &s, int64_t K)
{
   return (uintptr_t)s.codes % 16 == 0 && (s.rows == 1 || (s.ld % 16 == 0 && s.ld >= K && s.ld < ((int64_t)1 << 39))) &&
          s.rows < 0x7FFFFFFF - 256;
}

static int gemm(GemmArgs &a, cudaStream_t stream)
{
   DeviceInfo dev;
   if (current_device_info(&dev) != 0) return -1;
   if (a.K == 0 || a.K > 0x7FFFFF00 || !on_boundaries(a.p, a.K) || !on_boundaries(a.q, a.K)) {
      const int64_t pt = (a.p.rows + 63) / 64, qt = (a.q.rows + 63) / 64, tiles = pt * qt;
      if (pt > 0x7FFFFFFF / qt) SD_ERROR("block_gemm: matrix too large");
      gemm_plain<<<(unsigned)tiles, 256, 0, stream>>>(a);
      SD_LAUNCH_CHECK();
      return 0;
   }
   // Few tokens: the wider matrix on the lanes, the narrow one on just enough columns.  Many: the matrix with scales for
   // 128 rows on the columns, where they cost nothing.
   const int64_t narrow = std::min(a.p.rows, a.q.rows);
   const bool swap = narrow <= 128 ? a.q.rows > a.p.rows : (a.q.shift == 0 && a.p.shift == 7);
   if (swap) { std::swap(a.p, a.q); std::swap(a.cp, a.cq); }
   const int64_t ptiles = (a.p.rows + BM - 1) / BM;
   int bn = 256;
   if (a.q.rows <= 16) bn = 16; else if (a.q.rows <= 32) bn = 32; else if (a.q.rows <= 64) bn = 64; else if (a.q.rows <= 128) bn = 128;
   else {
      // A tile of 256 x 256 takes a pair of SMs about 1.5 times as long as a tile of 128 x 128 takes one (0.55 and 0.37 us
      // a depth block); the fewer rounds decide (8192 rows by 512 tokens: 38 and 49 us, by 256: 35 and 27 us).
      const int64_t pairs = std::max(1, dev.sms / 2), big = (a.p.rows + 255) / 256 * ((a.q.rows + 255) / 256);
      const int64_t small = ptiles * ((a.q.rows + 127) / 128);
      if (2 * ((small + dev.sms - 1) / dev.sms) < 3 * ((big + pairs - 1) / pairs)) bn = 128;
   }
   const int64_t qtiles = (a.q.rows + bn - 1) / bn, tiles = ptiles * qtiles, kblocks = (a.K + B8_BLOCK - 1) / B8_BLOCK;
   if (ptiles > 0x3FFFFFF / qtiles) SD_ERROR("block_gemm: matrix too large");
   // A tile is shared by up to eight blocks (the portable size of a cluster) while there is room on the GPU and two
   // depth blocks are left for each.
   int splits = 1;
   const int64_t room = (int64_t)dev.sms * (bn < 128 ? 2 : 1);
   while (splits < MAX_SPLITS && tiles * splits * 2 <= room && kblocks >= 4 * splits) splits *= 2;
   switch (bn) {
      case 16:  return launch_width<16>(a, splits, dev.sms, stream);
      case 32:  return launch_width<32>(a, splits, dev.sms, stream);
      case 64:  return launch_width<64>(a, splits, dev.sms, stream);
      case 128: return launch_width<128>(a, splits, dev.sms, stream);
      default:  return a.q.shift == 0 ? launch_tiles<256, true, true, false>(a, 1, dev.sms, stream)
                                      : launch_tiles<256, true, false, false>(a, 1, dev.sms, stream);
   }
}

static Side side_of(const solid_gpu_blocks *b, size_t rows)
{
   return { (const uint8_t *)b->codes, (int64_t)b->ld, b->scales, (int64_t)b->scale_stride0 / 4, (int64_t)b->scale_stride1 / 4,
            (int64_t)rows, b->block == 1 ? 0 : 7, b->format };
}

} // namespace sd

extern "C" int solid_gpu_block_gemm(int ctype, size_t M, size_t N, size_t K, const solid_gpu_blocks *a, const solid_gpu_blocks *b,
                                    const solid_gpu_matrix *c, cudaStream_t stream)
{
   const char *op = "block_gemm";
   if (ctype != SD_HALF && ctype != SD_FLOAT) SD_ERROR("%s: the result's type must be half or float", op);
   if (M > ((size_t)1 << 40) || N > ((size_t)1 << 40) || K > ((size_t)1 << 40)) SD_ERROR("%s: matrix too large", op);
   if (sd::check_blocks(a, op, "a", M == 0 || K == 0) != 0 || sd::check_blocks(b, op, "b", N == 0 || K == 0) != 0) return -1;
   if (c == nullptr || (c->ptr == nullptr && M != 0 && N != 0)) SD_ERROR("%s: missing matrix c", op);
   const ptrdiff_t es = solid_gpu_type_size[ctype];
   if ((uintptr_t)c->ptr % es != 0 || c->stride0 % es != 0 || c->stride1 % es != 0) SD_ERROR("%s: matrix c must be aligned to its element size", op);
   if (M == 0 || N == 0) return 0;
   sd::GemmArgs g = { sd::side_of(a, M), sd::side_of(b, N), (int64_t)K, (char *)c->ptr, (int64_t)c->stride0, (int64_t)c->stride1, ctype == SD_HALF };
   return sd::gemm(g, stream);
}
