// Root-mean-square norm over dimension 0 of an [n, rows] matrix, with the residual's addition in front of it, an output
// in 8 bits with scales, and its gradient:
//
//   solid_gpu_rms_norm            h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   solid_gpu_rms_norm_quantize   the same with y as 8-bit codes, one scale for 128 elements of a row
//   solid_gpu_rms_norm_grad       g = dy w,  dh = r g - h r^3 mean(g h) (+ dres),  dw = sum over rows of dy h r
//
// All of it is bound by memory: a row is read once and written once.  Sums are kept in 32 bits (double: 64) and y is
// formed from the unrounded h; h, y and dh are rounded once, to nearest even.  A row belongs to a warp or half a warp up
// to 512 elements (gradient: 256), to a block up to 16384, beyond that to a block that reads it twice.  Rows on 16-byte
// boundaries come through a ring in shared memory (norm_ring, grad_ring); others, and those too long for two places of a
// ring, are fetched by the threads themselves (norm_rows, grad_rows).  A row at a time in registers with the next one
// fetched ahead was the first form: its loads shared the registers with the sums, 62 % of the copy rate.
//
// Measured in a captured graph with inputs that rotate over more than the L2 cache, the copy's rate (6.57 TB/s) as 100 %,
// halves with residual: norm of 8192 rows of 4096 48.6 us (84 %), with 8-bit output of 4096 rows of 8192 50.4 us (71 %: the
// conversions want more warps than the loads), gradient of 4096 rows of 4096 33.2 us (61 %, 4.5 us of it the join of the
// weights' gradient, whose partial rows have to be written and read), one row of 4096 2.4 us (a launch).
// What the threads fetch themselves, 2^24 elements with residual: rows off 16-byte boundaries (4095 halves) norm 53.8 us
// (38 %), 8-bit output 68.7 (26 %), gradient 71.4 (29 %); floats off them 75, 50 and 61 %.  The gradient of 16384 floats, for
// which the ring has no room, holds 32 values of five arrays a thread and spills: 108 us (38 %); doubles of 8192 likewise,
// 199 us (41 %).  Rows above 16384, read twice: norm of 32768 halves 75 us (27 %), floats 83 (49 %), gradient 127 (16 %) and 90.
#include <atomic>
#include "block8.cuh"
#include "tcgen05.cuh"

namespace sd {

struct RowMatrix { char *p; int64_t s0, s1; };            // element (i, row) at p + i * s0 + row * s1; p null: absent

struct NormArgs {
   int64_t n, rows;
   int group;                                             // threads of a row where a row is a warp's part (16 or 32)
   RowMatrix x, res, h, y;                                // y: output in the type of x, or the codes
   const void *w;
   double eps;
   float *scale; int64_t ss0, ss1;                        // scale of (row, block) at row * ss0 + block * ss1 (floats)
   int format;
};

struct GradArgs {
   int64_t n, rows;
   int group;
   RowMatrix dy, h, res, dh;
   const void *w;
   double eps;
   void *part;                                            // one row of n partial sums for each block, null: no dw
};

// Where a thread's eight elements of a chunk lie.  VEC: side by side, one 16-byte access for halves.  Otherwise the
// warp takes 256 elements, lane after lane, so that scalar accesses of neighbouring lanes meet in one line.
template <bool VEC> __device__ __forceinline__ int64_t chunk_first(int v, int threads, int t)
{
   if (VEC) return ((int64_t)v * threads + t) * 8;
   return (int64_t)v * threads * 8 + (int64_t)(t >> 5) * 256 + (t & 31);
}
template <bool VEC> constexpr int chunk_step = VEC ? 1 : 32;

template <class T, bool VEC>
__device__ __forceinline__ void fetch(Eight<T> &c, const RowMatrix &m, int64_t row, int64_t i, int64_t n)
{
   const char *p = m.p + row * m.s1;
   if (VEC) {
      if (i < n) c = load_eight<T>(p + i * (int64_t)sizeof(T));
      else memset(&c, 0, sizeof(c));
   } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
         const int64_t k = i + 32 * j;
         if (k < n) c.e[j] = *reinterpret_cast<const T *>(p + k * m.s0); else from_acc(c.e[j], 0);
      }
   }
}

template <class T, bool VEC>
__device__ __forceinline__ void put(const RowMatrix &m, int64_t row, int64_t i, int64_t n, const typename Real<T>::acc *v)
{
   char *p = m.p + row * m.s1;
   if (VEC) {
      Eight<T> c;
#pragma unroll
      for (int j = 0; j < 8; j++) from_acc(c.e[j], v[j]);
      if (i < n) store_eight(p + i * (int64_t)sizeof(T), c);
   } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
         const int64_t k = i + 32 * j;
         if (k < n) from_acc(*reinterpret_cast<T *>(p + k * m.s0), v[j]);
      }
   }
}

// Weights of a chunk; absent weights are ones
template <class T, bool VEC>
__device__ __forceinline__ void fetch_weights(Eight<T> &c, const void *w, int64_t i, int64_t n)
{
   if (w != nullptr) { RowMatrix m = { (char *)w, (int64_t)sizeof(T), 0 }; fetch<T, VEC>(c, m, 0, i, n); }
   else {
#pragma unroll
      for (int j = 0; j < 8; j++) from_acc(c.e[j], 1);
   }
}

// Codes and scales of a chunk.  VEC: 16 neighbouring lanes hold the 128 elements of a block; otherwise the warp holds
// two blocks, elements 0-3 of every lane and elements 4-7.
template <bool VEC>
__device__ __forceinline__ void put_codes(const NormArgs &a, int64_t row, int64_t i, const float *v, int lane, unsigned int mask)
{
   char *p = a.y.p + row * a.y.s1;
   if (VEC) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) m = max(m, b8_magnitude(v[j]));
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(mask, m, d));
      if (i >= a.n) return;
      const float s = b8_scale(m, a.format), inv = 1.0f / s;
      *reinterpret_cast<uint2 *>(p + i) = make_uint2(b8_four(v, inv, a.format), b8_four(v + 4, inv, a.format));
      if ((lane & 15) == 0) a.scale[row * a.ss0 + i / B8_BLOCK * a.ss1] = s;
   } else {
#pragma unroll
      for (int half = 0; half < 2; half++) {
         uint32_t m = 0;
#pragma unroll
         for (int j = 0; j < 4; j++) m = max(m, b8_magnitude(v[4 * half + j]));
#pragma unroll
         for (int d = 16; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(mask, m, d));
         const float s = b8_scale(m, a.format), inv = 1.0f / s;
         const int64_t k0 = i + 128 * half;
#pragma unroll
         for (int j = 0; j < 4; j++)
            if (k0 + 32 * j < a.n) p[(k0 + 32 * j) * a.y.s0] = (char)b8_pair(v[4 * half + j] * inv, 0.0f, a.format);
         if (lane == 0 && k0 < a.n) a.scale[row * a.ss0 + k0 / B8_BLOCK * a.ss1] = s;
      }
   }
}

// Sum over the threads of a row, the same bits in each of them.  `buf` alternates from row to row, so that one barrier
// a row is enough.
template <bool BLOCK, class W>
__device__ __forceinline__ W row_sum(W s, int group, unsigned int mask, W *buf)
{
#pragma unroll
   for (int d = 16; d >= 1; d >>= 1) if (BLOCK || d < group) s += __shfl_xor_sync(mask, s, d);
   if (BLOCK) {
      const int warps = blockDim.x >> 5;
      if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = s;
      __syncthreads();
      s = 0;
      for (int k = 0; k < warps; k++) s += buf[k];
   }
   return s;
}

template <class T, int V, bool BLOCK, bool VEC, bool PIPE, bool QUANT, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_rows(const __grid_constant__ NormArgs a)
{
   using W = typename Real<T>::acc;
   __shared__ W sums[2][32];
   const int lane = threadIdx.x & 31;
   const int group = BLOCK ? (int)blockDim.x : a.group;
   const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x % group;
   const int per_block = BLOCK ? 1 : (int)blockDim.x / group;
   const unsigned int mask = BLOCK || group == 32 ? 0xFFFFFFFFu : 0xFFFFu << (lane & 16);
   const int64_t step = (int64_t)gridDim.x * per_block;
   int64_t row = (int64_t)blockIdx.x * per_block + (BLOCK ? 0 : (int)threadIdx.x / group);
   if (row >= a.rows) return;
   const bool has_res = a.res.p != nullptr;
   Eight<T> w[V], x[V], r[V];
   auto fetch_row = [&](int64_t q) {
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int64_t i = chunk_first<VEC>(v, group, t);
         fetch<T, VEC>(x[v], a.x, q, i, a.n);
         if (has_res) fetch<T, VEC>(r[v], a.res, q, i, a.n);
      }
   };
   fetch_row(row);
   if (PIPE) {
#pragma unroll
      for (int v = 0; v < V; v++) fetch_weights<T, VEC>(w[v], a.w, chunk_first<VEC>(v, group, t), a.n);
   }
   for (int odd = 0; row < a.rows; row += step, odd ^= 1) {
      W h[V][8];
      W s = 0;
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int j = 0; j < 8; j++) {
            h[v][j] = to_acc(x[v].e[j]);
            if (has_res) h[v][j] += to_acc(r[v].e[j]);
            s = fma(h[v][j], h[v][j], s);
         }
      if (PIPE && row + step < a.rows) fetch_row(row + step);
      if (!PIPE) {
#pragma unroll
         for (int v = 0; v < V; v++) fetch_weights<T, VEC>(w[v], a.w, chunk_first<VEC>(v, group, t), a.n);
      }
      s = row_sum<BLOCK>(s, group, mask, sums[odd]);
      const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int64_t i = chunk_first<VEC>(v, group, t);
         if (a.h.p != nullptr) put<T, VEC>(a.h, row, i, a.n, h[v]);
#pragma unroll
         for (int j = 0; j < 8; j++) h[v][j] = h[v][j] * rr * to_acc(w[v].e[j]);
         if (QUANT) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = (float)h[v][j];
#pragma unroll
            for (int j = 0; j < 8; j++) if (i + chunk_step<VEC> * j >= a.n) f[j] = 0.0f;     // zeros in their block's maximum
            put_codes<VEC>(a, row, i, f, lane, mask);
         } else put<T, VEC>(a.y, row, i, a.n, h[v]);
      }
      if (!PIPE && row + step < a.rows) fetch_row(row + step);
   }
}

// ---------------------------------------------------------------------------
// rows through a ring in shared memory
// ---------------------------------------------------------------------------
// Whole rows on 16-byte boundaries come by bulk copies into a ring of `stages` rows (of each operand), so that the loads in
// flight do not depend on registers or on the reduction's barrier: one thread refills a row's place after the barrier
// of the next row, by which time every thread has finished with it.  A wait that runs out makes the thread's elements NaN,
// what is stored of x + residual among them, and through the sums the row's results.
constexpr int RING_MAX = 4;

struct Ring {
   uint32_t bars, data, stage;                            // shared addresses, bytes of a stage
   int stages;
   bool ok;
   __device__ __forceinline__ void start(char *smem, uint64_t *bar, int bytes, int count)
   {
      bars = tc::smem_u32(bar); data = tc::smem_u32(smem); stage = bytes; stages = count; ok = true;
      if (threadIdx.x == 0) {
         for (int s = 0; s < stages; s++) tc::bar_init(bars + 8 * s, 1);
         asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      }
      __syncthreads();
   }
   // one row of an operand to its place in a stage
   __device__ __forceinline__ void copy(int s, int offset, const RowMatrix &m, int64_t row, uint32_t bytes)
   {
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   :: "r"(data + s * stage + offset), "l"(m.p + row * m.s1), "r"(bytes), "r"(bars + 8 * s) : "memory");
   }
   __device__ __forceinline__ void wait(int it) { if (ok) ok = tc::bar_wait(bars + 8 * (it % stages), (it / stages) & 1); }
};

template <class T, int V, bool QUANT, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_ring(const __grid_constant__ NormArgs a, int stages)
{
   using W = typename Real<T>::acc;
   extern __shared__ __align__(128) char smem[];
   __shared__ alignas(8) uint64_t bar[RING_MAX];
   __shared__ W sums[2][32];
   const int lane = threadIdx.x & 31, t = threadIdx.x, threads = blockDim.x;
   const bool has_res = a.res.p != nullptr;
   const int bytes = (int)(a.n * sizeof(T));
   Ring ring;
   ring.start(smem, bar, has_res ? 2 * bytes : bytes, stages);
   auto load = [&](int it) {
      const int64_t row = blockIdx.x + (int64_t)it * gridDim.x;
      if (row >= a.rows) return;
      const int s = it % stages;
      tc::bar_expect(ring.bars + 8 * s, ring.stage);
      ring.copy(s, 0, a.x, row, bytes);
      if (has_res) ring.copy(s, bytes, a.res, row, bytes);
   };
   if (t == 0) for (int it = 0; it < stages; it++) load(it);
   Eight<T> w[V];
#pragma unroll
   for (int v = 0; v < V; v++) fetch_weights<T, true>(w[v], a.w, chunk_first<true>(v, threads, t), a.n);
   int it = 0;
   for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, it++) {
      ring.wait(it);
      const char *place = smem + (it % stages) * ring.stage;
      W h[V][8];
      W s = 0;
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int i = (v * threads + t) * 8;
         if (i < a.n && ring.ok) {
            const Eight<T> x = load_eight<T>(place + i * sizeof(T));
#pragma unroll
            for (int j = 0; j < 8; j++) h[v][j] = to_acc(x.e[j]);
            if (has_res) {
               const Eight<T> r = load_eight<T>(place + bytes + i * sizeof(T));
#pragma unroll
               for (int j = 0; j < 8; j++) h[v][j] += to_acc(r.e[j]);
            }
         } else {
            const W none = ring.ok ? (W)0 : (W)NAN;
#pragma unroll
            for (int j = 0; j < 8; j++) h[v][j] = none;
         }
#pragma unroll
         for (int j = 0; j < 8; j++) s = fma(h[v][j], h[v][j], s);
      }
      s = row_sum<true>(s, threads, 0xFFFFFFFFu, sums[it & 1]);
      if (t == 0 && it > 0) load(it - 1 + stages);
      const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int64_t i = chunk_first<true>(v, threads, t);
         if (a.h.p != nullptr) put<T, true>(a.h, row, i, a.n, h[v]);
#pragma unroll
         for (int j = 0; j < 8; j++) h[v][j] = h[v][j] * rr * to_acc(w[v].e[j]);
         if (QUANT) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = i < a.n ? (float)h[v][j] : 0.0f;
            put_codes<true>(a, row, i, f, lane, 0xFFFFFFFFu);
         } else put<T, true>(a.y, row, i, a.n, h[v]);
      }
   }
   if (!ring.ok && t == 0) for (int k = max(0, it - stages); k < it; k++) tc::bar_wait(ring.bars + 8 * (k % stages), (k / stages) & 1);
}

// Rows too long for the registers of a block: the block reads the row twice (the second time from the L2 cache).  h is
// written in the second pass, each element by the thread that has just read it, so that h may stand in place of x or
// of the residual.
template <class T, bool QUANT>
__global__ void __launch_bounds__(512) norm_long(const __grid_constant__ NormArgs a)
{
   using W = typename Real<T>::acc;
   __shared__ W sums[2][32];
   const int t = threadIdx.x, lane = t & 31;
   const int chunk = 512 * 8;
   int odd = 0;
   for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, odd ^= 1) {
      W s = 0;
      Eight<T> x, r, w;
      auto element = [&](int j) { return a.res.p != nullptr ? to_acc(x.e[j]) + to_acc(r.e[j]) : to_acc(x.e[j]); };
      for (int64_t c = 0; c < a.n; c += chunk) {
         const int64_t i = c + chunk_first<false>(0, 512, t);
         fetch<T, false>(x, a.x, row, i, a.n);
         if (a.res.p != nullptr) fetch<T, false>(r, a.res, row, i, a.n);
#pragma unroll
         for (int j = 0; j < 8; j++) { const W h = element(j); s = fma(h, h, s); }
      }
      s = row_sum<true>(s, 512, 0xFFFFFFFFu, sums[odd]);
      const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
      for (int64_t c = 0; c < a.n; c += chunk) {
         const int64_t i = c + chunk_first<false>(0, 512, t);
         fetch<T, false>(x, a.x, row, i, a.n);
         if (a.res.p != nullptr) fetch<T, false>(r, a.res, row, i, a.n);
         fetch_weights<T, false>(w, a.w, i, a.n);
         W h[8];
#pragma unroll
         for (int j = 0; j < 8; j++) h[j] = element(j);
         if (a.h.p != nullptr) put<T, false>(a.h, row, i, a.n, h);
#pragma unroll
         for (int j = 0; j < 8; j++) h[j] = h[j] * rr * to_acc(w.e[j]);
         if (QUANT) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = i + 32 * j < a.n ? (float)h[j] : 0.0f;
            put_codes<false>(a, row, i, f, lane, 0xFFFFFFFFu);
         } else put<T, false>(a.y, row, i, a.n, h);
      }
   }
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
// With u = h r, the normalised row:  dh = r (g - u mean(g u)).  Each factor is then of the size of one of the operands;
// r^3 by itself would leave the range of 32 bits for rows above 1e13 or below 1e-13.
template <class T, int V, bool BLOCK, bool VEC, bool PIPE, int MAXT>
__global__ void __launch_bounds__(MAXT, BLOCK || sizeof(T) == 8 ? 1 : 3) grad_rows(const __grid_constant__ GradArgs a)
{
   using W = typename Real<T>::acc;
   __shared__ W sums[2][2][32];
   extern __shared__ char join_raw[];                     // warps' rows: n sums of the block
   const int lane = threadIdx.x & 31;
   const int group = BLOCK ? (int)blockDim.x : a.group;
   const int t = BLOCK ? (int)threadIdx.x : (int)threadIdx.x % group;
   const int per_block = BLOCK ? 1 : (int)blockDim.x / group;
   const int sub = BLOCK ? 0 : (int)threadIdx.x / group;
   const unsigned int mask = BLOCK || group == 32 ? 0xFFFFFFFFu : 0xFFFFu << (lane & 16);
   const int64_t step = (int64_t)gridDim.x * per_block;
   int64_t row = (int64_t)blockIdx.x * per_block + sub;
   const bool has_res = a.res.p != nullptr;
   Eight<T> w[V], g[V], h[V], r[V];
   W dw[V][8];
#pragma unroll
   for (int v = 0; v < V; v++)
#pragma unroll
      for (int j = 0; j < 8; j++) dw[v][j] = 0;
   auto fetch_row = [&](int64_t q) {
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int64_t i = chunk_first<VEC>(v, group, t);
         fetch<T, VEC>(g[v], a.dy, q, i, a.n);
         fetch<T, VEC>(h[v], a.h, q, i, a.n);
         if (has_res) fetch<T, VEC>(r[v], a.res, q, i, a.n);
      }
   };
   if (row < a.rows) fetch_row(row);
#pragma unroll
   for (int v = 0; v < V; v++) fetch_weights<T, VEC>(w[v], a.w, chunk_first<VEC>(v, group, t), a.n);
   const W inv_n = (W)1 / (W)a.n;
   for (int odd = 0; row < a.rows; row += step, odd ^= 1) {
      W s = 0, p = 0;
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int j = 0; j < 8; j++) {
            const W hv = to_acc(h[v].e[j]);
            s = fma(hv, hv, s);
            p = fma(to_acc(g[v].e[j]) * to_acc(w[v].e[j]), hv, p);
         }
      Eight<T> cg[V], ch[V], cr[V];
#pragma unroll
      for (int v = 0; v < V; v++) { cg[v] = g[v]; ch[v] = h[v]; if (has_res) cr[v] = r[v]; }
      if (PIPE && row + step < a.rows) fetch_row(row + step);
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) if (BLOCK || d < group) { s += __shfl_xor_sync(mask, s, d); p += __shfl_xor_sync(mask, p, d); }
      if (BLOCK) {
         if (lane == 0) { sums[odd][0][threadIdx.x >> 5] = s; sums[odd][1][threadIdx.x >> 5] = p; }
         __syncthreads();
         s = 0; p = 0;
         const int warps = blockDim.x >> 5;
         for (int k = 0; k < warps; k++) { s += sums[odd][0][k]; p += sums[odd][1][k]; }
      }
      const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
      const W c = rr * (p * inv_n);
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int64_t i = chunk_first<VEC>(v, group, t);
         W d[8];
#pragma unroll
         for (int j = 0; j < 8; j++) {
            const W gv = to_acc(cg[v].e[j]), u = to_acc(ch[v].e[j]) * rr;
            d[j] = rr * fma(-u, c, gv * to_acc(w[v].e[j]));
            if (has_res) d[j] += to_acc(cr[v].e[j]);
            dw[v][j] = fma(gv, u, dw[v][j]);
         }
         put<T, VEC>(a.dh, row, i, a.n, d);
      }
      if (!PIPE && row + step < a.rows) fetch_row(row + step);
   }
   if (a.part == nullptr) return;
   W *part = (W *)a.part + (int64_t)blockIdx.x * a.n;
   if (BLOCK) {
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int j = 0; j < 8; j++) {
            const int64_t k = chunk_first<VEC>(v, group, t) + chunk_step<VEC> * j;
            if (k < a.n) part[k] = dw[v][j];
         }
   } else {                                               // rows of the block join in the order of their warps
      W *join = (W *)join_raw;
      for (int q = 0; q < per_block; q++) {
         if (sub == q) {
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
               for (int j = 0; j < 8; j++) {
                  const int64_t k = chunk_first<VEC>(v, group, t) + chunk_step<VEC> * j;
                  if (k < a.n) join[k] = q == 0 ? dw[v][j] : join[k] + dw[v][j];
               }
         }
         __syncthreads();
      }
      for (int64_t k = threadIdx.x; k < a.n; k += blockDim.x) part[k] = join[k];
   }
}

template <class T, int V, int MAXT>
__global__ void __launch_bounds__(MAXT) grad_ring(const __grid_constant__ GradArgs a, int stages)
{
   using W = typename Real<T>::acc;
   extern __shared__ __align__(128) char smem[];
   __shared__ alignas(8) uint64_t bar[RING_MAX];
   __shared__ W sums[2][2][32];
   const int lane = threadIdx.x & 31, t = threadIdx.x, threads = blockDim.x;
   const bool has_res = a.res.p != nullptr;
   const int bytes = (int)(a.n * sizeof(T));
   Ring ring;
   ring.start(smem, bar, (has_res ? 3 : 2) * bytes, stages);
   auto load = [&](int it) {
      const int64_t row = blockIdx.x + (int64_t)it * gridDim.x;
      if (row >= a.rows) return;
      const int s = it % stages;
      tc::bar_expect(ring.bars + 8 * s, ring.stage);
      ring.copy(s, 0, a.dy, row, bytes);
      ring.copy(s, bytes, a.h, row, bytes);
      if (has_res) ring.copy(s, 2 * bytes, a.res, row, bytes);
   };
   if (t == 0) for (int it = 0; it < stages; it++) load(it);
   Eight<T> w[V];
   W dw[V][8];
#pragma unroll
   for (int v = 0; v < V; v++) {
      fetch_weights<T, true>(w[v], a.w, chunk_first<true>(v, threads, t), a.n);
#pragma unroll
      for (int j = 0; j < 8; j++) dw[v][j] = 0;
   }
   const W inv_n = (W)1 / (W)a.n;
   int it = 0;
   for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, it++) {
      ring.wait(it);
      const char *place = smem + (it % stages) * ring.stage;
      W s = 0, p = 0;
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int i = (v * threads + t) * 8;
         if (i < a.n) {
            const Eight<T> g = load_eight<T>(place + i * sizeof(T)), h = load_eight<T>(place + bytes + i * sizeof(T));
#pragma unroll
            for (int j = 0; j < 8; j++) {
               const W hv = to_acc(h.e[j]);
               s = fma(hv, hv, s);
               p = fma(to_acc(g.e[j]) * to_acc(w[v].e[j]), hv, p);
            }
         }
      }
      if (!ring.ok) s = (W)NAN;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) { s += __shfl_xor_sync(0xFFFFFFFFu, s, d); p += __shfl_xor_sync(0xFFFFFFFFu, p, d); }
      if (lane == 0) { sums[it & 1][0][t >> 5] = s; sums[it & 1][1][t >> 5] = p; }
      __syncthreads();
      if (t == 0 && it > 0) load(it - 1 + stages);
      s = 0; p = 0;
      for (int k = 0; k < threads / 32; k++) { s += sums[it & 1][0][k]; p += sums[it & 1][1][k]; }
      const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
      const W c = rr * (p * inv_n);
#pragma unroll
      for (int v = 0; v < V; v++) {                       // the row once more from shared memory: no registers between
         const int i = (v * threads + t) * 8;
         if (i < a.n) {
            const Eight<T> g = load_eight<T>(place + i * sizeof(T)), h = load_eight<T>(place + bytes + i * sizeof(T));
            W d[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
               const W gv = to_acc(g.e[j]), u = to_acc(h.e[j]) * rr;
               d[j] = rr * fma(-u, c, gv * to_acc(w[v].e[j]));
               dw[v][j] = fma(gv, u, dw[v][j]);
            }
            if (has_res) {
               const Eight<T> r = load_eight<T>(place + 2 * bytes + i * sizeof(T));
#pragma unroll
               for (int j = 0; j < 8; j++) d[j] += to_acc(r.e[j]);
            }
            put<T, true>(a.dh, row, i, a.n, d);
         }
      }
   }
   if (!ring.ok && t == 0) for (int k = max(0, it - stages); k < it; k++) tc::bar_wait(ring.bars + 8 * (k % stages), (k / stages) & 1);
   if (a.part != nullptr) {
      W *part = (W *)a.part + (int64_t)blockIdx.x * a.n;
#pragma unroll
      for (int v = 0; v < V; v++) {
         const int i = (v * threads + t) * 8;
         if (i < a.n) {
            Eight<W> o;
#pragma unroll
            for (int j = 0; j < 8; j++) o.e[j] = dw[v][j];
            store_eight(part + i, o);
         }
      }
   }
}

// dw = the sum of the blocks' partial rows: 32 columns a block, its warps a part of the rows each, in the order of the
// blocks within a warp and then of the warps
constexpr int JOIN_WARPS = 32;
template <class W>
__global__ void __launch_bounds__(JOIN_WARPS * 32) grad_join(const W *__restrict__ part, int64_t parts, int64_t n, W *__restrict__ dw)
{
   __shared__ W sums[JOIN_WARPS][33];
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
   const int64_t k = (int64_t)blockIdx.x * 32 + lane;
   W s = 0;
   if (k < n)
#pragma unroll 8
      for (int64_t p = warp; p < parts; p += JOIN_WARPS) s += part[p * n + k];
   sums[warp][lane] = s;
   __syncthreads();
   s = sums[lane][warp];                                  // column `warp` of the block's, a part each lane
#pragma unroll
   for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
   const int64_t c = (int64_t)blockIdx.x * 32 + warp;
   if (lane == 0 && c < n) dw[c] = s;
}

// Long rows: a first kernel forms each row's r and r mean(g h), a second one walks the columns
template <class T>
__global__ void __launch_bounds__(512) grad_long_sums(const __grid_constant__ GradArgs a, typename Real<T>::acc *rowsums)
{
   using W = typename Real<T>::acc;
   __shared__ W sums[2][2][32];
   int odd = 0;
   for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, odd ^= 1) {
      W s = 0, p = 0;
      for (int64_t c = 0; c < a.n; c += 512 * 8) {
         const int64_t i = c + chunk_first<false>(0, 512, threadIdx.x);
         Eight<T> g, h, w;
         fetch<T, false>(g, a.dy, row, i, a.n);
         fetch<T, false>(h, a.h, row, i, a.n);
         fetch_weights<T, false>(w, a.w, i, a.n);
#pragma unroll
         for (int j = 0; j < 8; j++) {
            const W hv = to_acc(h.e[j]);
            s = fma(hv, hv, s);
            p = fma(to_acc(g.e[j]) * to_acc(w.e[j]), hv, p);
         }
      }
      s = row_sum<true>(s, 512, 0xFFFFFFFFu, sums[odd][0]);
      p = row_sum<true>(p, 512, 0xFFFFFFFFu, sums[odd][1]);
      if (threadIdx.x == 0) {
         const W rr = (W)1 / sqrt(s / (W)a.n + (W)a.eps);
         rowsums[2 * row] = rr;
         rowsums[2 * row + 1] = rr * (p / (W)a.n);
      }
   }
}

template <class T>
__global__ void __launch_bounds__(256) grad_long_apply(const __grid_constant__ GradArgs a, const typename Real<T>::acc *rowsums)
{
   using W = typename Real<T>::acc;
   const int64_t i = (int64_t)blockIdx.x * 2048 + chunk_first<false>(0, 256, threadIdx.x);
   Eight<T> w;
   fetch_weights<T, false>(w, a.w, i, a.n);
   W dw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
   for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
      Eight<T> g, h, r;
      fetch<T, false>(g, a.dy, row, i, a.n);
      fetch<T, false>(h, a.h, row, i, a.n);
      if (a.res.p != nullptr) fetch<T, false>(r, a.res, row, i, a.n);
      const W rr = rowsums[2 * row], c = rowsums[2 * row + 1];
      W d[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
         const W gv = to_acc(g.e[j]), u = to_acc(h.e[j]) * rr;
         d[j] = rr * fma(-u, c, gv * to_acc(w.e[j]));
         if (a.res.p != nullptr) d[j] += to_acc(r.e[j]);
         dw[j] = fma(gv, u, dw[j]);
      }
      put<T, false>(a.dh, row, i, a.n, d);
   }
   if (a.part != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; j++) if (i + 32 * j < a.n) ((W *)a.part)[(int64_t)blockIdx.y * a.n + i + 32 * j] = dw[j];
   }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static bool whole(const RowMatrix &m, size_t elemsize, size_t align, int64_t rows)
{
   return m.p == nullptr || (m.s0 == (int64_t)elemsize && (uintptr_t)m.p % align == 0 && (rows == 1 || m.s1 % (int64_t)align == 0));
}

static int matrix_of(const solid_gpu_matrix *m, size_t elemsize, const char *what, const char *op, bool optional, RowMatrix *out)
{
   if (m == nullptr || m->ptr == nullptr) {
      if (!optional) SD_ERROR("%s: missing matrix %s", op, what);
      *out = { nullptr, 0, 0 };
      return 0;
   }
   if ((uintptr_t)m->ptr % elemsize != 0 || m->stride0 % (ptrdiff_t)elemsize != 0 || m->stride1 % (ptrdiff_t)elemsize != 0)
      SD_ERROR("%s: matrix %s must be aligned to its element size", op, what);
   *out = { (char *)m->ptr, (int64_t)m->stride0, (int64_t)m->stride1 };
   return 0;
}

// Resident blocks of a kernel on the current device, asked for once per kernel
template <class K> static int resident(K kernel, std::atomic<int> &cache, int threads, size_t smem, int sms)
{
   const int key = threads;                               // block size and blocks per SM in one word
   int v = cache.load(std::memory_order_relaxed);
   if (v / 64 != key) {
      int b = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, kernel, threads, smem) != cudaSuccess || b < 1) { cudaGetLastError(); b = 1; }
      v = key * 64 + (b < 63 ? b : 63);
      cache.store(v, std::memory_order_relaxed);
   }
   return (v % 64) * sms;
}

static int round32(int64_t v) { return (int)((v + 31) / 32 * 32); }
constexpr int64_t NORM_MAX = 16384;

template <class T, int V, bool BLOCK, bool VEC, bool PIPE, bool QUANT, int MAXT>
static int launch_norm(NormArgs &a, int threads, int sms, cudaStream_t stream)
{
   static std::atomic<int> cache{0};
   auto *kernel = norm_rows<T, V, BLOCK, VEC, PIPE, QUANT, MAXT>;
   const int64_t per_block = BLOCK ? 1 : threads / a.group;
   const int64_t want = (a.rows + per_block - 1) / per_block, most = resident(kernel, cache, threads, 0, sms);
   kernel<<<(unsigned)(want < most ? want : most), threads, 0, stream>>>(a);
   SD_LAUNCH_CHECK();
   return 0;
}

// Blocks of an SM and rows under way in each.  About 128 KB under way on an SM are enough for the memory's latency, more
// only disturbs (halves, n 4096 with residual: 45 us with 128 KB, 49 us with 190 KB); four rows a block spread over
// enough blocks for the arithmetic, which with 8-bit output is twice as much (n 4096: 58 us with 512 threads an SM, 47 us
// with 1024).
constexpr int64_t RING_ROOM = 225 * 1024, RING_STATIC = 2048;       // of an SM's shared memory; barriers and sums of a block
struct RingPlan { int per_sm, stages; size_t smem; };
static RingPlan ring_plan(int64_t stage_bytes, int threads, int threads_per_sm)
{
   constexpr int64_t UNDER_WAY = 128 * 1024, ROOM = RING_ROOM;
   RingPlan p;
   p.per_sm = (int)std::min<int64_t>(16, std::max<int64_t>(UNDER_WAY / (RING_MAX * stage_bytes), threads_per_sm / threads));
   p.per_sm = std::max(1, std::min(p.per_sm, 2048 / threads));
   while (p.per_sm > 1 && 2 * stage_bytes > ROOM / p.per_sm - RING_STATIC) p.per_sm--;
   p.stages = (int)std::max<int64_t>(2, std::min<int64_t>(RING_MAX, (p.per_sm > 1 ? UNDER_WAY : ROOM - RING_STATIC) / (p.per_sm * stage_bytes)));
   p.smem = (size_t)(p.stages * stage_bytes);
   if (2 * stage_bytes > ROOM - RING_STATIC) p.per_sm = 0;       // not even two rows: no ring
   return p;
}

// The limit on a kernel's shared memory belongs to the kernel, for all host threads.  So every call sets the same one, the
// most that a plan asks for: one of its own could be lowered by another thread's call between setting and launch.
template <class K> static int allow_ring(K kernel)
{
   SD_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(RING_ROOM - RING_STATIC)));
   return 0;
}

template <class T, int V, bool QUANT>
static int launch_norm_ring(NormArgs &a, const RingPlan &p, int threads, int sms, cudaStream_t stream)
{
   auto *kernel = norm_ring<T, V, QUANT, 512>;
   if (allow_ring(kernel) != 0) return -1;
   kernel<<<(unsigned)std::min<int64_t>(a.rows, (int64_t)p.per_sm * sms), threads, p.smem, stream>>>(a, p.stages);
   SD_LAUNCH_CHECK();
   return 0;
}

template <class T, bool VEC, bool QUANT>
static int norm_of(NormArgs &a, cudaStream_t stream)
{
   DeviceInfo dev;
   if (current_device_info(&dev) != 0) return -1;
   const int sms = dev.sms;
   const int64_t n = a.n, eights = (n + 7) / 8;
   constexpr bool WIDE = sizeof(T) == 8;                  // doubles: half as many elements fit the registers
   a.group = VEC && n <= 128 ? 16 : 32;
   if (n <= 256)  return launch_norm<T, 1, false, VEC, true, QUANT, 256>(a, 256, sms, stream);
   if (n <= 512)  return launch_norm<T, 2, false, VEC, true, QUANT, 256>(a, 256, sms, stream);
   // few rows: a thread takes eight elements, so that a row is one round of loads
   if (a.rows <= sms && n <= 8192) return launch_norm<T, 1, true, VEC, false, QUANT, 1024>(a, round32(eights), sms, stream);
   if constexpr (VEC) {
      if (n <= NORM_MAX) {
         const int threads = std::max(64, round32((eights + (n <= 8192 ? 1 : 3)) / (n <= 8192 ? 2 : 4)));
         const RingPlan p = ring_plan(n * (int64_t)sizeof(T) * (a.res.p != nullptr ? 2 : 1), threads, QUANT ? 1024 : 512);
         if (p.per_sm >= 1) return n <= 8192 ? launch_norm_ring<T, 2, QUANT>(a, p, threads, sms, stream)
                                             : launch_norm_ring<T, 4, QUANT>(a, p, threads, sms, stream);
      }
   }
   if constexpr (!VEC) {
      if (n <= 2048) return launch_norm<T, 1, true, VEC, true, QUANT, 256>(a, round32(eights), sms, stream);
   }
   // Of whole rows, two fit the ring for all halves, for floats up to 8192 elements and for most doubles
   if constexpr (!VEC || WIDE) {
      if (n <= 8192) return launch_norm<T, 2, true, VEC, !WIDE, QUANT, 512>(a, round32((eights + 1) / 2), sms, stream);
   }
   if constexpr (!WIDE && (!VEC || sizeof(T) == 4)) {
      if (n <= NORM_MAX) return launch_norm<T, 4, true, VEC, false, QUANT, 512>(a, round32((eights + 3) / 4), sms, stream);
   }
   norm_long<T, QUANT><<<(unsigned)(a.rows < 4 * sms ? a.rows : 4 * sms), 512, 0, stream>>>(a);
   SD_LAUNCH_CHECK();
   return 0;
}

template <class T, bool QUANT> static int norm_typed(NormArgs &a, cudaStream_t stream)
{
   const size_t es = sizeof(T);
   const bool vec = a.n % 8 == 0 && whole(a.x, es, 16, a.rows) && whole(a.res, es, 16, a.rows) && whole(a.h, es, 16, a.rows) &&
                    (uintptr_t)a.w % 16 == 0 && (QUANT ? whole(a.y, 1, 8, a.rows) : whole(a.y, es, 16, a.rows));
   return vec ? norm_of<T, true, QUANT>(a, stream) : norm_of<T, false, QUANT>(a, stream);
}

template <bool QUANT> static int norm_any(int dtype, NormArgs &a, cudaStream_t stream)
{
   if (dtype == SD_HALF)   return norm_typed<__half, QUANT>(a, stream);
   if (dtype == SD_FLOAT)  return norm_typed<float, QUANT>(a, stream);
   return norm_typed<double, QUANT>(a, stream);
}

static int check_norm(int dtype, size_t n, size_t rows, double eps, const void *w, const char *op, size_t *elemsize)
{
   if (dtype != SD_HALF && dtype != SD_FLOAT && dtype != SD_DOUBLE) SD_ERROR("%s: the type must be half, float or double", op);
   if (!(eps >= 0)) SD_ERROR("%s: eps must not be negative", op);
   if (n > ((size_t)1 << 40) || rows > ((size_t)1 << 40)) SD_ERROR("%s: matrix too large", op);
   *elemsize = (size_t)solid_gpu_type_size[dtype];
   if ((uintptr_t)w % *elemsize != 0) SD_ERROR("%s: the weights must be aligned to their element size", op);
   return 0;
}

static int fill_norm(int dtype, size_t n, size_t rows, const solid_gpu_matrix *x, const solid_gpu_matrix *residual,
                     const void *weight, double eps, const solid_gpu_matrix *h, const char *op, NormArgs *a)
{
   size_t es;
   if (check_norm(dtype, n, rows, eps, weight, op, &es) != 0) return -1;
   a->n = (int64_t)n; a->rows = (int64_t)rows; a->w = weight; a->eps = eps; a->group = 32;
   a->scale = nullptr; a->ss0 = a->ss1 = 0; a->format = 0;
   const bool empty = n == 0 || rows == 0;                // no element: no address needed
   if (matrix_of(x, es, "x", op, empty, &a->x) != 0 || matrix_of(residual, es, "residual", op, true, &a->res) != 0 ||
       matrix_of(h, es, "h", op, true, &a->h) != 0) return -1;
   return 0;
}

// ---- gradient ----
// kind: 1 a warp's row; 11, 12, 14 a block's, with 1, 2, 4 eights a thread; 20 long rows
struct GradPlan { int kind, threads, blocks; };

static int grad_stages(int64_t n, size_t elemsize, int operands, int per_sm)
{
   return (int)std::min<int64_t>(RING_MAX, (RING_ROOM / per_sm - RING_STATIC) / (n * (int64_t)elemsize * operands));
}

template <class T> static bool grad_vec(const GradArgs &a)
{
   const size_t es = sizeof(T);
   return a.n % 8 == 0 && whole(a.dy, es, 16, a.rows) && whole(a.h, es, 16, a.rows) && whole(a.res, es, 16, a.rows) &&
          whole(a.dh, es, 16, a.rows) && (uintptr_t)a.w % 16 == 0;
}

// The number of partial rows follows from sizes alone, so that the buffer's size can be asked for beforehand.  (A row's own
// sums are taken in another order where its elements come one by one, so the last bits do depend on alignment.)  Blocks
// of an SM: 1024 threads, as long as three operands' rows fit the ring twice (halves, n 4096: 34 us with 512 threads, 30
// us with 1024).
static GradPlan grad_plan(int64_t n, int64_t rows, size_t elemsize, int sms)
{
   const bool wide = elemsize == 8;
   const int64_t eights = (n + 7) / 8;
   GradPlan p;
   if (n <= 256)       { p.kind = 1; p.threads = 256; }
   else if (n <= 1024) { p.kind = 11; p.threads = round32(eights); }
   else if (n <= 8192) { p.kind = 12; p.threads = round32((eights + 1) / 2); }
   else if (n <= NORM_MAX && !wide) { p.kind = 14; p.threads = round32((eights + 3) / 4); }
   else                { p.kind = 20; p.threads = 256; }
   int per_sm = std::max(1, std::min(16, 1024 / p.threads));
   if (p.kind == 1) per_sm = 3;
   else while (per_sm > 1 && grad_stages(n, elemsize, 3, per_sm) < 2) per_sm--;
   const int64_t rows_at_once = p.kind < 10 ? 8 : 1;      // warps of a block
   const int64_t want = (rows + rows_at_once - 1) / rows_at_once;
   p.blocks = (int)std::max<int64_t>(1, std::min(want, p.kind == 20 ? 16 : (int64_t)sms * per_sm));
   return p;
}

template <class T, int V, bool BLOCK, bool VEC, bool PIPE, int MAXT>
static int launch_grad(GradArgs &a, const GradPlan &p, cudaStream_t stream)
{
   const size_t smem = BLOCK ? 0 : (size_t)a.n * sizeof(typename Real<T>::acc);
   grad_rows<T, V, BLOCK, VEC, PIPE, MAXT><<<p.blocks, p.threads, smem, stream>>>(a);
   SD_LAUNCH_CHECK();
   return 0;
}

template <class T, int V> static int launch_grad_ring(GradArgs &a, const GradPlan &p, int stages, size_t smem, cudaStream_t stream)
{
   auto *kernel = grad_ring<T, V, 512>;
   if (allow_ring(kernel) != 0) return -1;
   kernel<<<p.blocks, p.threads, smem, stream>>>(a, stages);
   SD_LAUNCH_CHECK();
   return 0;
}

template <class T, bool VEC> static int grad_of(GradArgs &a, const GradPlan &p, int sms, cudaStream_t stream)
{
   constexpr bool WIDE = sizeof(T) == 8;
   a.group = 32;
   if (p.kind == 1) return launch_grad<T, 1, false, VEC, true, 256>(a, p, stream);
   if constexpr (VEC) {
      const int per_sm = (p.blocks + sms - 1) / sms;
      const int operands = a.res.p != nullptr ? 3 : 2, stages = grad_stages(a.n, sizeof(T), operands, per_sm);
      if (stages >= 2) {
         const size_t smem = (size_t)(stages * operands * a.n * (int64_t)sizeof(T));
         if (p.kind == 11) return launch_grad_ring<T, 1>(a, p, stages, smem, stream);
         if (p.kind == 12) return launch_grad_ring<T, 2>(a, p, stages, smem, stream);
         if constexpr (!WIDE) return launch_grad_ring<T, 4>(a, p, stages, smem, stream);
      }
   }
   if constexpr (!VEC) { if (p.kind == 11) return launch_grad<T, 1, true, VEC, false, 256>(a, p, stream); }
   // Of whole rows, two of three operands fit the ring for all halves and for floats up to 8192 elements
   if constexpr (!VEC || WIDE) { if (p.kind == 12) return launch_grad<T, 2, true, VEC, false, 512>(a, p, stream); }
   if constexpr (!WIDE && (!VEC || sizeof(T) == 4)) { if (p.kind == 14) return launch_grad<T, 4, true, VEC, false, 512>(a, p, stream); }
   SD_ERROR("rms_norm_grad: no kernel for rows of %lld elements", (long long)a.n);
}

// Partial rows are stored 16 bytes at a time, so they start on the caller's buffer's first such boundary
constexpr size_t BUFFER_ALIGN = 16;

template <class T> static int grad_typed(GradArgs &a, void *dw, void *buffer, cudaStream_t stream)
{
   using W = typename Real<T>::acc;
   DeviceInfo dev;
   if (current_device_info(&dev) != 0) return -1;
   const GradPlan p = grad_plan(a.n, a.rows, sizeof(T), dev.sms);
   W *rowsums = (W *)(((uintptr_t)buffer + BUFFER_ALIGN - 1) / BUFFER_ALIGN * BUFFER_ALIGN);     // long rows only
   W *part = p.kind == 20 ? rowsums + 2 * a.rows : rowsums;
   a.part = dw != nullptr ? part : nullptr;
   if (p.kind == 20) {
      grad_long_sums<T><<<(unsigned)std::min<int64_t>(a.rows, 4 * dev.sms), 512, 0, stream>>>(a, rowsums);
      SD_LAUNCH_CHECK();
      grad_long_apply<T><<<dim3((unsigned)((a.n + 2047) / 2048), (unsigned)p.blocks), 256, 0, stream>>>(a, rowsums);
   }
   else if ((grad_vec<T>(a) ? grad_of<T, true>(a, p, dev.sms, stream) : grad_of<T, false>(a, p, dev.sms, stream)) != 0) return -1;
   SD_LAUNCH_CHECK();
   if (dw != nullptr) {
      grad_join<W><<<(unsigned)((a.n + 31) / 32), JOIN_WARPS * 32, 0, stream>>>(part, p.blocks, a.n, (W *)dw);
      SD_LAUNCH_CHECK();
   }
   return 0;
}

} // namespace sd

extern "C" int solid_gpu_rms_norm(int dtype, size_t n, size_t rows, const solid_gpu_matrix *x, const solid_gpu_matrix *residual,
                                  const void *weight, double eps, const solid_gpu_matrix *h, const solid_gpu_matrix *y,
                                  cudaStream_t stream)
{
   sd::NormArgs a;
   if (sd::fill_norm(dtype, n, rows, x, residual, weight, eps, h, "rms_norm", &a) != 0) return -1;
   const bool empty = n == 0 || rows == 0;
   if (sd::matrix_of(y, (size_t)solid_gpu_type_size[dtype], "y", "rms_norm", empty, &a.y) != 0) return -1;
   if (empty) return 0;
   return sd::norm_any<false>(dtype, a, stream);
}

extern "C" int solid_gpu_rms_norm_quantize(int dtype, size_t n, size_t rows, const solid_gpu_matrix *x, const solid_gpu_matrix *residual,
                                           const void *weight, double eps, const solid_gpu_matrix *h, const solid_gpu_blocks *y,
                                           cudaStream_t stream)
{
   sd::NormArgs a;
   if (sd::fill_norm(dtype, n, rows, x, residual, weight, eps, h, "rms_norm_quantize", &a) != 0) return -1;
   const bool empty = n == 0 || rows == 0;
   if (sd::check_blocks(y, "rms_norm_quantize", "y", empty) != 0) return -1;
   if (y->block != 1) SD_ERROR("rms_norm_quantize: a scale belongs to one row (block 1)");
   if (empty) return 0;
   a.y = { (char *)y->codes, 1, (int64_t)y->ld };
   a.scale = y->scales; a.ss0 = (int64_t)y->scale_stride0 / 4; a.ss1 = (int64_t)y->scale_stride1 / 4; a.format = y->format;
   return sd::norm_any<true>(dtype, a, stream);
}

extern "C" int solid_gpu_rms_norm_grad_buffer_size(int dtype, size_t n, size_t rows, int device, size_t *size)
{
   size_t es;
   if (sd::check_norm(dtype, n, rows, 0.0, nullptr, "rms_norm_grad", &es) != 0) return -1;
   if (size == nullptr) SD_ERROR("rms_norm_grad: missing size");
   const int sms = solid_gpu_multiprocessor_count(device);
   if (sms < 1) return -1;
   const sd::GradPlan p = sd::grad_plan((int64_t)n, (int64_t)rows, es, sms);
   *size = ((size_t)p.blocks * n + (p.kind == 20 ? 2 * rows : 0)) * (size_t)solid_gpu_worktype_size[dtype] + sd::BUFFER_ALIGN;
   return 0;
}

extern "C" int solid_gpu_rms_norm_grad(int dtype, size_t n, size_t rows, const solid_gpu_matrix *dy, const solid_gpu_matrix *h,
                                       const void *weight, double eps, const solid_gpu_matrix *dres, const solid_gpu_matrix *dh,
                                       void *dweight, void *buffer, cudaStream_t stream)
{
   sd::GradArgs a;
   size_t es;
   const char *op = "rms_norm_grad";
   if (sd::check_norm(dtype, n, rows, eps, weight, op, &es) != 0) return -1;
   const size_t ws = (size_t)solid_gpu_worktype_size[dtype];
   if ((uintptr_t)dweight % ws != 0 || (uintptr_t)buffer % ws != 0) SD_ERROR("%s: dweight and buffer must be aligned to their element size", op);
   a.n = (int64_t)n; a.rows = (int64_t)rows; a.w = weight; a.eps = eps; a.part = nullptr; a.group = 32;
   const bool empty = n == 0 || rows == 0;
   if (sd::matrix_of(dy, es, "dy", op, empty, &a.dy) != 0 || sd::matrix_of(h, es, "h", op, empty, &a.h) != 0 ||
       sd::matrix_of(dres, es, "dres", op, true, &a.res) != 0 || sd::matrix_of(dh, es, "dh", op, empty, &a.dh) != 0) return -1;
   if (n == 0) return 0;
   if (rows == 0) {                                       // no row: the weights' gradient is zero
      if (dweight != nullptr) SD_CUDA_CHECK(cudaMemsetAsync(dweight, 0, n * ws, stream));
      return 0;
   }
   if (buffer == nullptr) SD_ERROR("%s: missing scratch buffer", op);
   if (dtype == SD_HALF)  return sd::grad_typed<__half>(a, dweight, buffer, stream);
   if (dtype == SD_FLOAT) return sd::grad_typed<float>(a, dweight, buffer, stream);
   return sd::grad_typed<double>(a, dweight, buffer, stream);
}
