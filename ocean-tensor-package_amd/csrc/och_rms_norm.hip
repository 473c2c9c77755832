/* och_rms_norm and och_rms_norm_grad: the root-mean-square norm of the columns of a column-major n x rows matrix (one
 * column per token, n features), with the residual stream's addition in front and, behind it, an output in the input's
 * type or in 8-bit codes with one scale per 128 features; and its gradients. No counterpart in the reference.
 *
 *    h = round(x + r)          rstd = 1 / sqrt(mean(h^2) + eps)          y = (h rstd) w
 *    g = dy w,  u = h rstd     dx = rstd (g - u mean(g u)) + dh          dw = sum over the rows of dy u
 *
 * The norm is that of the sum as it is stored, so that the backward pass, which reads the stored sum, differentiates the
 * function that was computed. Sums are float. The gradient passes the 8-bit rounding straight through.
 */
#include "och_float8.h"

namespace och {

#define OCH_NORM_THREADS 256

/* x of the lane that the DPP control names, added */
template <int CTRL> __device__ __forceinline__ float dpp_add(float x)
{  const int i = __float_as_int(x); return x + __int_as_float(__builtin_amdgcn_update_dpp(0, i, CTRL, 0xF, 0xF, true)); }
__device__ __forceinline__ float row8_sum(float x)  { x = dpp_add<0xB1>(x); x = dpp_add<0x4E>(x); return dpp_add<0x141>(x); }
__device__ __forceinline__ float row16_sum(float x) { return dpp_add<0x140>(row8_sum(x)); }
__device__ __forceinline__ float lane_float(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }
/* sum over the wave, in all lanes: a fixed tree */
__device__ __forceinline__ float wave64_sum(float x)
{  x = row16_sum(x);
   return (lane_float(x, 0) + lane_float(x, 16)) + (lane_float(x, 32) + lane_float(x, 48));
}
/* sum over the workgroup, in all threads; `part` holds one float per wave and must not be in use */
__device__ __forceinline__ float block_sum(float x, float *part)
{  x = wave64_sum(x);
   if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
   __syncthreads();
   float s = 0;
   for (unsigned w = 0; w < blockDim.x / 64; w++) s += part[w];
   __syncthreads();
   return s;
}

/* sum over the T threads that share a row: 8, 16, 64 or the workgroup */
template <int T> __device__ __forceinline__ float group_sum(float x, float *part)
{  if (T == 8) return row8_sum(x);
   if (T == 16) return row16_sum(x);
   if (T == 64) return wave64_sum(x);
   return block_sum(x, part);
}

/* rows that a workgroup holds at a time when T threads share one */
constexpr int norm_rows(int T) { return T < OCH_NORM_THREADS ? OCH_NORM_THREADS / T : 1; }

struct NormParams
{
   const char *X, *R, *W; char *H, *Y; float *S, *rstd;
   int64_t  ldX, ldR, ldH, ldY, ldS;    /* in elements */
   int64_t  n, rows, first;             /* first: workgroup 0's place in the whole */
   float    eps, inverse;               /* inverse: 1 / n */
   int      w_float;                    /* the weights are float (else the type of X) */
};

/* 1 / sqrt(x): the instruction's result and one step of Newton's method; where that could leave the range of normal numbers,
   root and division */
__device__ __forceinline__ float inverse_root(float x)
{  if (!(x >= 0x1p-100f && x <= 0x1p100f)) return 1.0f / sqrtf(x);
   const float r = __builtin_amdgcn_rsqf(x);
   return __builtin_fmaf(0.5f * r, __builtin_fmaf(-x * r, r, 1.0f), r);
}

/* eight weights as floats (1 when there are none) */
template <int DT> __device__ __forceinline__ void load_weights(const char *W, int w_float, int64_t at, int64_t valid, float *w)
{  if (W == nullptr)
   {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = 1.0f;
   }
   else if (w_float)
   {  Wide8<OCH_FLOAT> v; v.load(reinterpret_cast<const float *>(W) + at, valid);
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = v.get(e);
   }
   else
   {  Wide8<DT> v; v.load(reinterpret_cast<const typename Wide<DT>::E *>(W) + at, valid);
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = v.get(e);
   }
}

/* eight values of the output: rounded to the input's type, or to codes with a scale that sixteen lanes share.
   Every lane of the wave calls it (CODE != 0 exchanges maxima between lanes). */
template <int DT, int CODE, bool NT> __device__ __forceinline__ void norm_store(const NormParams &p, int64_t row, int64_t at, int64_t valid, const float *y)
{
   if constexpr (CODE == 0)
   {  Wide8<DT> o;
#pragma unroll
      for (int e = 0; e < 8; e++) o.put(e, y[e]);
      o.template store<NT>(reinterpret_cast<typename Wide<DT>::E *>(p.Y) + at + row * p.ldY, valid);
   }
   else
   {  float m = 0;                                        /* a NaN stays; values behind the row's end are zero, or NaN with the row */
#pragma unroll
      for (int e = 0; e < 8; e++) m = __builtin_elementwise_maximum(m, fabsf(y[e]));
      float scale, factor; bool bad;
      block_scale<CODE>(row16_max(magnitude_bits(m)), scale, factor, bad);
      och_u32x2 q;
      q.x = code4<CODE>(y[0], y[1], y[2], y[3], factor, bad);
      q.y = code4<CODE>(y[4], y[5], y[6], y[7], factor, bad);
      store_codes<NT>(reinterpret_cast<uint8_t *>(p.Y) + at + row * p.ldY, q, valid);
      if (at % OCH_F8_BLOCK == 0 && valid > 0) p.S[at / OCH_F8_BLOCK + row * p.ldS] = scale;
   }
}

/* Rows of any length: a workgroup per row, two passes over it (the second finds it in the cache) */
template <int DT, int CODE>
__global__ __launch_bounds__(OCH_NORM_THREADS) void norm_long_kernel(const NormParams p)
{
   typedef typename Wide<DT>::E E;
   __shared__ float part[OCH_NORM_THREADS / 64];
   const int64_t row = p.first + blockIdx.x;
   const E *x = reinterpret_cast<const E *>(p.X) + row * p.ldX, *r = reinterpret_cast<const E *>(p.R) + row * p.ldR;
   E *h = reinterpret_cast<E *>(p.H) + row * p.ldH;
   float sum = 0;
   for (int64_t at = threadIdx.x * 8; at < p.n; at += OCH_NORM_THREADS * 8)
   {  Wide8<DT> v;
      v.load(x + at, p.n - at);
      if (p.R)
      {  Wide8<DT> a; a.load(r + at, p.n - at);
#pragma unroll
         for (int e = 0; e < 8; e++) v.put(e, v.get(e) + a.get(e));
      }
      if (p.H) v.store(h + at, p.n - at);
      float s = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) s = __builtin_fmaf(v.get(e), v.get(e), s);
      sum += s;
   }
   const float rstd = inverse_root(block_sum(sum, part) * p.inverse + p.eps);
   if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
   const E *again = p.H ? h : x;                           /* every thread reads what it wrote or read itself */
   for (int64_t at0 = 0; at0 < p.n; at0 += OCH_NORM_THREADS * 8)
   {  const int64_t at = at0 + threadIdx.x * 8;
      Wide8<DT> v; float w[8], y[8];
      v.load(again + at, p.n - at);
      load_weights<DT>(p.W, p.w_float, at, p.n - at, w);
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = v.get(e) * rstd * w[e];
      norm_store<DT, CODE, false>(p, row, at, p.n - at, y);
   }
}

/* Rows of at most 8 T V elements: T threads keep a row in registers, eight neighbouring elements in each of V vectors per
   thread, norm_rows(T) rows per workgroup. One pass over memory, which is what bounds it, then the instructions per element: with a
   general division for scale, factor, mean and root, 8192 rows of 8192 bfloat16 features to codes took 47.4 us, now 42.8.
   With the residual stream in and out: 82.2 us (5.7 TB/s of reads and writes); 5003 float features: 5.4 TB/s. */
template <int DT, int CODE, int T, int V, bool NT>
__global__ __launch_bounds__(T * norm_rows(T)) void norm_kernel(const NormParams p)
{
   typedef typename Wide<DT>::E E;
   __shared__ float part[T * norm_rows(T) / 64];
   const int64_t wanted = (p.first + blockIdx.x) * norm_rows(T) + threadIdx.x / T;
   const bool live = wanted < p.rows;
   const int64_t row = live ? wanted : p.rows - 1;
   const int first = (int)(threadIdx.x % T) * 8, n = live ? (int)p.n : 0;      /* a group without a row: no element is valid */
   const E *x = reinterpret_cast<const E *>(p.X) + row * p.ldX;
   Wide8<DT> h[V];
#pragma unroll
   for (int v = 0; v < V; v++) h[v].load(x + first + v * T * 8, n - first - v * T * 8);
   if (p.R)
   {  const E *r = reinterpret_cast<const E *>(p.R) + row * p.ldR;
      Wide8<DT> a[V];
#pragma unroll
      for (int v = 0; v < V; v++) a[v].load(r + first + v * T * 8, n - first - v * T * 8);
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int e = 0; e < 8; e++) h[v].put(e, h[v].get(e) + a[v].get(e));
   }
   if (p.H)
   {  E *to = reinterpret_cast<E *>(p.H) + row * p.ldH;
#pragma unroll
      for (int v = 0; v < V; v++) h[v].template store<NT>(to + first + v * T * 8, n - first - v * T * 8);
   }
   float sum = 0;
#pragma unroll
   for (int v = 0; v < V; v++)
   {  float s = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) s = __builtin_fmaf(h[v].get(e), h[v].get(e), s);
      sum += s;
   }
   const float rstd = inverse_root(group_sum<T>(sum, part) * p.inverse + p.eps);
   if (p.rstd && live && threadIdx.x % T == 0) p.rstd[row] = rstd;
#pragma unroll
   for (int v = 0; v < V; v++)
   {  const int at = first + v * T * 8;
      float w[8], y[8];
      load_weights<DT>(p.W, p.w_float, at, n - at, w);
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = h[v].get(e) * rstd * w[e];
      norm_store<DT, CODE, NT>(p, row, at, n - at, y);
   }
}

/* Threads and vectors by the row's length: as few threads as hold the row in two vectors each, because a group within a wave
   needs no barrier, but from there on more threads than vectors. 2^26 bfloat16 values with the residual stream, to codes:
      8192 features: 512 threads x 2 vectors 86.0 us, 256 x 4 90.2, 64 x 16 far behind;   16384: 512 x 4 91 us, 256 x 8 101;
      4096: 256 x 2 84.9 us, 512 x 1 83.4, but 48 against 58 without the residual stream;   5003 float: 256 x 3 15.3, 512 x 2 16.7;
   2^25 values in rows of 64, without it and without codes: 8 x 1 26.3 us, 16 x 1 39.8 */
template <int DT, int CODE> static int norm_launch(NormParams p, hipStream_t stream)
{
   auto go = [&](auto kernel, int rows, int threads) -> int
   {  const uint64_t groups = ((uint64_t)p.rows + rows - 1) / rows;
      for (p.first = 0; (uint64_t)p.first < groups; p.first += most_groups(threads))
      {  const uint64_t left = groups - p.first;
         hipLaunchKernelGGL(kernel, dim3((unsigned)(left < most_groups(threads) ? left : most_groups(threads))), dim3(threads), 0, stream, p);
         OCH_CHECK_LAUNCH();
      }
      return 0;
   };
   /* the rows with a workgroup of their own can be stored past the caches: 8192 rows of 8192 features 82.2 us against 84.8 */
   const uint64_t es = sizeof(typename Wide<DT>::E), values = (uint64_t)p.n * p.rows, ey = CODE == 0 ? es : 1;
   const bool nt = streams(p.Y, p.ldY * ey, values * ey) && (p.H == nullptr || streams(p.H, p.ldH * es, values * es));
#define OCH_GO(T, V) go(norm_kernel<DT, CODE, T, V, false>, norm_rows(T), T * norm_rows(T))
#define OCH_GO_NT(T, V) (nt ? go(norm_kernel<DT, CODE, T, V, true>, 1, T) : OCH_GO(T, V))
   if constexpr (CODE == 0) if (p.n <= 64) return OCH_GO(8, 1);          /* (codes: sixteen threads share a block's maximum) */
   if (p.n <= 128)   return OCH_GO(16, 1);
   if (p.n <= 256)   return OCH_GO(16, 2);
   if (p.n <= 512)   return OCH_GO(64, 1);
   if (p.n <= 1024)  return OCH_GO(64, 2);
   if (p.n <= 2048)  return OCH_GO_NT(256, 1);
   if (p.n <= 4096)  return OCH_GO_NT(256, 2);
   if (p.n <= 6144)  return OCH_GO_NT(256, 3);
   if (p.n <= 8192)  return OCH_GO_NT(512, 2);
   if (p.n <= 16384) return OCH_GO_NT(512, 4);
#undef OCH_GO_NT
#undef OCH_GO
   return go(norm_long_kernel<DT, CODE>, 1, OCH_NORM_THREADS);
}

/* ---- gradients ------------------------------------------------------------------------------------------------------ */
struct NormGradParams
{
   const char *dY, *H, *W, *dH; char *dX; const float *rstd; float *partial;   /* partial: n sums per workgroup, null when dW is not asked for */
   int64_t  lddY, ldH, lddH, lddX;
   int64_t  n, rows;
   float    inverse;                    /* 1 / n */
   int      w_float;
};

/* Rows of any length: workgroup b takes rows b, b + G, ... and keeps its sums for dw in its own n floats of the workspace
   (thread t always owns the same columns) */
template <int DT>
__global__ __launch_bounds__(OCH_NORM_THREADS) void norm_grad_long_kernel(const NormGradParams p)
{
   typedef typename Wide<DT>::E E;
   __shared__ float part[OCH_NORM_THREADS / 64];
   float *mine = p.partial ? p.partial + (int64_t)blockIdx.x * p.n : nullptr;
   for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x)
   {  const E *dy = reinterpret_cast<const E *>(p.dY) + row * p.lddY, *h = reinterpret_cast<const E *>(p.H) + row * p.ldH;
      const float rstd = p.rstd[row];
      float sum = 0;
      for (int64_t at = threadIdx.x * 8; at < p.n; at += OCH_NORM_THREADS * 8)
      {  Wide8<DT> a, b; float w[8], s = 0;
         a.load(dy + at, p.n - at); b.load(h + at, p.n - at);
         load_weights<DT>(p.W, p.w_float, at, p.n - at, w);
#pragma unroll
         for (int e = 0; e < 8; e++) s = __builtin_fmaf(a.get(e) * w[e], b.get(e) * rstd, s);
         sum += s;
      }
      const float mean = block_sum(sum, part) * p.inverse;
      for (int64_t at = threadIdx.x * 8; at < p.n; at += OCH_NORM_THREADS * 8)
      {  Wide8<DT> a, b, c, o; Wide8<OCH_FLOAT> d; float w[8];
         const int64_t valid = p.n - at;
         a.load(dy + at, valid); b.load(h + at, valid);
         if (p.dH) c.load(reinterpret_cast<const E *>(p.dH) + row * p.lddH + at, valid);
         load_weights<DT>(p.W, p.w_float, at, valid, w);
         if (mine && row != blockIdx.x) d.load(mine + at, valid);
         else
         {
#pragma unroll
            for (int e = 0; e < 8; e++) d.put(e, 0.0f);
         }
#pragma unroll
         for (int e = 0; e < 8; e++)
         {  const float u = b.get(e) * rstd;
            float x = rstd * (a.get(e) * w[e] - u * mean);
            if (p.dH) x += c.get(e);
            o.put(e, x);
            d.put(e, __builtin_fmaf(a.get(e), u, d.get(e)));
         }
         o.store(reinterpret_cast<E *>(p.dX) + row * p.lddX + at, valid);
         if (mine) d.store(mine + at, valid);
      }
   }
}

/* Rows of at most 8 T V elements: T threads keep a row in registers; a workgroup takes norm_rows(T) rows at a time,
   in steps of the grid, loads the next ones while it works, and its threads' sums for dw stay in registers until its last row;
   those of rows side by side meet in LDS then. 8192 rows of 4096 bfloat16 features with dh: 51.6 us (5.2 TB/s), 55.4 without
   the next row's loads; the second kernel's 3 us are part of it. */
template <int DT, int T, int V>
__global__ __launch_bounds__(T * norm_rows(T)) void norm_grad_kernel(const NormGradParams p)
{
   typedef typename Wide<DT>::E E;
   constexpr int ROWS = norm_rows(T);
   constexpr bool AHEAD = T < 1024;                         /* with 1024 threads there are not registers enough */
   __shared__ float part[T * ROWS / 64];
   __shared__ __align__(16) float meet[ROWS > 1 ? ROWS * T * V * 8 : 4];
   const int first = (int)(threadIdx.x % T) * 8, n = (int)p.n;
   float w[V][8], dw[V][8];
#pragma unroll
   for (int v = 0; v < V; v++)
   {  load_weights<DT>(p.W, p.w_float, first + v * T * 8, n - first - v * T * 8, w[v]);
#pragma unroll
      for (int e = 0; e < 8; e++) dw[v][e] = 0;
   }
   Wide8<DT> a[V], b[V], c[V];
   float rstd;
   bool live;
   int64_t row;
   /* the group's row of those that begin at row0 */
   auto load = [&](int64_t row0)
   {  const int64_t wanted = row0 + threadIdx.x / T;
      live = wanted < p.rows;
      row = live ? wanted : p.rows - 1;
#pragma unroll
      for (int v = 0; v < V; v++)
      {  const int at = first + v * T * 8, valid = (live ? n : 0) - at;
         a[v].load(reinterpret_cast<const E *>(p.dY) + row * p.lddY + at, valid);
         b[v].load(reinterpret_cast<const E *>(p.H) + row * p.ldH + at, valid);
         if (p.dH) c[v].load(reinterpret_cast<const E *>(p.dH) + row * p.lddH + at, valid);
      }
      rstd = p.rstd[row];
   };
   const int64_t step = (int64_t)gridDim.x * ROWS;
   int64_t row0 = (int64_t)blockIdx.x * ROWS;
   if (AHEAD && row0 < p.rows) load(row0);
   for (; row0 < p.rows; row0 += step)
   {  Wide8<DT> copy[3][AHEAD ? V : 1];                     /* this row; the next one's loads are under way beside it */
      const Wide8<DT> *dy = AHEAD ? copy[0] : a, *h = AHEAD ? copy[1] : b, *dh = AHEAD ? copy[2] : c;
      if (!AHEAD) load(row0);
      const float r = rstd;
      const int valid = live ? n : 0;
      E *to = reinterpret_cast<E *>(p.dX) + row * p.lddX;
      const bool mine = live;
      if (AHEAD)
      {
#pragma unroll
         for (int v = 0; v < V; v++) { copy[0][AHEAD ? v : 0] = a[v]; copy[1][AHEAD ? v : 0] = b[v]; copy[2][AHEAD ? v : 0] = c[v]; }
      }
      if (AHEAD && row0 + step < p.rows) load(row0 + step);
      float sum = 0;
#pragma unroll
      for (int v = 0; v < V; v++)
      {  float s = 0;
#pragma unroll
         for (int e = 0; e < 8; e++) s = __builtin_fmaf(dy[v].get(e) * w[v][e], h[v].get(e) * r, s);
         sum += s;
      }
      const float mean = group_sum<T>(sum, part) * p.inverse;
#pragma unroll
      for (int v = 0; v < V; v++)
      {  const int at = first + v * T * 8;
         Wide8<DT> o;
#pragma unroll
         for (int e = 0; e < 8; e++)
         {  const float u = h[v].get(e) * r;
            float x = r * (dy[v].get(e) * w[v][e] - u * mean);
            if (p.dH) x += dh[v].get(e);
            o.put(e, x);
            dw[v][e] = __builtin_fmaf(dy[v].get(e), mine ? u : 0.0f, dw[v][e]);
         }
         o.store(to + at, valid - at);
      }
   }
   if (p.partial == nullptr) return;
   if (ROWS > 1)
   {  float *mine = meet + threadIdx.x / T * (T * V * 8);
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int e = 0; e < 8; e++) mine[first + v * T * 8 + e] = dw[v][e];
      __syncthreads();
      if (threadIdx.x >= T) return;
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
         for (int e = 0; e < 8; e++)
         {  float s = 0;
            for (int g = 0; g < ROWS; g++) s += meet[g * (T * V * 8) + first + v * T * 8 + e];
            dw[v][e] = s;
         }
   }
   float *to = p.partial + (int64_t)blockIdx.x * p.n;
#pragma unroll
   for (int v = 0; v < V; v++)
   {  Wide8<OCH_FLOAT> d;
#pragma unroll
      for (int e = 0; e < 8; e++) d.put(e, dw[v][e]);
      d.store(to + first + v * T * 8, n - first - v * T * 8);
   }
}

/* dw: the workgroups' sums, added in a fixed order: sixteen threads per column take every sixteenth workgroup, their sums
   meet in LDS */
__global__ __launch_bounds__(1024) void norm_grad_finish_kernel(const float *partial, int64_t n, uint32_t groups, float *dW)
{
   __shared__ float meet[16][64];
   const uint32_t lane = threadIdx.x % 64, slice = threadIdx.x / 64;
   const int64_t at = (int64_t)blockIdx.x * 64 + lane;
   float s = 0;
   if (at < n)
   {  uint32_t g = slice;
      for (; g + 7 * 16 < groups; g += 8 * 16)
      {  float v[8];
#pragma unroll
         for (int u = 0; u < 8; u++) v[u] = partial[(int64_t)(g + 16 * u) * n + at];
#pragma unroll
         for (int u = 0; u < 8; u++) s += v[u];
      }
      for (; g < groups; g += 16) s += partial[(int64_t)g * n + at];
   }
   meet[slice][lane] = s;
   __syncthreads();
   if (slice != 0 || at >= n) return;
   for (int k = 1; k < 16; k++) s += meet[k][lane];
   dW[at] = s;
}

/* Workgroups: each costs n floats written and read again for dw, so as few as keep the memory busy. 2^25 bfloat16 values with
   dw: 8192 features 53.5 us with one per compute unit, 57.3 with two, 64.0 with four; 2048 features 68.2, 51.4,
   57.0; 256 features, sixteen threads a row, 52.8 with two, 58.3 with four; 64 features 51.6 with eight threads a row, 133 with
   sixteen. */
template <int DT> static int norm_grad_launch(NormGradParams p, float *dW, hipStream_t stream)
{
   const int rows_at_once = norm_rows(p.n <= 64 ? 8 : p.n <= 256 ? 16 : p.n <= 1024 ? 64 : OCH_NORM_THREADS);
   uint64_t groups = (p.n <= 2048 ? 2 : 1) * (uint64_t)gemm_compute_units();
   if (groups > ((uint64_t)p.rows + rows_at_once - 1) / rows_at_once) groups = ((uint64_t)p.rows + rows_at_once - 1) / rows_at_once;
   p.partial = nullptr;
   if (dW)
   {  const uint64_t fit = OCH_GEMM_WORKSPACE / ((uint64_t)p.n * sizeof(float));
      char *ws;
      if (fit == 0) return set_error("rms_norm_grad: rows of %lld features are too long for the weights' gradient", (long long)p.n);
      if (groups > fit) groups = fit;
      if (stream_gemm_workspace(stream, &ws) != 0) return -1;
      p.partial = reinterpret_cast<float *>(ws);
   }
#define OCH_GO(T, V) hipLaunchKernelGGL((norm_grad_kernel<DT, T, V>), dim3((unsigned)groups), dim3(T * norm_rows(T)), 0, stream, p)
   if (p.n <= 64)         OCH_GO(8, 1);
   else if (p.n <= 128)   OCH_GO(16, 1);
   else if (p.n <= 256)   OCH_GO(16, 2);
   else if (p.n <= 512)   OCH_GO(64, 1);
   else if (p.n <= 1024)  OCH_GO(64, 2);
   else if (p.n <= 2048)  OCH_GO(256, 1);
   else if (p.n <= 4096)  OCH_GO(256, 2);
   else if (p.n <= 6144)  OCH_GO(256, 3);
   else if (p.n <= 8192)  OCH_GO(512, 2);
   else if (p.n <= 16384) OCH_GO(1024, 2);
   else hipLaunchKernelGGL((norm_grad_long_kernel<DT>), dim3((unsigned)groups), dim3(OCH_NORM_THREADS), 0, stream, p);
#undef OCH_GO
   OCH_CHECK_LAUNCH();
   if (dW)
   {  hipLaunchKernelGGL(norm_grad_finish_kernel, dim3((unsigned)((p.n + 63) / 64)), dim3(1024), 0, stream, p.partial, p.n, (uint32_t)groups, dW);
      OCH_CHECK_LAUNCH();
   }
   return 0;
}

static int check_weights(const char *name, int dtype, int dtype_w, const void *W)
{
   if (W == nullptr) return 0;
   if (dtype_w != dtype && dtype_w != OCH_FLOAT) return set_error("%s: the weights are float or of the input's type (got %d)", name, dtype_w);
   if ((uintptr_t)W % wide_size(dtype_w) != 0) return set_error("%s: misaligned pointer", name);
   return 0;
}

} /* namespace och */

using namespace och;

extern "C" int och_rms_norm(int dtype, size_t n, size_t rows, const void *X, ptrdiff_t ldX, const void *R, ptrdiff_t ldR, void *H, ptrdiff_t ldH,
                            int dtype_w, const void *W, float eps, int dtype_y, void *Y, ptrdiff_t ldY, float *S, ptrdiff_t ldS, float *rstd, och_stream stream)
{
   if (!wide_type(dtype)) return set_error("rms_norm is available for half, bfloat16 and float (got %d)", dtype);
   if (dtype_y != dtype && !code_type(dtype_y)) return set_error("rms_norm: the output has the input's type, float8_e4m3 or float8_e5m2 (got %d)", dtype_y);
   if (!(eps >= 0.0f)) return set_error("rms_norm: eps is negative or not a number");
   const bool code = dtype_y != dtype;
   if (n == 0 || rows == 0) return 0;
   if (n > 0x7FFFFFFFull || rows > 0x7FFFFFFFull) return set_error("rms_norm: a side of %zu elements is too long", n > rows ? n : rows);
   if (X == nullptr || Y == nullptr || (R != nullptr && H == nullptr) || (code && S == nullptr)) return set_error("rms_norm: null pointer argument");
   const size_t blocks = (n + OCH_F8_BLOCK - 1) / OCH_F8_BLOCK;
   if (ldX < (ptrdiff_t)n || ldY < (ptrdiff_t)n || (R && ldR < (ptrdiff_t)n) || (H && ldH < (ptrdiff_t)n) || (code && ldS < (ptrdiff_t)blocks))
      return set_error("rms_norm: a leading dimension is smaller than the row (n = %zu)", n);
   if (check_weights("rms_norm", dtype, dtype_w, W) != 0) return -1;
   const size_t es = wide_size(dtype);
   if ((uintptr_t)X % es || (uintptr_t)R % es || (uintptr_t)H % es || (!code && (uintptr_t)Y % es) || (uintptr_t)S % 4 || (uintptr_t)rstd % 4)
      return set_error("rms_norm: misaligned pointer");
   if (H != nullptr && ((H == X && ldH != ldX) || (H == R && ldH != ldR))) return set_error("rms_norm: a sum in place needs its operand's leading dimension");
   if (Y == X && (code || R != nullptr || ldY != ldX)) return set_error("rms_norm: the output can take X's place only without a residual, in X's type and with its leading dimension");
   NormParams p;
   p.X = (const char *)X; p.R = (const char *)R; p.W = (const char *)W; p.H = (char *)H; p.Y = (char *)Y; p.S = S; p.rstd = rstd;
   p.ldX = ldX; p.ldR = ldR; p.ldH = ldH; p.ldY = ldY; p.ldS = ldS; p.n = (int64_t)n; p.rows = (int64_t)rows; p.eps = eps; p.inverse = 1.0f / (float)n; p.w_float = (dtype_w == OCH_FLOAT);
   hipStream_t s = as_stream(stream);
#define OCH_GO(DT) (!code ? norm_launch<DT, 0>(p, s) : dtype_y == OCH_FLOAT8_E4M3 ? norm_launch<DT, OCH_FLOAT8_E4M3>(p, s) : norm_launch<DT, OCH_FLOAT8_E5M2>(p, s))
   return OCH_BY_WIDE(dtype, OCH_GO);
#undef OCH_GO
}

extern "C" int och_rms_norm_grad(int dtype, size_t n, size_t rows, const void *dY, ptrdiff_t lddY, const void *H, ptrdiff_t ldH, const float *rstd,
                                 int dtype_w, const void *W, const void *dH, ptrdiff_t lddH, void *dX, ptrdiff_t lddX, float *dW, och_stream stream)
{
   if (!wide_type(dtype)) return set_error("rms_norm_grad is available for half, bfloat16 and float (got %d)", dtype);
   if (n == 0) return 0;
   if (n > 0x7FFFFFFFull || rows > 0x7FFFFFFFull) return set_error("rms_norm_grad: a side of %zu elements is too long", n > rows ? n : rows);
   if (check_weights("rms_norm_grad", dtype, dtype_w, W) != 0) return -1;
   if ((uintptr_t)dW % 4) return set_error("rms_norm_grad: misaligned pointer");
   if (rows == 0) return dW ? fill_bytes(dW, 0, n * sizeof(float), as_stream(stream)) : 0;      /* a sum over nothing */
   if (dY == nullptr || H == nullptr || rstd == nullptr || dX == nullptr) return set_error("rms_norm_grad: null pointer argument");
   if (lddY < (ptrdiff_t)n || ldH < (ptrdiff_t)n || lddX < (ptrdiff_t)n || (dH && lddH < (ptrdiff_t)n))
      return set_error("rms_norm_grad: a leading dimension is smaller than the row (n = %zu)", n);
   const size_t es = wide_size(dtype);
   if ((uintptr_t)dY % es || (uintptr_t)H % es || (uintptr_t)dH % es || (uintptr_t)dX % es || (uintptr_t)rstd % 4) return set_error("rms_norm_grad: misaligned pointer");
   if ((dX == dY && lddX != lddY) || (dX == dH && lddX != lddH)) return set_error("rms_norm_grad: dX in the place of dY or dH needs its leading dimension");
   NormGradParams p;
   p.dY = (const char *)dY; p.H = (const char *)H; p.W = (const char *)W; p.dH = (const char *)dH; p.dX = (char *)dX; p.rstd = rstd; p.partial = nullptr;
   p.lddY = lddY; p.ldH = ldH; p.lddH = lddH; p.lddX = lddX; p.n = (int64_t)n; p.rows = (int64_t)rows; p.inverse = 1.0f / (float)n; p.w_float = (dtype_w == OCH_FLOAT);
#define OCH_GO(DT) norm_grad_launch<DT>(p, dW, as_stream(stream))
   return OCH_BY_WIDE(dtype, OCH_GO);
#undef OCH_GO
}
