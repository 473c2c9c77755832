/* The block-scaled product on tiles of 128 x 128 for any operands: whatever their alignment, sizes and scales.
 *
 * Four waves own 64 x 64 of the tile each. A slab of 128 k of both operands and the slab's scales pass through registers
 * to one of two LDS buffers: the loads of slab s + 1 are issued before the matrix instructions of slab s and stored behind
 * them, one barrier per slab, two workgroups per compute unit. Chunks of 16 bytes are single loads whatever their
 * alignment; at the matrix's border they are put together from two that overlap.
 *
 * PAIR: where there are no more tiles than compute units, two groups of four waves share a tile, each with its half of K and
 * LDS of its own, as two workgroups would; their sums meet in LDS. The groups have their barriers in common, which is why every
 * slab but the last of K has to be pipelined. 2048 x 2048 x 4096 to bfloat16 40 -> 28.5 us, to float 57 -> 41; 1024^3 13.5 -> 10.2.
 *
 * ROWS: the scale of A differs between the rows of a wave (blockA = 1): a multiplication more per element and slab.
 *
 * A wave that multiplies goes before one that loads, stores or waits on the same SIMD, and the loads are issued in the first
 * row's step, behind the reads of the first fragments. 4096^3 to float: 156 -> 149 us with both operands contiguous along their
 * rows, 148 -> 133 contiguous along k with one scale of A per 128 rows; 4096 x 4096 x 4100, unaligned, to bfloat16 117 -> 112.
 *
 * Float results, 4096 x 5000 x 4001 with both operands contiguous along their rows: 205 us, 0.80 PFLOP/s; unaligned 11136 x
 * 2832 x 8716 to bfloat16: 477 us, 1.2 PFLOP/s. With float results a slab takes a wave about 4200 cycles, 1024 of them in
 * matrix instructions: 600 go into issuing its loads, 400 into B's fragments, 4 x 560 into the rows, whose conversions and
 * scaling are 1024 cycles of vector instructions, 900 into waiting for the loads and storing them. Loads and stores spread
 * over the rows gain nothing, 256 x 128 tiles filled straight from memory 8 % on full rounds: with two workgroups per unit the
 * clock falls from 1.9 to 1.5 GHz, power bounds it. */
#pragma once
#include "och_gemm_f8.h"

namespace och {

#define OCH_F8_TILE 128
#define OCH_F8_TILE_THREADS 256

/* Order of the tiles: workgroups go to the eight compute dies in turn, each with a cache of its own, so every die gets a
   contiguous run of tiles; inside the run tiles advance in strips of eight rows of tiles, so that the tiles of a die that
   are in flight together share operands */
__device__ __forceinline__ void f8_tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t &tm, uint32_t &tn)
{
   const uint32_t total = tiles_m * tiles_n, q = total / 8, r = total % 8, die = id % 8;
   id = die * q + (die < r ? die : r) + id / 8;
   const uint32_t strip = id / (8 * tiles_n), first = strip * 8, height = tiles_m - first < 8 ? tiles_m - first : 8, in = id - first * tiles_n;
   tm = first + in % height; tn = in / height;
}

typedef uint64_t f8_u64_any __attribute__((aligned(1)));
typedef uint32_t f8_u32_any __attribute__((aligned(1)));
static __device__ __forceinline__ och_u32x4 f8_pair(uint64_t lo, uint64_t hi)
{  och_u32x4 v;
   v.x = (uint32_t)lo; v.y = (uint32_t)(lo >> 32); v.z = (uint32_t)hi; v.w = (uint32_t)(hi >> 32);
   return v;
}
/* 16 bytes moved towards their start by `by` bytes (16 or more: zero), zeros behind */
static __device__ __forceinline__ och_u32x4 f8_shift(och_u32x4 v, uint32_t by)
{  uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
   const uint32_t bits = 8 * (by & 7);
   if (by & 8) { lo = hi; hi = 0; }
   lo = bits ? (lo >> bits | hi << (64 - bits)) : lo;
   hi >>= bits;
   if (by >= 16) lo = hi = 0;
   return f8_pair(lo, hi);
}
/* a chunk of which the first `valid` bytes exist (none when valid <= 0), the others zero; `length`: bytes of the run of
   memory that it ends (from 16 on, the 16 bytes up to its end are one load) */
static __device__ __forceinline__ och_u32x4 f8_border_chunk(const uint8_t *at, int64_t valid, uint32_t length)
{
   och_u32x4 v = { 0, 0, 0, 0 };
   if (valid >= 16) v = *reinterpret_cast<const och_u32x4_any *>(at);
   else if (valid > 0 && length >= 16) v = f8_shift(*reinterpret_cast<const och_u32x4_any *>(at + valid - 16), (uint32_t)(16 - valid));
   else if (valid >= 8)
   {  const uint64_t lo = *reinterpret_cast<const f8_u64_any *>(at), hi = *reinterpret_cast<const f8_u64_any *>(at + valid - 8);
      v = f8_pair(lo, valid > 8 ? hi >> (64 - 8 * (uint32_t)(valid - 8)) : 0);
   }
   else if (valid >= 4)
   {  const uint64_t lo = *reinterpret_cast<const f8_u32_any *>(at), hi = *reinterpret_cast<const f8_u32_any *>(at + valid - 4);
      v = f8_pair(lo | hi >> (32 - 8 * (uint32_t)(valid - 4)) << 32, 0);
   }
   else if (valid > 0)
   {  const uint32_t half = (uint32_t)valid / 2, last = (uint32_t)valid - 1;      /* the first, the second or last, the last */
      v.x = at[0] | (uint32_t)at[half] << 8 * half | (uint32_t)at[last] << 8 * last;
   }
   return v;
}

/* chunk q of a slab, wherever it lies with respect to the matrix's ends */
template <bool KC, int R> static __device__ __forceinline__ och_u32x4 f8_any_chunk(const uint8_t *mat, int64_t ld, uint32_t r0, uint32_t k0, uint32_t rows, uint32_t K, uint32_t q)
{  uint32_t row, k;
   F8Slab<KC, R>::where(q, row, k);
   const int64_t gr = (int64_t)r0 + row, gk = (int64_t)k0 + k;
   const int64_t valid = KC ? (gr < rows ? (int64_t)K - gk : 0) : (gk < K ? (int64_t)rows - gr : 0);
   return f8_border_chunk(mat + (KC ? gk + gr * ld : gr + gk * ld), valid, KC ? K : rows);
}

/* The chunks that thread t of THREADS moves: t + THREADS i of every slab. They differ by whole rows (KC) or whole k (!KC)
   with the same twist. Rows that do not exist are never loaded: KC repeats the last row instead; !KC loads the last 16
   rows where a chunk passes the end, and moves them into place on the way to LDS (so `rows` is at least 16 there). What
   these lanes hold for rows outside the matrix reaches only elements of C that are not written. */
template <bool KC, int R, int THREADS> struct F8Stage
{
   typedef F8Slab<KC, R> L;
   static constexpr int NV = (int)L::CHUNKS / THREADS;
   static constexpr uint32_t STEP = KC ? THREADS / 8 : THREADS / L::PER_K;       /* rows or k from a thread's chunk to its next */
   static_assert(STEP % 8 == 0, "the twist must not change from chunk to chunk");
   och_u32x4 v[NV];
   const uint8_t *slab;                  /* the next slab's first element: the same for all threads */
   uint32_t offset, most, move;          /* of the thread's first chunk from there, and (KC) of the same k of the last row; rows that a chunk is moved by */
   /* offsets within a slab are counted in 32 bits */
   static __device__ __forceinline__ bool pipelined(uint32_t rows, int64_t ld) { return (KC || rows >= 16) && ld < (1 << 24); }
   __device__ __forceinline__ void start(const uint8_t *mat, int64_t ld, uint32_t r0, uint32_t k0, uint32_t rows)
   {  uint32_t row, k;
      L::where(threadIdx.x % THREADS, row, k);
      slab = mat + (KC ? (int64_t)k0 + (int64_t)r0 * ld : (int64_t)r0 + (int64_t)k0 * ld);
      const uint32_t last = rows - r0 < R ? rows - r0 - 1 : R - 1;        /* the tile's last row */
      move = 0;
      most = last * (uint32_t)ld + k;
      if (KC) offset = row * (uint32_t)ld + k;
      else
      {  const int32_t from = (int32_t)row < (int32_t)last - 15 ? (int32_t)row : (int32_t)last - 15;      /* below zero: the chunk begins in front of the tile */
         slab -= 16;
         offset = (uint32_t)(from + 16) + k * (uint32_t)ld;
         move = (uint32_t)((int32_t)row - from);
      }
   }
   /* the next slab, whole along k */
   __device__ __forceinline__ void load(int64_t ld)
   {
#pragma unroll
      for (int i = 0; i < NV; i++)
      {  const uint32_t o = offset + i * STEP * (uint32_t)ld;
         v[i] = *reinterpret_cast<const och_u32x4_any *>(KC ? slab + (o < most ? o : most) : slab + i * (int64_t)STEP * ld + offset);
      }
      slab += KC ? OCH_F8_SLAB : OCH_F8_SLAB * ld;
   }
   /* any slab, chunk by chunk */
   __device__ __forceinline__ void load_border(const uint8_t *mat, int64_t ld, uint32_t r0, uint32_t k0, uint32_t rows, uint32_t K)
   {  move = 0;
      uint32_t thread = threadIdx.x % THREADS;
      asm volatile("" : "+v"(thread));   /* what follows from it is computed here, not kept in registers through the pipelined slabs */
#pragma unroll
      for (int i = 0; i < NV; i++) v[i] = f8_any_chunk<KC, R>(mat, ld, r0, k0, rows, K, thread + THREADS * i);
   }
   __device__ __forceinline__ void store(char *slab, bool border)
   {
#pragma unroll
      for (int i = 0; i < NV; i++)
      {  if (!KC && border) v[i] = f8_shift(v[i], move);
         *reinterpret_cast<och_u32x4 *>(slab + 16 * (threadIdx.x % THREADS + THREADS * i)) = v[i];
      }
   }
};

/* four neighbouring rows of one column of C */
template <int DT> __device__ __forceinline__ void f8_finish4(char *C, int64_t at, och_f32x4v s, float alpha, float beta, uint32_t valid)
{
   typedef typename Wide<DT>::E E;
   typedef E E4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));
   E *c = reinterpret_cast<E *>(C) + at;
   if (valid >= 4)
   {  E4 o;
      if (beta != 0.0f)
      {  const E4 old = *reinterpret_cast<const E4 *>(c);
#pragma unroll
         for (int r = 0; r < 4; r++) o[r] = Wide<DT>::put(__builtin_fmaf(beta, Wide<DT>::get(old[r]), alpha * s[r]));
      }
      else
      {
#pragma unroll
         for (int r = 0; r < 4; r++) o[r] = Wide<DT>::put(alpha * s[r]);
      }
      *reinterpret_cast<E4 *>(c) = o;
   }
   else
   {
#pragma unroll
      for (int r = 0; r < 3; r++) if ((uint32_t)r < valid) f8_finish<DT>(C, at + r, s[r], alpha, beta);
   }
}
/* COLUMNS columns of R rows of sums from LDS (PITCH bytes from column to column) to C, eight rows of a column at a time: memory
   sees runs of R elements */
template <int DT, int R, uint32_t PITCH, uint32_t COLUMNS, int THREADS> __device__ __forceinline__ void f8_store_columns(const F8GemmParams &p, const char *lds, uint32_t m0, uint32_t n0)
{
   typedef typename Wide<DT>::E E;
#pragma unroll 1
   for (uint32_t q = threadIdx.x; q < COLUMNS * (R / 8); q += THREADS)
   {  const uint32_t c = q / (R / 8), m = m0 + q % (R / 8) * 8, n = n0 + c;
      if (m >= p.M || n >= p.N) continue;
      const och_f32x4v *from = reinterpret_cast<const och_f32x4v *>(lds + c * PITCH + q % (R / 8) * 32);
      const och_f32x4v lo = from[0], hi = from[1];
      E *to = reinterpret_cast<E *>(p.C) + (int64_t)m + (int64_t)n * p.ldC;
      const int64_t valid = (int64_t)p.M - m;
      Wide8<DT> v;
      if (p.beta != 0.0f) v.load(to, valid);
#pragma unroll
      for (int e = 0; e < 8; e++)
      {  float x = p.alpha * (e < 4 ? lo[e % 4] : hi[e % 4]);
         if (p.beta != 0.0f) x = __builtin_fmaf(p.beta, v.get(e), x);
         v.put(e, x);
      }
      v.store(to, valid);
   }
}

template <bool AKC, bool BKC, bool E5A, bool E5B, bool WIDE, bool ROWS, bool PAIR>
__global__ __launch_bounds__(OCH_F8_TILE_THREADS * (PAIR ? 2 : 1), 2) void gemm_f8_tile_kernel(const F8GemmParams p)
{
   constexpr int R = OCH_F8_TILE, THREADS = OCH_F8_TILE_THREADS, OPERAND = R * OCH_F8_SLAB, BUF = 2 * OPERAND + 2 * R * 4;
   __shared__ __align__(16) char all_lds[(PAIR ? 4 : 2) * BUF];
   const uint32_t thread = threadIdx.x % THREADS, group = PAIR ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : 0;
   char *const lds = all_lds + group * (2 * BUF);
   uint32_t tm, tn;
   f8_tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
   const uint32_t m0 = tm * R, n0 = tn * R;
   const uint32_t lane = threadIdx.x & 63, wave = PAIR ? __builtin_amdgcn_readfirstlane(thread >> 6) : thread >> 6, wm = wave % 2 * 64, wn = wave / 2 * 64;
   const och_f32x4v zero = { 0, 0, 0, 0 };
   och_f32x4v acc[4][4];
#pragma unroll
   for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) acc[i][j] = zero;

   const uint32_t all = (p.K + OCH_F8_SLAB - 1) / OCH_F8_SLAB;
   uint32_t s = 0, end = all;
   if (p.share_slabs) { s = blockIdx.y * p.share_slabs; end = s + p.share_slabs < all ? s + p.share_slabs : all; }
   const uint32_t whole = p.K / OCH_F8_SLAB;
   uint32_t turns = end - s, rest = ~0u;                     /* rest: the turn in which one of the groups takes the slab inside which K ends */
   if (PAIR)
   {  const uint32_t half = (turns + 1) / 2, second = s + half;
      if (end > whole) rest = whole - (end > second ? second : s);
      if (group == 0) end = second; else s = second;         /* the second group may have one slab less */
      turns = half;
   }

   /* every thread brings one scale: waves 0 and 1 of A's rows, 2 and 3 of B's columns; those outside C repeat the last */
   const bool forA = __builtin_amdgcn_readfirstlane(wave) < 2;
   const uint32_t line = thread % R, most = (forA ? p.M - m0 : p.N - n0) - 1, shift = forA ? p.shiftA : p.shiftB, begin = forA ? m0 : n0;
   const uint32_t scale_of = ((begin + (line < most ? line : most)) >> shift) - (begin >> shift);
   const int64_t scale_line = forA ? p.sa_m : p.sb_n, scale_step = forA ? p.sa_k : p.sb_k;
   const float *scale = (forA ? p.SA : p.SB) + (int64_t)(begin >> shift) * scale_line + (int64_t)s * scale_step;
   auto next_scale = [&]() { const float x = scale[(int64_t)scale_of * scale_line]; scale += scale_step; return x; };

   /* slabs that are whole along k are pipelined; the rest of K, and everything of an operand of under 16 contiguous rows or
      of columns 16 MB apart, is not */
   const uint32_t piped = !F8Stage<AKC, R, THREADS>::pipelined(p.M, p.ldA) || !F8Stage<BKC, R, THREADS>::pipelined(p.N, p.ldB) ? s : end < whole ? end : whole;
   const bool borderA = m0 + R > p.M, borderB = n0 + R > p.N;
   F8Stage<AKC, R, THREADS> la; F8Stage<BKC, R, THREADS> lb; float ls = 0;
   la.start(p.A, p.ldA, m0, s * OCH_F8_SLAB, p.M); lb.start(p.B, p.ldB, n0, s * OCH_F8_SLAB, p.N);
   auto stash = [&](char *buf)
   {  la.store(buf, borderA); lb.store(buf + OPERAND, borderB);
      reinterpret_cast<float *>(buf + 2 * OPERAND)[thread] = ls;
   };
   if (s < piped)
   {  la.load(p.ldA); lb.load(p.ldB); ls = next_scale();
      stash(lds);
   }
   __syncthreads();
   for (uint32_t round = 0; round < turns; round++, s++)
   {  const uint32_t turn = round & 1;
      char *buf = lds + turn * BUF;
      const float *sA = reinterpret_cast<const float *>(buf + 2 * OPERAND), *sB = sA + R;
      if (PAIR ? round == rest : s >= piped)
      {  if (!PAIR || (s >= piped && s < end))
         {  la.load_border(p.A, p.ldA, m0, s * OCH_F8_SLAB, p.M, p.K); lb.load_border(p.B, p.ldB, n0, s * OCH_F8_SLAB, p.N, p.K); ls = next_scale();
            stash(buf);
         }
         __syncthreads();
      }
      if (PAIR && s >= end) { __syncthreads(); continue; }
      const bool more = s + 1 < piped;
      F8Operand<WIDE> b[4]; float t[4];
      {  och_i32x8 c[4];
#pragma unroll
         for (int j = 0; j < 4; j++) { c[j] = f8_fragment<BKC, R>(buf + OPERAND, wn + 16 * j); t[j] = sB[wn + 16 * j + lane % 16]; }
         const float whole_a = ROWS ? 1.0f : sA[wm];
         __builtin_amdgcn_sched_barrier(0);
#pragma unroll
         for (int j = 0; j < 4; j++)
         {  b[j].template set<E5B>(c[j]);
            if (!ROWS) t[j] *= whole_a;
            __builtin_amdgcn_sched_barrier(0);
         }
      }
      __builtin_amdgcn_s_setprio(1);
      /* step i: row i is multiplied while the sums of row i - 1 are scaled and added and the fragment of row i + 1 is read
         and made an operand. The fences keep the compiler from collecting more rows than registers hold. */
      F8Operand<WIDE> a;
      a.template set<E5A>(f8_fragment<AKC, R>(buf, wm));
      och_f32x4v part[2][4];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i <= 4; i++)
      {  och_i32x8 codes; F8Operand<WIDE> next = a; och_f32x4v rs;
         if (ROWS && i > 0) rs = *reinterpret_cast<const och_f32x4v *>(sA + wm + 16 * (i > 0 ? i - 1 : 0) + 4 * (lane / 16));
         if (i < 3) codes = f8_fragment<AKC, R>(buf, wm + 16 * (i + 1));
         if (i == 0 && more) { la.load(p.ldA); lb.load(p.ldB); ls = next_scale(); }
         if (i < 4)
            f8_row<E5A, E5B, 4>(a, b, part[i % 2]);
         if (i > 0)
         {  const int o = (i - 1) % 2, q = i > 0 ? i - 1 : 0;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
               for (int r = 0; r < 4; r++) acc[q][j][r] = __builtin_fmaf(part[o][j][r], ROWS ? rs[r] * t[j] : t[j], acc[q][j][r]);
#pragma unroll
            for (int j = 0; j < 4; j++) asm volatile("" : "+v"(acc[q][j]));      /* here, not behind the loop's last branch */
         }
         if (i < 3) next.template set<E5A>(codes);
         if (i < 4)
         {  /* matrix instructions and the vector instructions of their time in turn */
            constexpr int N = WIDE ? 16 : 4;
#pragma unroll
            for (int x = 0; x < N; x++)
            {  __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
               __builtin_amdgcn_sched_group_barrier(0x2, WIDE ? (ROWS ? 3 : 2) : (ROWS ? 8 : 4), 0);
            }
         }
         a = next;
         __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (more) stash(lds + (turn ^ 1) * BUF);
      __syncthreads();
   }
   /* the tile leaves through LDS, where the slabs were; a share of K as raw sums into the share's plane */
   constexpr uint32_t PITCH = R * 4 + 16;
   static_assert(R * PITCH <= 2 * BUF, "the tile fits where the slabs were");
   char *const mine = lds + (wn + lane % 16) * PITCH + (wm + 4 * (lane / 16)) * 4;
   auto put = [&]()
   {
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
         for (int i = 0; i < 4; i++) *reinterpret_cast<och_f32x4v *>(mine + 16 * j * PITCH + 64 * i) = acc[i][j];
   };
   if (PAIR)
   {  if (group == 1) put();
      __syncthreads();
      if (group == 0)
      {
#pragma unroll
         for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i][j] += *reinterpret_cast<const och_f32x4v *>(mine + 2 * BUF + 16 * j * PITCH + 64 * i);
      }
   }
   if (group == 0) put();
   __syncthreads();
   if (p.share_slabs)
   {  F8GemmParams q = p;
      q.ldC = f8_plane_pitch(p.M); q.C = reinterpret_cast<char *>(p.partial + (size_t)blockIdx.y * q.ldC * p.N); q.alpha = 1.0f; q.beta = 0.0f;
      f8_store_columns<OCH_FLOAT, R, PITCH, R, THREADS * (PAIR ? 2 : 1)>(q, all_lds, m0, n0);
   }
   else if (WIDE)                 f8_store_columns<OCH_FLOAT, R, PITCH, R, THREADS * (PAIR ? 2 : 1)>(p, all_lds, m0, n0);
   else if (p.dtypeC == OCH_HALF) f8_store_columns<OCH_HALF, R, PITCH, R, THREADS * (PAIR ? 2 : 1)>(p, all_lds, m0, n0);
   else                           f8_store_columns<OCH_BFLOAT16, R, PITCH, R, THREADS * (PAIR ? 2 : 1)>(p, all_lds, m0, n0);
}

template <bool E5A, bool E5B, bool WIDE, bool ROWS, bool PAIR> static int gemm_f8_tile_launch(const F8GemmParams &p, bool akc, bool bkc, dim3 grid, hipStream_t stream)
{
   const dim3 block(OCH_F8_TILE_THREADS * (PAIR ? 2 : 1));
   if (akc && bkc) hipLaunchKernelGGL((gemm_f8_tile_kernel<true, true, E5A, E5B, WIDE, ROWS, PAIR>), grid, block, 0, stream, p);
   else if (akc)   hipLaunchKernelGGL((gemm_f8_tile_kernel<true, false, E5A, E5B, WIDE, ROWS, PAIR>), grid, block, 0, stream, p);
   else if (bkc)   hipLaunchKernelGGL((gemm_f8_tile_kernel<false, true, E5A, E5B, WIDE, ROWS, PAIR>), grid, block, 0, stream, p);
   else            hipLaunchKernelGGL((gemm_f8_tile_kernel<false, false, E5A, E5B, WIDE, ROWS, PAIR>), grid, block, 0, stream, p);
   OCH_CHECK_LAUNCH();
   return 0;
}
template <bool E5A, bool E5B> static int gemm_f8_tile(const F8GemmParams &p, bool akc, bool bkc, bool pair, dim3 grid, hipStream_t stream)
{
   const bool wide = p.dtypeC == OCH_FLOAT, rows = p.shiftA == 0;
#define OCH_GO(WIDE, ROWS) (pair ? gemm_f8_tile_launch<E5A, E5B, WIDE, ROWS, true>(p, akc, bkc, grid, stream) : gemm_f8_tile_launch<E5A, E5B, WIDE, ROWS, false>(p, akc, bkc, grid, stream))
   return wide ? (rows ? OCH_GO(true, true) : OCH_GO(true, false)) : (rows ? OCH_GO(false, true) : OCH_GO(false, false));
#undef OCH_GO
}

} /* namespace och */
