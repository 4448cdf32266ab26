// Operators of the head over many positions, for gfx950: the cross entropy of hidden rows against a
// head's rows, its gradients, the rounding of rows to 8-bit integers and the product of such rows.
// None of their kernels waits for another workgroup; they may run beside anything.
#include <hip/hip_runtime.h>
#include <cstdint>
#include <tuple>
#include <type_traits>
#include <utility>

#include "qwen_megakernel.h"

#include "head_gemm.inc"

namespace hd {

constexpr int CUS = 256;
constexpr long CACHES = 32L << 20;  // the XCDs' L2 caches together
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

// targets as the caller holds them: 32- or 64-bit integers
struct Targets {
  const void* p;
  int wide;
  long long ignore;
  __device__ __forceinline__ long long operator[](int t) const {
    return wide ? ((const long long*)p)[t] : (long long)((const int*)p)[t];
  }
};

// the upstream gradient of each position: g[t stride], over *divisor where there is one
struct Upstream {
  const float* g;
  long stride;
  const float* divisor;
  __device__ __forceinline__ float operator[](int t) const {
    const float x = g[t * stride];
    if (!divisor) return x;
    const float d = *divisor;
    return d == 0.f ? 0.f : x / d;  // (a mean of no positions: none has a gradient)
  }
};

// ---- forward: running softmax statistics over the vocabulary ---------------------------

// First workgroup whose share of `items` holds item x, of `grid` (run_product's deal)
__host__ __device__ inline int owner(long x, long items, long grid) { return (int)(((x + 1) * grid - 1) / items); }

// Rows past the end of the head: logits of -inf, whose exponentials are 0
template <class C>
__device__ __forceinline__ void mask_rows(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, int lane, int wn, int rows) {
  const int n0 = at.tn * C::BN + 32 * C::NI * wn;
  if (n0 + 32 * C::NI <= rows) return;
  int left = rows - n0 - 4 * (lane >> 5);
#pragma unroll
  for (int j = 0; j < C::NJ; ++j)
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        asm volatile("" : "+v"(left));  // (one comparison at a time: all masks at once do not fit the scalar registers)
        acc[i][j][k] = 32 * i + 8 * (k >> 2) + (k & 3) >= left ? -INFINITY : acc[i][j][k];
      }
}

// two running sums over disjoint rows into one
__device__ __forceinline__ void join(float& m, float& s, float mo, float so) {
  const float to = fmaxf(m, mo), ref = to == -INFINITY ? 0.f : to;
  s = s * __builtin_amdgcn_exp2f(m - ref) + so * __builtin_amdgcn_exp2f(mo - ref);
  m = to;
}

// Each lane keeps, for each of its tokens, the maximum m of the logits it has seen (in units of log 2) and
// the sum of 2^(logit log2(e) - m), the target's own left out; at the end of a workgroup's rows for a
// token tile they go to `part`, one slot per workgroup and row half. The logits themselves stay in the
// accumulators. Against a head of 151936 rows of 1024, fp16: 1 position 57 us and 61 positions 60 us (the head's
// rows at 5.4 TB/s), 1919 positions 558 us (1070 TFLOP/s; the matrix cores 59% busy at the clock that they leave, the
// library's product of 2048 without a softmax 587).
template <class C>
struct Stats : FromZero<C> {
  f32x2* part;  // [slot][tokens]
  float* tl;    // [tokens] target's logit
  Targets targets;
  int tokens, vocab, tiles_t, tiles_n;
  float m[C::NJ], s[C::NJ];
  int tile_t = -1;  // the token tile whose targets the lanes hold
  int row[C::NJ];   // (-1: none that counts)

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      m[j] = -INFINITY;
      s[j] = 0.f;
    }
  }
  __device__ __forceinline__ void tile(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, bool last, int lane, int wn, int wt) {
    asm volatile("" : "+v"(lane));  // (as in Stores)
    const int n0 = at.tn * C::BN + 32 * C::NI * wn + 4 * (lane >> 5);  // register (i, q, r): row n0 + 32 i + 8 q + r
    const int t0 = at.tt * C::BT + 32 * C::NJ * wt + (lane & 31);
    mask_rows<C>(acc, at, lane, wn, vocab);
    if (at.tt != tile_t) {
      tile_t = at.tt;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const long long y = t0 + 32 * j < tokens ? targets[t0 + 32 * j] : targets.ignore;
        row[j] = y != targets.ignore && y >= 0 && y < vocab ? (int)y : -1;
      }
    }
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      const int t = t0 + 32 * j;
      int d = row[j] >= n0 && row[j] < n0 + 32 * C::NI ? row[j] - n0 : -1;
      if (__any(d >= 0)) {
        // the target's logit goes to `tl` and leaves the sum: see head_join_kernel
        float x = 0.f;
        bool here = false;
#pragma unroll
        for (int i = 0; i < C::NI; ++i)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            asm volatile("" : "+v"(d));  // (one comparison at a time: 64 masks kept at once do not fit the scalar registers)
            const bool hit = d == 32 * i + 8 * (k >> 2) + (k & 3);
            x = hit ? acc[i][j][k] : x;
            here |= hit;
            acc[i][j][k] = hit ? -INFINITY : acc[i][j][k];
          }
        if (here) tl[t] = x;
      }
      float top = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < C::NI; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) top = fmaxf(top, acc[i][j][k]);
      const float to = fmaxf(m[j], top * LOG2E);
      // all logits so far -inf: measured from 0, the exponentials are 0 (from -inf they would be NaN)
      const float ref = to == -INFINITY ? 0.f : to;
      float sum = s[j] * __builtin_amdgcn_exp2f(m[j] - ref);
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        float part_sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 16; ++k) part_sum[k & 3] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][k], LOG2E, -ref));
        sum += (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
      }
      m[j] = to;
      s[j] = sum;
    }
    if (last || at.tn + 1 == tiles_n) {
      const long items = (long)tiles_t * tiles_n;
      const int slot = ((int)blockIdx.x - owner((long)at.tt * tiles_n, items, gridDim.x)) * C::WN + wn;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const float mo = __shfl_xor(m[j], 32), so = __shfl_xor(s[j], 32);
        join(m[j], s[j], mo, so);
        if (lane < 32 && t0 + 32 * j < tokens) part[(long)slot * tokens + t0 + 32 * j] = f32x2{m[j], s[j]};
      }
      reset();
    }
  }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) head_stats_kernel(Product P, Stats<C> epi) {
  __shared__ __align__(16) char ring[C::RING];
  epi.reset();
  run_product<C>(P, ring, epi);
}

// Joins the slots of each token: 8 tokens per workgroup, 32 lanes' worth of slots each
constexpr int JT = 8, JS = 32;
__global__ void __launch_bounds__(JT* JS) head_join_kernel(const f32x2* part, const float* tl, Targets targets, int tokens,
                                                           int vocab, int bt, int tiles_t, int tiles_n, int grid, int wn,
                                                           float* loss, float* lse) {
  __shared__ f32x2 sm[JS / 8][JT];
  const int i = threadIdx.x % JT, g = threadIdx.x / JT, t = blockIdx.x * JT + i;
  float m = -INFINITY, s = 0.f;
  if (t < tokens) {
    const int tt = t / bt;
    const long items = (long)tiles_t * tiles_n, a = (long)tt * tiles_n;
    const int slots = (owner(a + tiles_n - 1, items, grid) - owner(a, items, grid) + 1) * wn;
#pragma unroll 4
    for (int k = g; k < slots; k += JS) {
      const f32x2 v = part[(long)k * tokens + t];
      join(m, s, v[0], v[1]);
    }
  }
#pragma unroll
  for (int d = JT; d < 64; d *= 2) join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
  if ((threadIdx.x & 63) < JT) sm[threadIdx.x >> 6][i] = f32x2{m, s};
  __syncthreads();
  if (g != 0 || t >= tokens) return;
#pragma unroll
  for (int k = 1; k < JS / 8; ++k) join(m, s, sm[k][i][0], sm[k][i][1]);
  const long long y = targets[t];
  if (y == targets.ignore || y < 0 || y >= vocab) {
    lse[t] = (m + log2f(s)) * LN2;
    loss[t] = y == targets.ignore ? 0.f : NAN;  // neither a row of the head nor ignore_index
    return;
  }
  // With the sum S of the other rows' exponentials apart, the loss log(S + e^l) - l is log1p(S e^-l) where l is large:
  // the loss of a target that the model is sure of is not the difference of two numbers that are nearly equal.
  const float l = tl[t], d = fmaf(l, LOG2E, -m);  // the target's logit above the others' largest, in units of log 2
  if (d > 0.f) {
    const float x = log1pf(s * __builtin_amdgcn_exp2f(-d));
    loss[t] = l == INFINITY ? NAN : x;
    lse[t] = l + x;
  } else {
    const float all = s + __builtin_amdgcn_exp2f(d);  // (at least 1)
    loss[t] = (log2f(all) - d) * LN2;
    lse[t] = (m + log2f(all)) * LN2;
  }
}

// sum of the losses (in a fixed order), number of the positions that count, mean
__global__ void __launch_bounds__(1024) head_total_kernel(const float* loss, Targets targets, int tokens, float* total) {
  __shared__ float sm[16];
  __shared__ int cn[16];
  float s = 0.f;
  int n = 0;
  for (int t = threadIdx.x; t < tokens; t += 1024) {
    s += loss[t];
    n += targets[t] != targets.ignore;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    s += __shfl_xor(s, d);
    n += __shfl_xor(n, d);
  }
  if ((threadIdx.x & 63) == 0) {
    sm[threadIdx.x >> 6] = s;
    cn[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 1; k < 16; ++k) {
    s += sm[k];
    n += cn[k];
  }
  total[0] = s;
  total[1] = (float)n;
  total[2] = s / (float)n;
}

// ---- stores of a tile ------------------------------------------------------------------

// A wave's accumulators to memory as numbers of type T, 16 bytes per lane along the rows, by way of 4 KB of
// LDS of its own: straight from the accumulators a store instruction would touch 32 lines for 16 bytes
// each. make(i, q, j, v) turns the 4 accumulators of rows 32 i + 8 q + 4 (lane / 32) .. + 3 of the wave's (v, in
// place) into what is stored; patch(ib, j) may then change numbers in LDS, and last(j, token, x) changes the
// 16 bytes that go out for one of the wave's 32 tokens. Tokens from t_end and rows from n_end on are not stored.
// STREAM: past the caches, for arrays that do not stay in them anyway (8-bit logits of 1919 positions, 583 MB,
// 400 -> 348 us; the logits' gradient, which the next kernels read, is stored the ordinary way: 4% faster in all).
// (The stores take a scalar base and a vector offset: with buffer stores that take a scalar offset of their own, now
// and then 16 bytes of a tile were wrong.)
struct Nothing {
  __device__ void operator()(int, int) const {}
  __device__ void operator()(int, int, u32x4&) const {}
};
template <class C, class T, bool STREAM>
struct Stores {
  static constexpr int FIT = 4 / (int)sizeof(T);
  static constexpr int NB = C::NI < FIT ? C::NI : FIT;            // tiles of 32 rows staged at a time
  static constexpr int PER = 16 / sizeof(T), CH = 32 * NB / PER;  // numbers per 16 bytes, 16 bytes per token
  static_assert(C::NI % NB == 0 && NB >= 1, "a wave's staging area");
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef T tp __attribute__((ext_vector_type(PER)));
  // where the wave's LDS holds chunk c of token t
  static __device__ __forceinline__ u32 place(int t, int c) { return (u32)(t * CH * 16 + ((c ^ (t & (CH - 1))) << 4)); }

  template <class Make, class Patch, class Last>
  static __device__ __forceinline__ void store(typename C::E::acc (&acc)[C::NI][C::NJ], const Cursor& at, int lane, int wn,
                                               int wt, char* lds, T* out, long ld, int t_end, int n_end, Make&& make,
                                               Patch&& patch, Last&& last) {
    // (what follows from `lane` is computed here, item by item, rather than kept in registers through the K loop)
    asm volatile("" : "+v"(lane));
    const bool whole = n_end % PER == 0 && ld % PER == 0 && ((size_t)out & 15) == 0;  // 16-byte stores are aligned and end with the row
    const int t0 = at.tt * C::BT + 32 * C::NJ * wt, n0 = at.tn * C::BN + 32 * C::NI * wn;  // the wave's first token and row
    const bool inner = whole && t0 + 32 * C::NJ <= t_end && n0 + 32 * C::NI <= n_end;
    char* base = (char*)uniform((const char*)(out + (long)t0 * ld + n0));
    const int tl = lane & 31;
    const u32 to = place(tl, 0) + 8 * (sizeof(T) == 2 ? lane >> 5 : 0);  // (chunk c: to ^ 16 c)
    // reading back, a lane has 16 bytes of token 64 / CH p + lane / CH
    constexpr int TP = 64 / CH;
    const int tr = lane / CH, cr = lane % CH;
    const u32 off = (u32)(tr * (int)ld + PER * cr) * (u32)sizeof(T);
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
#pragma unroll
      for (int ib = 0; ib < C::NI; ib += NB) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (float)acc[ib + i][j][4 * q + r];
            make(ib + i, q, j, v);
            const u32 c = sizeof(T) == 2 ? 16 * (4 * i + q) : 16 * (8 * i + 2 * q + (lane >> 5));
            *(t4*)(lds + (to ^ c)) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          }
        asm volatile("" ::: "memory");
        patch(ib, j);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int p = 0; p < 32 / TP; ++p) {
          const int t = TP * p + tr;
          u32x4 x = *(const u32x4*)(lds + place(t, cr));
          last(j, t, x);
          if (inner) {
            typedef __attribute__((address_space(1))) u32x4 global_u32x4;  // (made of integers, `base` could be in any memory)
            global_u32x4* dst = (global_u32x4*)(base + ((long)(32 * j + TP * p) * ld + 32 * ib) * (long)sizeof(T) + off);
            if (STREAM)
              __builtin_nontemporal_store(x, dst);
            else
              *dst = x;
          } else if (t0 + 32 * j + t < t_end && n0 + 32 * ib + PER * cr < n_end) {
            const int n = n0 + 32 * ib + PER * cr;
            T* dst = out + (long)(t0 + 32 * j + t) * ld + n;
            if (n + PER <= n_end) {
              __builtin_memcpy(dst, &x, 16);
            } else {
              const tp y = __builtin_bit_cast(tp, x);
#pragma unroll
              for (int k = 0; k < PER; ++k)
                if (n + k < n_end) dst[k] = y[k];
            }
          }
        }
        asm volatile("" ::: "memory");
      }
    }
  }
};

// ---- gradients -------------------------------------------------------------------------

// The softmax's gradient of one piece of the vocabulary, G[t][v] = (2^(logit log2(e) - lse) - [v is the target])
// * SCALE, in the inputs' 16-bit type: the next products take it as a matrix operand. fp16's SCALE (a power of
// two, taken back at the end) keeps probabilities from 2^-29 on at full precision; without it those of a vocabulary
// of 151936 would be subnormal. Tokens that do not count, and v past the vocabulary, get zeros.
// The target's own entry is the largest of its token by far: its rounding is what one sees of G's. own_entry is that entry,
// own_rest what its rounding leaves, which the gradients take up again (grad_hidden always, grad_weight for few tokens).
template <class E>
constexpr float grad_scale() { return sizeof(typename E::elem) == 2 && std::is_same<E, Half>::value ? 32768.f : 1.f; }

template <class E>
__device__ __forceinline__ float own_entry(float loss) { return expm1f(-loss) * grad_scale<E>(); }  // p - 1, also where p is nearly 1
template <class E>
__device__ __forceinline__ float own_rest(float loss) {
  const float own = own_entry<E>(loss);
  return own - (float)(typename E::elem)own;
}

// 4096 positions, bf16: 132 us for 16384 rows (1040 TFLOP/s); the stores, all workgroups' at once, are 16 of them.
template <class C>
struct Softgrad : FromZero<C> {
  typedef typename C::E::elem T;
  typedef Stores<C, T, false> St;
  T* out;  // [tokens_pad][ld]
  long ld;
  const float *loss, *lse;
  Targets targets;
  int tokens, tokens_pad, v0, rows, rows_pad;  // the piece: vocabulary rows v0 .. v0 + rows - 1
  char* lds;
  // what the lanes hold of their tokens, loaded when the token tile changes
  int tile_t = -1;
  float l2[C::NJ], own[C::NJ];
  int row[C::NJ];     // the target's row of the piece, or out of it
  u32 counts[C::NJ];  // a bit per token
  __device__ __forceinline__ void tile(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, bool, int lane, int wn, int wt) {
    constexpr float SCALE = grad_scale<typename C::E>();
    if (at.tt != tile_t) {
      tile_t = at.tt;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const int t = at.tt * C::BT + 32 * (C::NJ * wt + j) + (lane & 31);
        const long long target = t < tokens ? targets[t] : targets.ignore, far = target - v0;
        const bool c = t < tokens && target != targets.ignore;
        counts[j] = (u32)__ballot(c);
        row[j] = c && lane < 32 && far >= 0 && far < rows ? (int)far : -1;
        const float x = c ? loss[t] : 0.f;
        // (a NaN loss: a target that is no row of the head, or logits that are NaN)
        l2[j] = c ? (x == x ? fmaf(lse[t], LOG2E, -__builtin_log2f(SCALE)) : NAN) : 0.f;
        own[j] = own_entry<typename C::E>(x);
      }
    }
    const int n0 = at.tn * C::BN + 32 * C::NI * wn;
    mask_rows<C>(acc, at, lane, wn, rows);
    St::store(
        acc, at, lane, wn, wt, lds, out, ld, tokens_pad, rows_pad,
        [&](int, int, int j, float (&v)[4]) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = __builtin_amdgcn_exp2f(fmaf(v[r], LOG2E, -l2[j]));
        },
        [&](int ib, int j) {
          const int n = row[j] - n0 - 32 * ib;
          if (row[j] >= 0 && n >= 0 && n < 32 * St::NB) *(T*)(lds + St::place(lane & 31, n / St::PER) + (int)sizeof(T) * (n % St::PER)) = (T)own[j];
        },
        [&](int j, int t, u32x4& x) {
          // (a mask: what a token that does not count holds may be NaN)
          x &= (u32)__builtin_amdgcn_sbfe((int)counts[j], t, 1);
        });
  }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) head_softgrad_kernel(Product P, Softgrad<C> epi) {
  __shared__ __align__(16) char ring[C::RING];
  __shared__ __align__(16) char stage[C::STAGING];
  epi.lds = stage + (threadIdx.x >> 6) * 4096;
  run_product<C>(P, ring, epi);
}

// Partial sums of grad_hidden: the accumulators of each item as the lanes hold them (fp32, 16 bytes per lane, 1 KB
// per wave and store), carried on from one piece of the vocabulary to the next. 4096 positions, bf16: 117 us for 16384
// rows (1170 TFLOP/s), 10 of them for reading and writing the sums.
template <class C>
struct Partials {
  float* out;  // [item][wave][i][j][q][lane][4]
  bool add;
  static __host__ __device__ __forceinline__ long place(long item, int wave, int i, int j) {
    return ((item * C::WAVES + wave) * C::NI * C::NJ + i * C::NJ + j) * 1024;
  }
  __device__ __forceinline__ void begin(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, int lane, int wave) {
    asm volatile("" : "+v"(lane));  // (as in Stores)
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v = {0.f, 0.f, 0.f, 0.f};
          if (add) v = *(const f32x4*)(out + place(at.item, wave, i, j) + 256 * q + 4 * lane);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][4 * q + r] = v[r];
        }
  }
  __device__ __forceinline__ void tile(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, bool, int lane, int wn, int wt) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(f32x4*)(out + place(at.item, wt * C::WN + wn, i, j) + 256 * q + 4 * lane) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
  }
};
template <class C>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) head_partials_kernel(Product P, Partials<C> epi) {
  __shared__ __align__(16) char ring[C::RING];
  run_product<C>(P, ring, epi);
}

// grad_hidden: the splits' sums in order and what the target's entry lost to rounding, times the position's upstream gradient;
// a thread has 4 numbers of one row
template <class C>
__global__ void __launch_bounds__(256) head_grad_hidden_kernel(const float* part, int splits, int tiles_t, int tiles_n,
                                                               int tokens, int width, Targets targets, Upstream grad,
                                                               float unscale, const float* loss, int vocab,
                                                               const typename C::E::elem* weight, long weight_ld,
                                                               typename C::E::elem* out) {
  typedef typename C::E::elem T;
  constexpr int PER_TILE = C::BN * C::BT / 4;
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  const int tile = (int)(e / PER_TILE), o = (int)(e % PER_TILE);
  const int wave = o / (C::NI * C::NJ * 256), ij = o / 256 % (C::NI * C::NJ), q = o / 64 % 4, lane = o % 64;
  const int t = tile / tiles_n * C::BT + 32 * (C::NJ * (wave / C::WN) + ij % C::NJ) + (lane & 31);
  const int n = tile % tiles_n * C::BN + 32 * (C::NI * (wave % C::WN) + ij / C::NJ) + 8 * q + 4 * (lane >> 5);
  if (tile >= tiles_t * tiles_n || t >= tokens || n >= width) return;
  typedef T t4 __attribute__((ext_vector_type(4)));
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  const long long y = targets[t];
  if (y != targets.ignore) {
    if (y >= 0 && y < vocab) {
      const t4 w = *(const t4*)(weight + y * weight_ld + n);
      const float rest = own_rest<typename C::E>(loss[t]);
      // (none: nothing is added, also where the row holds the infinity that made the target impossible)
      if (rest != 0.f) a = f32x4{rest * (float)w[0], rest * (float)w[1], rest * (float)w[2], rest * (float)w[3]};
    }
#pragma unroll 8
    for (int s = 0; s < splits; ++s) a += *(const f32x4*)(part + ((long)s * tiles_t * tiles_n * PER_TILE + e) * 4);
    a *= grad[t] * unscale;
  }
  *(t4*)(out + (long)t * width + n) = t4{(T)a[0], (T)a[1], (T)a[2], (T)a[3]};
}

// max |upstream gradient| of the positions that count
__global__ void __launch_bounds__(1024) head_grad_max_kernel(Upstream grad, Targets targets, int tokens, float* out) {
  __shared__ float sm[16];
  float m = 0.f;
  for (int t = threadIdx.x; t < tokens; t += 1024)
    if (targets[t] != targets.ignore) m = fmaxf(m, fabsf(grad[t]));
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 1; k < 16; ++k) m = fmaxf(m, sm[k]);
  *out = m;
}

// The hidden rows as grad_weight's product takes them: each times its upstream gradient over the largest one
// (1 or -1, and no rounding, where all positions weigh the same), zeros for positions that do not count
// and up to a whole number of K steps. top: the largest, or null where there is only one.
template <class T>
__global__ void __launch_bounds__(256) head_weighted_rows_kernel(const T* hidden, long ld, Targets targets, Upstream grad,
                                                                 const float* top, int tokens, int tokens_pad, int width,
                                                                 T* out) {
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e >= (long)tokens_pad * width) return;
  const int t = (int)(e / width), c = (int)(e % width);
  typedef T t8 __attribute__((ext_vector_type(8)));
  t8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (T)0.f;
  if (t < tokens && targets[t] != targets.ignore) {
    const float m = top ? *top : fabsf(grad[0]), g = m == 0.f ? 0.f : grad[t] / m;
    const t8 h = *(const t8*)(hidden + t * ld + c);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (T)((float)h[k] * g);
  }
  *(t8*)(out + e) = v;
}

// grad_weight's rows of a piece. 4096 positions, bf16: 104 us for 16384 rows (1320 TFLOP/s, the matrix cores 63% busy).
// Of up to FEW tokens the target's entries are added what their rounding left; the lanes hold whose targets are
// where, a wave adds a token's hidden row to the accumulators of the target's row. (Of more tokens the roundings'
// errors are a fifth on top of the output's own.)
// It is a kernel of its own (RESTS): it takes 19 (fp16) or 26 (bf16) of the 27 registers that the 256x256 tile leaves.
constexpr int FEW = 256;  // (four targets a lane)
template <class C, bool RESTS>
struct WeightGrad : FromZero<C> {
  typedef typename C::E::elem T;
  T* out;  // [rows][width]
  Upstream grad;
  const float* top;  // as in head_weighted_rows_kernel
  int rows, width;
  const T* weighted;  // [tokens][width]
  const float* loss;
  Targets targets;
  int tokens, v0;  // (the piece's first row)
  char* lds;
  bool looked = false;
  int row0, row1, row2, row3;  // of tokens lane, 64 + lane, ..: the target's row of the piece, or -1 (a field each: an array would be in memory)
  __device__ __forceinline__ void add_rests(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, int lane, int wn, int wt) {
    if (!looked) {
      looked = true;
      const auto look = [&](int t) {
        const long long y = t < tokens ? targets[t] : targets.ignore, far = y - v0;
        return y != targets.ignore && far >= 0 && far < rows ? (int)far : -1;
      };
      row0 = look(lane), row1 = look(64 + lane), row2 = look(128 + lane), row3 = look(192 + lane);
    }
    const int r0 = at.tt * C::BT + 32 * C::NJ * wt;  // the wave's first row
    const int n0 = at.tn * C::BN + 32 * C::NI * wn + 4 * (lane >> 5);
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      const int mine = q == 0 ? row0 : q == 1 ? row1 : q == 2 ? row2 : row3;
      unsigned long long hits = __ballot(mine >= r0 && mine < r0 + 32 * C::NJ);
      while (hits) {
        const int l = __builtin_ctzll(hits);
        hits &= hits - 1;
        const int t = 64 * q + l, r = __builtin_amdgcn_readlane(mine, l) - r0;
        const float rest = own_rest<typename C::E>(loss[t]);
        const T* h = weighted + (long)t * width;
        if ((lane & 31) != (r & 31)) continue;
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
          if (j == r >> 5) {
#pragma unroll
            for (int i = 0; i < C::NI; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int n = n0 + 32 * i + 8 * k;
                const t4 x = *(const t4*)(h + (n < width ? n : 0));  // (columns past the width are not stored)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][4 * k + e] = fmaf(rest, (float)x[e], acc[i][j][4 * k + e]);
              }
          }
      }
    }
  }
  __device__ __forceinline__ void tile(f32x16 (&acc)[C::NI][C::NJ], const Cursor& at, bool, int lane, int wn, int wt) {
    if constexpr (RESTS) add_rests(acc, at, lane, wn, wt);
    const float f = (top ? *top : fabsf(grad[0])) * (1.f / grad_scale<typename C::E>());
    Stores<C, T, true>::store(
        acc, at, lane, wn, wt, lds, out, width, rows, width,
        [&](int, int, int, float (&v)[4]) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] *= f;
        },
        Nothing(), Nothing());
  }
};
template <class C, bool RESTS>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) head_weight_grad_kernel(Product P, WeightGrad<C, RESTS> epi) {
  __shared__ __align__(16) char ring[C::RING];
  __shared__ __align__(16) char stage[C::STAGING];
  epi.lds = stage + (threadIdx.x >> 6) * 4096;
  run_product<C>(P, ring, epi);
}

// ---- 8-bit integers --------------------------------------------------------------------

// The int32 sums times both scales. Tokens 1 by a head of 151936 rows of 1024: 27 us (the head's rows at 5.7 TB/s);
// 1919: 343 us (1740 TOP/s; the library's largest products reach 2110), 12% of it for the stores of 583 MB.
template <class C, class T, bool STREAM>
struct Dequant : FromZero<C> {
  T* out;  // [tokens][rows]
  const float *xs, *ws;
  int tokens, rows;
  char* lds;
  int tile_t = -1;  // the token tile whose scales the lanes hold
  float sx[C::NJ];
  __device__ __forceinline__ void tile(i32x16 (&acc)[C::NI][C::NJ], const Cursor& at, bool, int lane, int wn, int wt) {
    const int n0 = at.tn * C::BN + 32 * C::NI * wn + 4 * (lane >> 5);
    if (at.tt != tile_t) {
      tile_t = at.tt;
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) sx[j] = xs[min(at.tt * C::BT + 32 * (C::NJ * wt + j) + (lane & 31), tokens - 1)];
    }
    // the rows' scales, 4 together (the wave's rows may end before its tile does)
    f32x4 sw[C::NI][4];
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + 32 * i + 8 * q;
        if (at.tn * C::BN + 32 * (C::NI * wn + i + 1) <= rows) {
          __builtin_memcpy(&sw[i][q], ws + n, 16);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) sw[i][q][r] = ws[min(n + r, rows - 1)];
        }
      }
    Stores<C, T, STREAM>::store(
        acc, at, lane, wn, wt, lds, out, rows, tokens, rows,
        [&](int i, int q, int j, float (&v)[4]) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] *= sx[j] * sw[i][q][r];
        },
        Nothing(), Nothing());
  }
};
template <class C, class T, bool STREAM>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) matmul_i8_kernel(Product P, Dequant<C, T, STREAM> epi) {
  __shared__ __align__(16) char ring[C::RING];
  __shared__ __align__(16) char stage[C::STAGING];
  epi.lds = stage + (threadIdx.x >> 6) * 4096;
  run_product<C>(P, ring, epi);
}

// Rows to 8-bit integers: scale = max |x| / 127, q = 127 x / max |x| rounded to the nearest integer, ties to even:
// exactly, without a division per number. x and max |x| have at most 11 significant bits, so a quotient that is
// not k + 1/2 itself differs from it by more than 2^-19 of its size (|254 x - (2 k + 1) max| is a whole number of
// steps of x or max, and 254 * 2047 < 2^19). t = x * fl(127 / max) is good to 2^-23; rounded to 20 bits it is k + 1/2 where
// the quotient is, and on the quotient's side of it where it is not. A row of zeros gets scale 0; one with an
// infinity or a NaN scale NaN and zeros, so that what is computed from it is NaN. One wave per row, the row
// in registers up to 2048 numbers. Bound by memory: 151936 rows of 1024 in 80 us, 5.8 TB/s (127 us with a
// division per number and the row read twice).
template <class T, int CHUNKS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long ld, int rows, int width, signed char* q,
                                                            float* scale) {
#pragma clang fp contract(off)
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  typedef T t8 __attribute__((ext_vector_type(8)));
  const T* p = x + row * ld;
  signed char* out = q + (long)row * width;
  float top = 0.f;
  bool bad = false;
  auto look = [&](const t8& v) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = fabsf((float)v[k]);
      bad |= !(a < INFINITY);
      top = fmaxf(top, a);
    }
  };
  t8 held[CHUNKS > 0 ? CHUNKS : 1];
  if (CHUNKS > 0) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) held[c] = *(const t8*)(p + min(8 * lane + 512 * c, width - 8));
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) look(held[c]);
  } else {
    for (int c = 8 * lane; c < width; c += 512) look(*(const t8*)(p + c));
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  bad = __any(bad);
  if (lane == 0) scale[row] = bad ? NAN : top / 127.f;
  // powers of two keep 127 / max and x in fp32's range at both ends of bf16's, and leave every quotient as it is
  const float f = top > 0x1p60f ? 0x1p-60f : top < 0x1p-60f ? 0x1p66f : 1.f;
  const float r = top == 0.f || bad ? 0.f : 127.f / (top * f);
  auto round = [&](const t8& v, int at) {
    u32 w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32 b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float t = (float)v[4 * h + k] * f * r, c = 17.f * t, t20 = c - (c - t);
        b[k] = __float_as_uint(t20 + 12582912.f);  // (1.5 * 2^23: the sum's low byte is the integer)
      }
      w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                   0x05040100u);
      if (bad) w[h] = 0;
    }
    *(unsigned long long*)(out + at) = (unsigned long long)w[1] << 32 | w[0];
  };
  if (CHUNKS > 0) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (8 * lane + 512 * c < width) round(held[c], 8 * lane + 512 * c);
  } else {
    for (int c = 8 * lane; c < width; c += 512) round(*(const t8*)(p + c), c);
  }
}
template <class T>
const void* quantize_kernel(int width) {
  return width <= 1024 ? (const void*)quantize_rows_kernel<T, 2>
         : width <= 2048 ? (const void*)quantize_rows_kernel<T, 4> : (const void*)quantize_rows_kernel<T, 0>;
}

// ---- the engine's final norm over many rows --------------------------------------------

// fp16(x / rms * gain) of fp32 rows of 1024, one wave per row
__global__ void __launch_bounds__(256) norm_rows_kernel(const float* x, const _Float16* gain, int rows, _Float16* out) {
  constexpr int H = 1024;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  f32x4 v[4];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = *(const f32x4*)(x + (long)row * H + 8 * lane + 512 * (k >> 1) + 4 * (k & 1));
    s += (v[k][0] * v[k][0] + v[k][1] * v[k][1]) + (v[k][2] * v[k][2] + v[k][3] * v[k][3]);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  const float r = rsqrtf(s * (1.f / H) + 1e-6f);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = 8 * lane + 512 * k;
    const f16x8 g = *(const f16x8*)(gain + c);
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)(v[2 * k + (e >> 2)][e & 3] * r * (float)g[e]);
    *(f16x8*)(out + (long)row * H + c) = y;
  }
}

// ====================================================================================
// host side

namespace {

int launch(const void* kernel, long grid, int threads, void** args, hipStream_t stream) {
  if (grid <= 0 || grid > 0x7fffffffL) return QWEN_ERR_ARG;
  return hipLaunchKernel(kernel, dim3((unsigned)grid), dim3(threads), args, 0, stream) == hipSuccess ? QWEN_OK : QWEN_ERR_LAUNCH;
}
template <class P, class E>
int launch_product(void (*kernel)(P, E), long grid, int threads, P product, E epi, hipStream_t stream) {
  void* args[] = {&product, &epi};
  return launch((const void*)kernel, grid, threads, args, stream);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
long round_up(long x, long m) { return (x + m - 1) / m * m; }

// The tiles a product can be cut into. Large ones do the most per byte that they bring to LDS, small ones leave no
// CU idle where there are few, and two workgroups on a CU hide each other's waits (few tokens: the
// head's rows then arrive as fast as memory gives them). SMALL is sized for the LDS that an epilogue leaves.
enum TileKind : int { SMALL, MIDDLE, LARGE };
template <class E, int LW = ROWS, int LX = ROWS>
struct Tiles {
  typedef Config<E, 128, 64, 2, 2, 2, 2, LW, LX> Small;
  typedef Config<E, 128, 128, 2, 2, 2, 2, LW, LX> Middle;
  typedef Config<E, 256, 256, 2, 4, 2, 1, LW, LX> Large;
};
template <>
struct Tiles<Int8, ROWS, ROWS> {
  typedef Config<Int8, 64, 64, 2, 2, 3, 2> Small;
  typedef Config<Int8, 128, 128, 2, 2, 2, 2> Middle;
  typedef Config<Int8, 256, 256, 2, 4, 2, 1> Large;
};
template <class E>
struct StatsTiles {  // (no stores through LDS: a deeper ring)
  typedef Config<E, 128, 64, 2, 2, 3, 2> Small;
  typedef Config<E, 128, 128, 2, 2, 2, 2> Middle;
  typedef Config<E, 256, 256, 2, 4, 2, 1> Large;
};

// How long a product takes, in units of what a CU multiplies by large tiles: whole rounds of tiles over
// the chip, each as long as its numbers at the rate that this tile reaches (measured on 1919 positions: 16-bit 1622, 921
// and 562 us, 8-bit 909, 510 and 343).
template <class C>
long cost(int tokens, int rows, int percent) {
  const long items = (long)((tokens + C::BT - 1) / C::BT) * ((rows + C::BN - 1) / C::BN);
  const long rounds = (items + CUS * C::OCC - 1) / (CUS * C::OCC);
  return rounds * C::OCC * C::BN * C::BT * 100 / percent;
}
template <class TS>
long tile_cost(TileKind k, int tokens, int rows) {
  return k == SMALL ? cost<typename TS::Small>(tokens, rows, 36) : k == MIDDLE ? cost<typename TS::Middle>(tokens, rows, 62)
                                                                                : cost<typename TS::Large>(tokens, rows, 100);
}
template <class TS>
TileKind pick(int tokens, int rows) {
  const long s = tile_cost<TS>(SMALL, tokens, rows), m = tile_cost<TS>(MIDDLE, tokens, rows), l = tile_cost<TS>(LARGE, tokens, rows);
  return l <= m && l <= s ? LARGE : m <= s ? MIDDLE : SMALL;
}
// f(tile) for the tile of this kind
template <class TS, class F>
auto with_tile(TileKind k, F&& f) {
  return k == SMALL ? f(typename TS::Small()) : k == MIDDLE ? f(typename TS::Middle()) : f(typename TS::Large());
}

// a product's tiles over [tokens][rows]
template <class C>
Product make_product(Operand x, Operand w, int steps) {
  Product P;
  P.x = x;
  P.w = w;
  P.tiles_t = (x.n + C::BT - 1) / C::BT;
  P.tiles_n = (w.n + C::BN - 1) / C::BN;
  P.steps = steps;
  P.splits = 1;
  P.split_steps = steps;
  return P;
}
template <class C>
long grid_of(const Product& P) {
  const long items = (long)P.splits * P.tiles_t * P.tiles_n;
  return items < CUS * C::OCC ? items : CUS * C::OCC;
}
int k_steps(long bytes) { return (int)((bytes + STEP - 1) / STEP); }

struct Head {
  const void* hidden;
  long hidden_ld;
  const void* weight;
  long weight_ld;
  Targets targets;
  int tokens, vocab, width;
};

constexpr long MAX_ROW_BYTES = 4L << 20;  // a tile's offsets stay below 2^31
constexpr int MAX_TOKENS = 1 << 20, MAX_VOCAB = 1 << 24, MAX_CHANNELS = 1 << 22;

int check_head(const Head& h, int target_bits, int dtype) {
  if (h.tokens < 0 || h.tokens > MAX_TOKENS || h.vocab < 1 || h.vocab > MAX_VOCAB || h.width < 8 || h.width % 8 != 0)
    return QWEN_ERR_ARG;
  if (dtype != QWEN_F16 && dtype != QWEN_BF16) return QWEN_ERR_ARG;
  if (target_bits != 32 && target_bits != 64) return QWEN_ERR_ARG;
  if (h.hidden_ld < h.width || h.weight_ld < h.width || h.hidden_ld % 8 != 0 || h.weight_ld % 8 != 0 ||
      2 * h.hidden_ld > MAX_ROW_BYTES || 2 * h.weight_ld > MAX_ROW_BYTES)
    return QWEN_ERR_ARG;
  if (h.tokens > 0 && (!h.hidden || !h.targets.p || !aligned16(h.hidden) || ((uintptr_t)h.targets.p & (target_bits / 8 - 1)) != 0))
    return QWEN_ERR_ARG;
  if (!h.weight || !aligned16(h.weight)) return QWEN_ERR_ARG;
  return QWEN_OK;
}

Operand rows_of(const void* p, long ld, int n, int width) { return Operand{(const char*)p, 2 * ld, n, 2 * width}; }

struct ForwardPlan {
  Product P;
  long grid;
  int wn, slots;
};
template <class C>
ForwardPlan forward_plan(const Head& h) {
  ForwardPlan f;
  f.P = make_product<C>(rows_of(h.hidden, h.hidden_ld, h.tokens, h.width), rows_of(h.weight, h.weight_ld, h.vocab, h.width),
                        k_steps(2L * h.width));
  f.grid = grid_of<C>(f.P);
  f.wn = C::WN;
  f.slots = 0;
  const long items = (long)f.P.tiles_t * f.P.tiles_n;
  for (long t = 0; t < f.P.tiles_t; ++t) {
    const int n = owner((t + 1) * f.P.tiles_n - 1, items, f.grid) - owner(t * f.P.tiles_n, items, f.grid) + 1;
    if (n > f.slots) f.slots = n;
  }
  f.slots *= C::WN;
  return f;
}
template <class C>
long forward_bytes(const Head& h) {
  const ForwardPlan f = forward_plan<C>(h);
  return round_up(8L * f.slots * h.tokens, 256) + round_up(4L * h.tokens, 256);
}

template <class C>
int forward(const Head& h, float* loss, float* lse, float* total, char* ws, long ws_bytes, hipStream_t stream) {
  if (ws_bytes < forward_bytes<C>(h)) return QWEN_ERR_ARG;
  const ForwardPlan f = forward_plan<C>(h);
  Stats<C> epi;
  epi.part = (f32x2*)ws;
  epi.tl = (float*)(ws + round_up(8L * f.slots * h.tokens, 256));
  epi.targets = h.targets;
  epi.tokens = h.tokens;
  epi.vocab = h.vocab;
  epi.tiles_t = f.P.tiles_t;
  epi.tiles_n = f.P.tiles_n;
  int rc = launch_product(head_stats_kernel<C>, f.grid, C::THREADS, f.P, epi, stream);
  if (rc != QWEN_OK) return rc;
  const f32x2* part = epi.part;
  const float* tl = epi.tl;
  Targets targets = h.targets;
  int tokens = h.tokens, vocab = h.vocab, bt = C::BT, tt = f.P.tiles_t, tn = f.P.tiles_n, grid = (int)f.grid, wn = f.wn;
  void* join[] = {&part, &tl, &targets, &tokens, &vocab, &bt, &tt, &tn, &grid, &wn, &loss, &lse};
  rc = launch((const void*)head_join_kernel, (h.tokens + JT - 1) / JT, JT * JS, join, stream);
  if (rc != QWEN_OK || !total) return rc;
  void* sum[] = {&loss, &targets, &tokens, &total};
  return launch((const void*)head_total_kernel, 1, 1024, sum, stream);
}

// ---- backward: pieces of the vocabulary

struct BackwardPlan {
  int tokens_pad;   // K of grad_weight's product
  int rows;         // vocabulary rows per piece (a multiple of 256)
  TileKind kind;    // of grad_hidden's product (its partial sums are laid out by tile)
  int splits;
  long g, weighted, partial, top, bytes;  // places in the workspace
};
// K steps in at most `most` parts: their length, their number
std::pair<int, int> split(int steps, int most) {
  const int length = (steps + most - 1) / most;
  return {length, (steps + length - 1) / length};
}

// the cost of one piece's products, and of what comes with a piece (launches, partial sums read and written)
long piece_cost(const Head& h, int rows, bool want_weight) {
  typedef Tiles<Half> G;
  typedef Tiles<Half, COLS, COLS> W;
  const long k = 1024 / 16;  // in units of 16 numbers of k
  return tile_cost<G>(pick<G>(h.tokens, rows), h.tokens, rows) * (h.width / 8) / 2 +
         (want_weight ? tile_cost<W>(pick<W>(rows, h.width), rows, h.width) * (h.tokens + 15) / 16 : 0) + 256 * 256 * k / 3;
}
BackwardPlan backward_plan(const Head& h, bool want_hidden, bool want_weight) {
  typedef Tiles<Half, COLS, ROWS> TS;
  BackwardPlan b;
  b.tokens_pad = (int)round_up(h.tokens, 64);
  // The gradient of the logits is kept for a piece of the vocabulary: at most 128 MB, half of the 256 MB cache before HBM
  // (4096 positions: 64 MB 4380 us, 128 MB 3845, 256 MB 3977). Within that, the size whose products leave the
  // fewest CUs idle in their last rounds (999 positions 1104 -> 986 us). Pieces of which the head's rows fit the
  // cache too, for the second product that reads them, are no faster (20 positions 224 us instead of 207).
  constexpr long PIECE = 64L << 20;
  const long all = round_up(h.vocab, 256);
  long most = PIECE / b.tokens_pad / 256 * 256;
  most = most < 256 ? 256 : most > all ? all : most;
  b.rows = (int)most;
  long least = -1;
  for (long rows = most; rows >= 256 && rows > most / 2; rows -= 256 * (1 + most / 65536)) {
    const long full = h.vocab / rows;
    const int last = (int)(h.vocab - full * rows);
    const long c = full * piece_cost(h, (int)rows, want_weight) + (last ? piece_cost(h, last, want_weight) : 0);
    if (least < 0 || c < least) {
      least = c;
      b.rows = (int)rows;
    }
  }
  // of grad_hidden's sums over the vocabulary, as many parts as give every workgroup one, of 8 K steps at least (each
  // is written and read again)
  const int steps = (int)(round_up(b.rows < h.vocab ? b.rows : h.vocab, 64) / 64);  // of the first piece; no other has more
  b.kind = h.tokens <= 64 ? SMALL : h.tokens <= 128 ? MIDDLE : LARGE;
  const long tile_numbers = with_tile<TS>(b.kind, [&](auto c) {
    typedef decltype(c) C;
    const long tiles = (long)((h.tokens + C::BT - 1) / C::BT) * ((h.width + C::BN - 1) / C::BN), s = CUS * C::OCC / tiles;
    b.splits = (int)(s > steps / 8 ? steps / 8 : s);
    if (b.splits < 1) b.splits = 1;
    return tiles * C::BN * C::BT;
  });
  b.splits = split(steps, b.splits).second;
  long at = 0;
  auto take = [&](long bytes) {
    const long p = at;
    at += round_up(bytes, 256);
    return p;
  };
  b.top = take(4);
  b.g = take(2L * b.tokens_pad * b.rows);
  b.weighted = take(want_weight ? 2L * b.tokens_pad * h.width : 0);
  b.partial = take(want_hidden ? 4L * b.splits * tile_numbers : 0);
  b.bytes = at;
  return b;
}

template <class E>
int backward(const Head& h, Upstream grad, const float* loss, const float* lse, void* grad_hidden,
             void* grad_weight, char* ws, long ws_bytes, hipStream_t stream) {
  typedef typename E::elem T;
  const BackwardPlan b = backward_plan(h, grad_hidden, grad_weight);
  if (ws_bytes < b.bytes) return QWEN_ERR_ARG;
  T* g = (T*)(ws + b.g);
  T* weighted = (T*)(ws + b.weighted);
  float* partial = (float*)(ws + b.partial);
  float* top = (float*)(ws + b.top);
  Targets targets = h.targets;
  int tokens = h.tokens, tokens_pad = b.tokens_pad, width = h.width;
  int rc = QWEN_OK;
  if (grad_weight) {
    if (grad.stride == 0) {
      top = nullptr;  // one number for all positions
    } else {
      void* a[] = {&grad, &targets, &tokens, &top};
      if ((rc = launch((const void*)head_grad_max_kernel, 1, 1024, a, stream)) != QWEN_OK) return rc;
    }
    const T* hidden = (const T*)h.hidden;
    long ld = h.hidden_ld;
    void* c[] = {&hidden, &ld, &targets, &grad, &top, &tokens, &tokens_pad, &width, &weighted};
    rc = launch((const void*)head_weighted_rows_kernel<T>, ((long)tokens_pad * width / 8 + 255) / 256, 256, c, stream);
    if (rc != QWEN_OK) return rc;
  }
  for (int v0 = 0; v0 < h.vocab; v0 += b.rows) {
    const int rows = h.vocab - v0 < b.rows ? h.vocab - v0 : b.rows, rows_pad = (int)round_up(rows, 64);
    const char* w = (const char*)h.weight + 2 * (long)v0 * h.weight_ld;
    rc = with_tile<Tiles<E>>(pick<Tiles<E>>(tokens, rows), [&](auto c) {
      typedef decltype(c) C;
      Product P = make_product<C>(rows_of(h.hidden, h.hidden_ld, tokens, width), rows_of(w, h.weight_ld, rows, width),
                                  k_steps(2L * width));
      Softgrad<C> e;
      e.out = g;
      e.ld = b.rows;
      e.loss = loss;
      e.lse = lse;
      e.targets = targets;
      e.tokens = tokens;
      e.tokens_pad = tokens_pad;
      e.v0 = v0;
      e.rows = rows;
      e.rows_pad = rows_pad;
      return launch_product(head_softgrad_kernel<C>, grid_of<C>(P), C::THREADS, P, e, stream);
    });
    if (rc != QWEN_OK) return rc;
    if (grad_hidden) {
      rc = with_tile<Tiles<E, COLS, ROWS>>(b.kind, [&](auto c) {
        typedef decltype(c) C;
        Product P = make_product<C>(Operand{(const char*)g, 2L * b.rows, tokens, 2 * rows_pad},
                                    Operand{w, 2 * h.weight_ld, width, rows}, rows_pad / 64);
        std::tie(P.split_steps, P.splits) = split(P.steps, b.splits);
        Partials<C> e;
        e.out = partial;
        e.add = v0 > 0;
        return launch_product(head_partials_kernel<C>, grid_of<C>(P), C::THREADS, P, e, stream);
      });
      if (rc != QWEN_OK) return rc;
    }
    if (grad_weight) {
      rc = with_tile<Tiles<E, COLS, COLS>>(pick<Tiles<E, COLS, COLS>>(rows, width), [&](auto c) {
        typedef decltype(c) C;
        Product P = make_product<C>(Operand{(const char*)g, 2L * b.rows, rows_pad, tokens_pad},
                                    Operand{(const char*)weighted, 2L * width, width, tokens_pad}, tokens_pad / 64);
        const auto run = [&](auto rests) {
          constexpr bool RESTS = decltype(rests)::value;
          WeightGrad<C, RESTS> e;
          e.out = (T*)grad_weight + (long)v0 * width;
          e.grad = grad;
          e.top = top;
          e.rows = rows;
          e.width = width;
          e.weighted = weighted;
          e.loss = loss;
          e.targets = targets;
          e.tokens = tokens;
          e.v0 = v0;
          return launch_product(head_weight_grad_kernel<C, RESTS>, grid_of<C>(P), C::THREADS, P, e, stream);
        };
        return tokens <= FEW ? run(std::true_type()) : run(std::false_type());
      });
      if (rc != QWEN_OK) return rc;
    }
  }
  if (!grad_hidden) return rc;
  return with_tile<Tiles<E, COLS, ROWS>>(b.kind, [&](auto c) {
    typedef decltype(c) C;
    int splits = b.splits, tiles_t = (tokens + C::BT - 1) / C::BT, tiles_n = (width + C::BN - 1) / C::BN;
    float unscale = 1.f / grad_scale<E>();
    const void* weight = h.weight;
    long weight_ld = h.weight_ld;
    int vocab = h.vocab;
    void* a[] = {&partial, &splits, &tiles_t, &tiles_n, &tokens, &width, &targets, &grad, &unscale, &loss, &vocab, &weight, &weight_ld,
                 &grad_hidden};
    return launch((const void*)head_grad_hidden_kernel<C>, (long)tiles_t * tiles_n * (C::BN * C::BT / 1024), 256, a, stream);
  });
}

}  // namespace
}  // namespace hd

using namespace hd;

extern "C" long long qwen_cross_entropy_workspace(int tokens, int vocab, int width) {
  if (tokens < 1 || tokens > MAX_TOKENS || vocab < 1 || vocab > MAX_VOCAB || width < 8) return 0;
  Head h = {nullptr, 0, nullptr, 0, {}, tokens, vocab, width};
  return with_tile<StatsTiles<Half>>(pick<StatsTiles<Half>>(tokens, vocab), [&](auto c) { return forward_bytes<decltype(c)>(h); });
}

extern "C" int qwen_cross_entropy(const void* hidden, long long hidden_stride, const void* weight, long long weight_stride,
                                  const void* targets, int target_bits, int tokens, int vocab, int width, int dtype,
                                  long long ignore_index, float* loss, float* lse, float* total, void* workspace,
                                  long long workspace_bytes, hipStream_t stream) {
  const Head h = {hidden, (long)hidden_stride, weight, (long)weight_stride, {targets, target_bits == 64, ignore_index},
                  tokens, vocab, width};
  const int rc = check_head(h, target_bits, dtype);
  if (rc != QWEN_OK) return rc;
  if (tokens == 0) return QWEN_OK;
  if (!loss || !lse || !workspace || !aligned16(workspace)) return QWEN_ERR_ARG;
  char* ws = (char*)workspace;
  const TileKind k = pick<StatsTiles<Half>>(tokens, vocab);
  auto run = [&](auto c) { return forward<decltype(c)>(h, loss, lse, total, ws, workspace_bytes, stream); };
  return dtype == QWEN_F16 ? with_tile<StatsTiles<Half>>(k, run) : with_tile<StatsTiles<Bfloat>>(k, run);
}

extern "C" long long qwen_cross_entropy_backward_workspace(int tokens, int vocab, int width, int want_hidden, int want_weight) {
  if (tokens < 1 || tokens > MAX_TOKENS || vocab < 1 || vocab > MAX_VOCAB || width < 8) return 0;
  Head h = {nullptr, 0, nullptr, 0, {}, tokens, vocab, width};
  return backward_plan(h, want_hidden != 0, want_weight != 0).bytes;
}

extern "C" int qwen_cross_entropy_backward(const float* grad_loss, long long grad_stride, const float* grad_divisor,
                                           const void* hidden, long long hidden_stride, const void* weight, long long weight_stride,
                                           const void* targets, int target_bits, int tokens, int vocab, int width,
                                           int dtype, long long ignore_index, const float* loss, const float* lse,
                                           void* grad_hidden, void* grad_weight, void* workspace,
                                           long long workspace_bytes, hipStream_t stream) {
  const Head h = {hidden, (long)hidden_stride, weight, (long)weight_stride, {targets, target_bits == 64, ignore_index},
                  tokens, vocab, width};
  const int rc = check_head(h, target_bits, dtype);
  if (rc != QWEN_OK) return rc;
  if (tokens < 1 || !grad_loss || grad_stride < 0 || !loss || !lse || (!grad_hidden && !grad_weight) || !aligned16(grad_hidden) ||
      !aligned16(grad_weight) || !workspace || !aligned16(workspace))
    return QWEN_ERR_ARG;
  char* ws = (char*)workspace;
  const Upstream grad = {grad_loss, (long)grad_stride, grad_divisor};
  return dtype == QWEN_F16 ? backward<Half>(h, grad, loss, lse, grad_hidden, grad_weight, ws, workspace_bytes, stream)
                           : backward<Bfloat>(h, grad, loss, lse, grad_hidden, grad_weight, ws, workspace_bytes, stream);
}

extern "C" int qwen_quantize_rows(const void* x, long long stride, int rows, int width, int dtype, signed char* q,
                                  float* scale, hipStream_t stream) {
  if (rows < 0 || width < 16 || width % 16 != 0 || stride < width || stride % 8 != 0 || (dtype != QWEN_F16 && dtype != QWEN_BF16))
    return QWEN_ERR_ARG;
  if (rows == 0) return QWEN_OK;
  if (!x || !q || !scale || !aligned16(x) || !aligned16(q)) return QWEN_ERR_ARG;
  long ld = (long)stride;
  void* args[] = {&x, &ld, &rows, &width, &q, &scale};
  return launch(dtype == QWEN_F16 ? quantize_kernel<_Float16>(width) : quantize_kernel<__bf16>(width), ((long)rows + 3) / 4, 256,
                args, stream);
}

namespace hd {
namespace {
template <class C, class T, bool STREAM>
int product_i8(const signed char* a, const float* as, const signed char* b, const float* bs, void* out, int tokens,
               int channels, int width, hipStream_t stream) {
  Product P = make_product<C>(Operand{(const char*)a, width, tokens, width}, Operand{(const char*)b, width, channels, width},
                              k_steps(width));
  Dequant<C, T, STREAM> e;
  e.out = (T*)out;
  e.xs = as;
  e.ws = bs;
  e.tokens = tokens;
  e.rows = channels;
  return launch_product(matmul_i8_kernel<C, T, STREAM>, grid_of<C>(P), C::THREADS, P, e, stream);
}
template <class T>
int product_i8(const signed char* a, const float* as, const signed char* b, const float* bs, void* out, int tokens,
               int channels, int width, hipStream_t stream) {
  typedef Tiles<Int8> TS;
  return with_tile<TS>(pick<TS>(tokens, channels), [&](auto c) {
    typedef decltype(c) C;
    if ((long)tokens * channels * (long)sizeof(T) > CACHES)
      return product_i8<C, T, true>(a, as, b, bs, out, tokens, channels, width, stream);
    return product_i8<C, T, false>(a, as, b, bs, out, tokens, channels, width, stream);
  });
}
}  // namespace

// rows of the engine's residual stream through its final norm (called by qwen_prefill_hidden)
int norm_rows(const float* x, const void* gain, int rows, void* out, hipStream_t stream) {
  const _Float16* g = (const _Float16*)gain;
  _Float16* o = (_Float16*)out;
  void* args[] = {&x, &g, &rows, &o};
  return launch((const void*)norm_rows_kernel, ((long)rows + 3) / 4, 256, args, stream);
}
}  // namespace hd

extern "C" int qwen_matmul_i8(const signed char* a, const float* a_scale, const signed char* b, const float* b_scale,
                              void* out, int out_dtype, int tokens, int channels, int width, hipStream_t stream) {
  // 65536 products of 8-bit numbers stay within 2^30
  if (tokens < 0 || tokens > MAX_TOKENS || channels < 0 || channels > MAX_CHANNELS || width < 16 || width % 16 != 0 || width > 65536) return QWEN_ERR_ARG;
  if (out_dtype != QWEN_F16 && out_dtype != QWEN_BF16 && out_dtype != QWEN_F32) return QWEN_ERR_ARG;
  if (tokens == 0 || channels == 0) return QWEN_OK;
  if (!a || !a_scale || !b || !b_scale || !out || !aligned16(a) || !aligned16(b) || !aligned16(out)) return QWEN_ERR_ARG;
  if (out_dtype == QWEN_F16) return product_i8<_Float16>(a, a_scale, b, b_scale, out, tokens, channels, width, stream);
  if (out_dtype == QWEN_BF16) return product_i8<__bf16>(a, a_scale, b, b_scale, out, tokens, channels, width, stream);
  return product_i8<float>(a, a_scale, b, b_scale, out, tokens, channels, width, stream);
}
