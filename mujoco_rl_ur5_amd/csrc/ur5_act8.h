// ur5_act8.h -- device code of the 8-bit activation checkpoints (include/ur5learn.h): packing, restoring, and a pointwise convolution's weight gradient that reads the
// codes as they are.
#pragma once
#include "ur5_policy.h"

namespace ur5act8 {
using ur5policy::load8; using ur5policy::store8; using ur5policy::widen; using ur5policy::narrow; using ur5policy::lanes_sum;
using ur5policy::f32_t; using ur5policy::f16_t; using ur5policy::bf16_t;

constexpr int GROUP = 64, THREADS = 256, LANES = 8;   // 8 lanes of 8 neighbouring values per group
constexpr float ZERO_BELOW = 1e-30f;
constexpr float MOST_SCALE = 0x1.020406p+121f;            // the largest fp32 s with a finite 127 s: a group of fp32's largest values stays finite

// ---- pack: reads each value once, writes a byte and 1/16 of a scale's byte for it; bound by the reads.
// code = the integer nearest to x / s, exactly: the quotient by a reciprocal is right to 1e-4, so the code is floor or floor + 1 of it, and the sign of
// fma(-(floor + 1/2), s, x) -- one rounding, never through zero -- says which.
__device__ __forceinline__ int nearest_code(float x, float s, float per) {
  const float f = floorf(x * per), over = fmaf(-(f + 0.5f), s, x);
  const int c = (int)f;
  return c + (over > 0.f || (over == 0.f && (c & 1)));
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_act8_pack(const typename T::raw* x, unsigned groups, unsigned total, long long size, int8_t* codes, float* scales) {
  const unsigned g = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  if (g >= total) return;                                     // all 8 lanes of a group leave together
  const unsigned plane = g / groups, at = (g - plane * groups) * GROUP + lane * 8;
  const auto* p = x + plane * size + at;
  float v[8];
  if (at + 8 <= size) load8(T{}, p, v);
  else for (int i = 0; i < 8; i++) v[i] = at + i < size ? widen(T{}, p[i]) : 0.f;
  uint32_t most = 0;                                          // magnitudes compare as integers, a NaN above everything
#pragma unroll
  for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  for (int o = LANES / 2; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
  const float amax = __uint_as_float(most);
  const bool finite = most < 0x7f800000u, some = finite && amax >= ZERO_BELOW;
  const float s = some ? fminf(amax / 127.f, MOST_SCALE) : finite ? 0.f : NAN, per = some ? __builtin_amdgcn_rcpf(s) : 0.f;
  uint64_t c = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) c |= (uint64_t)(uint8_t)(some ? nearest_code(v[i], s, per) : 0) << (8 * i);
  *(uint64_t*)(codes + (size_t)g * GROUP + lane * 8) = c;
  if (lane == 0) scales[g] = s;
}

template <typename T> __global__ void __launch_bounds__(THREADS) ur5_act8_unpack(const int8_t* codes, const float* scales, unsigned groups, unsigned total, long long size, typename T::raw* x) {
  const unsigned g = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  if (g >= total) return;
  const unsigned plane = g / groups, at = (g - plane * groups) * GROUP + lane * 8;
  const uint64_t c = *(const uint64_t*)(codes + (size_t)g * GROUP + lane * 8);
  const float s = scales[g];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)(int8_t)(c >> (8 * i)) * s;
  auto* p = x + plane * size + at;
  if (at + 8 <= size) store8(T{}, p, v);
  else for (int i = 0; i < 8; i++) if (at + i < size) p[i] = narrow(T{}, v[i]);
}

// ---- weight gradient: dw[o][c] = sum over (image, pixel) of dy[o] x[c], a matrix product whose long axis is the pixels (both operands have them neighbouring).
// Codes are small integers, exact in 16-bit floats, and a group's scale is a factor of 64 pixels of one input channel: v_mfma_f32_32x32x16 runs over the 64 pixels on
// plain codes, and its 32 x 32 result is multiplied by the scales once -- a lane holds one column (one input channel) of it, so the scale is one register.
// fp32 gradients go in as three bf16 terms whose sum is the value exactly (8 + 8 + 8 bits, cut off, not rounded), 16-bit gradients as they are.
// A wavefront owns 64 output x TC input channels of a range of groups and loads its operands straight into the instruction's lane layout: lane l holds channel l % 32
// and pixels 32 (l / 32) .. + 31 of the group (the order of the pixels is free as long as both operands agree). Four wavefronts split a workgroup's range and add up
// through LDS; workgroups split the pixels `splits` ways and ur5_act8_wgrad_sum adds their parts in order: no atomics, the same result every time.
typedef float F16 __attribute__((ext_vector_type(16)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef uint32_t U4a __attribute__((ext_vector_type(4)));
__device__ __forceinline__ F16 mfma(bf16_t, U4a a, U4a b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0); }
__device__ __forceinline__ F16 mfma(f16_t, U4a a, U4a b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0); }
template <typename T> struct Terms { static constexpr int N = 1; using kind = T; };
template <> struct Terms<f32_t> { static constexpr int N = 3; using kind = bf16_t; };

// 32 gradients of a lane as they come from memory
template <typename T> struct Raw { uint32_t w[16]; };
template <> struct Raw<f32_t> { uint32_t w[32]; };
// first: the row's 32 values; left: how many of them lie inside the plane
template <typename T> __device__ __forceinline__ void fetch(Raw<T>& r, const typename T::raw* first, int left, bool whole) {
  constexpr int PER = 4 / sizeof(typename T::raw), WORDS = 32 / PER;
  if (whole) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const ur5policy::U4 v = *(const ur5policy::U4*)(first + i * PER);
#pragma unroll
      for (int k = 0; k < 4; k++) r.w[i + k] = v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
      if (PER == 1) r.w[i] = i < left ? __builtin_bit_cast(uint32_t, (float)widen(T{}, first[i])) : 0u;
      else r.w[i] = (2 * i < left ? (uint32_t)first[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)first[2 * i + 1] << 16 : 0u);
    }
  }
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }   // {a's high half, b's high half}
// matrix operand of pixels 8 step .. 8 step + 7, and what it adds to the bias
__device__ __forceinline__ float operand(const Raw<f32_t>& r, int step, U4a* term) {
  float sum = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t part[3][2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float v = __uint_as_float(r.w[8 * step + 2 * i + k]);
      sum += v;
#pragma unroll
      for (int n = 0; n < 3; n++) {
        part[n][k] = __float_as_uint(v) & 0xffff0000u;
        v -= __uint_as_float(part[n][k]);
      }
    }
#pragma unroll
    for (int n = 0; n < 3; n++) term[n][i] = high_halves(part[n][0], part[n][1]);
  }
  return sum;
}
template <typename T> __device__ __forceinline__ float operand(const Raw<T>& r, int step, U4a* term) {
  float sum = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t w = r.w[4 * step + i];
    term[0][i] = w;
    sum += widen(T{}, (uint16_t)w) + widen(T{}, (uint16_t)(w >> 16));
  }
  return sum;
}
// 8 codes as 16-bit floats
template <typename K> __device__ __forceinline__ U4a code_operand(uint32_t lo, uint32_t hi) {
  U4a out;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t w = i < 2 ? lo : hi;
    const int sh = 16 * (i & 1);
    const float a = (float)(int8_t)(w >> sh), b = (float)(int8_t)(w >> (sh + 8));
    out[i] = (uint32_t)narrow(K{}, a) | (uint32_t)narrow(K{}, b) << 16;
  }
  return out;
}

struct Wgrad {
  const int8_t* codes; const float* scales; const void* dy;
  long long size; int groups, n, cin, cout, splits, o_tiles, c_tiles;
  float* part; float* part_bias;      // [splits][cout][cin], [splits][4][cout]
};
constexpr int TO = 64;
template <typename T, int TC> __global__ void __launch_bounds__(THREADS, 1) ur5_act8_wgrad(Wgrad W) {
  using K = typename Terms<T>::kind;
  constexpr int N = Terms<T>::N, A = TO / 32, B = TC / 32;
  // workgroups of one pixel range sit on one XCD and run together: they share the range's gradients and codes in its L2
  const int tiles = W.o_tiles * W.c_tiles, b = blockIdx.x;
  const int split = (b & 7) + 8 * ((b >> 3) / tiles), tile = (b >> 3) % tiles;
  if (split >= W.splits) return;
  const int o0 = tile / W.c_tiles * TO, c0 = tile % W.c_tiles * TC;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
  const long long all = (long long)W.n * W.groups, ranges = 4ll * W.splits;
  long long g = all * (4 * split + wave) / ranges;
  const long long end = all * (4 * split + wave + 1) / ranges;
  F16 acc[A][B] = {};
  float bias[A] = {};
  int image = (int)(g / W.groups), at = (int)(g % W.groups);
  for (; g < end; g++) {
    Raw<T> raw[A];
    const bool whole = (at + 1) * (long long)GROUP <= W.size;
    const long long pixel = (long long)at * GROUP + 32 * half;
    const int left = (int)min(32ll, max(0ll, W.size - pixel));
#pragma unroll
    for (int a = 0; a < A; a++) {
      const int o = min(o0 + 32 * a + col, W.cout - 1);                  // channels behind the last: its values again, their results are not kept
      fetch<T>(raw[a], (const typename T::raw*)W.dy + ((long long)image * W.cout + o) * W.size + pixel, left, whole);
    }
    uint32_t code[B][8];
    float scale[B];
#pragma unroll
    for (int k = 0; k < B; k++) {
      const int c = min(c0 + 32 * k + col, W.cin - 1);
      const long long group = ((long long)image * W.cin + c) * W.groups + at;
      const U4a* p = (const U4a*)(W.codes + group * GROUP + 32 * half);
      const U4a u = p[0], v = p[1];
#pragma unroll
      for (int i = 0; i < 4; i++) { code[k][i] = u[i]; code[k][4 + i] = v[i]; }
      scale[k] = W.scales[group];
    }
    U4a term[A][4][N];
#pragma unroll
    for (int a = 0; a < A; a++)
#pragma unroll
      for (int s = 0; s < 4; s++) bias[a] += operand(raw[a], s, term[a][s]);
#pragma unroll
    for (int k = 0; k < B; k++) {
      F16 sum[A] = {};
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const U4a x = code_operand<K>(code[k][2 * s], code[k][2 * s + 1]);
#pragma unroll
        for (int n = N - 1; n >= 0; n--)
#pragma unroll
          for (int a = 0; a < A; a++) sum[a] = mfma(K{}, term[a][s][n], x, sum[a]);
      }
#pragma unroll
      for (int a = 0; a < A; a++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[a][k][i] = fmaf(scale[k], sum[a][i], acc[a][k][i]);
    }
    if (++at == W.groups) { at = 0; image++; }
  }
  // the four wavefronts' tiles, 32 x 32 at a time
  __shared__ float block[4][32][33];
#pragma unroll
  for (int a = 0; a < A; a++)
#pragma unroll
    for (int k = 0; k < B; k++) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; i++) block[wave][(i & 3) + 8 * (i >> 2) + 4 * half][col] = acc[a][k][i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = (threadIdx.x >> 5) + 8 * i, c = threadIdx.x & 31, o = o0 + 32 * a + r, ci = c0 + 32 * k + c;
        if (o < W.cout && ci < W.cin) W.part[((size_t)split * W.cout + o) * W.cin + ci] = block[0][r][c] + block[1][r][c] + block[2][r][c] + block[3][r][c];
      }
    }
  if (W.part_bias && c0 == 0) {
#pragma unroll
    for (int a = 0; a < A; a++) {
      const float v = bias[a] + __shfl_xor(bias[a], 32);
      const int o = o0 + 32 * a + col;
      if (half == 0 && o < W.cout) W.part_bias[((size_t)split * 4 + wave) * W.cout + o] = v;
    }
  }
}
// parts in order, in 64 bits
__global__ void __launch_bounds__(THREADS) ur5_act8_wgrad_sum(const float* part, const float* part_bias, int splits, int weights, int cout, float* dw, float* db) {
  const int i = blockIdx.x * THREADS + threadIdx.x;
  if (i < weights) {
    double s = 0;
    for (int k = 0; k < splits; k++) s += part[(size_t)k * weights + i];
    dw[i] = (float)s;
  } else if (db && i - weights < cout) {
    double s = 0;
    for (int k = 0; k < 4 * splits; k++) s += part_bias[(size_t)k * cout + i - weights];
    db[i - weights] = (float)s;
  }
}
}  // namespace ur5act8
