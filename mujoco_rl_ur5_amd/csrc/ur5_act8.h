// ur5_act8.h -- device code of the 8-bit activation checkpoints (include/ur5learn.h): packing, restoring, and a pointwise convolution's weight gradient that reads the
// codes as they are.
#pragma once
#include "ur5_policy.h"

namespace ur5act8 {
using ur5policy::store8; using ur5policy::widen; using ur5policy::narrow;
using ur5policy::f32_t; using ur5policy::f16_t; using ur5policy::bf16_t; using ur5policy::yes; using ur5policy::no;

constexpr int GROUP = 64, THREADS = 256;
constexpr float ZERO_BELOW = 1e-30f;
constexpr float MOST_SCALE = 0x1.020406p+121f;            // the largest fp32 s with a finite 127 s: a group of fp32's largest values stays finite

// ---- pack and unpack move 4 (2) + 1.06 bytes per value and are bound by them: 164 M fp32 values, one MI355X, 133 + 113 us, 6.3 and 7.4 TB/s (with 8 fp32 values per lane,
// so that a wavefront's 16-byte loads skip every second 16 bytes, and plain accesses: 168 + 150).
// code = the integer nearest to x / s, exactly: the quotient by a reciprocal is right to 1e-4, so the code is floor or floor + 1 of it, and the sign of
// fma(-(floor + 1/2), s, x) -- one rounding, never through zero -- says which.
__device__ __forceinline__ int nearest_code(float x, float s, float per) {
  const float f = floorf(x * per), over = fmaf(-(f + 0.5f), s, x);
  const int c = (int)f;
  return c + (over > 0.f || (over == 0.f && (c & 1)));
}
// A lane holds as many neighbouring values as a 16-byte load brings, so that a wavefront's load or store is one run of memory; each thread has two groups under way.
template <typename T> struct Lane {
  static constexpr int PER = 16 / sizeof(typename T::raw), LANES = GROUP / PER, GROUPS = 2 * THREADS / LANES;   // values per lane, lanes per group, groups per workgroup
};
__device__ __forceinline__ void take(f32_t, const float* p, float* v) {
  const ur5policy::F4 a = __builtin_nontemporal_load((const ur5policy::F4*)p);     // read once
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = a[i];
}
template <typename T> __device__ __forceinline__ void take(T tag, const uint16_t* p, float* v) { ur5policy::unpack8(ur5policy::fetch8_last<T>(p), v); }
template <typename Past> __device__ __forceinline__ void put(f32_t, float* p, const float* v, Past past) {
  ur5policy::F4 a;
#pragma unroll
  for (int i = 0; i < 4; i++) a[i] = v[i];
  ur5policy::put((ur5policy::F4*)p, a, past);
}
template <typename T, typename Past> __device__ __forceinline__ void put(T tag, uint16_t* p, const float* v, Past past) { store8(tag, p, v, past); }

// where this thread's two groups lie: group, first value of the lane, and how many of the lane's values exist (0: no such group)
struct Where { unsigned g; long long at; int left; };
template <typename T> __device__ __forceinline__ void locate(unsigned groups, unsigned total, long long size, Where* w) {
  using L = Lane<T>;
  const unsigned lane = threadIdx.x % L::LANES, g = blockIdx.x * L::GROUPS + threadIdx.x / L::LANES;
  if (size == (long long)groups * GROUP) {                    // planes of whole groups lie like one
#pragma unroll
    for (int k = 0; k < 2; k++) {
      w[k].g = g + k * (L::GROUPS / 2);
      w[k].at = (long long)w[k].g * GROUP + lane * L::PER;
      w[k].left = w[k].g < total ? L::PER : 0;
    }
    return;
  }
  unsigned plane = g / groups, at = g - plane * groups;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    w[k].g = g + k * (L::GROUPS / 2);
    if (k) for (at += L::GROUPS / 2; at >= groups; at -= groups) plane++;
    const long long first = (long long)at * GROUP + lane * L::PER;
    w[k].at = plane * size + first;
    w[k].left = w[k].g < total ? (int)min((long long)L::PER, max(0ll, size - first)) : 0;
  }
}
// the largest of the lanes of a group, in all of them
template <int LANES> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
  using ur5policy::dpp;
  v = max(v, (uint32_t)dpp<0xB1>((int)v));
  v = max(v, (uint32_t)dpp<0x4E>((int)v));
  v = max(v, (uint32_t)dpp<0x141>((int)v));
  return LANES == 16 ? max(v, (uint32_t)dpp<0x140>((int)v)) : v;
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_act8_pack(const typename T::raw* x, unsigned groups, unsigned total, long long size, int8_t* codes, float* scales) {
  using L = Lane<T>;
  const unsigned lane = threadIdx.x % L::LANES;
  Where w[2];
  locate<T>(groups, total, size, w);
  float v[2][L::PER];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (w[k].left == L::PER) take(T{}, x + w[k].at, v[k]);
    else for (int i = 0; i < L::PER; i++) v[k][i] = i < w[k].left ? widen(T{}, x[w[k].at + i]) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    uint32_t most = 0;                                        // magnitudes compare as integers, a NaN above everything
#pragma unroll
    for (int i = 0; i < L::PER; i++) most = max(most, __float_as_uint(v[k][i]) & 0x7fffffffu);
    most = group_max<L::LANES>(most);
    const float amax = __uint_as_float(most);
    const bool finite = most < 0x7f800000u, some = finite && amax >= ZERO_BELOW;
    const float s = some ? fminf(amax / 127.f, MOST_SCALE) : finite ? 0.f : NAN, per = some ? __builtin_amdgcn_rcpf(s) : 0.f;
    if (w[k].g >= total) return;                              // all lanes of a group leave together
    uint32_t c[L::PER / 4] = {};
    if (some) {
#pragma unroll
      for (int i = 0; i < L::PER; i++) c[i / 4] |= (uint32_t)(uint8_t)nearest_code(v[k][i], s, per) << (8 * (i % 4));
    }
    int8_t* to = codes + (size_t)w[k].g * GROUP + lane * L::PER;
    if (L::PER == 4) *(uint32_t*)to = c[0];
    else *(uint2*)to = uint2{c[0], c[L::PER / 4 - 1]};
    if (lane == 0) scales[w[k].g] = s;
  }
}

template <typename T, typename Past> __global__ void __launch_bounds__(THREADS) ur5_act8_unpack(const int8_t* codes, const float* scales, unsigned groups, unsigned total, long long size, typename T::raw* x) {
  using L = Lane<T>;
  const unsigned lane = threadIdx.x % L::LANES;
  Where w[2];
  locate<T>(groups, total, size, w);
  uint2 c[2];
  float s[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const unsigned g = min(w[k].g, total - 1);
    const int8_t* from = codes + (size_t)g * GROUP + lane * L::PER;
    if (L::PER == 4) c[k].x = *(const uint32_t*)from;
    else c[k] = *(const uint2*)from;
    s[k] = scales[g];
  }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    float v[L::PER];
#pragma unroll
    for (int i = 0; i < L::PER; i++) v[i] = (float)(int8_t)((i < 4 ? c[k].x : c[k].y) >> (8 * (i % 4))) * s[k];
    auto* p = x + w[k].at;
    if (w[k].left == L::PER) put(T{}, p, v, Past{});
    else for (int i = 0; i < L::PER; i++) if (i < w[k].left) p[i] = narrow(T{}, v[i]);
  }
}

// ---- ReLU whose backward pass needs a bit per value: 64 neighbouring lanes hold 64 PER values, word i of theirs has a bit per lane, for value i of each. Bound by memory: 2 x 4 (2)
// + 1/8 bytes per value in both directions (41 M fp32 values, one MI355X: 54 us each way, 6.2 TB/s; bf16 30 and 33 us).
template <typename T> struct Run { long long at; int left; long long word; };   // this thread's values: the first, how many exist, and the first word of its wavefront
template <typename T> __device__ __forceinline__ Run<T> run_of(int k, long long count) {
  const long long wave = ((long long)blockIdx.x * 2 + k) * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int PER = Lane<T>::PER;
  const long long at = (wave * 64 + (threadIdx.x & 63)) * PER;
  return Run<T>{at, (int)min((long long)PER, max(0ll, count - at)), wave * 64 * PER < count ? wave * PER : -1};
}
template <typename T> __device__ __forceinline__ void take_some(const typename T::raw* p, int left, float* v) {
  if (left == Lane<T>::PER) take(T{}, p, v);
  else for (int i = 0; i < Lane<T>::PER; i++) v[i] = i < left ? widen(T{}, p[i]) : 0.f;
}
template <typename T, typename Past> __device__ __forceinline__ void put_some(typename T::raw* p, int left, const float* v, Past past) {
  if (left == Lane<T>::PER) put(T{}, p, v, past);
  else for (int i = 0; i < Lane<T>::PER; i++) if (i < left) p[i] = narrow(T{}, v[i]);
}
template <typename T, typename Past> __global__ void __launch_bounds__(THREADS) ur5_act8_relu(const typename T::raw* x, long long count, typename T::raw* y, uint64_t* bits) {
  constexpr int PER = Lane<T>::PER;
  float v[2][PER];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const Run<T> r = run_of<T>(k, count);
    take_some<T>(x + r.at, r.left, v[k]);
  }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const Run<T> r = run_of<T>(k, count);
    if (r.word < 0) return;                                   // (a wavefront together)
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const bool passes = !(v[k][i] <= 0.f);                  // a NaN passes
      const uint64_t word = __ballot(passes);
      if ((threadIdx.x & 63) == i) mine = word;
      v[k][i] = passes ? v[k][i] : 0.f;
    }
    put_some<T>(y + r.at, r.left, v[k], Past{});
    if ((threadIdx.x & 63) < PER) bits[r.word + (threadIdx.x & 63)] = mine;
  }
}
template <typename T, typename Past> __global__ void __launch_bounds__(THREADS) ur5_act8_relu_grad(const typename T::raw* dy, const uint64_t* bits, long long count, typename T::raw* dx) {
  constexpr int PER = Lane<T>::PER;
  float v[2][PER];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const Run<T> r = run_of<T>(k, count);
    take_some<T>(dy + r.at, r.left, v[k]);
  }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const Run<T> r = run_of<T>(k, count);
    if (r.word < 0) return;
#pragma unroll
    for (int i = 0; i < PER; i++) v[k][i] = bits[r.word + i] >> (threadIdx.x & 63) & 1 ? v[k][i] : 0.f;
    put_some<T>(dx + r.at, r.left, v[k], Past{});
  }
}

// ---- weight gradient: dw[o][c] = sum over (image, pixel) of dy[o] x[c], a matrix product whose long axis is the pixels (both operands have them neighbouring).
// Codes are small integers, exact in 16-bit floats, and a group's scale is a factor of 64 pixels of one input channel: v_mfma_f32_32x32x16 runs over the 64 pixels on
// plain codes, and its 32 x 32 result is multiplied by the scales once -- a lane holds one column (one input channel) of it, so the scale is one register.
// fp32 gradients go in as three bf16 terms whose sum is the value exactly (8 + 8 + 8 bits, cut off, not rounded), 16-bit gradients as they are.
// A workgroup owns TO output x TC input channels of a range of groups; its WO x WC wavefronts own A x B results of 32 x 32 each. Per group, its threads read the TO x 64
// gradients in whole rows (256 bytes), cut them into terms and put them into LDS in the instruction's order -- 8 pixels of a channel are 16 bytes, channels next to each
// other, so that writes and reads of 16 bytes are free of bank conflicts --, once instead of once per wavefront. Codes go straight from memory into the lanes that need
// them: lane l holds channel l % 32 and pixels 32 (l / 32) .. + 31 of the group (the order of the pixels is free as long as both operands agree). Two buffers in LDS: while
// the matrix instructions run over group g, group g + 1 is cut into the other buffer and group g + 2 is on its way; one barrier per group.
// Ranges are `splits` in number, and ur5_act8_wgrad_sum adds their parts in order: no atomics, the same result every time.
// 12 images of 64 -> 128 channels and 100 x 100 fp32 pixels: 21 us (bf16 16). 61 MB of gradients and 8 MB of codes are 3.3 TB/s; 75 MB are fetched and 8 MB of parts written, 3.9. A
// workgroup's 99 KB of LDS leave one per CU, it has seven or eight groups in all, and one of them on its way: latency, not the memory's rate.
// 64 images of 256 -> 512 and 50 x 50: 148 us at 2.1 GHz, 176 in a loop, where the card holds its power by its clock (2.1 -> 1.75 GHz); the cycles are the same 310 k. The three bf16 products
// are 123 k of them per SIMD, the vector instructions that cut, convert and scale another 118 k, LDS reads about 60 k, and they add up instead of overlapping: the matrix pipes are busy for 44 %
// of a CU's busy cycles. (bf16 gradients, a third of the products and two thirds of the vector instructions: 108 and 115 us.)
typedef float F16 __attribute__((ext_vector_type(16)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef uint32_t U4a __attribute__((ext_vector_type(4)));
__device__ __forceinline__ F16 mfma(bf16_t, U4a a, U4a b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0); }
__device__ __forceinline__ F16 mfma(f16_t, U4a a, U4a b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0); }
template <typename T> struct Terms { static constexpr int N = 1; using kind = T; };
template <> struct Terms<f32_t> { static constexpr int N = 3; using kind = bf16_t; };

// 8 neighbouring gradients of a thread as they come from memory
template <typename T> struct Raw { uint32_t w[4]; };
template <> struct Raw<f32_t> { uint32_t w[8]; };
// first: where the 8 lie; left: how many of them lie inside the plane
template <typename T> __device__ __forceinline__ void fetch(Raw<T>& r, const typename T::raw* first, int left, bool whole) {
  constexpr int PER = 4 / sizeof(typename T::raw), WORDS = 8 / PER;
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
// the terms of 8 gradients, and what they add to the bias
__device__ __forceinline__ float cut(const Raw<f32_t>& r, U4a* term) {
  float sum = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t part[3][2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float v = __uint_as_float(r.w[2 * i + k]);
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
template <typename T> __device__ __forceinline__ float cut(const Raw<T>& r, U4a* term) {
  float sum = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    term[0][i] = r.w[i];
    sum += widen(T{}, (uint16_t)r.w[i]) + widen(T{}, (uint16_t)(r.w[i] >> 16));
  }
  return sum;
}
// 8 codes as 16-bit floats (a bf16 is the high half of the fp32 that holds so small an integer)
__device__ __forceinline__ uint32_t pair(bf16_t, float a, float b) { return high_halves(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ uint32_t pair(f16_t, float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }
template <typename K> __device__ __forceinline__ U4a code_operand(uint32_t lo, uint32_t hi) {
  U4a out;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t w = i < 2 ? lo : hi;
    const int sh = 16 * (i & 1);
    out[i] = pair(K{}, (float)(int8_t)(w >> sh), (float)(int8_t)(w >> (sh + 8)));
  }
  return out;
}

struct Wgrad {
  const int8_t* codes; const float* scales; const void* dy;
  long long size; int groups, n, cin, cout, splits, o_tiles, c_tiles;
  float* part; float* part_bias;      // [splits][cout][cin], [splits][cout]
};
// Groups that a plane fills come first; the planes' last, shorter groups are a second, plain loop.
template <typename T, int A, int B, int WO, int WC> __global__ void __launch_bounds__(64 * WO * WC, 2) ur5_act8_wgrad(Wgrad W) {
  using K = typename Terms<T>::kind;
  using R = typename T::raw;
  constexpr int N = Terms<T>::N, TO = 32 * A * WO, TC = 32 * B * WC, COUNT = 64 * WO * WC, ROWS = TO * 8 / COUNT;
  __shared__ U4a shared[2][N][8][TO + 1];                                // [buffer][term][8 pixels][output channel]
  // workgroups of one range sit on one XCD and run together: they share the range's gradients and codes in its L2 (less than 8 ranges: one after the other)
  const int tiles = W.o_tiles * W.c_tiles, b = blockIdx.x, xcds = W.splits & 7 ? 1 : 8;
  const int split = b % xcds + xcds * (b / xcds / tiles), tile = b / xcds % tiles;
  const int o0 = tile / W.c_tiles * TO, c0 = tile % W.c_tiles * TC;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
  const int wave_o = wave / WC * 32 * A, wave_c = wave % WC * 32 * B;
  const bool with_bias = W.part_bias && c0 == 0;

  // this thread's share of the gradients: 8 pixels of ROWS rows; channels behind the last: its values again, their results are not kept
  const int eight = threadIdx.x & 7, row = threadIdx.x >> 3;
  const R* dy[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) dy[i] = (const R*)W.dy + min(o0 + row + COUNT / 8 * i, W.cout - 1) * W.size + 8 * eight;
  long long group[B];
#pragma unroll
  for (int k = 0; k < B; k++) group[k] = (long long)min(c0 + wave_c + 32 * k + col, W.cin - 1) * W.groups;

  F16 acc[A][B] = {};
  float bias[ROWS] = {};
  struct Place { int image, at; };
  const auto cut_rows = [&](const Raw<T>* raw, int buffer, bool counts) {
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      U4a term[N];
      const float v = cut(raw[i], term);
      bias[i] += counts ? v : 0.f;
#pragma unroll
      for (int n = 0; n < N; n++) shared[buffer][n][eight][row + COUNT / 8 * i] = term[n];
    }
  };
  const auto fetch_rows = [&](const Place& p, Raw<T>* raw) {
    const long long plane = (long long)p.image * W.cout * W.size + (long long)p.at * GROUP;
#pragma unroll
    for (int i = 0; i < ROWS; i++) fetch<T>(raw[i], dy[i] + plane, 8, true);
  };
  struct Codes { U4a lo[B], hi[B]; float scale[B]; };
  const auto fetch_codes = [&](const Place& p, Codes& c) {
    const long long first = (long long)p.image * W.cin * W.groups + p.at;
#pragma unroll
    for (int k = 0; k < B; k++) {
      const U4a* at = (const U4a*)(W.codes + (first + group[k]) * GROUP + 32 * half);
      c.lo[k] = at[0]; c.hi[k] = at[1];
      c.scale[k] = W.scales[first + group[k]];
    }
  };
  const auto multiply = [&](int buffer, const Codes& c) {
    F16 sum[A][B] = {};
#pragma unroll
    for (int q = 0; q < 4; q++) {
      U4a term[A][N], v[B];
#pragma unroll
      for (int a = 0; a < A; a++)
#pragma unroll
        for (int n = 0; n < N; n++) term[a][n] = shared[buffer][n][4 * half + q][wave_o + 32 * a + col];
#pragma unroll
      for (int k = 0; k < B; k++) {
        const U4a& w = q < 2 ? c.lo[k] : c.hi[k];
        v[k] = code_operand<K>(w[2 * (q & 1)], w[2 * (q & 1) + 1]);
      }
#pragma unroll
      for (int n = N - 1; n >= 0; n--)
#pragma unroll
        for (int a = 0; a < A; a++)
#pragma unroll
          for (int k = 0; k < B; k++) sum[a][k] = mfma(K{}, term[a][n], v[k], sum[a][k]);
    }
#pragma unroll
    for (int a = 0; a < A; a++)
#pragma unroll
      for (int k = 0; k < B; k++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[a][k][i] = fmaf(c.scale[k], sum[a][k][i], acc[a][k][i]);
  };

  const int wholes = (int)(W.size / GROUP);
  const long long all = (long long)W.n * wholes, first = all * split / W.splits, last = all * (split + 1) / W.splits;
  if (first < last) {
    const auto next = [&](Place& p, long long g) {                       // the group after p, or p again at the range's end (a load too many, of something that is there)
      if (g + 1 < last && ++p.at == wholes) { p.at = 0; p.image++; }
    };
    Place ahead{(int)(first / wholes), (int)(first % wholes)}, now = ahead;
    Raw<T> raw[ROWS];
    Codes codes[2];
    fetch_rows(ahead, raw);
    fetch_codes(now, codes[0]);
    cut_rows(raw, 0, true);
    next(ahead, first);
    fetch_rows(ahead, raw);
    const auto step = [&](long long g, auto odd) {
      constexpr int me = decltype(odd)::value ? 1 : 0;
      __syncthreads();                                                   // group g is in its buffer, and everybody has read the other one
      next(now, g);
      fetch_codes(now, codes[me ^ 1]);
      cut_rows(raw, me ^ 1, g + 1 < last);                               // (behind the last group: once more, not counted)
      next(ahead, g + 1);
      fetch_rows(ahead, raw);
      multiply(me, codes[me]);
    };
    for (long long g = first; g < last; g += 2) {                        // by twos: what is on its way lands in registers of its own, nothing is moved (a move would wait for it)
      step(g, no{});
      if (g + 1 < last) step(g + 1, yes{});
    }
  }
  if (W.size % GROUP) {                                                  // the planes' last groups
    const int left = (int)min(8, max(0, (int)(W.size % GROUP) - 8 * eight));
    for (Place p{(int)((long long)W.n * split / W.splits), wholes}; p.image < (int)((long long)W.n * (split + 1) / W.splits); p.image++) {
      Raw<T> raw[ROWS];
      Codes codes;
      const long long plane = (long long)p.image * W.cout * W.size + (long long)p.at * GROUP;
#pragma unroll
      for (int i = 0; i < ROWS; i++) fetch<T>(raw[i], dy[i] + plane, left, false);
      fetch_codes(p, codes);
      __syncthreads();
      cut_rows(raw, 0, true);
      __syncthreads();
      multiply(0, codes);
    }
  }
#pragma unroll
  for (int a = 0; a < A; a++)
#pragma unroll
    for (int k = 0; k < B; k++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int o = o0 + wave_o + 32 * a + (i & 3) + 8 * (i >> 2) + 4 * half, c = c0 + wave_c + 32 * k + col;
        if (o < W.cout && c < W.cin) W.part[((size_t)split * W.cout + o) * W.cin + c] = acc[a][k][i];
      }
  if (with_bias) {
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      float v = bias[i];
      for (int o = 4; o; o >>= 1) v += __shfl_xor(v, o);
      const int o = o0 + row + COUNT / 8 * i;
      if (eight == 0 && o < W.cout) W.part_bias[(size_t)split * W.cout + o] = v;
    }
  }
}
// parts in order, in 64 bits: 32 outputs per workgroup, eight threads each (few outputs and many parts want many loads at once: 128 parts of 8192 weights 120 us with one thread each)
__global__ void __launch_bounds__(THREADS) ur5_act8_wgrad_sum(const float* part, const float* part_bias, int splits, int weights, int cout, float* dw, float* db) {
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  const bool is_weight = i < weights, is_bias = !is_weight && db && i - weights < cout;
  const float* p = is_weight ? part + i : part_bias + (i - weights);
  const size_t step = is_weight ? weights : cout;
  double s = 0;
  if (is_weight || is_bias)
#pragma unroll 4
    for (int k = share; k < splits; k += 8) s += p[k * step];
  __shared__ double sums[8][32];
  sums[share][threadIdx.x & 31] = s;
  __syncthreads();
  if (share) return;
  for (int k = 1; k < 8; k++) s += sums[k][threadIdx.x];
  if (is_weight) dw[i] = (float)s;
  else if (is_bias) db[i - weights] = (float)s;
}
}  // namespace ur5act8
