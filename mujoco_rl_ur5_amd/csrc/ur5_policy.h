// ur5_policy.h -- device code of the policy operators (include/ur5learn.h): softmax statistics over rows of logits, sampling, log-probabilities, the clipped policy
// loss and the preference loss with their gradients.
//
// A row holds one logit per action, action = rotation * pixels + pixel, and a mask of the pixels that every rotation shares (mask[j % mask_len]). Rows are long
// (240 000 actions) and few (1 .. some thousands), so a row is cut into `splits` pieces of `per` tiles; each piece is one workgroup that reads its logits ONCE and
// leaves a record of running sums relative to the piece's own maximum; whoever needs the row joins its records. All of it is bound by the bytes of the logits.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace ur5policy {

constexpr int THREADS = 256, VEC = 8, TILE = THREADS * VEC;   // a thread takes 8 neighbouring actions per tile: 2 (fp32) or 1 (16-bit) loads of 16 bytes, 8 mask bytes
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LOWEST = -3.402823466e38f;                    // start of a running maximum: finite, so -inf logits give exp2(-inf) = 0 and never inf - inf

enum { F32 = 0, F16 = 1, BF16 = 2 };

struct Rows {                       // rows of logits as the kernels see them
  const void* logits; const void* ref; const uint8_t* mask;
  long long stride, ref_stride, mask_stride;   // elements between rows
  int rows, actions, mask_len, splits, per;
};

struct Sums {                       // of (a piece of) a row, with e = exp(z - m)
  float m, mq;                      // maximum of the logits and of the reference's
  double s, t, k, sq;               // sum of e, of e (z - m) (the entropy's), of e (z - q) (the KL's), of exp(q - mq)
};
struct alignas(16) Part { Sums sums; double pad; };                  // what a piece of a row leaves in the workspace
struct alignas(16) Draw { double score, s; float m; int best; };    // the same for sampling: best noisy score and its action
static_assert(sizeof(Part) == 48 && sizeof(Draw) <= sizeof(Part), "records of the workspace");

// ---- loads. Rows start anywhere (odd strides, odd lengths), so 16-byte loads are declared with the element's alignment: gfx950 serves unaligned global loads.
typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint64_t U8 __attribute__((aligned(1)));

struct f32_t { using raw = float; };
struct f16_t { using raw = uint16_t; };
struct bf16_t { using raw = uint16_t; };
__device__ __forceinline__ float widen(f32_t, float v) { return v; }
__device__ __forceinline__ float widen(f16_t, uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ float widen(bf16_t, uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
__device__ __forceinline__ float narrow(f32_t, float v) { return v; }
__device__ __forceinline__ uint16_t narrow(f16_t, float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ uint16_t narrow(bf16_t, float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest, ties to even

__device__ __forceinline__ void load8(f32_t, const float* p, float* v) {
  const F4 a = *(const F4*)p, b = *(const F4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
}
template <typename T> __device__ __forceinline__ void load8(T tag, const uint16_t* p, float* v) {
  const U4 a = *(const U4*)p;
#pragma unroll
  for (int i = 0; i < 4; i++) { v[2 * i] = widen(tag, (uint16_t)a[i]); v[2 * i + 1] = widen(tag, (uint16_t)(a[i] >> 16)); }
}
__device__ __forceinline__ void store8(f32_t, float* p, const float* v) {
  F4 a, b;
#pragma unroll
  for (int i = 0; i < 4; i++) { a[i] = v[i]; b[i] = v[4 + i]; }
  *(F4*)p = a; *(F4*)(p + 4) = b;
}
template <typename T> __device__ __forceinline__ void store8(T tag, uint16_t* p, const float* v) {
  U4 a;
#pragma unroll
  for (int i = 0; i < 4; i++) a[i] = (uint32_t)narrow(tag, v[2 * i]) | (uint32_t)narrow(tag, v[2 * i + 1]) << 16;
  *(U4*)p = a;
}

// a thread's place in a row: action j and its mask position j mod mask_len, advanced without a division
struct Place {
  int j, p;
  __device__ __forceinline__ void next(int step_mod, int len) { j += TILE; p += step_mod; if (p >= len) p -= len; }
};
// one byte per action of the 8 at the place: may it be taken? Positions wrap inside the 8 where the mask does.
__device__ __forceinline__ uint64_t allowed8(const uint8_t* mask, int p, int len) {
  if (p + VEC <= len) return *(const U8*)(mask + p);
  uint64_t b = 0;
  for (int i = 0; i < VEC; i++) {
    b |= (uint64_t)(mask[p] != 0) << (8 * i);
    if (++p == len) p = 0;
  }
  return b;
}
// which of the 8 actions at the place may be taken, and logits with -inf where not; actions behind the row's end (!FULL) are not allowed either
template <bool MASK, bool FULL> __device__ __forceinline__ uint64_t allowed_at(const Rows& R, const uint8_t* mask, const Place& at) {
  return MASK && (FULL || at.j < R.actions) ? allowed8(mask, at.p, R.mask_len) : ~0ull;
}
template <typename T, bool MASK, bool FULL> __device__ __forceinline__ void take8(const Rows& R, const typename T::raw* row, uint64_t ok, const Place& at, float* z) {
  if (FULL) {
    load8(T{}, row + at.j, z);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) z[i] = at.j + i < R.actions ? widen(T{}, row[at.j + i]) : -INFINITY;
  }
  if (MASK) {
#pragma unroll
    for (int i = 0; i < VEC; i++) z[i] = (ok >> (8 * i)) & 0xff ? z[i] : -INFINITY;
  }
}
// whether the row's action counts: inside the row, allowed, and of a logit above -inf (a NaN counts: it has to show)
template <typename T> __device__ __forceinline__ bool action_counts(const Rows& R, int row, long long a, float* z_out) {
  if (a < 0 || a >= R.actions) return false;
  if (R.mask && !R.mask[row * R.mask_stride + a % R.mask_len]) return false;
  const float z = widen(T{}, ((const typename T::raw*)R.logits)[row * R.stride + a]);
  *z_out = z;
  return !(z == -INFINITY);
}

// ---- reductions over lanes
__device__ __forceinline__ float lanes_max(float v, int width = 64) { for (int o = width >> 1; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o)); return v; }
template <typename S> __device__ __forceinline__ S lanes_sum(S v, int width = 64) { for (int o = width >> 1; o; o >>= 1) v += __shfl_xor(v, o); return v; }
// exp(d) for d <= 0 by the hardware's 2^x (results below 2^-126 are 0)
__device__ __forceinline__ float fall(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
__device__ __forceinline__ float shrink(float from, float to) { return fall(from - to); }

// ---- SplitMix64's finaliser over a counter: the draws of sharding.scene_uniform, keyed by (seed, scene id, round, stream)
constexpr uint64_t GOLD = 0x9E3779B97F4A7C15ull;
__device__ __forceinline__ uint64_t mix64(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
// the noisy score whose argmax over a row is a draw from its softmax: z - log(-log u), in 64 bits so that two near scores are told apart
__device__ __forceinline__ double noisy_score(float z, uint64_t key, int j) {
  const uint64_t bits = mix64(key + (uint64_t)(j + 1) * GOLD) >> 11;
  const double u = fmax((double)bits * 0x1p-53, 0x1p-54);
  return (double)z - log(-log(u));
}
__device__ __forceinline__ bool better(double s, int i, double than, int at) { return s > than || (s == than && i < at); }

// running sums of one thread: fp32, over at most a few hundred terms
struct Running { float m, s, t, k, mq, sq; };
__device__ __forceinline__ Running nothing() { return Running{LOWEST, 0, 0, 0, LOWEST, 0}; }
// z (and q): 8 logits, -inf where not allowed. One maximum per 8, one rescaling, then the sums relative to it.
template <bool REF, bool ENTROPY> __device__ __forceinline__ void add8(Running& a, const float* z, const float* q, float* e) {
  float m = a.m;
#pragma unroll
  for (int i = 0; i < VEC; i++) m = fmaxf(m, z[i]);
  const float f = shrink(a.m, m);
  if (ENTROPY) a.t = f * (a.t + a.s * fmaxf(a.m - m, -1e30f));   // the sums move to the new maximum; an empty sum meets LOWEST - m: kept finite
  a.s *= f;
  if (REF) a.k *= f;
  a.m = m;
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const float d = z[i] - m;
    e[i] = fall(d);
    a.s += e[i];
    if (ENTROPY) a.t += e[i] * fmaxf(d, -1e4f);                 // e is 0 long before -1e4: 0 * -inf does not arise
    if (REF) a.k += e[i] == 0.f ? 0.f : e[i] * (z[i] - q[i]);
  }
  if (REF) {
    float mq = a.mq;
#pragma unroll
    for (int i = 0; i < VEC; i++) mq = fmaxf(mq, q[i]);
    a.sq *= shrink(a.mq, mq);
    a.mq = mq;
#pragma unroll
    for (int i = 0; i < VEC; i++) a.sq += fall(q[i] - mq);
  }
}
// From here on sums are 64 bits wide: a KL is a difference of two logarithms of sums, and what a few last additions lose in 32 bits (5e-8 of a sum, measured) would be
// 1e-6 of it. Their factors come from the precise exp where a single one weighs (joining wavefronts and records).
__device__ __forceinline__ double moved(double s, double t, float from, float to) { return t + s * fmaxf(from - to, -1e30f); }
// sums of `width` neighbouring lanes joined, in every one of them
__device__ __forceinline__ void join_lanes(Sums& a, int width, bool ref, bool entropy) {
  const float m = lanes_max(a.m, width);
  const double f = exp((double)a.m - m);
  if (entropy) a.t = lanes_sum(f * moved(a.s, a.t, a.m, m), width);
  a.s = lanes_sum(a.s * f, width);
  if (ref) {
    a.k = lanes_sum(a.k * f, width);
    const float mq = lanes_max(a.mq, width);
    a.sq = lanes_sum(a.sq * exp((double)a.mq - mq), width);
    a.mq = mq;
  }
  a.m = m;
}
// a wavefront's running sums joined, in every lane
__device__ __forceinline__ Sums join_wave(const Running& r, bool ref, bool entropy) {
  Sums a{lanes_max(r.m), r.mq, 0, 0, 0, 0};
  const float f = shrink(r.m, a.m);
  a.s = lanes_sum((double)(r.s * f));
  if (entropy) a.t = lanes_sum((double)(f * (r.t + r.s * fmaxf(r.m - a.m, -1e30f))));
  if (ref) {
    a.k = lanes_sum((double)(r.k * f));
    a.mq = lanes_max(r.mq);
    a.sq = lanes_sum((double)(r.sq * shrink(r.mq, a.mq)));
  }
  return a;
}

// what a piece of a row is to its threads
template <typename T, bool MASK> struct Piece {
  const typename T::raw* z_row; const uint8_t* mask;
  int tiles, whole, step_mod;       // tiles of the piece, and how many of them the row fills
  Place at;
  __device__ __forceinline__ Piece(const Rows& R, int row, int piece) {
    z_row = (const typename T::raw*)R.logits + row * R.stride;
    mask = MASK ? R.mask + row * R.mask_stride : nullptr;
    const int begin = piece * R.per * TILE, left = R.actions - begin;
    tiles = min(R.per, (left + TILE - 1) / TILE); whole = min(R.per, left / TILE);
    at.j = begin + (int)threadIdx.x * VEC;
    at.p = MASK ? at.j % R.mask_len : 0;
    step_mod = MASK ? TILE % R.mask_len : 0;
  }
};
// the workgroup's sums joined, in the first lanes of every wavefront
__device__ __forceinline__ Sums join_workgroup(const Running& r, bool ref, bool entropy) {
  __shared__ Sums wave[THREADS / 64];
  Sums a = join_wave(r, ref, entropy);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = a;
  __syncthreads();
  a = wave[threadIdx.x & (THREADS / 64 - 1)];
  join_lanes(a, THREADS / 64, ref, entropy);
  return a;
}

// ---- statistics of the pieces of rows. Grid: rows * splits workgroups, the pieces of a row next to each other. fp32 sums: a thread adds at most 8 * per terms,
// lanes and pieces join in trees.
template <typename T, bool MASK, bool REF, bool ENTROPY> __device__ __forceinline__ Sums piece_sums(const Rows& R, int row, int piece) {
  Piece<T, MASK> P(R, row, piece);
  const auto* q_row = REF ? (const typename T::raw*)R.ref + row * R.ref_stride : nullptr;
  Running a = nothing();
  float z[VEC], q[VEC], e[VEC];
#pragma unroll 2
  for (int i = 0; i < P.whole; i++) {
    const uint64_t ok = allowed_at<MASK, true>(R, P.mask, P.at);
    take8<T, MASK, true>(R, P.z_row, ok, P.at, z);
    if (REF) take8<T, MASK, true>(R, q_row, ok, P.at, q);
    add8<REF, ENTROPY>(a, z, q, e);
    P.at.next(P.step_mod, R.mask_len);
  }
  if (P.whole < P.tiles) {
    const uint64_t ok = allowed_at<MASK, false>(R, P.mask, P.at);
    take8<T, MASK, false>(R, P.z_row, ok, P.at, z);
    if (REF) take8<T, MASK, false>(R, q_row, ok, P.at, q);
    add8<REF, ENTROPY>(a, z, q, e);
  }
  return join_workgroup(a, REF, ENTROPY);
}

template <typename T, bool MASK, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_stats(Rows R, const int64_t* action, Part* parts, int* counts) {
  const int row = blockIdx.x / R.splits, piece = blockIdx.x % R.splits;
  const Sums a = piece_sums<T, MASK, REF, true>(R, row, piece);
  if (threadIdx.x == 0) {
    parts[blockIdx.x] = Part{a, 0};
    float z;
    if (piece == 0) counts[row] = action_counts<T>(R, row, action[row], &z);
  }
}

// the records of a row joined by `width` neighbouring lanes (`lane`: this one's place among them), in every one of them
__device__ __forceinline__ Sums join_row(const Part* parts, int splits, int lane, int width, bool ref) {
  Sums a{LOWEST, LOWEST, 0, 0, 0, 0};
  for (int i = lane; i < splits; i += width) {
    const Sums p = parts[i].sums;
    const float m = fmaxf(a.m, p.m), mq = fmaxf(a.mq, p.mq);
    const double f = exp((double)a.m - m), g = exp((double)p.m - m);
    a.t = f * moved(a.s, a.t, a.m, m) + g * moved(p.s, p.t, p.m, m);
    a.s = f * a.s + g * p.s;
    if (ref) {
      a.k = f * a.k + g * p.k;
      a.sq = a.sq * exp((double)a.mq - mq) + p.sq * exp((double)p.mq - mq);
    }
    a.m = m; a.mq = mq;
  }
  join_lanes(a, width, ref, true);
  return a;
}

// ---- log-probability of an action and entropy per row: a wavefront joins a row's records. logp 0 where the action lies outside the row (no action), -inf where it
// may not be taken; entropy 0 where nothing may.
template <typename T> __device__ __forceinline__ void write_logp(const Rows& R, int row, const Sums& a, const int64_t* action, float* logp, float* entropy) {
  const long long at = action[row];
  float z = 0;
  const bool counts = action_counts<T>(R, row, at, &z);
  const double ls = a.s > 0 ? log(a.s) : a.s - a.s;   // a NaN sum stays NaN
  logp[row] = counts ? (float)((double)z - a.m - ls) : at < 0 || at >= R.actions ? 0.f : -INFINITY;
  if (entropy) entropy[row] = a.s == 0 ? 0.f : (float)(ls - a.t / a.s);
}
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_logp(Rows R, const int64_t* action, Part* parts, float* logp, float* entropy) {
  const int row = blockIdx.x / R.splits, piece = blockIdx.x % R.splits;
  const Sums a = piece_sums<T, MASK, false, true>(R, row, piece);
  if (threadIdx.x) return;
  if (R.splits == 1) write_logp<T>(R, row, a, action, logp, entropy);
  else parts[blockIdx.x] = Part{a, 0};
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_policy_logp_rows(Rows R, const int64_t* action, const Part* parts, float* logp, float* entropy) {
  const int row = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= R.rows) return;
  const Sums a = join_row(parts + (size_t)row * R.splits, R.splits, lane, 64, false);
  if (lane == 0) write_logp<T>(R, row, a, action, logp, entropy);
}

// ---- sampling. argmax_j z_j - log(-log u_j) is a draw from softmax(z). Two logarithms in 64 bits per action would cost more than reading it, and nearly every action
// is far from winning: with E = -log u >= 1 - u, action j can only reach score `bar` if 1 - u_j <= exp(z_j - bar) -- one product and one comparison on the exp that the
// softmax's sum needs anyway. `bar` is the best score any thread of the workgroup has seen (less a margin over every rounding below), so about one action per
// piece passes and is scored in 64 bits; equal scores go to the lower action, so the result does not depend on who was first.
__device__ __forceinline__ int ordered(float v) { const int b = __float_as_int(v); return b ^ ((b >> 31) & 0x7fffffff); }
__device__ __forceinline__ float unordered(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }
__device__ __forceinline__ float below(double score) { return (float)score - (1e-4f + 1e-6f * fabsf((float)score)); }

struct Best { double score; int at; };
__device__ __forceinline__ void join_best(Best& b, int width) {
  for (int o = width >> 1; o; o >>= 1) {
    const double s = __shfl_xor(b.score, o);
    const int i = __shfl_xor(b.at, o);
    if (better(s, i, b.score, b.at)) { b.score = s; b.at = i; }
  }
}
// 1 - u of 8 neighbouring draws, rounded down to 32 bits
__device__ __forceinline__ void missing8(uint64_t key, int j, uint32_t* w) {
  uint64_t c = key + (uint64_t)(j + 1) * GOLD;
#pragma unroll
  for (int i = 0; i < VEC; i++, c += GOLD) {
    uint64_t x = (c ^ (c >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    const uint32_t hi = (uint32_t)(x >> 32);
    w[i] = ~(hi ^ (hi >> 31));
  }
}
template <typename T> __device__ __forceinline__ void draw8(const Rows& R, const typename T::raw* row, uint64_t key, const Place& at, const Running& a, const float* z,
                                                            const float* e, bool first, int* bar, Best& best) {
  uint32_t w[VEC];
  missing8(key, at.j, w);
  if (first) {   // no score yet: a bound from below, E <= (1 - u) / u, one fast logarithm per action
    float low = -INFINITY;
#pragma unroll
    for (int i = 0; i < VEC; i++) low = fmaxf(low, z[i] - 0.693147181f * __log2f(((float)w[i] + 1.f) / (float)~w[i]));
    low = lanes_max(low);
    if ((threadIdx.x & 63) == 0) atomicMax(bar, ordered(below(low)));
  }
  const float reach = fminf(__builtin_amdgcn_exp2f((a.m - unordered(__hip_atomic_load(bar, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP))) * LOG2E), 1e30f) * (1.0001f * 4294967296.f);
  uint32_t near = 0;
#pragma unroll
  for (int i = 0; i < VEC; i++) near |= (e[i] > 0 && (float)w[i] <= e[i] * reach) ? 1u << i : 0u;
  while (near) {
    const int j = at.j + __ffs(near) - 1;
    near &= near - 1;
    const double s = noisy_score(widen(T{}, row[j]), key, j);
    if (better(s, j, best.score, best.at)) {
      best = Best{s, j};
      atomicMax(bar, ordered(below(s)));
    }
  }
}
// the drawn action (-1: nothing may be taken, log-probability 0) and its log-probability
template <typename T> __device__ __forceinline__ void write_draw(const Rows& R, int row, float m, double s, const Best& b, int64_t* action, float* logp) {
  const bool some = b.at >= 0 && b.at < R.actions;
  action[row] = some ? b.at : -1;
  logp[row] = some ? (float)((double)widen(T{}, ((const typename T::raw*)R.logits)[row * R.stride + b.at]) - m - log(s)) : s == 0 ? 0.f : NAN;
}
constexpr int NOBODY = 0x7fffffff;
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_sample(Rows R, uint64_t offset, const int64_t* gids, Draw* draws, int64_t* action, float* logp) {
  const int row = blockIdx.x / R.splits, piece = blockIdx.x % R.splits;
  const uint64_t key = mix64((uint64_t)gids[row] * GOLD + offset);
  __shared__ int bar;
  __shared__ Best wave[THREADS / 64];
  if (threadIdx.x == 0) bar = ordered(-INFINITY);
  __syncthreads();
  Piece<T, MASK> P(R, row, piece);
  Running a = nothing();
  Best best{-INFINITY, NOBODY};
  float z[VEC], e[VEC];
  for (int i = 0; i < P.whole; i++) {
    take8<T, MASK, true>(R, P.z_row, allowed_at<MASK, true>(R, P.mask, P.at), P.at, z);
    add8<false, false>(a, z, nullptr, e);
    draw8<T>(R, P.z_row, key, P.at, a, z, e, i == 0, &bar, best);
    P.at.next(P.step_mod, R.mask_len);
  }
  if (P.whole < P.tiles) {
    take8<T, MASK, false>(R, P.z_row, allowed_at<MASK, false>(R, P.mask, P.at), P.at, z);
    add8<false, false>(a, z, nullptr, e);
    draw8<T>(R, P.z_row, key, P.at, a, z, e, P.whole == 0, &bar, best);
  }
  join_best(best, 64);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = best;
  const Sums sums = join_workgroup(a, false, false);   // (its barrier stands between the wavefronts' bests and their join)
  best = wave[threadIdx.x & (THREADS / 64 - 1)];
  join_best(best, THREADS / 64);
  if (threadIdx.x) return;
  if (R.splits == 1) write_draw<T>(R, row, sums.m, sums.s, best, action, logp);
  else draws[blockIdx.x] = Draw{best.score, sums.s, sums.m, best.at};
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_policy_sample_rows(Rows R, const Draw* draws, int64_t* action, float* logp) {
  const int row = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= R.rows) return;
  Sums a{LOWEST, LOWEST, 0, 0, 0, 0};
  Best best{-INFINITY, NOBODY};
  for (int i = lane; i < R.splits; i += 64) {
    const Draw d = draws[(size_t)row * R.splits + i];
    const float m = fmaxf(a.m, d.m);
    a.s = a.s * exp((double)a.m - m) + d.s * exp((double)d.m - m);
    a.m = m;
    if (better(d.score, d.best, best.score, best.at)) best = Best{d.score, d.best};
  }
  join_lanes(a, 64, false, false);
  join_best(best, 64);
  if (lane == 0) write_draw<T>(R, row, a.m, a.s, best, action, logp);
}

// ---- gradients. Both losses have, per row, dL/dz_j = p_j (c0 + kl_coef (z_j - q_j - gap) + entropy_coef (z_j - m - level)) + [j = action] take, times one factor.
struct Slope { float m, rs, c0, kl, gap, entropy, level, take; };

template <typename T, bool MASK, bool REF, bool FULL>
__device__ __forceinline__ void slope8(const Rows& R, const Piece<T, MASK>& P, const typename T::raw* q_row, const Slope& S, int action, typename T::raw* out) {
  const Place& at = P.at;
  float z[VEC], q[VEC], g[VEC];
  const uint64_t ok = allowed_at<MASK, FULL>(R, P.mask, at);
  take8<T, MASK, FULL>(R, P.z_row, ok, at, z);
  if (REF) take8<T, MASK, FULL>(R, q_row, ok, at, q);
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const float d = z[i] - S.m, p = fall(d) * S.rs;
    float v = S.c0 + S.entropy * (d - S.level);
    if (REF) v += S.kl * (z[i] - q[i] - S.gap);
    g[i] = p == 0.f ? 0.f : p * v;                       // not allowed, or too unlikely for 32 bits: the limit, whatever q holds
    if (at.j + i == action) g[i] += S.take;
  }
  if (FULL) {
    store8(T{}, out + at.j, g);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) if (at.j + i < R.actions) out[at.j + i] = narrow(T{}, g[i]);
  }
}
// a piece of a row of the gradient; a row that does not count is zero and its logits are not read
template <typename T, bool MASK, bool REF> __device__ __forceinline__ void write_slope(const Rows& R, int row, int piece, const Slope& S, long long action, bool counts, void* grad) {
  typename T::raw* out = (typename T::raw*)grad + (long long)row * R.actions;
  Piece<T, MASK> P(R, row, piece);
  if (!counts) {
    const float zero[VEC] = {};
    for (int i = 0; i < P.tiles; i++, P.at.j += TILE) {
      if (P.at.j + VEC <= R.actions) store8(T{}, out + P.at.j, zero);
      else for (int n = P.at.j; n < R.actions; n++) out[n] = narrow(T{}, 0.f);
    }
    return;
  }
  const auto* q_row = REF ? (const typename T::raw*)R.ref + row * R.ref_stride : nullptr;
#pragma unroll 2
  for (int i = 0; i < P.whole; i++) {
    slope8<T, MASK, REF, true>(R, P, q_row, S, (int)action, out);
    P.at.next(P.step_mod, R.mask_len);
  }
  if (P.whole < P.tiles) slope8<T, MASK, REF, false>(R, P, q_row, S, (int)action, out);
}

// ---- clipped policy loss. Per row: ratio r = exp(logp - old), L = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl_coef KL(p || q) - entropy_coef H; the mean over the rows that count.
struct Clip {
  const int64_t* action; const float* old_logp; const float* advantage;
  float lo, hi, kl_coef, entropy_coef, scale;   // scale: a factor of the gradient
  const float* upstream;                        // another, on the device (autograd's), or null
};
struct ClipRow { float logp, kl, entropy, loss, take; double shift, ls; };
// normalisers in 64 bits: KL = k / s - (lse - lse_q) is a small difference of large numbers
template <typename T, bool REF> __device__ __forceinline__ ClipRow clip_row(const Rows& R, const Clip& C, int row, const Sums& a) {
  ClipRow c{};
  c.ls = log(a.s);
  c.shift = REF ? (double)a.m - a.mq + c.ls - log(a.sq) : 0;
  const float z = widen(T{}, ((const typename T::raw*)R.logits)[row * R.stride + C.action[row]]), adv = C.advantage[row];
  c.logp = (float)((double)z - a.m - c.ls);
  c.kl = REF ? (float)(a.k / a.s - c.shift) : 0;
  c.entropy = (float)(c.ls - a.t / a.s);
  const float ratio = expf(c.logp - C.old_logp[row]), free = ratio * adv, held = fminf(fmaxf(ratio, 1 - C.lo), 1 + C.hi) * adv;
  c.take = held < free ? 0.f : -adv * ratio;     // the clipped branch has no slope; NaN stays
  c.loss = -(held < free ? held : free) + (REF ? C.kl_coef * c.kl : 0.f) - C.entropy_coef * c.entropy;
  return c;
}
__device__ __forceinline__ int count_rows(const int* counts, int rows) {   // of the workgroup, in every thread
  __shared__ int wave[THREADS / 64];
  int n = 0;
  for (int i = threadIdx.x; i < rows; i += THREADS) n += counts[i];
  n = lanes_sum(n);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
  for (int i = 0; i < THREADS / 64; i++) n += wave[i];
  return n;
}
// loss and per-row terms, by one workgroup: groups of `width` lanes join a row's records; row losses add up in 64 bits in a fixed order
template <typename T, bool REF> __device__ __forceinline__ void clip_loss(const Rows& R, const Clip& C, const Part* parts, const int* counts, float* loss, float* logp, float* kl, float* entropy) {
  int width = 1;
  while (width < 64 && width < R.splits) width *= 2;
  const int lane = threadIdx.x & (width - 1);
  double sum = 0;
  for (int base = 0; base < R.rows; base += THREADS / width) {     // every lane takes every turn: the joins shuffle
    const int row = base + threadIdx.x / width;
    const bool in = row < R.rows;
    const Sums a = join_row(parts + (size_t)(in ? row : 0) * R.splits, R.splits, lane, width, REF);
    if (!in || lane) continue;
    ClipRow c{};
    if (counts[row]) c = clip_row<T, REF>(R, C, row, a);
    logp[row] = c.logp; kl[row] = c.kl; entropy[row] = c.entropy;
    sum += c.loss;
  }
  __shared__ double wave[THREADS / 64];
  sum = lanes_sum(sum);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = sum;
  const int n = count_rows(counts, R.rows);      // (its barrier)
  if (threadIdx.x == 0) {
    sum = 0;
    for (int i = 0; i < THREADS / 64; i++) sum += wave[i];
    *loss = (float)(sum / (n > 1 ? n : 1));
  }
}
template <typename T, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_clip_loss(Rows R, Clip C, const Part* parts, const int* counts, float* loss, float* logp, float* kl, float* entropy) {
  clip_loss<T, REF>(R, C, parts, counts, loss, logp, kl, entropy);
}
// the gradient's pieces, in the statistics' order and, as 8 workgroups come before them, on the same XCD (whose L2 then holds a piece's logits if they fit). The first
// of the 8 writes the loss, if asked for, while the others run.
constexpr int FIRST = 8;
template <typename T, bool MASK, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_clip_grad(Rows R, Clip C, const Part* parts, const int* counts, void* grad, float* loss, float* logp, float* kl, float* entropy) {
  const int block = (int)blockIdx.x - FIRST;
  if (block < 0) {
    if (loss && blockIdx.x == 0) clip_loss<T, REF>(R, C, parts, counts, loss, logp, kl, entropy);
    return;
  }
  const int row = block / R.splits, piece = block % R.splits;
  const bool on = counts[row];
  __shared__ Slope shared;
  const int n = count_rows(counts, R.rows);
  if (on) {
    const Sums a = join_row(parts + (size_t)row * R.splits, R.splits, threadIdx.x & 63, 64, REF);
    if (threadIdx.x == 0) {
      const ClipRow c = clip_row<T, REF>(R, C, row, a);
      const float w = (C.upstream ? *C.upstream : 1.f) * C.scale / (float)n;
      shared = Slope{a.m, (float)(w / a.s), -c.take, C.kl_coef, (float)(c.shift + c.kl), C.entropy_coef, (float)(c.ls - c.entropy), w * c.take};
    }
  }
  __syncthreads();
  write_slope<T, MASK, REF>(R, row, piece, shared, C.action[row], on, grad);
}

// ---- preference loss. Episodes are runs of rows: episode k holds the rows offsets[k] .. offsets[k + 1]. S_k = sum over its counting rows of logp - ref_logp,
// margin_i = beta (S_2i - S_2i+1), loss = mean over pairs of (1 - eps) softplus(-margin) + eps softplus(margin).
struct Prefer {
  const int64_t* action; const float* ref_logp; const int64_t* offsets;
  int pairs; double beta, eps; float scale; const float* upstream;
};
struct RowState { float m, rs, weight; int counts; };   // weight: d loss / d logp of the row
constexpr int PAIR_THREADS = 1024;
// one workgroup: log-probabilities of all rows, then a wavefront per pair
template <typename T> __global__ void __launch_bounds__(PAIR_THREADS) ur5_policy_prefer_pairs(Rows R, Prefer P, const Part* parts, const int* counts, RowState* state, double* ratio, float* loss, float* margin) {
  int width = 1;
  while (width < 64 && width < R.splits) width *= 2;
  const int sub = threadIdx.x & (width - 1);
  for (int base = 0; base < R.rows; base += PAIR_THREADS / width) {
    const int row = base + threadIdx.x / width;
    const bool in = row < R.rows;
    const Sums a = join_row(parts + (size_t)(in ? row : 0) * R.splits, R.splits, sub, width, false);
    if (!in || sub) continue;
    double l = 0;
    if (counts[row]) l = (double)widen(T{}, ((const typename T::raw*)R.logits)[row * R.stride + P.action[row]]) - a.m - log(a.s) - P.ref_logp[row];
    ratio[row] = l;
    state[row] = RowState{a.m, (float)(1 / a.s), 0.f, counts[row]};
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ double sums[PAIR_THREADS / 64];
  double total = 0;
  for (int i = wave; i < P.pairs; i += PAIR_THREADS / 64) {
    long long end[3];
    for (int k = 0; k < 3; k++) end[k] = min(max(P.offsets[2 * i + k], 0ll), (long long)R.rows);   // offsets outside the rows are taken as their ends
    double d = 0;
    for (long long r = end[0] + lane; r < end[1]; r += 64) d += ratio[r];
    for (long long r = end[1] + lane; r < end[2]; r += 64) d -= ratio[r];
    const double mg = P.beta * lanes_sum(d);
    const double up = 1 / (1 + exp(mg));                                       // sigmoid(-margin)
    const double soft = fmax(mg, 0.0) + log1p(exp(-fabs(mg)));                 // softplus(margin)
    if (lane == 0) { margin[i] = (float)mg; total += (1 - P.eps) * (soft - mg) + P.eps * soft; }
    const float w = (float)(-P.beta * ((1 - P.eps) * up - P.eps * (1 - up)) / P.pairs);
    for (long long r = end[0] + lane; r < end[1]; r += 64) state[r].weight = w;
    for (long long r = end[1] + lane; r < end[2]; r += 64) state[r].weight = -w;
  }
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0;
    for (int k = 0; k < PAIR_THREADS / 64; k++) total += sums[k];
    *loss = (float)(total / P.pairs);
  }
}
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_prefer_grad(Rows R, Prefer P, const RowState* state, void* grad) {
  const int row = blockIdx.x / R.splits, piece = blockIdx.x % R.splits;
  const RowState s = state[row];
  const float w = s.weight * (P.upstream ? *P.upstream : 1.f) * P.scale;
  const Slope S{s.m, s.rs, -w, 0, 0, 0, 0, w};
  write_slope<T, MASK, false>(R, row, piece, S, P.action[row], s.counts && s.weight != 0.f, grad);
}

}  // namespace ur5policy
