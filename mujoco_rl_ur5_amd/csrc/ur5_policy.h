// ur5_policy.h -- device code of the policy operators (include/ur5learn.h): softmax statistics over rows of logits, sampling, log-probabilities, the clipped policy
// loss and the preference loss with their gradients.
//
// A row holds one logit per action, action = map * pixels + pixel (a map per wrist rotation), and a mask of the pixels that all maps share (mask[j % pixels]). Rows are long
// (240 000 actions) and few (1 .. some thousands), so a row is cut into pieces, a workgroup each: some pixels of some maps. A piece reads its logits ONCE and leaves a record
// of running sums relative to its own maximum; whoever needs the row joins its records. All of it is bound by the bytes of the logits and, next, by the instructions per logit.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace ur5policy {

constexpr int THREADS = 256, VEC = 8;                         // a thread takes 8 neighbouring actions at a time: 2 (fp32) or 1 (16-bit) loads of 16 bytes, 8 mask bytes
constexpr int TILE = THREADS * VEC;                           // pixels of a piece: `per` tiles of 2048
constexpr int MOST_PER = 16, MOST_PER_MASKED = 4;             // (a masked piece lists its allowed pixels in LDS)
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LOWEST = -3.402823466e38f;                    // start of a running maximum: finite, so -inf logits give 2^-inf = 0 and never inf - inf

struct yes { static constexpr bool value = true; };
struct no { static constexpr bool value = false; };

struct Rows {                       // rows of logits as the kernels see them
  const void* logits; const void* ref; const uint8_t* mask;
  long long stride, ref_stride, mask_stride;   // elements between rows
  int rows, actions;
  int pixels, maps;                 // actions = pixels * maps; without a mask one map of all actions
  int per, maps_per;                // a piece: per * TILE pixels of maps_per maps
  int pieces_x, pieces;             // pieces along the pixels, and of a row
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

// Non-temporal accesses. Logits at their last use need not stay in the caches. What is written goes past them (`past`) only in calls over more memory than the 256 MB cache
// holds: its reader would not find it there anyway, and it would push out what this kernel still reads; a small result stays for its reader. (The gradient of 513 bf16 rows
// with plain stores 194 us a call, past the caches 171, with last reads too 161.) A lane's 8 fp32 logits are two loads of half a sector each: their line has to stay until the
// second (323 fp32 rows: 117 us, with such reads 127).
constexpr int64_t CACHE_BYTES = 256ll << 20;
__device__ __forceinline__ void put(F4* p, F4 v, yes) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void put(F4* p, F4 v, no) { *p = v; }
__device__ __forceinline__ void put(U4* p, U4 v, yes) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void put(U4* p, U4 v, no) { *p = v; }

// 8 values as they lie in memory: what is loaded ahead of its use
template <typename T> struct Eight { U4 w; };
template <> struct Eight<f32_t> { F4 a, b; };
template <typename T> __device__ __forceinline__ Eight<T> fetch8(const typename T::raw* p) { return Eight<T>{*(const U4*)p}; }
template <> __device__ __forceinline__ Eight<f32_t> fetch8<f32_t>(const float* p) { return Eight<f32_t>{*(const F4*)p, *(const F4*)(p + 4)}; }
template <typename T> __device__ __forceinline__ Eight<T> fetch8_last(const typename T::raw* p) { return Eight<T>{__builtin_nontemporal_load((const U4*)p)}; }
template <> __device__ __forceinline__ Eight<f32_t> fetch8_last<f32_t>(const float* p) { return fetch8<f32_t>(p); }
__device__ __forceinline__ void unpack8(const Eight<f32_t>& e, float* v) {
#pragma unroll
  for (int i = 0; i < 4; i++) { v[i] = e.a[i]; v[4 + i] = e.b[i]; }
}
template <typename T> __device__ __forceinline__ void unpack8(const Eight<T>& e, float* v) {
#pragma unroll
  for (int i = 0; i < 4; i++) { v[2 * i] = widen(T{}, (uint16_t)e.w[i]); v[2 * i + 1] = widen(T{}, (uint16_t)(e.w[i] >> 16)); }
}
template <typename Past> __device__ __forceinline__ void store8(f32_t, float* p, const float* v, Past past) {
  F4 a, b;
#pragma unroll
  for (int i = 0; i < 4; i++) { a[i] = v[i]; b[i] = v[4 + i]; }
  put((F4*)p, a, past);
  put((F4*)(p + 4), b, past);
}
template <typename T, typename Past> __device__ __forceinline__ void store8(T tag, uint16_t* p, const float* v, Past past) {
  U4 a;
#pragma unroll
  for (int i = 0; i < 4; i++) a[i] = (uint32_t)narrow(tag, v[2 * i]) | (uint32_t)narrow(tag, v[2 * i + 1]) << 16;
  put((U4*)p, a, past);
}

// 8 values from p on, of which the first `left` exist
template <typename T> __device__ __forceinline__ void take8(const typename T::raw* p, int left, float* v) {
#pragma unroll
  for (int i = 0; i < VEC; i++) v[i] = i < left ? widen(T{}, p[i]) : -INFINITY;
}
template <typename T, typename Past> __device__ __forceinline__ void put8(typename T::raw* p, int left, bool whole, const float* v, Past past) {
  if (whole) { store8(T{}, p, v, past); return; }
#pragma unroll
  for (int i = 0; i < VEC; i++) if (i < left) p[i] = narrow(T{}, v[i]);
}
// -inf where an action may not be taken: bit i of `allowed` is value i's. By the bits (v_bfe, v_bfi): a select would become eight branches round the loads.
__device__ __forceinline__ float barred(uint32_t allowed, int i, float v) {
  const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)allowed, i, 1);
  return __uint_as_float((__float_as_uint(v) & keep) | (0xff800000u & ~keep));
}
__device__ __forceinline__ void bar8(uint32_t allowed, float* v) {
#pragma unroll
  for (int i = 0; i < VEC; i++) v[i] = barred(allowed, i, v[i]);
}
// whether the row's action counts: inside the row, allowed, and of a logit above -inf (a NaN counts: it has to show)
template <typename T> __device__ __forceinline__ float logit(const Rows& R, int row, long long a) { return widen(T{}, ((const typename T::raw*)R.logits)[row * R.stride + a]); }
template <typename T> __device__ __forceinline__ bool action_counts(const Rows& R, int row, long long a) {
  if (a < 0 || a >= R.actions || (R.mask && !R.mask[row * R.mask_stride + a % R.pixels])) return false;
  return !(logit<T>(R, row, a) == -INFINITY);
}

// ---- the 8s of a piece. For every 8 pixels of every map of the piece that hold an allowed one: use(first action, allowed bits, fetch(first action)), or
// part(first action, allowed bits, values that exist) where the mask ends inside the 8; with NONE, none(piece, 8, map, step) for the others: every step-th map from that one on.
// A thread fetches its next 8 before it uses one: what a workgroup does is a chain of latencies. Logits that may not be taken are not read: the allowed 8s of the piece's
// pixels are listed in LDS once (the maps share them) and dealt to the threads from the list, so that no lane idles where the mask has holes.
struct Piece { int first, pixels, map0, maps; };   // pixels first .. of maps map0 ..
__device__ __forceinline__ Piece piece_of(const Rows& R, int piece) {
  const int x = piece % R.pieces_x, y = piece / R.pieces_x;
  Piece P{x * R.per * TILE, 0, y * R.maps_per, 0};
  P.pixels = min(R.per * TILE, R.pixels - P.first);
  P.maps = min(R.maps_per, R.maps - P.map0);
  return P;
}
__device__ __forceinline__ uint32_t four(uint32_t bytes) {      // a byte per pixel, non-zero = allowed -> a bit per pixel
  const uint32_t ones = (((bytes & 0x7f7f7f7fu) + 0x7f7f7f7fu) | bytes) >> 7 & 0x01010101u;
  return __builtin_amdgcn_udot4(ones, 0x08040201u, 0, false);
}
__device__ __forceinline__ uint32_t allowed8(const uint8_t* mask, int left, bool whole) {
  uint64_t b = 0;
  if (whole) b = *(const U8*)mask;
  else for (int i = 0; i < left; i++) b |= (uint64_t)mask[i] << (8 * i);
  return four((uint32_t)b) | four((uint32_t)(b >> 32)) << 4;
}
template <typename A, typename F, typename U> __device__ __forceinline__ void in_turns(int all, A at, F fetch, U use) {   // items threadIdx.x, + THREADS, .. below all
  int i = threadIdx.x;
  if (i >= all) return;
  auto one = at(i);
  auto a = fetch(one);
  for (;;) {
    const bool more = (i += THREADS) < all;
    auto other = one;
    auto b = a;
    if (more) { other = at(i); b = fetch(other); }
    use(one, a);
    if (!more) return;
    const bool again = (i += THREADS) < all;
    if (again) { one = at(i); a = fetch(one); }
    use(other, b);
    if (!again) return;
  }
}
template <bool MASK, bool NONE, typename F, typename U, typename P8, typename N> __device__ __forceinline__ void for_piece(const Rows& R, int row, int piece, F fetch, U use, P8 part, N none) {
  const Piece P = piece_of(R, piece);
  struct At { int j; uint32_t allowed; };
  const auto fetch_at = [&](const At& a) { return fetch(a.j); };
  const auto use_at = [&](const At& a, const auto& e) { use(a.j, a.allowed, e); };
  const int tail = P.pixels % VEC, last = P.first + P.pixels - tail;      // the row's or the mask's last, shorter 8
  if (!MASK) {                      // one map: pixel = action
    in_turns(P.pixels / VEC, [&](int i) { return At{P.first + i * VEC, 0xffu}; }, fetch_at, use_at);
    if (tail && threadIdx.x == 0) part(last, (1u << tail) - 1, tail);
    return;
  }
  const uint8_t* mask = R.mask + row * R.mask_stride + P.first;
  if (tail) {                       // a thread per map
    const uint32_t bits = allowed8(mask + P.pixels - tail, tail, false);
    if (!bits) { if (NONE) none(P, P.pixels / VEC, threadIdx.x, THREADS); }
    else for (int m = threadIdx.x; m < P.maps; m += THREADS) part((P.map0 + m) * R.pixels + last, bits, tail);
  }
  // A small batch, cut into pieces of an 8 per thread: latency counts, so the logits are asked for together with their mask (17 masked f16 rows of 131 x 93, statistics and
  // gradient: 9.1 -> 8.0 us; one fp32 row of 6 x 200 x 200, sampling: 7.7 -> 7.1).
  if (R.per == 1 && R.maps_per == 1) {
    const int g = threadIdx.x, j = P.map0 * R.pixels + P.first + g * VEC;
    if (g < P.pixels / VEC) {
      const auto e = fetch(j);
      use(j, allowed8(mask + g * VEC, VEC, true), e);
    }
    return;
  }
  __shared__ uint32_t list[MOST_PER_MASKED * THREADS];      // group of 8 << 8 | bits, in the order of the pixels
  __shared__ int4 share[MOST_PER_MASKED];                   // entries of the four wavefronts of each tile
  static_assert(THREADS / 64 == 4, "an int4 of wavefronts");
  const bool narrow = P.pixels / VEC < THREADS;             // few 8s of many maps: all threads share each
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t bits[MOST_PER_MASKED];
  int before[MOST_PER_MASKED];
#pragma unroll
  for (int t = 0; t < MOST_PER_MASKED; t++) {
    if (t >= R.per) break;
    const int g = t * THREADS + threadIdx.x;
    const bool in = g < P.pixels / VEC;
    bits[t] = in ? allowed8(mask + g * VEC, VEC, true) : 0;
    const uint64_t some = __ballot(bits[t] != 0);
    before[t] = __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
    if (lane == 0) ((int*)&share[t])[wave] = __popcll(some);
    if (NONE && in && !bits[t] && !narrow) none(P, g, 0, 1);
  }
  if (NONE && narrow)
    for (int i = threadIdx.x, groups = P.pixels / VEC; i < groups * P.maps; i += THREADS)
      if (!allowed8(mask + i % groups * VEC, VEC, true)) none(P, i % groups, i / groups, P.maps);
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int t = 0; t < MOST_PER_MASKED; t++) {
    if (t >= R.per) break;
    const int4 w = share[t];
    const int mine = n + (wave > 0 ? w.x : 0) + (wave > 1 ? w.y : 0) + (wave > 2 ? w.z : 0);
    if (bits[t]) list[mine + before[t]] = (uint32_t)(t * THREADS + threadIdx.x) << 8 | bits[t];
    n += w.x + w.y + w.z + w.w;
  }
  __syncthreads();
  const float per = __builtin_amdgcn_rcpf((float)n);
  in_turns(n * P.maps, [&](int i) {
    int m = (int)(((float)i + 0.5f) * per), k = i - m * n;               // map and list entry of item i; the estimate is off by at most one
    if (k < 0) { m--; k += n; }
    if (k >= n) { m++; k -= n; }
    const uint32_t e = list[k];
    return At{(P.map0 + m) * R.pixels + P.first + (int)(e >> 8) * VEC, e & 0xff};
  }, fetch_at, use_at);
}

// ---- reductions over 64 or 4 neighbouring lanes, in every lane, in a fixed order: lanes of a row of 16 exchange through DPP, the four rows through scalar registers
// (through LDS, one exchange costs as much as all of a reduction here)
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
  const int2 w = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, int2{dpp<CTRL>(w.x), dpp<CTRL>(w.y)});
}
__device__ __forceinline__ int at_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float at_lane(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double at_lane(double v, int lane) {
  const int2 w = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, int2{at_lane(w.x, lane), at_lane(w.y, lane)});
}
template <int WIDTH, typename S, typename F> __device__ __forceinline__ S lanes_fold(S v, F f) {
  static_assert(WIDTH == 64 || WIDTH == 4, "widths in use");
  v = f(v, dpp<0xB1>(v));             // quad_perm 1 0 3 2
  v = f(v, dpp<0x4E>(v));             // quad_perm 2 3 0 1
  if (WIDTH == 4) return v;
  v = f(v, dpp<0x141>(v));            // row_half_mirror
  v = f(v, dpp<0x140>(v));            // row_mirror
  return f(f(at_lane(v, 0), at_lane(v, 16)), f(at_lane(v, 32), at_lane(v, 48)));
}
template <int WIDTH = 64> __device__ __forceinline__ float lanes_max(float v) { return lanes_fold<WIDTH>(v, [](float x, float y) { return fmaxf(x, y); }); }
template <int WIDTH = 64, typename S> __device__ __forceinline__ S lanes_sum(S v) { return lanes_fold<WIDTH>(v, [](S x, S y) { return x + y; }); }
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

// a sum times the factor of a new maximum: a KL sum that met a reference of probability 0 is infinite, and stays out where its share of the row vanishes
template <typename S> __device__ __forceinline__ S scaled(S sum, S f) { return f > 0 ? sum * f : f; }

// running sums of one thread: fp32, over at most a few hundred terms
struct Running { float m, s, t, k, mq, sq; };
__device__ __forceinline__ Running nothing() { return Running{LOWEST, 0, 0, 0, LOWEST, 0}; }
// z (and q): 8 logits, -inf where not allowed. One maximum per 8; the sums move to it where it is new (rare after a few 8s).
template <bool REF, bool ENTROPY> __device__ __forceinline__ void add8(Running& a, const float* z, const float* q, float* e) {
  float m = a.m, mq = a.mq;
#pragma unroll
  for (int i = 0; i < VEC; i++) { m = fmaxf(m, z[i]); if (REF) mq = fmaxf(mq, q[i]); }
  if (m > a.m) {
    const float f = shrink(a.m, m);
    if (ENTROPY) a.t = f * (a.t + a.s * fmaxf(a.m - m, -1e30f));   // an empty sum meets LOWEST - m: kept finite
    a.s *= f;
    if (REF) a.k = scaled(a.k, f);
    a.m = m;
  }
  if (REF && mq > a.mq) { a.sq *= shrink(a.mq, mq); a.mq = mq; }
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const float d = z[i] - a.m;
    e[i] = fall(d);
    a.s += e[i];
    if (ENTROPY) a.t += e[i] * fmaxf(d, -1e4f);                   // e is 0 long before -1e4: 0 * -inf does not arise
    if (REF) {
      a.k += e[i] * (e[i] > 0 ? z[i] - q[i] : 0.f);               // what is not allowed or too unlikely for 32 bits adds nothing, whatever q holds
      a.sq += fall(q[i] - a.mq);
    }
  }
}
// From here on sums are 64 bits wide: a KL is a difference of two logarithms of sums, and what a few last additions lose in 32 bits (5e-8 of a sum, measured) would be
// 1e-6 of it. Their factors come from the precise exp where a single one weighs (joining wavefronts and records).
__device__ __forceinline__ double moved(double s, double t, float from, float to) { return t + s * fmaxf(from - to, -1e30f); }
// sums of neighbouring lanes joined, in every one of them
template <int WIDTH> __device__ __forceinline__ void join_lanes(Sums& a, bool ref, bool entropy) {
  const float m = lanes_max<WIDTH>(a.m);
  const double f = exp((double)a.m - m);
  if (entropy) a.t = lanes_sum<WIDTH>(f * moved(a.s, a.t, a.m, m));
  a.s = lanes_sum<WIDTH>(a.s * f);
  if (ref) {
    a.k = lanes_sum<WIDTH>(scaled(a.k, f));
    const float mq = lanes_max<WIDTH>(a.mq);
    a.sq = lanes_sum<WIDTH>(a.sq * exp((double)a.mq - mq));
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
    a.k = lanes_sum((double)scaled(r.k, f));
    a.mq = lanes_max(r.mq);
    a.sq = lanes_sum((double)(r.sq * shrink(r.mq, a.mq)));
  }
  return a;
}
// the workgroup's sums joined, in every thread
__device__ __forceinline__ Sums join_workgroup(const Running& r, bool ref, bool entropy) {
  __shared__ Sums wave[THREADS / 64];
  Sums a = join_wave(r, ref, entropy);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = a;
  __syncthreads();
  a = wave[threadIdx.x & (THREADS / 64 - 1)];
  join_lanes<THREADS / 64>(a, ref, entropy);
  return a;
}

// ---- statistics of the pieces of rows: log-probability and entropy of 2000 bf16 rows of 40 000 actions 35 us (4.6 TB/s, what a large copy reaches).
template <typename T, bool REF> struct Both {       // 8 logits, and the reference's
  Eight<T> z, q;
  __device__ __forceinline__ Both(const typename T::raw* z_row, const typename T::raw* q_row, int j, no) : z(fetch8<T>(z_row + j)) { if (REF) q = fetch8<T>(q_row + j); }
  __device__ __forceinline__ Both(const typename T::raw* z_row, const typename T::raw* q_row, int j, yes) : z(fetch8_last<T>(z_row + j)) { if (REF) q = fetch8_last<T>(q_row + j); }
  __device__ __forceinline__ void get(float* a, float* b) const { unpack8(z, a); if (REF) unpack8(q, b); }
};
template <typename T, bool MASK, bool REF, bool ENTROPY> __device__ __forceinline__ Sums piece_sums(const Rows& R, int row, int piece) {
  const auto* z_row = (const typename T::raw*)R.logits + row * R.stride;
  const auto* q_row = REF ? (const typename T::raw*)R.ref + row * R.ref_stride : nullptr;
  Running a = nothing();
  const auto add = [&](uint32_t allowed, float* z, float* q) {
    float e[VEC];
    if (MASK) { bar8(allowed, z); if (REF) bar8(allowed, q); }
    add8<REF, ENTROPY>(a, z, q, e);
  };
  for_piece<MASK, false>(R, row, piece, [&](int j) { return Both<T, REF>(z_row, q_row, j, no{}); },
    [&](int, uint32_t allowed, const Both<T, REF>& b) { float z[VEC], q[VEC]; b.get(z, q); add(allowed, z, q); },
    [&](int j, uint32_t allowed, int left) { float z[VEC], q[VEC]; take8<T>(z_row + j, left, z); if (REF) take8<T>(q_row + j, left, q); add(allowed, z, q); },
    [](const Piece&, int, int, int) {});
  return join_workgroup(a, REF, ENTROPY);
}

// ---- what both losses have in common. Per row, dL/dz_j = p_j (c0 + kl (z_j - q_j - gap) + entropy (z_j - m - level)) + [j = action] take; p_j = exp(z_j - m) rs.
// Three launches: statistics of the pieces -- a Slope per row and a term per row or pair of the loss -- the gradient, of which the first workgroup adds the terms up.
// (Joining a row's records in every workgroup of the gradient saves a launch and costs each of them 3 us of double arithmetic before its first load: ur5_policy_clip_few.)
// Bound by memory where rows are many -- 513 masked bf16 rows of 6 x 200 x 200 with their reference: 71 + 5 + 89 us; the mask's runs end inside 128-byte lines, 281 MB are
// fetched for 199 MB of allowed logits --, by the latency of the launches where they are few (12 fp32 rows: 9 + 14 us).
struct Slope { float m, rs, c0, kl, gap, entropy, level, take; int on; };   // on: the row counts; anything else is unset where it does not
struct Span { const int64_t* ends; int last; };   // the preference loss: rows outside [ends[0], ends[last]) belong to no episode and do not count; ends == null: all rows
__device__ __forceinline__ bool in_span(const Span& s, int row) { return !s.ends || (row >= s.ends[0] && row < s.ends[s.last]); }
// The pieces come after `front` workgroups (a multiple of 8, so that pieces keep their XCDs from kernel to kernel) that write which rows count, a thread each.
template <typename T, bool MASK, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_stats(Rows R, Span span, int front, const int64_t* action, Part* parts, Slope* slopes, int* counts) {
  if ((int)blockIdx.x < front) {
    const int row = blockIdx.x * THREADS + threadIdx.x;
    const bool on = row < R.rows && in_span(span, row) && action_counts<T>(R, row, action[row]);
    if (row < R.rows) slopes[row] = Slope{0, 0, 0, 0, 0, 0, 0, 0, on};
    const int n = __syncthreads_count(on);
    if (threadIdx.x == 0 && row < R.rows) counts[blockIdx.x] = n;
    return;
  }
  const int block = (int)blockIdx.x - front, row = block / R.pieces, piece = block % R.pieces;
  const int64_t a = action[row];
  if (a < 0 || a >= R.actions || !in_span(span, row)) return;
  const Sums sums = piece_sums<T, MASK, REF, true>(R, row, piece);
  if (threadIdx.x == 0) parts[block] = Part{sums, 0};
}
// the records of a row joined by a wavefront, in every lane
__device__ __forceinline__ Sums join_row(const Part* parts, int pieces, bool ref) {
  Sums a{LOWEST, LOWEST, 0, 0, 0, 0};
  for (int i = threadIdx.x & 63; i < pieces; i += 64) {
    const Sums p = parts[i].sums;
    const float m = fmaxf(a.m, p.m), mq = fmaxf(a.mq, p.mq);
    const double f = exp((double)a.m - m), g = exp((double)p.m - m);
    a.t = f * moved(a.s, a.t, a.m, m) + g * moved(p.s, p.t, p.m, m);
    a.s = f * a.s + g * p.s;
    if (ref) {
      a.k = scaled(a.k, f) + scaled(p.k, g);
      a.sq = a.sq * exp((double)a.mq - mq) + p.sq * exp((double)p.mq - mq);
    }
    a.m = m; a.mq = mq;
  }
  join_lanes<64>(a, ref, true);
  return a;
}
constexpr int WAVES = THREADS / 64;
// sums over the workgroup in a fixed order, in every thread
template <typename S> __device__ __forceinline__ S workgroup_sum(S v) {
  __shared__ S wave[WAVES];
  v = lanes_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = wave[0];
  for (int i = 1; i < WAVES; i++) v += wave[i];
  return v;
}
// loss = sum of n terms / what they are a mean over: *counting (the rows that count), or n without it
struct Terms { const double* term; int n; const int* counting; float* loss; };
__device__ __forceinline__ void add_terms(const Terms& t) {
  double sum = 0;
  for (int i = threadIdx.x; i < t.n; i += THREADS) sum += t.term[i];
  sum = workgroup_sum(sum);
  if (threadIdx.x == 0) *t.loss = (float)(sum / max(1, t.counting ? *t.counting : t.n));
}
// (a forward pass without a gradient)
static __global__ void __launch_bounds__(THREADS) ur5_policy_loss(Terms t) { add_terms(t); }
// the gradient of a piece of a row; factor: of the whole gradient
template <typename T, bool MASK, bool REF, typename Past> __device__ __forceinline__ void grad_piece(const Rows& R, int row, int piece, Slope S, float factor, int a, void* grad, Past past) {
  typename T::raw* out = (typename T::raw*)grad + (long long)row * R.actions;
  const float zero[VEC] = {};
  const auto clear = [&](const Piece& P, int g, int map, int step) {   // 8 pixels of maps of the piece
    const int p = P.first + g * VEC, left = R.pixels - p;
    for (int m = map; m < P.maps; m += step) put8<T>(out + (P.map0 + m) * R.pixels + p, left, left >= VEC, zero, past);
  };
  if (!S.on) {                                             // zeros; the logits are not read
    const Piece P = piece_of(R, piece);
    const int groups = (P.pixels + VEC - 1) / VEC;
    if (groups < THREADS) for (int i = threadIdx.x; i < groups * P.maps; i += THREADS) clear(P, i % groups, i / groups, P.maps);
    else for (int g = threadIdx.x; g < groups; g += THREADS) clear(P, g, 0, 1);
    return;
  }
  S.rs *= factor; S.take *= factor;
  const auto* z_row = (const typename T::raw*)R.logits + row * R.stride;
  const auto* q_row = REF ? (const typename T::raw*)R.ref + row * R.ref_stride : nullptr;
  const auto slope = [&](int j, uint32_t allowed, float* z, const float* q, float* g) {
    if (MASK) bar8(allowed, z);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float d = z[i] - S.m, p = fall(d) * S.rs;
      float v = S.c0 + S.entropy * (d - S.level);
      if (REF) v += S.kl * (z[i] - q[i] - S.gap);
      g[i] = p == 0.f ? 0.f : p * v;                       // not allowed, or too unlikely for 32 bits: the limit, whatever q holds
    }
    if ((unsigned)(a - j) < VEC)
#pragma unroll
      for (int i = 0; i < VEC; i++) g[i] += a - j == i ? S.take : 0.f;
  };
  for_piece<MASK, true>(R, row, piece, [&](int j) { return Both<T, REF>(z_row, q_row, j, yes{}); },
    [&](int j, uint32_t allowed, const Both<T, REF>& b) { float z[VEC], q[VEC], g[VEC]; b.get(z, q); slope(j, allowed, z, q, g); store8(T{}, out + j, g, past); },
    [&](int j, uint32_t allowed, int left) {
      float z[VEC], q[VEC], g[VEC];
      take8<T>(z_row + j, left, z);
      if (REF) take8<T>(q_row + j, left, q);
      slope(j, allowed, z, q, g);
      put8<T>(out + j, left, false, g, past);
    }, clear);
}
__device__ __forceinline__ float grad_factor(float scale, const float* upstream, const int* counting) { return scale * (upstream ? *upstream : 1.f) / (counting ? max(1, *counting) : 1); }
constexpr int FIRST = 8;             // workgroups before the pieces, as in the statistics; the first of them writes the loss if t.loss
template <typename T, bool MASK, bool REF, typename Past> __global__ void __launch_bounds__(THREADS) ur5_policy_grad(Rows R, Terms t, const int64_t* action, const Slope* slopes, float scale, const float* upstream, void* grad) {
  constexpr Past past;
  const int block = (int)blockIdx.x - FIRST;
  if (block < 0) {
    if (t.loss && blockIdx.x == 0) add_terms(t);
    return;
  }
  const int row = R.rows - 1 - block / R.pieces, piece = block % R.pieces;   // the rows that the statistics read last, and the 256 MB memory-side cache may hold, come first (259 fp32 rows: 80.0 us in their order, 78.7 in this; 513 bf16 rows: 91.6 and 90.3)
  grad_piece<T, MASK, REF>(R, row, piece, slopes[row], grad_factor(scale, upstream, t.counting), (int)action[row], grad, past);
}

// ---- clipped policy loss. Per row: ratio r = exp(logp - old), L = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl_coef KL(p || q) - entropy_coef H; the mean over the rows that count.
struct Clip { const int64_t* action; const float* old_logp; const float* advantage; float lo, hi, kl_coef, entropy_coef; };
// The end of a row that counts, by a wavefront, in every lane. Normalisers in 64 bits: KL = k / s - (lse - lse_q) is a small difference of large numbers.
struct ClipRow { Slope slope; double term; float logp, kl, entropy; };
template <typename T, bool REF> __device__ __forceinline__ ClipRow clip_row(const Rows& R, const Clip& C, const Part* parts, int pieces, int row) {
  const Sums a = join_row(parts + (size_t)row * pieces, pieces, REF);
  const double ls = log(a.s), shift = REF ? (double)a.m - a.mq + ls - log(a.sq) : 0;
  const float adv = C.advantage[row], lp = (float)((double)logit<T>(R, row, C.action[row]) - a.m - ls), k = REF ? (float)(a.k / a.s - shift) : 0.f, h = (float)(ls - a.t / a.s);
  const float ratio = expf(lp - C.old_logp[row]), free = ratio * adv, held = fminf(fmaxf(ratio, 1 - C.lo), 1 + C.hi) * adv;
  const float take = held < free ? 0.f : -adv * ratio;   // the clipped branch has no slope; NaN stays
  const double term = -(double)(held < free ? held : free) + (REF && C.kl_coef > 0 ? (double)C.kl_coef * k : 0.0) - (double)C.entropy_coef * h;   // (an infinite KL that has no weight is only reported)
  return ClipRow{Slope{a.m, (float)(1 / a.s), -take, C.kl_coef, (float)(shift + k), C.entropy_coef, (float)(ls - h), take, 1}, term, lp, k, h};
}
struct ClipOut { float* logp; float* kl; float* entropy; };
__device__ __forceinline__ int rows_that_count(const int* counts, int rows) {   // by the workgroup
  int n = 0;
  for (int i = threadIdx.x; i < (rows + THREADS - 1) / THREADS; i += THREADS) n += counts[i];
  return workgroup_sum(n);
}
template <typename T, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_clip_rows(Rows R, Clip C, const Part* parts, Slope* slopes, const int* counts, int* counting, double* term, ClipOut out) {
  if (blockIdx.x == 0) {
    const int n = rows_that_count(counts, R.rows);
    if (threadIdx.x == 0) *counting = n;
  }
  const int row = blockIdx.x * WAVES + (threadIdx.x >> 6);   // a wavefront per row
  if (row >= R.rows) return;
  ClipRow end{};
  if (slopes[row].on) end = clip_row<T, REF>(R, C, parts, R.pieces, row);
  if (threadIdx.x & 63) return;
  term[row] = end.term; out.logp[row] = end.logp; out.kl[row] = end.kl; out.entropy[row] = end.entropy;
  if (end.slope.on) slopes[row] = end.slope;
}
// Few rows: the gradient ends them by itself, every workgroup its own (its wavefronts all the same), the first one all of them for the loss: two launches instead of three.
// `pieces`: the statistics' of a row. The first workgroup's wavefronts take the rows in turns, some 2.5 us each, while the others write the gradient: at most FEW rows, or as many
// fewer as a lane has records of one. A call on fp32 rows with their reference, two launches against three: 12 of 6 x 200 x 200 (120 records) 22.1 us, 23.9; 16 of them 24.6, 24.0;
// 24 of 131 x 93 21.5, 24.6; 48 of them 28.6, 24.5.
constexpr int FEW = 24;
template <typename T, bool MASK, bool REF> __global__ void __launch_bounds__(THREADS) ur5_policy_clip_few(Rows R, int pieces, Clip C, const Part* parts, const Slope* slopes, const int* counts, float* loss, ClipOut out, float scale,
                                                                                                          const float* upstream, void* grad) {
  const int block = (int)blockIdx.x - FIRST;
  if (block < 0) {
    if (blockIdx.x) return;
    __shared__ double term[FEW];
    for (int row = threadIdx.x >> 6; row < R.rows; row += WAVES) {
      ClipRow end{};
      if (slopes[row].on) end = clip_row<T, REF>(R, C, parts, pieces, row);
      if ((threadIdx.x & 63) == 0) { term[row] = end.term; out.logp[row] = end.logp; out.kl[row] = end.kl; out.entropy[row] = end.entropy; }
    }
    __syncthreads();
    add_terms(Terms{term, R.rows, counts, loss});          // (so few rows are one part of the counts)
    return;
  }
  const int row = R.rows - 1 - block / R.pieces, piece = block % R.pieces;
  Slope S{};
  if (slopes[row].on) S = clip_row<T, REF>(R, C, parts, pieces, row).slope;
  grad_piece<T, MASK, REF>(R, row, piece, S, grad_factor(scale, upstream, counts), (int)C.action[row], grad, no{});
}
static_assert(FEW <= THREADS, "one part of the counts");

// ---- preference loss. Episodes are runs of rows: episode k holds the rows offsets[k] .. offsets[k + 1]. S_k = sum over its counting rows of logp - ref_logp,
// margin_i = beta (S_2i - S_2i+1), loss = mean over pairs of (1 - eps) softplus(-margin) + eps softplus(margin).
struct Prefer { const int64_t* action; const float* ref_logp; const int64_t* offsets; int pairs; double beta, eps; };
// the end of a row that counts, by a wavefront, in every lane: what it adds to its episode, and its slope's m and rs
struct PreferRow { double l; float m, rs; };
template <typename T> __device__ __forceinline__ PreferRow prefer_row(const Rows& R, const Prefer& P, const Part* parts, int pieces, int row) {
  const Sums a = join_row(parts + (size_t)row * pieces, pieces, false);
  return PreferRow{(double)logit<T>(R, row, P.action[row]) - a.m - log(a.s) - P.ref_logp[row], a.m, (float)(1 / a.s)};
}
struct Ends { int at[3]; };            // a pair's rows: at[0] .. of the preferred episode, at[1] .. at[2] of the other; offsets outside the rows are taken as their ends
__device__ __forceinline__ Ends ends_of(const Rows& R, const Prefer& P, int pair) {
  Ends e;
  for (int k = 0; k < 3; k++) e.at[k] = (int)min(max((long long)P.offsets[2 * pair + k], 0ll), (long long)R.rows);
  return e;
}
// from the sum over a pair: its margin, its term of the loss, and d loss / d logp of the preferred episode's rows
struct PairEnd { float margin, w; double term; };
__device__ __forceinline__ PairEnd pair_end(const Prefer& P, double d) {
  const double mg = P.beta * d, up = 1 / (1 + exp(mg));                      // sigmoid(-margin)
  const double rest = log1p(exp(-fabs(mg)));                                 // softplus(x) = max(x, 0) + this, of margin and -margin
  const double other = P.eps > 0 ? P.eps * (fmax(mg, 0.0) + rest) : 0.0;     // (an infinite margin that has no weight adds nothing)
  return PairEnd{(float)mg, (float)(-P.beta * ((1 - P.eps) * up - P.eps * (1 - up)) / P.pairs), (1 - P.eps) * (fmax(-mg, 0.0) + rest) + other};
}
// long episodes: all rows in a launch of their own, a wavefront each; what a row adds stays in its first record (10 000 rows of 2400 actions in one pair, us a call: 1985 with its
// workgroup alone, 99 so)
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_policy_prefer_rows(Rows R, Prefer P, Part* parts, Slope* slopes) {
  const int row = blockIdx.x * WAVES + (threadIdx.x >> 6);
  if (row >= R.rows || !slopes[row].on) return;
  const PreferRow end = prefer_row<T>(R, P, parts, R.pieces, row);
  if (threadIdx.x & 63) return;
  slopes[row].m = end.m; slopes[row].rs = end.rs;
  parts[(size_t)row * R.pieces].sums.s = end.l;
}
// a workgroup per pair; of rows that are not ended yet a wavefront each
template <typename T, bool ENDED> __global__ void __launch_bounds__(THREADS) ur5_policy_prefer_pairs(Rows R, Prefer P, const Part* parts, Slope* slopes, double* term, float* margin) {
  const Ends e = ends_of(R, P, blockIdx.x);
  double d = 0;
  for (int half = 0; half < 2; half++)
    for (int row = e.at[half] + (ENDED ? threadIdx.x : threadIdx.x >> 6); row < e.at[half + 1]; row += ENDED ? THREADS : WAVES) {
      if (!slopes[row].on) continue;
      double l;
      if (ENDED) l = parts[(size_t)row * R.pieces].sums.s;
      else {
        const PreferRow end = prefer_row<T>(R, P, parts, R.pieces, row);
        if ((threadIdx.x & 63) == 0) { slopes[row].m = end.m; slopes[row].rs = end.rs; }
        l = end.l;
      }
      d += half ? -l : l;
    }
  const PairEnd pair = pair_end(P, workgroup_sum(ENDED || (threadIdx.x & 63) == 0 ? d : 0.0));
  if (threadIdx.x == 0) { margin[blockIdx.x] = pair.margin; term[blockIdx.x] = pair.term; }
  for (int half = 0; half < 2; half++)
    for (int row = e.at[half] + threadIdx.x; row < e.at[half + 1]; row += THREADS) {
      Slope& S = slopes[row];
      S.take = half ? -pair.w : pair.w;
      S.rs *= S.take;
      S.c0 = -1.f;
    }
}
// Few rows and pairs: the gradient ends them by itself, every workgroup its row's pair, the first one all of them for the loss. The sums run as in ur5_policy_prefer_pairs, wavefront
// by wavefront: the same bits. 17 f16 rows of 131 x 93, us a call: 20.2 in three launches, 18.4 in two; 8 fp32 rows of 9600 in one pair 18.8, 16.2.
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_prefer_few(Rows R, int pieces, Prefer P, const Part* parts, const Slope* slopes, float* loss, float* margin, float scale, const float* upstream, void* grad) {
  const int block = (int)blockIdx.x - FIRST, wave = threadIdx.x >> 6;
  if (block < 0) {
    if (blockIdx.x) return;
    __shared__ double l[FEW], term[FEW];
    for (int row = wave; row < R.rows; row += WAVES) {
      const double v = slopes[row].on ? prefer_row<T>(R, P, parts, pieces, row).l : 0.0;
      if ((threadIdx.x & 63) == 0) l[row] = v;
    }
    __syncthreads();
    if ((int)threadIdx.x < P.pairs) {
      const Ends e = ends_of(R, P, threadIdx.x);
      double d[WAVES] = {};
      for (int w = 0; w < WAVES; w++)
        for (int half = 0; half < 2; half++)
          for (int row = e.at[half] + w; row < e.at[half + 1]; row += WAVES) if (slopes[row].on) d[w] += half ? -l[row] : l[row];
      static_assert(WAVES == 4, "the order of workgroup_sum");
      const PairEnd pair = pair_end(P, ((d[0] + d[1]) + d[2]) + d[3]);
      margin[threadIdx.x] = pair.margin;
      term[threadIdx.x] = pair.term;
    }
    __syncthreads();
    add_terms(Terms{term, P.pairs, nullptr, loss});
    return;
  }
  const int mine = R.rows - 1 - block / R.pieces, piece = block % R.pieces;
  int pair = 0;
  Ends e{};
  for (; pair < P.pairs; pair++) {
    e = ends_of(R, P, pair);
    if (mine >= e.at[0] && mine < e.at[2]) break;
  }
  __shared__ Slope S;
  if (threadIdx.x == 0) S = Slope{};
  __syncthreads();
  if (pair < P.pairs && slopes[mine].on) {
    double d = 0;
    for (int half = 0; half < 2; half++)
      for (int row = e.at[half] + wave; row < e.at[half + 1]; row += WAVES) {
        if (!slopes[row].on) continue;
        const PreferRow end = prefer_row<T>(R, P, parts, pieces, row);
        d += half ? -end.l : end.l;
        if (row == mine && (threadIdx.x & 63) == 0) { S.m = end.m; S.rs = end.rs; S.take = half ? -1.f : 1.f; S.c0 = -1.f; S.on = 1; }
      }
    const float w = pair_end(P, workgroup_sum((threadIdx.x & 63) == 0 ? d : 0.0)).w;
    if (threadIdx.x == 0) { S.take *= w; S.rs *= S.take; }
    __syncthreads();
  }
  grad_piece<T, MASK, false>(R, mine, piece, S, grad_factor(scale, upstream, nullptr), (int)P.action[mine], grad, no{});
}

// ---- log-probability of an action and entropy per row. logp 0 where the action lies outside the row (no action), -inf where it may not be taken; entropy 0 where
// nothing may. A row of one piece is finished by its workgroup, others by a wavefront each.
template <typename T> __device__ __forceinline__ void write_logp(const Rows& R, int row, const Sums& a, const int64_t* action, float* logp, float* entropy) {
  const long long at = action[row];
  const double ls = a.s > 0 ? log(a.s) : a.s - a.s;   // a NaN sum stays NaN
  logp[row] = action_counts<T>(R, row, at) ? (float)((double)logit<T>(R, row, at) - a.m - ls) : at < 0 || at >= R.actions ? 0.f : -INFINITY;
  if (entropy) entropy[row] = a.s == 0 ? 0.f : (float)(ls - a.t / a.s);
}
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_logp(Rows R, const int64_t* action, Part* parts, float* logp, float* entropy) {
  const int row = blockIdx.x / R.pieces, piece = blockIdx.x % R.pieces;
  const Sums a = piece_sums<T, MASK, false, true>(R, row, piece);
  if (threadIdx.x) return;
  if (R.pieces == 1) write_logp<T>(R, row, a, action, logp, entropy);
  else parts[blockIdx.x] = Part{a, 0};
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_policy_logp_rows(Rows R, const int64_t* action, const Part* parts, float* logp, float* entropy) {
  const int row = blockIdx.x * WAVES + (threadIdx.x >> 6);
  if (row >= R.rows) return;
  const Sums a = join_row(parts + (size_t)row * R.pieces, R.pieces, false);
  if ((threadIdx.x & 63) == 0) write_logp<T>(R, row, a, action, logp, entropy);
}

// ---- sampling. argmax_j z_j - log(-log u_j) is a draw from softmax(z). Two logarithms in 64 bits per action would cost more than reading it, and nearly every action
// is far from winning: with E = -log u >= 1 - u, action j can only reach score `bar` if 1 - u_j <= exp(z_j - bar) -- one product and one comparison on the exp that the
// softmax's sum needs anyway. `bar` is the best score any thread of the workgroup has seen (less a margin over every rounding below), so a few actions per
// piece pass and are scored in 64 bits; equal scores go to the lower action, so the result does not depend on who was first.
// What is left per action is the hash: two products of 64 bits, six of the slow integer instructions, which is what bounds it (512 masked fp32 rows of 6 x 200 x 200: 88 us,
// log-probability and entropy of the same rows 51).
__device__ __forceinline__ int ordered(float v) { const int b = __float_as_int(v); return b ^ ((b >> 31) & 0x7fffffff); }
__device__ __forceinline__ float unordered(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }
__device__ __forceinline__ float below(double score) { return (float)score - (1e-4f + 1e-6f * fabsf((float)score)); }

struct Best { double score; int at; };
__device__ __forceinline__ void join_best(Best& b) {   // over a wavefront, in every lane
  for (int o = 32; o; o >>= 1) {
    const double s = __shfl_xor(b.score, o);
    const int i = __shfl_xor(b.at, o);
    if (better(s, i, b.score, b.at)) { b.score = s; b.at = i; }
  }
}
// 1 - u of 8 neighbouring draws in units of 2^-32, off by at most 1 from what it is rounded down (the finaliser's last shift, left out, may flip the lowest bit)
__device__ __forceinline__ void missing8(uint64_t key, int j, uint32_t* w) {
  uint64_t c = key + (uint64_t)(j + 1) * GOLD;
#pragma unroll
  for (int i = 0; i < VEC; i++, c += GOLD) {
    uint64_t x = (c ^ (c >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    w[i] = ~(uint32_t)(x >> 32);
  }
}
// What the workgroup has found: the bar, and the actions that passed it, whose scores are computed together at the end (64 bits of two logarithms cost 250 instructions, for one
// lane as for all). Where more pass -- logits so large that the margin covers many -- the rest are scored as they come.
constexpr int LISTED = 64;
struct Found { int bar, listed; int at[LISTED]; };
template <typename T> __device__ __forceinline__ void score(const typename T::raw* row, uint64_t key, int at, Best& best) {
  const float v = widen(T{}, row[at]);
  const double s = noisy_score(v, key, at);
  if (v > -INFINITY && better(s, at, best.score, best.at)) best = Best{s, at};
}
// a score from below in 32 bits: E <= (1 - u) / u
__device__ __forceinline__ float at_least(float z, uint32_t w) { return z - 0.693147181f * __log2f(((float)w + 2.f) * __builtin_amdgcn_rcpf((float)~w)); }
template <typename T> __device__ __forceinline__ void draw8(const typename T::raw* row, uint64_t key, int j, const Running& a, uint32_t allowed, const float* z, const float* e, bool first, Found& found, Best& best) {
  uint32_t w[VEC];
  missing8(key, j, w);
  if (first) {   // no score yet
    float low = -INFINITY;
#pragma unroll
    for (int i = 0; i < VEC; i++) low = fmaxf(low, at_least(z[i], w[i]));
    atomicMax(&found.bar, ordered(below(low)));
  }
  const float reach = fminf(__builtin_amdgcn_exp2f((a.m - unordered(__hip_atomic_load(&found.bar, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP))) * LOG2E), 1e30f) * (1.0001f * 4294967296.f);
  bool some = false;                                           // of all lanes, on the scalar side; which one it was is asked only where there is one
#pragma unroll
  for (int i = 0; i < VEC; i++) some |= (float)w[i] <= fmaf(e[i], reach, 1.f);
  if (!some) return;
  uint32_t near = 0;
  float low = -INFINITY;
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const bool passes = (allowed >> i & 1) && (float)w[i] <= fmaf(e[i], reach, 1.f);
    near |= passes ? 1u << i : 0u;
    low = passes ? fmaxf(low, at_least(z[i], w[i])) : low;
  }
  if (!near) return;
  if (!first) atomicMax(&found.bar, ordered(below(low)));
  int to = atomicAdd(&found.listed, __popc(near));
  for (; near; near &= near - 1, to++) {
    const int at = j + __ffs(near) - 1;
    if (to < LISTED) found.at[to] = at;
    else score<T>(row, key, at, best);
  }
}
// the drawn action (-1: nothing may be taken, log-probability 0) and its log-probability
template <typename T> __device__ __forceinline__ void write_draw(const Rows& R, int row, float m, double s, const Best& b, int64_t* action, float* logp) {
  const bool some = b.at >= 0 && b.at < R.actions;
  action[row] = some ? b.at : -1;
  logp[row] = some ? (float)((double)logit<T>(R, row, b.at) - m - log(s)) : s == 0 ? 0.f : NAN;
}
constexpr int NOBODY = 0x7fffffff;
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) ur5_policy_sample(Rows R, uint64_t offset, const int64_t* gids, Draw* draws, int64_t* action, float* logp) {
  const int row = blockIdx.x / R.pieces, piece = blockIdx.x % R.pieces;
  const uint64_t key = mix64((uint64_t)gids[row] * GOLD + offset);
  __shared__ Found found;
  __shared__ Best wave[WAVES];
  if (threadIdx.x == 0) { found.bar = ordered(-INFINITY); found.listed = 0; }
  __syncthreads();
  const auto* z_row = (const typename T::raw*)R.logits + row * R.stride;
  Running a = nothing();
  Best best{-INFINITY, NOBODY};
  bool first = true;
  const auto draw = [&](int j, uint32_t allowed, float* z) {
    float e[VEC];
    if (MASK) bar8(allowed, z);
    add8<false, false>(a, z, nullptr, e);
    draw8<T>(z_row, key, j, a, allowed, z, e, first, found, best);
    first = false;
  };
  for_piece<MASK, false>(R, row, piece, [&](int j) { return fetch8<T>(z_row + j); }, [&](int j, uint32_t allowed, const Eight<T>& w) { float z[VEC]; unpack8(w, z); draw(j, allowed, z); },
    [&](int j, uint32_t allowed, int left) { float z[VEC]; take8<T>(z_row + j, left, z); draw(j, allowed, z); }, [](const Piece&, int, int, int) {});
  const Sums sums = join_workgroup(a, false, false);   // (its barrier stands between the list and its readers)
  const int listed = found.listed;
  if (listed > LISTED) {                               // the others' bests, too
    join_best(best);
    if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = best;
    __syncthreads();
    best = wave[threadIdx.x & (WAVES - 1)];
  }
  if (threadIdx.x >= 64) return;
  if ((int)threadIdx.x < listed) score<T>(z_row, key, found.at[threadIdx.x], best);
  join_best(best);
  if (threadIdx.x) return;
  if (R.pieces == 1) write_draw<T>(R, row, sums.m, sums.s, best, action, logp);
  else draws[blockIdx.x] = Draw{best.score, sums.s, sums.m, best.at};
}
template <typename T> __global__ void __launch_bounds__(THREADS) ur5_policy_sample_rows(Rows R, const Draw* draws, int64_t* action, float* logp) {
  const int row = blockIdx.x * WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= R.rows) return;
  Sums a{LOWEST, LOWEST, 0, 0, 0, 0};
  Best best{-INFINITY, NOBODY};
  for (int i = lane; i < R.pieces; i += 64) {
    const Draw d = draws[(size_t)row * R.pieces + i];
    const float m = fmaxf(a.m, d.m);
    a.s = a.s * exp((double)a.m - m) + d.s * exp((double)d.m - m);
    a.m = m;
    if (better(d.score, d.best, best.score, best.at)) best = Best{d.score, d.best};
  }
  join_lanes<64>(a, false, false);
  join_best(best);
  if (lane == 0) write_draw<T>(R, row, a.m, a.s, best, action, logp);
}

}  // namespace ur5policy
