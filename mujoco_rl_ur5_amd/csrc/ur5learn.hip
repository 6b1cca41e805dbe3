// ur5learn.hip -- C ABI of include/ur5learn.h: argument checks, launch shapes and dispatch over types for the device code of ur5_policy.h and ur5_act8.h. Nothing of the
// simulation engine is touched; the entry points share libur5sim.so and its error text.
#include <hip/hip_runtime.h>
#include <cstdint>
#include <cstdio>
#include "../../include/ur5learn.h"
#include "ur5_act8.h"
#include "ur5_policy.h"

extern "C" int ur5_learn_fail(int code, const char* text);   // ur5sim.hip: the library's error text

namespace {
using namespace ur5policy;

int fail(int code, const char* entry, const char* text) {
  char line[256];
  snprintf(line, sizeof line, "%s: %s", entry, text);
  return ur5_learn_fail(code, line);
}
// the caller's current device stays what it was
struct OnDevice {
  int before = -1;
  hipError_t error = hipSuccess;
  explicit OnDevice(int device) {
    int now = -1;
    error = hipGetDevice(&now);
    if (error == hipSuccess && now != device && (error = hipSetDevice(device)) == hipSuccess) before = now;
  }
  ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
int launched(const char* entry) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(UR5_ERR_DEVICE, entry, hipGetErrorString(e));
}
int no_device(const char* entry, hipError_t e) {
  return e == hipErrorNoDevice ? fail(UR5_ERR_NOGPU, entry, "no HIP device visible: libur5sim.so runs on an MI355X (gfx950) only, there is no CPU fallback") : fail(UR5_ERR_DEVICE, entry, hipGetErrorString(e));
}

// ---- how rows are cut. Pieces grow from one turn of 256 threads first over the maps, which share a list of allowed pixels, then along the pixels, up to 64 turns, so that a
// thread's fp32 sums stay short (512 terms); images of less than 2048 pixels take as many maps as fill a workgroup. How many pieces a call aims at: more fill the card's 256 CUs
// (8 workgroups each) more evenly, fewer share what a piece costs before and after its loads. us of the kernel at 2048 / 4096 / 8192 / 16384 pieces wanted:
// sample (512 fp32 rows) 96 / 88 / 102 / 138, logp (2000 x 40 000 bf16) 45 / 36 / 38 / 47, statistics (513 bf16 rows) 70 / 66 / 75 / 99, gradient 123 / 113 / 103 / 90, at
// 24576 89, at 32768 123 (259 fp32 rows: 78, 73, 75).
// A row of few turns is one piece of the calls that end with it: their second launch costs 3 us more than 5 turns (12 rows of 6 x 40 x 40, us a call: logp 14.4 -> 11.6, sample
// 13.9 -> 11.8; of 11 turns: logp 13.7 -> 10.7, sample 14.0 -> 17.7).
struct Aim { int64_t pieces, whole; };
constexpr Aim SAMPLE{4096, 6}, LOGP{4096, 10}, LOSS{4096, 0}, GRADIENT{24576, 0};
constexpr int64_t MOST_TURNS = 64;
int64_t clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }
void cut(int64_t rows, int64_t actions, int64_t mask_len, const Aim& aim, Rows* R) {
  const int64_t pixels = mask_len ? mask_len : actions, maps = actions / pixels, tiles = (pixels + TILE - 1) / TILE, groups = (pixels + VEC - 1) / VEC;
  const int64_t turns = clamp(rows * tiles * maps / aim.pieces, 1, MOST_TURNS);
  int64_t maps_per = clamp(turns, 1, maps), per = clamp(turns / maps_per, 1, mask_len ? MOST_PER_MASKED : MOST_PER);
  if (groups < THREADS) maps_per = clamp(THREADS / groups * maps_per, 1, maps);
  if (tiles <= (mask_len ? MOST_PER_MASKED : MOST_PER) && (groups * maps + THREADS - 1) / THREADS <= aim.whole) { per = tiles; maps_per = maps; }
  R->rows = (int)rows; R->actions = (int)actions; R->pixels = (int)pixels; R->maps = (int)maps; R->per = (int)per; R->maps_per = (int)maps_per;
  R->pieces_x = (int)((tiles + per - 1) / per);
  R->pieces = (int)(R->pieces_x * ((maps + maps_per - 1) / maps_per));
}
// workspace: records | slopes | terms of the loss (one per row; one per pair where there are more pairs than rows) | rows that count, of all and of every 256
struct Work { Part* parts; Slope* slopes; double* term; int* counting; int* counts; };
int64_t lay_out(const Rows& R, int64_t terms, void* base, Work* w) {
  char* p = (char*)base;
  const int64_t n = R.rows, parts = n * R.pieces * (int64_t)sizeof(Part), slopes = (n * (int64_t)sizeof(Slope) + 15) / 16 * 16, sums = (terms > n ? terms : n) * 8;
  int* counting = (int*)(p + parts + slopes + sums);
  if (w) *w = Work{(Part*)p, (Slope*)(p + parts), (double*)(p + parts + slopes), counting, counting + 1};
  return parts + slopes + sums + (1 + (n + THREADS - 1) / THREADS) * 4;
}
constexpr int64_t ENDS = -1;                         // in the place of pairs: sampling and log-probabilities, which leave records of rows of several pieces and nothing else
int64_t need(const Rows& R, int64_t pairs) { return pairs != ENDS ? lay_out(R, pairs, nullptr, nullptr) : R.pieces > 1 ? (int64_t)R.rows * R.pieces * (int64_t)sizeof(Part) : 0; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t MOST = 0x7fffffff;
constexpr int64_t MOST_LAUNCHED = (1 << 24) - 1;     // workgroups of 256 threads: a launch holds less than 2^32 threads

const char* check_size(int64_t rows, int64_t actions, int64_t mask_len, int64_t pairs, const Aim& aim, Rows* R) {
  if (rows < 0 || actions < 1) return "rows must be at least 0 and actions at least 1";
  if (actions > MOST - 2 * TILE * MOST_PER || rows > MOST_LAUNCHED || pairs > MOST_LAUNCHED) return "too many rows, pairs (2^24 - 1) or actions (2^31 - 65537)";
  if (mask_len < 0 || (mask_len && actions % mask_len)) return "mask_len must divide actions";
  cut(rows, actions, mask_len, GRADIENT, R);
  const int64_t most = R->pieces;                    // the finest of the cuts
  cut(rows, actions, mask_len, aim, R);
  if (rows * most > MOST_LAUNCHED - rows / THREADS - 2 * FIRST) return "too many logits in one call";
  return nullptr;
}
// checks what every entry point over rows checks; launches nothing
const char* check_rows(const ur5_rows* r, int64_t pairs, const Aim& aim, Rows* R, Work* w) {
  if (!r) return "no rows";
  if (r->dtype != UR5_F32 && r->dtype != UR5_F16 && r->dtype != UR5_BF16) return "dtype must be UR5_F32, UR5_F16 or UR5_BF16";
  if (r->mask && (r->mask_len < 1 || r->mask_stride < 0)) return "mask_len must be at least 1 and mask_stride at least 0";
  if (const char* why = check_size(r->rows, r->actions, r->mask ? r->mask_len : 0, pairs, aim, R)) return why;
  if (r->stride < r->actions && r->rows > 1) return "the row stride is smaller than a row";
  if (r->ref && r->ref_stride < r->actions && r->rows > 1) return "the reference's row stride is smaller than a row";
  if (r->rows && !r->logits) return "no logits";
  const int64_t bytes = r->rows || pairs > 0 ? need(*R, pairs) : 0;
  if (bytes && (!r->work || !aligned16(r->work) || r->work_bytes < bytes)) return "the workspace is missing, not 16-byte aligned, or smaller than ur5_policy_work_bytes";
  R->logits = r->logits; R->ref = r->ref; R->mask = r->mask; R->stride = r->stride; R->ref_stride = r->ref_stride; R->mask_stride = r->mask_stride;
  lay_out(*R, pairs, r->work, w);                    // (the records come first)
  return nullptr;
}

template <typename F> void by_type(int dtype, F f) { dtype == UR5_F32 ? f(f32_t{}) : dtype == UR5_F16 ? f(f16_t{}) : f(bf16_t{}); }
template <typename F> void by_flag(bool b, F f) { b ? f(yes{}) : f(no{}); }

const char* check_clip(const ur5_rows* r, const ur5_clip* c) {
  if (!c || (r->rows && (!c->action || !c->old_logp || !c->advantage))) return "action, old_logp and advantage are needed";
  if (!(c->clip_low >= 0 && c->clip_low <= 1) || !(c->clip_high >= 0)) return "clip_low must lie in [0, 1] and clip_high be at least 0";
  if (!(c->kl_coef >= 0) || c->entropy_coef != c->entropy_coef) return "kl_coef must be at least 0 and entropy_coef a number";
  if (c->kl_coef > 0 && !r->ref && r->rows) return "kl_coef needs reference logits";
  return nullptr;
}
Clip clip_of(const ur5_clip* c) { return Clip{c->action, c->old_logp, c->advantage, c->clip_low, c->clip_high, c->kl_coef, c->entropy_coef}; }
const char* check_prefer(const ur5_rows* r, const ur5_prefer* p) {
  if (!p || (r->rows && (!p->action || !p->ref_logp))) return "action and ref_logp are needed";
  if (p->pairs < 1 ||  !p->offsets) return "pairs must be at least 1, with 2 pairs + 1 offsets";
  if (!(p->beta > 0) || !(p->label_smoothing >= 0 && p->label_smoothing <= 0.5)) return "beta must be above 0 and label_smoothing lie in [0, 0.5]";
  return nullptr;
}
Prefer prefer_of(const ur5_prefer* p) { return Prefer{p->action, p->ref_logp, p->offsets, (int)p->pairs, p->beta, p->label_smoothing}; }

void stats(const Rows& R, int dtype, hipStream_t s, const Span& span, const int64_t* action, const Work& w) {
  if (!R.rows) return;
  const int front = (R.rows + 8 * THREADS - 1) / (8 * THREADS) * 8;
  by_type(dtype, [&](auto t) { by_flag(R.mask, [&](auto m) { by_flag(R.ref, [&](auto q) {
    ur5_policy_stats<decltype(t), decltype(m)::value, decltype(q)::value><<<front + R.rows * R.pieces, THREADS, 0, s>>>(R, span, front, action, w.parts, w.slopes, w.counts);
  }); }); });
}
// the rows of the clipped loss, or the pairs of the preference loss: slopes and terms
void clip_rows(const Rows& R, int dtype, hipStream_t s, const Clip& C, const Work& w, const ClipOut& out) {
  stats(R, dtype, s, Span{}, C.action, w);
  if (R.rows) by_type(dtype, [&](auto t) { by_flag(R.ref, [&](auto q) {
    ur5_policy_clip_rows<decltype(t), decltype(q)::value><<<(R.rows + WAVES - 1) / WAVES, THREADS, 0, s>>>(R, C, w.parts, w.slopes, w.counts, w.counting, w.term, out);
  }); });
}
// A pair's workgroup ends its rows by itself, four at a time, unless pairs are long, or so many rows come that a launch more does not count and some pair may be long.
// us a call without the launch and with it, rows of 9600 fp32 actions: 32 rows of one pair 19.6, 22.8, 64 27.6, 22.8, 512 167, 23.7; 2048 rows of 64 pairs 54, 49.
constexpr int64_t LONG_PAIR = 32, MANY_ROWS = 4096;
void prefer_pairs(const Rows& R, int dtype, hipStream_t s, const Prefer& P, const Work& w, float* margin) {
  stats(R, dtype, s, Span{P.offsets, 2 * P.pairs}, P.action, w);
  const bool ended = R.rows > LONG_PAIR * (int64_t)P.pairs || R.rows > MANY_ROWS;
  by_type(dtype, [&](auto t) {
    if (ended) ur5_policy_prefer_rows<decltype(t)><<<(R.rows + WAVES - 1) / WAVES, THREADS, 0, s>>>(R, P, w.parts, w.slopes);
    by_flag(ended, [&](auto e) { ur5_policy_prefer_pairs<decltype(t), decltype(e)::value><<<P.pairs, THREADS, 0, s>>>(R, P, w.parts, w.slopes, w.term, margin); });
  });
}
// rows that the gradient's workgroups end by themselves: FEW, or as many fewer as a lane has records of one
bool few(const Rows& R) { return R.rows * (((int64_t)R.pieces + 63) / 64) <= FEW; }
// The preference loss: a workgroup ends every row of its pair, its wavefronts a quarter each. Rows of up to 64 records gain to the edge of the rule (24 rows of 6 x 40 x 40 in one pair, two
// launches and three: 18.7 and 21.5 us a call, 14.7 and 15.4 in a graph; 24 f16 rows of 131 x 93 18.8, 21.6, 15.3, 17.2). Rows of more than that only in short pairs: 8 fp32 rows of
// 6 x 200 x 200 (120 records) in one pair 18.2 and 21.0 (16.1 and 14.6 in a graph), 12 rows in three 18.4 and 20.8 (18.0, 17.6), but 12 in one 25.1 and 21.1 (25.3, 19.5).
bool few_pairs(const Rows& R, int64_t pairs) { return few(R) && pairs <= FEW && (R.pieces <= 64 || R.rows <= 8 || R.rows <= 4 * pairs); }
// a call over more memory than the caches hold
bool past_caches(const Rows& R, int dtype) { return (int64_t)R.rows * R.actions * (dtype == UR5_F32 ? 4 : 2) * (R.ref ? 3 : 2) > CACHE_BYTES; }
void gradient(Rows R, int dtype, hipStream_t s, const Terms& t, const int64_t* action, const Work& w, float scale, const float* upstream, void* grad) {
  cut(R.rows, R.actions, R.mask ? R.pixels : 0, GRADIENT, &R);      // it leaves no records
  by_type(dtype, [&](auto k) { by_flag(R.mask, [&](auto m) { by_flag(R.ref, [&](auto q) { by_flag(past_caches(R, dtype), [&](auto p) {
    ur5_policy_grad<decltype(k), decltype(m)::value, decltype(q)::value, decltype(p)><<<FIRST + R.rows * R.pieces, THREADS, 0, s>>>(R, t, action, w.slopes, scale, upstream, grad);
  }); }); }); });
}
Terms clip_terms(const Rows& R, const Work& w, float* loss) { return Terms{w.term, R.rows, R.rows ? w.counting : nullptr, loss}; }
// the gradient of the clipped loss; the reference has no part in it without a KL term
void clip_gradient(Rows R, const ur5_rows* r, const ur5_clip* c, const Terms& t, const Work& w, void* grad) {
  if (!(c->kl_coef > 0)) R.ref = nullptr;
  gradient(R, r->dtype, (hipStream_t)r->stream, t, c->action, w, c->grad_scale, c->upstream, grad);
}
}  // namespace

#define CHECK(text) do { const char* why_ = (text); if (why_) return fail(UR5_ERR_ARG, __func__, why_); } while (0)
#define ON(device) OnDevice on_(device); if (on_.error != hipSuccess) return no_device(__func__, on_.error)

extern "C" {

int64_t ur5_policy_work_bytes(int64_t rows, int64_t actions, int64_t mask_len, int64_t pairs) {
  Rows R, L;
  if (pairs < ENDS || check_size(rows, actions, mask_len, pairs, pairs == ENDS ? SAMPLE : LOSS, &R)) return 0;
  if (pairs != ENDS) return need(R, pairs);
  cut(rows, actions, mask_len, LOGP, &L);
  return need(R.pieces > L.pieces ? R : L, ENDS);
}

int ur5_policy_sample(const ur5_rows* r, uint64_t offset, const int64_t* gids, int64_t* action, float* logp) {
  Rows R; Work w;
  CHECK(check_rows(r, ENDS, SAMPLE, &R, &w));
  if (!R.rows) return 0;
  if (!gids || !action || !logp) return fail(UR5_ERR_ARG, __func__, "gids, action and logp are needed");
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  Draw* draws = (Draw*)w.parts;
  by_type(r->dtype, [&](auto t) {
    by_flag(R.mask, [&](auto m) { ur5_policy_sample<decltype(t), decltype(m)::value><<<R.rows * R.pieces, THREADS, 0, s>>>(R, offset, gids, draws, action, logp); });
    if (R.pieces > 1) ur5_policy_sample_rows<decltype(t)><<<(R.rows + WAVES - 1) / WAVES, THREADS, 0, s>>>(R, draws, action, logp);
  });
  return launched(__func__);
}

int ur5_policy_logp(const ur5_rows* r, const int64_t* action, float* logp, float* entropy) {
  Rows R; Work w;
  CHECK(check_rows(r, ENDS, LOGP, &R, &w));
  if (!R.rows) return 0;
  if (!action || !logp) return fail(UR5_ERR_ARG, __func__, "action and logp are needed");
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  by_type(r->dtype, [&](auto t) {
    by_flag(R.mask, [&](auto m) { ur5_policy_logp<decltype(t), decltype(m)::value><<<R.rows * R.pieces, THREADS, 0, s>>>(R, action, w.parts, logp, entropy); });
    if (R.pieces > 1) ur5_policy_logp_rows<decltype(t)><<<(R.rows + WAVES - 1) / WAVES, THREADS, 0, s>>>(R, action, w.parts, logp, entropy);
  });
  return launched(__func__);
}

int ur5_policy_clip_loss(const ur5_rows* r, const ur5_clip* c, float* loss, float* logp, float* kl, float* entropy) {
  Rows R; Work w;
  CHECK(check_rows(r, 0, LOSS, &R, &w));
  CHECK(check_clip(r, c));
  if (!loss || (R.rows && (!logp || !kl || !entropy))) return fail(UR5_ERR_ARG, __func__, "loss, logp, kl and entropy are needed");
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  clip_rows(R, r->dtype, s, clip_of(c), w, ClipOut{logp, kl, entropy});
  ur5_policy_loss<<<1, THREADS, 0, s>>>(clip_terms(R, w, loss));
  return launched(__func__);
}
int ur5_policy_clip_grad(const ur5_rows* r, const ur5_clip* c, void* grad) {
  Rows R; Work w;
  CHECK(check_rows(r, 0, LOSS, &R, &w));
  CHECK(check_clip(r, c));
  if (!R.rows) return 0;
  if (!grad) return fail(UR5_ERR_ARG, __func__, "grad is needed");
  ON(r->device);
  clip_gradient(R, r, c, clip_terms(R, w, nullptr), w, grad);
  return launched(__func__);
}
int ur5_policy_clip_loss_grad(const ur5_rows* r, const ur5_clip* c, float* loss, float* logp, float* kl, float* entropy, void* grad) {
  Rows R; Work w;
  CHECK(check_rows(r, 0, LOSS, &R, &w));
  CHECK(check_clip(r, c));
  if (!loss || (R.rows && (!logp || !kl || !entropy || !grad))) return fail(UR5_ERR_ARG, __func__, "loss, logp, kl, entropy and grad are needed");
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  const ClipOut out{logp, kl, entropy};
  if (R.rows && few(R) && (!R.ref || c->kl_coef > 0) && !past_caches(R, r->dtype)) {
    const Clip C = clip_of(c);
    const int pieces = R.pieces;
    stats(R, r->dtype, s, Span{}, C.action, w);
    cut(R.rows, R.actions, R.mask ? R.pixels : 0, GRADIENT, &R);
    by_type(r->dtype, [&](auto t) { by_flag(R.mask, [&](auto m) { by_flag(R.ref, [&](auto q) {
      ur5_policy_clip_few<decltype(t), decltype(m)::value, decltype(q)::value><<<FIRST + R.rows * R.pieces, THREADS, 0, s>>>(R, pieces, C, w.parts, w.slopes, w.counts, loss, out, c->grad_scale, c->upstream, grad);
    }); }); });
    return launched(__func__);
  }
  clip_rows(R, r->dtype, s, clip_of(c), w, out);
  clip_gradient(R, r, c, clip_terms(R, w, loss), w, grad);
  return launched(__func__);
}

int ur5_policy_prefer_loss(const ur5_rows* r, const ur5_prefer* p, float* loss, float* margin) {
  Rows R; Work w;
  CHECK(check_rows(r, p ? p->pairs : 0, LOSS, &R, &w));
  CHECK(check_prefer(r, p));
  if (!loss || !margin) return fail(UR5_ERR_ARG, __func__, "loss and margin are needed");
  R.ref = nullptr;
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  prefer_pairs(R, r->dtype, s, prefer_of(p), w, margin);
  ur5_policy_loss<<<1, THREADS, 0, s>>>(Terms{w.term, (int)p->pairs, nullptr, loss});
  return launched(__func__);
}
int ur5_policy_prefer_grad(const ur5_rows* r, const ur5_prefer* p, void* grad) {
  Rows R; Work w;
  CHECK(check_rows(r, p ? p->pairs : 0, LOSS, &R, &w));
  CHECK(check_prefer(r, p));
  if (!R.rows) return 0;
  if (!grad) return fail(UR5_ERR_ARG, __func__, "grad is needed");
  R.ref = nullptr;
  ON(r->device);
  gradient(R, r->dtype, (hipStream_t)r->stream, Terms{}, p->action, w, p->grad_scale, p->upstream, grad);
  return launched(__func__);
}
int ur5_policy_prefer_loss_grad(const ur5_rows* r, const ur5_prefer* p, float* loss, float* margin, void* grad) {
  Rows R; Work w;
  CHECK(check_rows(r, p ? p->pairs : 0, LOSS, &R, &w));
  CHECK(check_prefer(r, p));
  if (!loss || !margin || (R.rows && !grad)) return fail(UR5_ERR_ARG, __func__, "loss, margin and grad are needed");
  R.ref = nullptr;
  ON(r->device);
  const hipStream_t s = (hipStream_t)r->stream;
  if (R.rows && few_pairs(R, p->pairs) && !past_caches(R, r->dtype)) {
    const Prefer P = prefer_of(p);
    const int pieces = R.pieces;
    stats(R, r->dtype, s, Span{P.offsets, 2 * P.pairs}, P.action, w);
    cut(R.rows, R.actions, R.mask ? R.pixels : 0, GRADIENT, &R);
    by_type(r->dtype, [&](auto t) { by_flag(R.mask, [&](auto m) {
      ur5_policy_prefer_few<decltype(t), decltype(m)::value><<<FIRST + R.rows * R.pieces, THREADS, 0, s>>>(R, pieces, P, w.parts, w.slopes, loss, margin, p->grad_scale, p->upstream, grad);
    }); });
    return launched(__func__);
  }
  prefer_pairs(R, r->dtype, s, prefer_of(p), w, margin);
  gradient(R, r->dtype, s, Terms{w.term, (int)p->pairs, nullptr, loss}, p->action, w, p->grad_scale, p->upstream, grad);
  return launched(__func__);
}

// ---- 8-bit checkpoints
static const char* check_planes(int dtype, int64_t planes, int64_t size) {
  if (dtype != UR5_F32 && dtype != UR5_F16 && dtype != UR5_BF16) return "dtype must be UR5_F32, UR5_F16 or UR5_BF16";
  if (planes < 0 || size < 1 || size > MOST - ur5act8::GROUP || planes > MOST || planes * ((size + ur5act8::GROUP - 1) / ur5act8::GROUP) > MOST_LAUNCHED * ur5act8::Lane<f32_t>::GROUPS) return "planes must be at least 0, a plane of 1 .. 2^31 - 65 values, and all groups below 2^29 - 31";
  return nullptr;
}
int ur5_act8_pack(const void* x, int dtype, int64_t planes, int64_t size, int8_t* codes, float* scales, int device, void* stream) {
  CHECK(check_planes(dtype, planes, size));
  if (!planes) return 0;
  if (!x || !codes || !scales || !aligned16(codes)) return fail(UR5_ERR_ARG, __func__, "x, codes (16-byte aligned) and scales are needed");
  ON(device);
  const unsigned groups = (unsigned)((size + ur5act8::GROUP - 1) / ur5act8::GROUP), total = (unsigned)(planes * groups);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr unsigned per = ur5act8::Lane<T>::GROUPS;
    ur5act8::ur5_act8_pack<T><<<(total + per - 1) / per, ur5act8::THREADS, 0, (hipStream_t)stream>>>((const typename T::raw*)x, groups, total, size, codes, scales);
  });
  return launched(__func__);
}
int ur5_act8_unpack(const int8_t* codes, const float* scales, int64_t planes, int64_t size, void* x, int dtype, int device, void* stream) {
  CHECK(check_planes(dtype, planes, size));
  if (!planes) return 0;
  if (!x || !codes || !scales || !aligned16(codes)) return fail(UR5_ERR_ARG, __func__, "x, codes (16-byte aligned) and scales are needed");
  ON(device);
  const unsigned groups = (unsigned)((size + ur5act8::GROUP - 1) / ur5act8::GROUP), total = (unsigned)(planes * groups);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr unsigned per = ur5act8::Lane<T>::GROUPS;
    by_flag(planes * size * (int64_t)(sizeof(typename T::raw) + 1) > CACHE_BYTES, [&](auto p) {
      ur5act8::ur5_act8_unpack<T, decltype(p)><<<(total + per - 1) / per, ur5act8::THREADS, 0, (hipStream_t)stream>>>(codes, scales, groups, total, size, (typename T::raw*)x);
    });
  });
  return launched(__func__);
}

static const char* check_relu(int dtype, int64_t count) {
  if (dtype != UR5_F32 && dtype != UR5_F16 && dtype != UR5_BF16) return "dtype must be UR5_F32, UR5_F16 or UR5_BF16";
  if (count < 0 || count > MOST_LAUNCHED * 2 * ur5act8::THREADS * ur5act8::Lane<f32_t>::PER) return "count must be at least 0 and below 2^35 - 2047";
  return nullptr;
}
static unsigned relu_grid(int64_t count, int per) { return (unsigned)((count + 2 * ur5act8::THREADS * per - 1) / (2 * ur5act8::THREADS * per)); }
int ur5_act8_relu(const void* x, int dtype, int64_t count, void* y, uint64_t* bits, int device, void* stream) {
  CHECK(check_relu(dtype, count));
  if (!count) return 0;
  if (!x || !y || !bits || ((uintptr_t)bits & 7)) return fail(UR5_ERR_ARG, __func__, "x, y and bits (8-byte aligned) are needed");
  ON(device);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_flag(count * 2 * (int64_t)sizeof(typename T::raw) > CACHE_BYTES, [&](auto p) {
      ur5act8::ur5_act8_relu<T, decltype(p)><<<relu_grid(count, ur5act8::Lane<T>::PER), ur5act8::THREADS, 0, (hipStream_t)stream>>>((const typename T::raw*)x, count, (typename T::raw*)y, bits);
    });
  });
  return launched(__func__);
}
int ur5_act8_relu_grad(const void* dy, int dtype, const uint64_t* bits, int64_t count, void* dx, int device, void* stream) {
  CHECK(check_relu(dtype, count));
  if (!count) return 0;
  if (!dy || !dx || !bits || ((uintptr_t)bits & 7)) return fail(UR5_ERR_ARG, __func__, "dy, dx and bits (8-byte aligned) are needed");
  ON(device);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_flag(count * 2 * (int64_t)sizeof(typename T::raw) > CACHE_BYTES, [&](auto p) {
      ur5act8::ur5_act8_relu_grad<T, decltype(p)><<<relu_grid(count, ur5act8::Lane<T>::PER), ur5act8::THREADS, 0, (hipStream_t)stream>>>((const typename T::raw*)dy, bits, count, (typename T::raw*)dx);
    });
  });
  return launched(__func__);
}

// ---- weight gradient: how the work is split. Tiles of 128 output x 256 input channels (of half the outputs, and of half or a quarter of the inputs where there are no more),
// and as many ranges of the pixels as give every CU a workgroup (two of the smaller ones): less than 8, or a multiple of 8, one set per XCD. A larger tile reads and converts
// each operand less often: 256 -> 512 channels 183 us with 128 x 256, 229 with 128 x 128, 233 with 64 x 256. One that reaches past the channels multiplies for nothing: 64 -> 128
// channels 22 us with 128 x 64, 36 with 128 x 256.
constexpr int64_t WORKGROUPS = 256;
struct WgradPlan { int to, tc, o_tiles, c_tiles, splits; int64_t part, bytes; };
static WgradPlan wgrad_plan(int64_t n, int64_t cin, int64_t cout, int64_t size) {
  WgradPlan p;
  p.to = cout > 64 ? 128 : 64; p.tc = cin > 128 ? 256 : cin > 64 ? 128 : 64;
  p.o_tiles = (int)((cout + p.to - 1) / p.to); p.c_tiles = (int)((cin + p.tc - 1) / p.tc);
  const int64_t groups = n * ((size + ur5act8::GROUP - 1) / ur5act8::GROUP), tiles = (int64_t)p.o_tiles * p.c_tiles;
  const int64_t s = clamp((WORKGROUPS * (p.to == 64 ? 2 : 1) + tiles - 1) / tiles, 1, groups > 0 ? groups : 1);
  p.splits = (int)(s < 8 ? s : (s + 7) / 8 * 8);
  p.part = ((int64_t)p.splits * cin * cout * 4 + 15) / 16 * 16;
  p.bytes = p.part + (int64_t)p.splits * cout * 4;
  return p;
}
static const char* check_wgrad(int64_t n, int64_t cin, int64_t cout, int64_t size) {
  if (n < 0 || cin < 1 || cout < 1 || cin > 65536 || cout > 65536 || cin * cout > MOST / 8) return "n must be at least 0, channels 1 .. 65536 and their product below 2^28";
  if (n > 65536) return "n must be at most 65536";
  return check_planes(UR5_F32, n * (cin > cout ? cin : cout), size);
}
int64_t ur5_act8_wgrad_work_bytes(int64_t n, int64_t cin, int64_t cout, int64_t size) { return check_wgrad(n, cin, cout, size) ? 0 : wgrad_plan(n, cin, cout, size).bytes; }
int ur5_act8_wgrad(const int8_t* codes, const float* scales, const void* dy, int dtype, int64_t n, int64_t cin, int64_t cout, int64_t size, float* dw, float* db,
                   void* work, int64_t work_bytes, int device, void* stream) {
  CHECK(check_planes(dtype, n, size));
  CHECK(check_wgrad(n, cin, cout, size));
  const WgradPlan p = wgrad_plan(n, cin, cout, size);
  if (!dw || (n && (!codes || !scales || !dy || !aligned16(codes)))) return fail(UR5_ERR_ARG, __func__, "codes (16-byte aligned), scales, dy and dw are needed");
  if (!work || !aligned16(work) || work_bytes < p.bytes) return fail(UR5_ERR_ARG, __func__, "the workspace is missing, not 16-byte aligned, or smaller than ur5_act8_wgrad_work_bytes");
  ON(device);
  const hipStream_t s = (hipStream_t)stream;
  float* part = (float*)work;
  float* part_bias = db ? (float*)((char*)work + p.part) : nullptr;
  const ur5act8::Wgrad W{codes, scales, dy, size, (int)((size + ur5act8::GROUP - 1) / ur5act8::GROUP), (int)n, (int)cin, (int)cout, p.splits, p.o_tiles, p.c_tiles, part, part_bias};
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int grid = p.splits * p.o_tiles * p.c_tiles;
    const auto run = [&](auto kernel, int threads) { kernel<<<grid, threads, 0, s>>>(W); };
    if (p.to == 128) p.tc == 256 ? run(ur5act8::ur5_act8_wgrad<T, 2, 2, 2, 4>, 512) : p.tc == 128 ? run(ur5act8::ur5_act8_wgrad<T, 1, 2, 4, 2>, 512) : run(ur5act8::ur5_act8_wgrad<T, 1, 1, 4, 2>, 512);
    else p.tc == 256 ? run(ur5act8::ur5_act8_wgrad<T, 1, 2, 2, 4>, 512) : p.tc == 128 ? run(ur5act8::ur5_act8_wgrad<T, 1, 1, 2, 4>, 512) : run(ur5act8::ur5_act8_wgrad<T, 1, 1, 2, 2>, 256);
  });
  const int weights = (int)(cin * cout), outs = weights + (db ? (int)cout : 0);
  ur5act8::ur5_act8_wgrad_sum<<<(outs + 31) / 32, ur5act8::THREADS, 0, s>>>(part, part_bias, p.splits, weights, (int)cout, dw, db);
  return launched(__func__);
}
}
