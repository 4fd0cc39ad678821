// Causal flash attention (head_dim 64) on the Blackwell tensor cores.
//
// Both kernels are persistent: one CTA per SM walks a list of work items and
// keeps its shared-memory rings and TMEM handshakes running from one item into
// the next (see the item comments at each kernel).
// Forward (attn_fwd_tc): work item = (pair of 128-query tiles, batch*head).
// 11 warps, all of TMEM: warp 0 loads both Q tiles of an item (two item
// slots) and 128-key K/V blocks into a 4-stage ring (4-D tensor maps over
// (e, t, h, b), so any [b, t, h, e] strides work and rows past the sequence
// end arrive as zeros); one MMA thread per tile issues S_x = Q_x K^T (128x128
// fp32 in TMEM) and O_x += P_x V (P_x read from TMEM, V an MN-major shared
// operand); two softmax warpgroups own one tile each (thread = query row =
// TMEM lane) and turn S_x into bf16 P_x in TMEM, so the two tiles ping-pong:
// while one warpgroup exponentiates, the tensor core runs the other tile's
// MMAs.
// Backward (attn_bwd_tc): work item = (128-key tile, batch*head), looping over
// 64-query tiles from the diagonal down. 23 warps: TMA (K, V per item in two
// slots; Q/dO into a 4-stage ring with the tile's lse/delta copied in by
// cp.async), a scores MMA thread (S^T = K Q^T and dP^T = V dO^T into one
// of three 128-column TMEM buffers, as far ahead as the buffers allow), a
// gradient MMA thread (dV += P^T dO and dK += dS^T Q with P^T / dS^T read
// straight from TMEM; dQ = dS K per pair of tiles, dS^T read MN-major from a
// shared-memory ring), 16 softmax warps that take every tile together
// (thread = key row, 16 query columns per warp: P^T = exp2(S^T c - lse),
// dS^T = P^T (dP^T - delta), written over the warp's own S^T columns as bf16
// pairs), and four dQ warps. Two issuing threads keep the tensor pipe fed
// while either waits on a barrier. The dQ warps read each pair's dQ out of
// TMEM as soon as its MMA completes and reduce it into an fp32 accumulator by
// TMA; at the end of an item they also write dK and dV.
// q and k arrive already rotated (RoPE runs in the QKV projection epilogue);
// with RoPE tables the backward rotates dq and dk back so they are gradients
// of the unrotated inputs.
// Every mbarrier wait is bounded (common.cuh). Semantics follow
// rig/kernels/tpu_flash_attention.py:171-207 (fp32 statistics, bf16 P).
//
// Score-modified attention (gptb200_score_attention_fwd/bwd) has a forward of its own,
// score_fwd_tc, and shares the backward, whose MODE kClassic is the plain causal
// attention above:
//   s'_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i - j|,
// with key/value heads shared by heads / kv_heads query heads, a per-sequence
// prefix whose keys every query sees, and segment ids whose negative values
// mark padding (a row that sees nothing gets o = 0, lse = -inf and no
// gradients). What they add to the softmax warps:
//  * tanh. The exponentials hold the MUFU pipe for 8 clocks a score (of a warp's
//    32 rows), so tanh runs on the FMA pipe beside it, 8 clocks for a score too:
//    z P(z^2) with five terms, relative error 7e-6 (seven and 5e-8 for caps above
//    kShortCap), where a warp's scores have |z| <= 1; only a warp that holds a larger
//    one takes 1 - 2 / (1 + e^(2z)), two more MUFU operations per score.
//  * the bias. Linear in the key up to the query, so it is one packed FMA for
//    two scores; |i - j| itself only near the diagonal and in the prefix.
// Masks are words of 32 keys, made once per block and warp; blocks that no mask
// reaches run code without them (tests that are predicated off still take issue
// slots). The forward's rows go through one streaming pass against the reference
// they have so far, the diagonal block first. In the backward an
// item is a key tile of a key/value head: it walks the query tiles of every query
// head that shares it, so dK and dV of the group add up in TMEM, in a fixed order.
// Roundings: P to bf16 before P.V and P^T dO, dS to bf16 before dK and dQ, delta
// from O as stored (exact for one key tile); sums, maxima, lse, dQ's accumulator
// and everything between are fp32.
// What bounds them, 1 x 12 x 8192 (us, forward | backward):
//    plain causal kernels 230 | 395; without cap and bias 181 | 343; bias
//    192 | 358; cap 238 | 429; both 259 | 454 (398 and 568 TFLOP/s).
//  Forward: the latency of two softmax warps a scheduler. Without any arithmetic
//  (raw scores packed as P) it takes 123 us; with it a warp spends 4,100 of 5,080
//  clocks a block on its 64 pairs of scores a row, where the FMA pipe needs 1,024
//  and two warps share a scheduler, and 830 waiting for the next block's scores,
//  which are issued when it has finished with this block's. Splitting blocks in
//  halves to issue them earlier halves that wait, but MMAs of 64 columns and twice
//  the handshakes cost more (293 us against 279).
//  Backward: shared memory. Without any arithmetic it takes 309 us, 1,510 clocks a
//  tile of 128 x 64; the MMAs' operands (88 KB), dS^T, the Q and dO tiles and dQ's
//  way out are 152 KB a tile, 1,190 clocks at 128 bytes a clock.
#include <algorithm>
#include <mutex>
#include <new>
#include <shared_mutex>
#include <type_traits>
#include <unordered_map>
#include <vector>

#include "common.cuh"

namespace gptb200 {

static __device__ int g_attn_error;


constexpr int HD = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Modes of the score-modified kernels (bits: 1 always, 2 cap, 4 bias, 8 a cap above
// kShortCap); kClassic is the plain attention's backward.
enum { kClassic = 0, kGeneral = 1, kCap = 2, kBias = 4, kWide = 8 };
// An error of tanh counts cap times in a score. Its five terms (7e-6 relative) are up
// to 7e-4 of a probability at this cap, a third of the rounding to bf16; larger caps
// take seven (5e-8). 1 x 12 x 8192 capped (us, forward | backward): 238 | 429 with
// five, 278 | 443 with seven.
constexpr float kShortCap = 128.f;

struct AttnParams {
  int B, H, T;         // H: query heads
  int KVH, group;      // key/value heads, query heads per key/value head (score-modified)
  float scale;
  float cap;           // tanh cap of the scaled scores (kCap)
  const float* slopes; // [H] distance slopes (kBias)
  const int* prefix;   // [B] keys every query sees, or null (score-modified)
  int by_weight;       // items of all heads by falling weight (score-modified)
  // output / saved tensors
  bf16* o;
  int64_t osb, osh, ost;
  float* o32;          // [B, H, T, 64] fp32 instead of o and lse, or null (score-modified)
  float* lse;          // [B, H, T], natural log
  const bf16* dout;
  const float* delta;  // [B, H, T] (score-modified: negated)
  const float* neg_lse2;  // [B, H, T] -lse log2(e) (score-modified)
  float* dq_acc;       // [B, H, T, 64] fp32
  bf16* dk;
  bf16* dv;
  int64_t sb, sh, st;  // q/k/v (and dq/dk/dv) strides
  const bf16* rcos;    // RoPE tables [T, 32] or null
  const bf16* rsin;
  const int* seg;      // document segment ids [B, T] or null (causal only)
  unsigned* sched;     // this launch's work counter {next item, finished CTAs}
};

__device__ __forceinline__ uint32_t swz128(int row, int chunk) {
  return (uint32_t)(row * 128 + (((chunk ^ (row & 7)) & 7) << 4));
}

// Rotates 4 interleaved pairs (one 16-byte chunk holding elements 8c..8c+7 of
// position t) by the transpose of the RoPE rotation.
__device__ __forceinline__ void rope_back(float* v, const bf16* rcos, const bf16* rsin, int t,
                                          int c) {
  const bf16* cs = rcos + (int64_t)t * (HD / 2) + c * 4;
  const bf16* sn = rsin + (int64_t)t * (HD / 2) + c * 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float cv = __bfloat162float(cs[j]), sv = __bfloat162float(sn[j]);
    float ge = v[2 * j], go = v[2 * j + 1];
    v[2 * j] = ge * cv + go * sv;
    v[2 * j + 1] = -ge * sv + go * cv;
  }
}

// ------------------------------------------------------------------ segments
// Document masking (rig/kernels/tpu_flash_attention.py:171-207 with segment
// ids): a query sees a key only if the key is not later and both carry the same
// segment id. Each CTA first reduces the ids of every 64-position chunk of its
// sequence to a (min, max) range in shared memory; a key block and a query tile
// whose ranges are disjoint never meet, and when both ranges are one and the
// same single id no per-element test is needed. Both hold for any ids; with the
// nondecreasing ids of document_segments (rig/attention.py:205-208) the blocks
// before a query tile's first document are exactly the ones skipped.
constexpr int kSegChunk = 64;
constexpr int kMaxSegChunks = 1024;  // segment ids are supported up to T = 65536

__device__ __forceinline__ int2 rng_merge(int2 a, int2 b) {
  return make_int2(min(a.x, b.x), max(a.y, b.y));
}
__device__ __forceinline__ bool rng_meet(int2 a, int2 b) { return a.x <= b.y && b.x <= a.y; }
__device__ __forceinline__ bool rng_single(int2 a, int2 b) {
  return a.x == a.y && b.x == b.y && a.x == b.x;
}

// Range of the ids in table entries [c, c + n) (entries at or past nch are empty).
__device__ __forceinline__ int2 seg_range(const int2* tab, int nch, int c, int n) {
  int2 r = make_int2(INT_MAX, INT_MIN);
  for (int i = c; i < c + n && i < nch; ++i) r = rng_merge(r, tab[i]);
  return r;
}

// Dynamic work distribution of the persistent kernels: the TMA warp of each
// CTA takes the next item index from a per-launch counter (the items are laid
// out head by head, heaviest first within a head, so the items in flight at
// once cover a few heads whose K/V or Q/dO tiles come from DRAM about once and
// are then served from L2, and a CTA that finishes early takes more work).
// The counters live in a device array of slots. Launches that may overlap on the
// GPU have different slots (SchedSlot), and the last CTA of a launch to finish
// puts its slot back to zero.
constexpr int kSchedSlots = 1 << 16;
__device__ unsigned g_attn_sched[kSchedSlots][2];

// Called by the whole producer warp: the next item index (lane 0 fetches).
__device__ __forceinline__ int next_item(unsigned* sched, int lane) {
  int v = 0;
  if (lane == 0) v = (int)atomicAdd(sched, 1u);
  return __shfl_sync(0xffffffffu, v, 0);
}

// Called by thread 0 of each CTA after all of the CTA's work: the last CTA
// resets the launch's counter slot.
__device__ __forceinline__ void sched_finish(unsigned* sched) {
  __threadfence();
  if (atomicAdd(sched + 1, 1u) == gridDim.x - 1) {
    sched[0] = 0;
    sched[1] = 0;
    __threadfence();
  }
}

// ------------------------------------------------------------------ scores
// tanh(z) / z in u = z^2 on |z| <= 1: minimax in relative error (7e-6 and 5e-8) by
// reweighted least squares over Chebyshev points.
#define GPTB200_TANH_COEFS \
  {0.999993085861206f, -0.3329806327819824f, 0.13036808371543884f, -0.04481752589344978f, \
   0.009036410599946976f}
#define GPTB200_TANH_WIDE_COEFS \
  {0.9999999403953552f, -0.33332839608192444f, 0.13325203955173492f, -0.053457025438547134f, \
   0.02028997428715229f, -0.006203373894095421f, 0.0010410209652036428f}

// Any z: 1 - 2 / (1 + e^(2z)), an absolute error of a few 2^-24. WIDE: that on |z| > 1
// only, the seven terms below, a few 2^-24 of the result.
template <bool WIDE>
GPTB200_DEV float tanh_any(float z) {
  const float far = fmaf(-2.f, __fdividef(1.f, 1.f + ex2(2.f * kLog2e * z)), 1.f);
  if constexpr (!WIDE) return far;
  constexpr float c[7] = GPTB200_TANH_WIDE_COEFS;
  const float u = z * z;
  float a = c[6];
#pragma unroll
  for (int e = 5; e >= 0; --e) a = fmaf(u, a, c[e]);
  return u <= 1.f ? z * a : far;
}

GPTB200_DEV float fmax3_abs(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A query row's raw scores, 32 columns (keys) at a time, and their way to the
// probabilities exp2(s' log2(e) - m), packed as bf16 pairs. The callers loop over
// the chunks of a block without unrolling: two warps of a scheduler at different
// places of a block-long sequence of instructions fetch more than they compute.
template <int MODE>
struct Score {
  static constexpr bool CAP = (MODE & kCap) != 0, BIAS = (MODE & kBias) != 0;
  static constexpr bool WIDE = (MODE & kWide) != 0;
  static constexpr int TERMS = WIDE ? 7 : 5;
  // A row keeps its reference m until a block's probabilities against it add up to
  // more than this: 128 keys at the 2^8 that the plain kernels allow one. bf16 and
  // the fp32 sums lose nothing below that. O before its division by l is at most the
  // sum of the probabilities times max |v|: finite for |v| up to 2^113 / blocks.
  static constexpr float kSlack = 0x1p15f;
  // A reference is set this far (log2) above the maximum that asks for it, so that
  // later keys seldom reach the limit: a row's first block is its diagonal one, and
  // its first rows see few keys. Without it 10% more time at 8 x 12 x 1024 (general
  // 45.0 us, with 6 41.7, 8 40.1, 10 and 12 39.7); smaller probabilities are as exact.
  static constexpr float kRoom = 12.f;
  float z_per_s;  // tanh's argument per raw score
  float out;      // s' log2(e) per tanh, or per raw score
  float slope2;   // slope * log2(e)
  float far_max;  // the largest raw score squared (WIDE: z squared) with |z| <= 1
  GPTB200_DEV Score(const AttnParams& p, float slope2_) : slope2(slope2_) {
    // (finite for the smallest caps too: a score of 0 stays 0)
    z_per_s = CAP ? fminf(p.scale / p.cap, 0x1p100f) : 1.f;
    out = (CAP ? p.cap : p.scale) * kLog2e;
    // below 2^-13 the ninth power in stream_coefs may underflow: never stream
    far_max = WIDE ? 1.f : z_per_s < 0x1p-13f ? -1.f : 1.f / (z_per_s * z_per_s);
  }
  static GPTB200_DEV float2 both(float x) { return make_float2(x, x); }
  static GPTB200_DEV float2 pair(const uint32_t (&v)[32], int i) {
    return make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
  }
  // The polynomial's coefficients, times `by`.
  static GPTB200_DEV void coefs(float2 (&k)[TERMS], float by) {
    constexpr float c[5] = GPTB200_TANH_COEFS, w[7] = GPTB200_TANH_WIDE_COEFS;
#pragma unroll
    for (int u = 0; u < TERMS; ++u) k[u] = both(by * (WIDE ? w[u] : c[WIDE ? 0 : u]));
  }
  // Four pairs at a time, so that their dependent steps interleave.
  static GPTB200_DEV void poly4(const float2 (&k)[TERMS], const float2 (&u)[4], float2 (&a)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = ffma2(u[q], k[TERMS - 1], k[TERMS - 2]);
#pragma unroll
    for (int e = TERMS - 3; e >= 0; --e) {
#pragma unroll
      for (int q = 0; q < 4; ++q) a[q] = ffma2(u[q], a[q], k[e]);
    }
  }

  // Without masks, keys before the query, against the reference m: arithmetic (FMA
  // pipe) and exponentials (MUFU) of different columns overlap, with nothing to
  // wait for in between. 16 columns at a time; the callers have the next ones on
  // their way from TMEM meanwhile. far collects the largest raw score squared; the
  // caller discards the block if it, or the sum of the probabilities, does not do. The tanh's
  // argument is not formed: its factor is in the coefficients (stream_coefs; WIDE forms
  // it, as the factor's powers would underflow). The
  // bias, slope (key - query), with -m folded in, runs in four pairs that step by
  // eight keys: one addition for two scores. `at`: first key - query.
  GPTB200_DEV void stream_coefs(float2 (&k)[TERMS]) const {
    if constexpr (WIDE) return coefs(k, out);
    constexpr float c[5] = GPTB200_TANH_COEFS;
    float f = out * z_per_s;
#pragma unroll
    for (int u = 0; u < 5; ++u) {
      k[u] = both(f * c[u]);
      f *= z_per_s * z_per_s;
    }
  }
  GPTB200_DEV void stream_bias(float at, float m, float2 (&off)[4]) const {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      off[q] = BIAS ? make_float2(fmaf(slope2, at + (float)(2 * q), -m),
                                  fmaf(slope2, at + (float)(2 * q + 1), -m))
                    : both(-m);
  }
  GPTB200_DEV void stream(const uint32_t (&v)[16], const float2 (&k)[TERMS], float2 (&off)[4],
                          uint32_t* pk, float2 (&acc)[2], float& far) const {
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      float2 s[4], y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        s[q] = make_float2(__uint_as_float(v[i + 2 * q]), __uint_as_float(v[i + 2 * q + 1]));
      if constexpr (CAP) {
        float2 u[4], a[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (WIDE) s[q] = fmul2(s[q], both(z_per_s));
          u[q] = fmul2(s[q], s[q]);
        }
        poly4(k, u, a);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          far = fmax3(far, u[q].x, u[q].y);
          y[q] = ffma2(s[q], a[q], off[q]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = ffma2(s[q], both(out), off[q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (BIAS) off[q] = fadd2(off[q], both(8.f * slope2));
        y[q] = make_float2(ex2(y[q].x), ex2(y[q].y));
        acc[q & 1] = fadd2(acc[q & 1], y[q]);
        pk[i / 2 + q] = pack_bf16x2(y[q].x, y[q].y);
      }
    }
  }
  // Whether a block that went through stream() has to be done in steps.
  GPTB200_DEV bool discard(float sum, float far) const {
    // (m = -inf lifts everything to +inf)
    return __any_sync(0xffffffffu, !(sum <= kSlack) || (CAP && !(far <= far_max)));
  }

  // Modified scores in place of the raw ones, in log2, and their maximum; those
  // not in `see` become -inf (and do not choose tanh's form).
  GPTB200_DEV float modify(uint32_t (&v)[32], float at, uint32_t see, bool full) const {
    bool large = false;
    if constexpr (CAP) {
      float far = 0.f;
      if (!full) hide(v, see, 0.f);
#pragma unroll
      for (int i = 0; i < 32; i += 2) far = fmax3_abs(far, pair(v, i).x, pair(v, i).y);
      large = __any_sync(0xffffffffu, far * z_per_s > 1.f);
    }
    if (large) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[i] = __float_as_uint(
            biased(out * tanh_any<WIDE>(__uint_as_float(v[i]) * z_per_s), at + (float)i));
    } else {
      float2 k[TERMS];
      if constexpr (CAP) coefs(k, out);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        float2 y[4];
        if constexpr (CAP) {
          float2 z[4], u[4], a[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) z[q] = fmul2(pair(v, i + 2 * q), both(z_per_s));
#pragma unroll
          for (int q = 0; q < 4; ++q) u[q] = fmul2(z[q], z[q]);
          poly4(k, u, a);
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = fmul2(z[q], a[q]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = fmul2(pair(v, i + 2 * q), both(out));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[i + 2 * q] = __float_as_uint(biased(y[q].x, at + (float)(i + 2 * q)));
          v[i + 2 * q + 1] = __float_as_uint(biased(y[q].y, at + (float)(i + 2 * q + 1)));
        }
      }
    }
    if (!full) hide(v, see, -INFINITY);
    float t[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; i += 2) t[(i >> 1) & 1] = fmax3(t[(i >> 1) & 1], pair(v, i).x, pair(v, i).y);
    return fmaxf(t[0], t[1]);
  }
  GPTB200_DEV float biased(float y, float distance) const {
    return BIAS ? fmaf(-slope2, fabsf(distance), y) : y;
  }
  static GPTB200_DEV void hide(uint32_t (&v)[32], uint32_t see, float to) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = (see >> i) & 1u ? v[i] : __float_as_uint(to);
  }
  // Backward, transposed: one key against 16 queries. stat: the queries' -lse
  // log2(e) at [0, 16) and -delta at [64, 80). P = exp2(s' log2(e) - lse log2(e))
  // and dS = P (dP - delta) ds'/ds, packed; zero at queries not in `see`.
  // at: key - query of column 0. EDGE: with hidden queries or keys past a query;
  // apart, because its tests would be issued (predicated off) in every chunk.
  template <bool EDGE>
  GPTB200_DEV void gradients(uint32_t (&s)[16], const uint32_t (&d)[16], const float* stat, float at,
                             uint32_t see, uint32_t (&pk)[8], uint32_t (&dk)[8]) const {
    bool large = false;
    if constexpr (CAP) {
      float far[2] = {0.f, 0.f};
      if constexpr (EDGE) {  // hidden scores do not choose tanh's form
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = (see >> j) & 1u ? s[j] : 0u;
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2)
        far[(j >> 1) & 1] =
            fmax3_abs(far[(j >> 1) & 1], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
      large = __any_sync(0xffffffffu, fmaxf(far[0], far[1]) * z_per_s > 1.f);
    }
    float2 k[TERMS];
    if constexpr (CAP) coefs(k, 1.f);
    float2 b = make_float2(slope2 * at, slope2 * (at - 1.f));  // the bias, key up to the query
#pragma unroll
    for (int j = 0; j < 16; j += 8) {
      float2 t[4], w[4];  // tanh (without a cap: the raw score), ds' / ds
#pragma unroll
      for (int q = 0; q < 4; ++q)
        t[q] = make_float2(__uint_as_float(s[j + 2 * q]), __uint_as_float(s[j + 2 * q + 1]));
      if constexpr (CAP) {
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q] = fmul2(t[q], both(z_per_s));
        if (large) {
#pragma unroll
          for (int q = 0; q < 4; ++q) t[q] = make_float2(tanh_any<WIDE>(t[q].x), tanh_any<WIDE>(t[q].y));
        } else {
          float2 u[4], a[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) u[q] = fmul2(t[q], t[q]);
          poly4(k, u, a);
#pragma unroll
          for (int q = 0; q < 4; ++q) t[q] = fmul2(t[q], a[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = ffma2(fmul2(t[q], t[q]), both(-1.f), both(1.f));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = j + 2 * q;
        const float4 n4 = *reinterpret_cast<const float4*>(stat + (i & ~3));
        const float4 g4 = *reinterpret_cast<const float4*>(stat + 64 + (i & ~3));
        float2 n = q & 1 ? make_float2(n4.z, n4.w) : make_float2(n4.x, n4.y);
        const float2 g = q & 1 ? make_float2(g4.z, g4.w) : make_float2(g4.x, g4.y);
        if constexpr (BIAS) {
          if constexpr (EDGE) {
            n.x = fmaf(-slope2, fabsf(at - (float)i), n.x);
            n.y = fmaf(-slope2, fabsf(at - (float)(i + 1)), n.y);
          } else {
            n = fadd2(n, b);
            b = fadd2(b, both(-2.f * slope2));
          }
        }
        float2 x = ffma2(t[q], both(out), n);
        x = make_float2(ex2(x.x), ex2(x.y));
        float2 y = fmul2(x, fadd2(make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), g));
        if constexpr (CAP) y = fmul2(y, w[q]);
        pk[i / 2] = pack_bf16x2(x.x, x.y);
        dk[i / 2] = pack_bf16x2(y.x, y.y);
      }
    }
    if constexpr (EDGE) {  // halves of the packed pairs
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t keep = ((see >> (2 * i)) & 1u ? 0x0000ffffu : 0u) |
                              ((see >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
        pk[i] &= keep;
        dk[i] &= keep;
      }
    }
  }
  // Probabilities of modified scores.
  static GPTB200_DEV void exponentials(const uint32_t (&v)[32], float m, uint32_t (&pk)[16],
                                       float2 (&acc)[2]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float2 y = fadd2(pair(v, i), both(-m));
      y = make_float2(ex2(y.x), ex2(y.y));
      acc[(i >> 1) & 1] = fadd2(acc[(i >> 1) & 1], y);
      pk[i / 2] = pack_bf16x2(y.x, y.y);
    }
  }
};

// Bits of the keys 0..lim of a key block.
GPTB200_DEV void causal_words(int lim, uint32_t (&see)[4]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int n = lim - 32 * w;  // the word's last visible key
    see[w] = n >= 31 ? 0xffffffffu : n < 0 ? 0u : (2u << n) - 1u;
  }
}
// ANDs in the keys that carry the row's id: one ballot per word for every
// distinct id among the warp's 32 rows (packed documents have one or two).
// kid[w]: the id of key 32 w + lane.
GPTB200_DEV void segment_words(const int (&kid)[4], int sq, uint32_t (&see)[4]) {
  uint32_t same[4] = {0, 0, 0, 0};
  uint32_t left = 0xffffffffu;
  while (left) {
    const int id = __shfl_sync(0xffffffffu, sq, __ffs(left) - 1);
    const bool mine = sq == id;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t b = __ballot_sync(0xffffffffu, kid[w] == id);
      if (mine) same[w] = b;
    }
    left &= ~__ballot_sync(0xffffffffu, mine);
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) see[w] &= same[w];
}

// Bits of the 16 queries that carry the key's id; id: of query `lane % 16`. One
// ballot for every distinct id among the warp's 32 keys.
GPTB200_DEV uint32_t segment_columns(int id, int key_id) {
  uint32_t same = 0, left = 0xffffffffu;
  while (left) {
    const int one = __shfl_sync(0xffffffffu, key_id, __ffs(left) - 1);
    const uint32_t b = __ballot_sync(0xffffffffu, id == one);
    const bool mine = key_id == one;
    if (mine) same = b & 0xffffu;
    left &= ~__ballot_sync(0xffffffffu, mine);
  }
  return same;
}

// Padding (a negative id) never equals another id: queries carry -2, keys -1.
GPTB200_DEV int seg_query_id(int v) { return v < 0 ? -2 : v; }
GPTB200_DEV int seg_key_id(int v) { return v < 0 ? -1 : v; }
// Ranges of ids with padding as -1: it is part of its chunk's (and so of its
// tile's) range, but what meets, or is one id without a test, is an id >= 0.
GPTB200_DEV int2 seg_chunk(int mn, int mx) { return make_int2(max(mn, -1), max(mx, -1)); }
GPTB200_DEV bool seg_meet(int2 a, int2 b) { return rng_meet(a, b) && min(a.y, b.y) >= 0; }
GPTB200_DEV bool seg_single(int2 a, int2 b) { return rng_single(a, b) && a.x >= 0; }

// ------------------------------------------------------------------ forward
// Persistent: one CTA per SM walks work items (pair of 128-query tiles pr,
// batch*head bh), item = bh * npair + (npair-1-pr), handed out by next_item.
// Every role keeps running
// counters across items, so the K/V ring and the per-tile S/P/O handshakes
// flow from one item into the next; Q tiles are double-buffered per item.
constexpr int FQ = 128;                 // queries per tile (TMEM lanes); two tiles per item
constexpr int FK = 128;                 // keys per K/V block
constexpr int Q_BYTES = FQ * 128;       // 128 rows x 64 bf16
constexpr int KV_BYTES = FK * 128;      // 128 rows x 64 bf16
constexpr int kKvStages = 4;
constexpr int kFwdMma1Warp = 10;       // MMA thread of tile 1 (warp 1 serves tile 0)
constexpr int kFwdThreads = 32 * 11;
// score_fwd_tc: whole warpgroups, so that registers can move from the one
// that loads and issues (warps 0-3, the last one idle) to the two softmax ones
// (4-7: tile 0, 8-11: tile 1), which keep a block's raw scores beside its
// probabilities. The shares add up to what the launch gives.
constexpr int kFwdGeneralThreads = 32 * 12;
constexpr int kFwdRegs = 168, kFwdRegsIssue = 56, kFwdRegsSoftmax = 224;
static_assert(kFwdRegsIssue + 2 * kFwdRegsSoftmax == 3 * kFwdRegs, "register shares");
constexpr int kFwdItemUsers = 2 + 8;   // both MMA threads, the 8 softmax warps

// Item slot written by the TMA warp: pair, batch*head, key blocks the pair
// visits (tile 0 the first n0 of them), whether tile 1 lies inside the sequence.
struct FwdItem {
  int pr, bh, nkv, n0, has1;
  int nch;     // chunks of the segment table (score_fwd_tc)
  int prefix;  // keys every query sees (score_fwd_tc)
  int pad;
};

template <bool SEG>
struct FwdSmem {
  static constexpr int Q = 0;                                 // 2 item slots x 2 tiles
  static constexpr int K = Q + 4 * Q_BYTES;                   // kKvStages
  static constexpr int V = K + kKvStages * KV_BYTES;          // kKvStages
  static constexpr int ITEM = V + kKvStages * KV_BYTES;       // 2 FwdItem slots
  // segment ids only: per slot, (min, max) id per 64-position chunk and the
  // key blocks the pair visits; per tile, two buffers of a block's key ids
  static constexpr int SEGTAB = ITEM + 64;
  static constexpr int BLOCKS = SEGTAB + (SEG ? 2 * kMaxSegChunks * 8 : 0);
  static constexpr int KSEG = BLOCKS + (SEG ? 2 * (kMaxSegChunks / 2) * 4 : 0);
  static constexpr int BAR = KSEG + (SEG ? 2 * 2 * FK * 4 : 0);
  // the dynamic shared memory base is 1024-byte aligned (checked at entry)
  static constexpr int TOTAL = BAR + 256;
};

template <bool SEG>
__global__ void __launch_bounds__(kFwdThreads, 1)
    attn_fwd_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const AttnParams p) {
  using L = FwdSmem<SEG>;
  extern __shared__ __align__(1024) uint8_t smem_fwd[];
  uint8_t* sm = smem_fwd;
  if (smem_u32(sm) & 1023) {  // the layout needs 1024-byte aligned tiles: give up, flagged
    if (threadIdx.x == 0) {
      atomicCAS(&g_attn_error, 0, kErrSmemAlign);
      sched_finish(p.sched);
    }
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BAR);
  uint64_t* q_full = bars + 0;                 // [2 item slots]
  uint64_t* q_empty = bars + 2;                // [2]
  uint64_t* kv_full = bars + 4;                // [kKvStages]
  uint64_t* kv_empty = kv_full + kKvStages;    // [kKvStages]
  uint64_t* s_full = kv_empty + kKvStages;     // [2 tiles]: S of the current block is in TMEM
  uint64_t* p_full = s_full + 2;               // [2]: P written to TMEM
  uint64_t* pv_done = p_full + 2;              // [2]: the tile's P.V MMA has completed
  uint64_t* s_free = pv_done + 2;              // [2]: S has been loaded into registers
  uint64_t* kseg_full = s_free + 2;            // [2 tiles][2]: a block's key ids are in smem
  uint64_t* item_full = kseg_full + 4;         // [2]
  uint64_t* item_empty = item_full + 2;        // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(item_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  FwdItem* items = reinterpret_cast<FwdItem*>(sm + L::ITEM);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int BH = p.B * p.H;
  const int npair = (p.T + 2 * FQ - 1) / (2 * FQ);
  const int n_items = npair * BH;  // item = bh * npair + (npair - 1 - pair)
  int* err = &g_attn_error;
  auto segtab_of = [&](int slot) {
    return reinterpret_cast<int2*>(sm + L::SEGTAB) + slot * kMaxSegChunks;
  };
  // key block of list entry j of the item in `slot`
  auto kblock = [&](int slot, int j) -> int {
    if constexpr (SEG)
      return reinterpret_cast<const int*>(sm + L::BLOCKS)[slot * (kMaxSegChunks / 2) + j];
    else
      return j;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 2);  // released by each tile's MMA thread
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], kFwdItemUsers);
    }
    for (int s = 0; s < kKvStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);  // released by each tile's MMA thread
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
      mbar_init(&pv_done[x], 1);
      mbar_init(&s_free[x], 4);
      mbar_init(&kseg_full[2 * x], FQ);
      mbar_init(&kseg_full[2 * x + 1], FQ);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // TMEM columns: S[2] (128 fp32 each) | O[2] (64 fp32) | P[2] (128 keys as bf16 pairs)
  const uint32_t tmem = *tmem_slot;
  auto tS = [&](int x) { return tmem + 128 * x; };
  auto tO = [&](int x) { return tmem + 256 + 64 * x; };
  auto tP = [&](int x) { return tmem + 384 + 64 * x; };

  if (warp == 0) {
    // Item producer: publishes each item's slot (with segment ids also the
    // chunk ranges and the key-block list), then loads its two Q tiles and its
    // K/V blocks into the ring.
    bool ok = true;
    int gk = 0;
    for (int ii = 0; ok; ++ii) {
      const int slot = ii & 1;
      const int item = next_item(p.sched, lane);
      if (!(ok = mbar_wait(&item_empty[slot], ((ii >> 1) & 1) ^ 1, abort_flag, err))) break;
      if (item >= n_items) {  // no more work: an empty slot ends every role's loop
        if (lane == 0) {
          items[slot].nkv = -1;
          mbar_arrive(&item_full[slot]);
        }
        break;
      }
      const int bh = item / npair, pr = npair - 1 - (item - bh * npair);
      const int b = bh / p.H, h = bh - b * p.H;
      const int q0 = pr * 2 * FQ;
      // tile x's diagonal key block is d0 + x; tile 1 of the last pair may lie
      // wholly past the sequence end
      const int d0 = q0 / FK;
      const int has1 = q0 + FQ < p.T;
      const int dmax = has1 ? d0 + 1 : d0;
      int nkv = dmax + 1, n0 = d0 + 1;
      if constexpr (SEG) {
        // The key blocks 0..dmax either query tile can see, in order. Both
        // tiles walk this one list (tile 0 its prefix up to d0); a block only
        // the other tile needs is fully masked for a tile, at most costing its
        // exps.
        const int* segrow = p.seg + (int64_t)b * p.T;
        int2* tab = segtab_of(slot);
        const int nch = min((p.T + kSegChunk - 1) / kSegChunk, 2 * (dmax + 1));
        for (int c = 0; c < nch; ++c) {
          int mn = INT_MAX, mx = INT_MIN;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t = c * kSegChunk + u * 32 + lane;
            if (t < p.T) {
              const int v = segrow[t];
              mn = min(mn, v);
              mx = max(mx, v);
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          }
          if (lane == 0) tab[c] = make_int2(mn, mx);
        }
        __syncwarp();
        if (lane == 0) {
          int* bl = reinterpret_cast<int*>(sm + L::BLOCKS) + slot * (kMaxSegChunks / 2);
          const int2 qr0 = seg_range(tab, nch, 2 * d0, 2);
          const int2 qr1 = seg_range(tab, nch, 2 * d0 + 2, 2);
          int n = 0, n_le0 = 0;
          for (int j = 0; j <= dmax; ++j) {
            const int2 kr = seg_range(tab, nch, 2 * j, 2);
            if ((j <= d0 && rng_meet(kr, qr0)) || (has1 && rng_meet(kr, qr1))) {
              bl[n++] = j;
              if (j <= d0) ++n_le0;
            }
          }
          nkv = n;
          n0 = n_le0;
        }
        nkv = __shfl_sync(0xffffffffu, nkv, 0);
        n0 = __shfl_sync(0xffffffffu, n0, 0);
      }
      if (lane == 0) {
        items[slot] = FwdItem{pr, bh, nkv, n0, has1, 0, 0, 0};
        mbar_arrive(&item_full[slot]);
        if ((ok = mbar_wait(&q_empty[slot], ((ii >> 1) & 1) ^ 1, abort_flag, err))) {
          uint8_t* qd = sm + L::Q + slot * 2 * Q_BYTES;
          mbar_arrive_expect_tx(&q_full[slot], 2 * Q_BYTES);
          tma_load_4d(qd, &tmQ, &q_full[slot], 0, q0, h, b);
          tma_load_4d(qd + Q_BYTES, &tmQ, &q_full[slot], 0, q0 + FQ, h, b);
        }
        for (int j = 0; ok && j < nkv; ++j, ++gk) {
          const int s = gk % kKvStages;
          if (!(ok = mbar_wait(&kv_empty[s], ((gk / kKvStages) & 1) ^ 1, abort_flag, err))) break;
          mbar_arrive_expect_tx(&kv_full[s], 2 * KV_BYTES);
          const int key0 = kblock(slot, j) * FK;
          tma_load_4d(sm + L::K + s * KV_BYTES, &tmK, &kv_full[s], 0, key0, h, b);
          tma_load_4d(sm + L::V + s * KV_BYTES, &tmV, &kv_full[s], 0, key0, h, b);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
  } else if (warp == 1 || warp == kFwdMma1Warp) {
    // One MMA thread per tile: S_x = Q_x K_j^T (128 x 128 fp32) for the next
    // block as soon as the softmax holds S_x in registers, O_x += P_x V_j
    // once P_x is in TMEM. The two tiles progress independently; each walks
    // every block of the item's list and releases the ones it does not use.
    const int x = warp == 1 ? 0 : 1;
    if (lane == 0) {
      constexpr uint32_t idS = umma_idesc_bf16(128, FK, 0, 0);
      constexpr uint32_t idO = umma_idesc_bf16(128, HD, 0, 1);  // A = P in TMEM, B = V MN-major
      bool ok = true;
      int gk = 0, jx = 0, ii = 0;  // ring block, this tile's running block, item
      for (; ok; ++ii) {
        const int slot = ii & 1;
        if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
        const FwdItem inf = items[slot];
        if (inf.nkv < 0) break;  // no more items
        const int nb = x == 0 ? inf.n0 : (inf.has1 ? inf.nkv : 0);
        const uint32_t sQ = smem_u32(sm + L::Q + (slot * 2 + x) * Q_BYTES);
        auto issue_s = [&](int s) {
          const uint32_t sK = smem_u32(sm + L::K + s * KV_BYTES);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            umma_bf16(tS(x), umma_smem_desc(sQ + k * 32, 16, 1024),
                      umma_smem_desc(sK + k * 32, 16, 1024), idS, k > 0);
          umma_commit(&s_full[x]);
        };
        if (nb > 0) {
          // S of the item's first block: Q loaded, the block loaded, and the
          // previous item's last S taken out of TMEM by the softmax
          ok = mbar_wait(&q_full[slot], (ii >> 1) & 1, abort_flag, err) &&
               mbar_wait(&kv_full[gk % kKvStages], (gk / kKvStages) & 1, abort_flag, err) &&
               (jx == 0 || mbar_wait(&s_free[x], (jx - 1) & 1, abort_flag, err));
          if (!ok) break;
          tc_fence_after();
          issue_s(gk % kKvStages);
        }
        for (int j = 0; ok && j < inf.nkv; ++j) {
          const int s = (gk + j) % kKvStages;
          if (j >= nb) {  // a block this tile skips: release it once it has arrived
            if (!(ok = mbar_wait(&kv_full[s], ((gk + j) / kKvStages) & 1, abort_flag, err))) break;
            mbar_arrive(&kv_empty[s]);
            continue;
          }
          const int jj = jx + j;  // running block index of this tile
          if (j + 1 < nb) {
            const int s1 = (gk + j + 1) % kKvStages;
            if (!(ok = mbar_wait(&kv_full[s1], ((gk + j + 1) / kKvStages) & 1, abort_flag, err)) ||
                !(ok = mbar_wait(&s_free[x], jj & 1, abort_flag, err)))
              break;
            tc_fence_after();
            issue_s(s1);
          }
          if (!(ok = mbar_wait(&p_full[x], jj & 1, abort_flag, err))) break;
          tc_fence_after();
          const uint32_t sV = smem_u32(sm + L::V + s * KV_BYTES);
          // O_x += P_x V_j, P read from TMEM (keys 16k..16k+15 at column 8k)
#pragma unroll
          for (int k = 0; k < FK / 16; ++k)
            umma_bf16_ts(tO(x), tP(x) + k * 8, umma_smem_desc(sV + k * 2048, KV_BYTES, 1024), idO,
                         (j > 0 || k > 0));
          umma_commit(&pv_done[x]);
          umma_commit(&kv_empty[s]);
        }
        if (!ok) break;
        // the item's Q tile is free once its last S MMA has completed
        if (nb > 0)
          umma_commit(&q_empty[slot]);
        else
          mbar_arrive(&q_empty[slot]);
        mbar_arrive(&item_empty[slot]);
        gk += inf.nkv;
        jx += nb;
      }
    }
  } else if (warp < kFwdMma1Warp) {
    // Softmax warpgroup x (warps 2-5: tile 0, 6-9: tile 1); thread = query
    // row r of the tile (TMEM lane r). Per block: the S row into registers,
    // its max, then exp + row sum + P, with a running max that is only raised
    // when the row max grows by more than 2^8; O is then rescaled in TMEM.
    // Otherwise the stale max is exact because O and the row sum share it.
    const int x = (warp - 2) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const float c = p.scale * kLog2e;
    int* kseg = reinterpret_cast<int*>(sm + L::KSEG) + x * 2 * FK;
    int nseg = 0;  // blocks of this tile that needed the per-element test so far
    bool ok = true;
    int jx = 0, ii = 0;
    for (; ok; ++ii) {
      const int slot = ii & 1;
      if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
      const FwdItem inf = items[slot];
      if (inf.nkv < 0) break;  // no more items
      const int nb = x == 0 ? inf.n0 : (inf.has1 ? inf.nkv : 0);
      const int bh = inf.bh, b = bh / p.H, h = bh - b * p.H;
      const int q0 = inf.pr * 2 * FQ;
      const int d0 = q0 / FK;
      const int qrow = q0 + x * FQ + r;
      const int* segrow = SEG ? p.seg + (int64_t)b * p.T : nullptr;
      const int2* segtab = SEG ? segtab_of(slot) : nullptr;
      const int nch = min((p.T + kSegChunk - 1) / kSegChunk, 2 * (d0 + inf.has1 + 1));
      // this row's segment id (rows past T take an id no key has)
      const int sq = segrow ? (qrow < p.T ? segrow[qrow] : INT_MIN) : 0;
      const int2 qrng = segrow ? seg_range(segtab, nch, 2 * (d0 + x), 2) : make_int2(0, 0);
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < nb && ok; ++j) {
        const int jj = jx + j;
        if (!(ok = mbar_wait(&s_full[x], jj & 1, abort_flag, err))) break;
        tc_fence_after();
        const int jb = kblock(slot, j);
        const bool diag = (jb == d0 + x);  // keys past the query (and past T) are masked
        // Per-element segment test unless keys and queries all share one id;
        // the block's key ids then come through shared memory (double-buffered,
        // one mbarrier handshake across the warpgroup).
        const bool segmask = segrow && !rng_single(seg_range(segtab, nch, 2 * jb, 2), qrng);
        const int* ks = kseg + (nseg & 1) * FK;
        if (segmask) {
          const int key = jb * FK + r;
          kseg[(nseg & 1) * FK + r] = key < p.T ? segrow[key] : INT_MAX;
          mbar_arrive(&kseg_full[2 * x + (nseg & 1)]);
          if (!(ok = mbar_wait(&kseg_full[2 * x + (nseg & 1)], (nseg >> 1) & 1, abort_flag, err)))
            break;
          ++nseg;
        }
        // The whole 128-column S row in one batch of TMEM loads, then S_x is
        // handed back so the next block's scores overlap this block's exps.
        uint32_t v[FK];
#pragma unroll
        for (int cc = 0; cc < FK / 32; ++cc) tmem_ld32_nw(tS(x) + lane_off + cc * 32, v + 32 * cc);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[x]);
        // Row max of the raw scores (c > 0 commutes with the max), eight
        // independent chains; on the diagonal block keys past the query are out.
        float m8[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) m8[u] = -INFINITY;
        auto visible = [&](int i) { return (!diag || i <= r) && (!segmask || ks[i] == sq); };
        if (diag || segmask) {
#pragma unroll
          for (int i = 0; i < FK; i += 2)
            m8[(i >> 1) & 7] = fmax3(m8[(i >> 1) & 7], visible(i) ? __uint_as_float(v[i]) : -INFINITY,
                                     visible(i + 1) ? __uint_as_float(v[i + 1]) : -INFINITY);
        } else {
#pragma unroll
          for (int i = 0; i < FK; i += 2)
            m8[(i >> 1) & 7] =
                fmax3(m8[(i >> 1) & 7], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        }
        const float mx =
            fmaxf(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], fmaxf(m8[5], fmaxf(m8[6], m8[7])))) * c;
        // The rescale decision is made per warp: the TMEM loads/stores of O are
        // warp-collective and must not run in a divergent branch. Rows whose
        // max did not move rescale by exactly 1.
        const bool rescale = __any_sync(0xffffffffu, mx > m_used + 8.0f);
        float alpha = 1.f;
        if (rescale) {
          // 0 on a row's first visible block (m_used = -inf); a row with no
          // visible key yet (document masking) keeps its -inf max and alpha 1
          const float m_new = fmaxf(m_used, mx);
          alpha = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
          m_used = m_new;
        }
        // P = exp2(s*c - m) packed to bf16 pairs in registers (the S registers
        // die as P is produced); four packed partial row sums.
        const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_used, -m_used);
        float2 acc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
        uint32_t pk[FK / 2];
#pragma unroll
        for (int i = 0; i < FK; i += 2) {
          const float2 t = ffma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), c2, nm2);
          float p0 = ex2(t.x), p1 = ex2(t.y);
          if (diag || segmask) {
            if (!visible(i)) p0 = 0.f;
            if (!visible(i + 1)) p1 = 0.f;
          }
          acc[(i >> 1) & 3] = fadd2(acc[(i >> 1) & 3], make_float2(p0, p1));
          pk[i / 2] = pack_bf16x2(p0, p1);
        }
        const float2 s01 = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        const float sum = s01.x + s01.y;
        // P and O of the previous block must have been consumed by its P.V
        // MMA (the previous item's last block was waited for at its end).
        if (j > 0) {
          if (!(ok = mbar_wait(&pv_done[x], (jj - 1) & 1, abort_flag, err))) break;
          tc_fence_after();
        }
#pragma unroll
        for (int g = 0; g < FK / 16; ++g) tmem_st8_nw(tP(x) + lane_off + g * 8, pk + 8 * g);
        l = l * alpha + sum;
        if (rescale && j > 0) {
          float o[32];
#pragma unroll
          for (int cc = 0; cc < HD / 32; ++cc) {
            tmem_ld32(tO(x) + lane_off + cc * 32, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(tO(x) + lane_off + cc * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (ok && nb > 0) {
        if (!(ok = mbar_wait(&pv_done[x], (jx + nb - 1) & 1, abort_flag, err))) break;
        tc_fence_after();
        const float inv = 1.f / l;
        float o[32];
        bf16* orow = p.o + b * p.osb + h * p.osh + (int64_t)qrow * p.ost;
#pragma unroll
        for (int cc = 0; cc < HD / 32; ++cc) {
          tmem_ld32(tO(x) + lane_off + cc * 32, o);
          if (qrow < p.T) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint4 q;
              q.x = pack_bf16x2(o[8 * g] * inv, o[8 * g + 1] * inv);
              q.y = pack_bf16x2(o[8 * g + 2] * inv, o[8 * g + 3] * inv);
              q.z = pack_bf16x2(o[8 * g + 4] * inv, o[8 * g + 5] * inv);
              q.w = pack_bf16x2(o[8 * g + 6] * inv, o[8 * g + 7] * inv);
              *reinterpret_cast<uint4*>(orow + cc * 32 + 8 * g) = q;
            }
          }
        }
        if (qrow < p.T) p.lse[(int64_t)bh * p.T + qrow] = (m_used + __log2f(l)) * kLn2;
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      jx += nb;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) sched_finish(p.sched);
}

// The forward of the score-modified attention. A kernel of its own: with the roles of
// both as functions of one template, the plain kernel took 1 to 2.7% more time.
template <bool SEG, int MODE>
__global__ void __launch_bounds__(kFwdGeneralThreads, 1)
    score_fwd_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const AttnParams p) {
  using L = FwdSmem<SEG>;
  extern __shared__ __align__(1024) uint8_t smem_fwd[];
  uint8_t* sm = smem_fwd;
  if (smem_u32(sm) & 1023) {  // the layout needs 1024-byte aligned tiles: give up, flagged
    if (threadIdx.x == 0) {
      atomicCAS(&g_attn_error, 0, kErrSmemAlign);
      sched_finish(p.sched);
    }
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BAR);
  uint64_t* q_full = bars + 0;                 // [2 item slots]
  uint64_t* q_empty = bars + 2;                // [2]
  uint64_t* kv_full = bars + 4;                // [kKvStages]
  uint64_t* kv_empty = kv_full + kKvStages;    // [kKvStages]
  uint64_t* s_full = kv_empty + kKvStages;     // [2 tiles]: S of the current block is in TMEM
  uint64_t* p_full = s_full + 2;               // [2]: P written to TMEM
  uint64_t* pv_done = p_full + 2;              // [2]: the tile's P.V MMA has completed
  uint64_t* s_free = pv_done + 2;              // [2]: S has been loaded into registers
  uint64_t* item_full = s_free + 2;            // [2]
  uint64_t* item_empty = item_full + 2;        // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(item_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  FwdItem* items = reinterpret_cast<FwdItem*>(sm + L::ITEM);

  constexpr int kMma1Warp = 2;  // MMA thread of tile 1 (warp 1 serves tile 0)
  constexpr int kSoftmaxWarp = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int BH = p.B * p.H;
  const int npair = (p.T + 2 * FQ - 1) / (2 * FQ);
  const int n_items = npair * BH;  // item = bh * npair + (npair - 1 - pair)
  int* err = &g_attn_error;
  auto segtab_of = [&](int slot) {
    return reinterpret_cast<int2*>(sm + L::SEGTAB) + slot * kMaxSegChunks;
  };
  // Key block of list entry j of the item in `slot` (nkv entries). The list is walked
  // from its end: the diagonal comes first and sets the rows' maxima, which a bias
  // that falls with the distance then never raises.
  auto kblock = [&](int slot, int j, int nkv) -> int {
    j = nkv - 1 - j;
    if constexpr (SEG)
      return reinterpret_cast<const int*>(sm + L::BLOCKS)[slot * (kMaxSegChunks / 2) + j];
    else
      return j;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 2);  // released by each tile's MMA thread
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], kFwdItemUsers);
    }
    for (int s = 0; s < kKvStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);  // released by each tile's MMA thread
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
      mbar_init(&pv_done[x], 1);
      mbar_init(&s_free[x], 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // TMEM columns: S[2] (128 fp32 each) | O[2] (64 fp32) | P[2] (128 keys as bf16 pairs)
  const uint32_t tmem = *tmem_slot;
  auto tS = [&](int x) { return tmem + 128 * x; };
  auto tO = [&](int x) { return tmem + 256 + 64 * x; };
  auto tP = [&](int x) { return tmem + 384 + 64 * x; };

  auto produce = [&]() {
    // Item producer: publishes each item's slot (with segment ids also the
    // chunk ranges and the key-block list), then loads its two Q tiles and its
    // K/V blocks into the ring.
    bool ok = true;
    int gk = 0;
    for (int ii = 0; ok; ++ii) {
      const int slot = ii & 1;
      const int item = next_item(p.sched, lane);
      if (!(ok = mbar_wait(&item_empty[slot], ((ii >> 1) & 1) ^ 1, abort_flag, err))) break;
      if (item >= n_items) {  // no more work: an empty slot ends every role's loop
        if (lane == 0) {
          items[slot].nkv = -1;
          mbar_arrive(&item_full[slot]);
        }
        break;
      }
      int bh = item / npair, pr = npair - 1 - (item - bh * npair);
      if (p.by_weight) {
        pr = npair - 1 - item / BH;
        bh = item % BH;
      }
      const int b = bh / p.H, h = bh - b * p.H;
      const int q0 = pr * 2 * FQ;
      // tile x's diagonal key block is d0 + x; tile 1 of the last pair may lie
      // wholly past the sequence end
      const int d0 = q0 / FK;
      const int has1 = q0 + FQ < p.T;
      const int dmax = has1 ? d0 + 1 : d0;
      int nkv = dmax + 1, n0 = d0 + 1;
      const int hk = h / p.group;
      int pf = 0, nch = 0;
      if (p.prefix) {  // the prefix's blocks are seen by both tiles
        pf = min(max(p.prefix[b], 0), p.T);
        nkv = max(nkv, (pf + FK - 1) / FK);
        n0 = max(n0, (pf + FK - 1) / FK);
      }
      if constexpr (SEG) {
        // The key blocks up to the diagonal or the prefix's end that either query
        // tile can see, in order; both tiles walk this one list (tile 0 the first n0).
        // A tile's diagonal block stays in it even if nothing meets there (padding
        // alone), so that every tile has a block and writes its rows.
        const int* segrow = p.seg + (int64_t)b * p.T;
        int2* tab = segtab_of(slot);
        nch = min((p.T + kSegChunk - 1) / kSegChunk, 2 * nkv);
        for (int c = 0; c < nch; ++c) {
          int mn = INT_MAX, mx = INT_MIN;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t = c * kSegChunk + u * 32 + lane;
            if (t < p.T) {
              const int v = segrow[t];
              mn = min(mn, v);
              mx = max(mx, v);
            }
          }
          mn = __reduce_min_sync(0xffffffffu, mn);
          mx = __reduce_max_sync(0xffffffffu, mx);
          if (lane == 0) tab[c] = seg_chunk(mn, mx);
        }
        __syncwarp();
        if (lane == 0) {
          int* bl = reinterpret_cast<int*>(sm + L::BLOCKS) + slot * (kMaxSegChunks / 2);
          const int2 qr0 = seg_range(tab, nch, 2 * d0, 2);
          const int2 qr1 = seg_range(tab, nch, 2 * d0 + 2, 2);
          int n = 0, n_le0 = 0;
          for (int j = 0; j < nkv; ++j) {
            const int2 kr = seg_range(tab, nch, 2 * j, 2);
            if (j == d0 || j == dmax || (j < n0 && seg_meet(kr, qr0)) ||
                (has1 && seg_meet(kr, qr1))) {
              bl[n++] = j;
              if (j < n0) ++n_le0;
            }
          }
          nkv = n;
          n0 = n_le0;
        }
        nkv = __shfl_sync(0xffffffffu, nkv, 0);
        n0 = __shfl_sync(0xffffffffu, n0, 0);
      }
      if (lane == 0) {
        items[slot] = FwdItem{pr, bh, nkv, n0, has1, nch, pf, 0};
        mbar_arrive(&item_full[slot]);
        if ((ok = mbar_wait(&q_empty[slot], ((ii >> 1) & 1) ^ 1, abort_flag, err))) {
          uint8_t* qd = sm + L::Q + slot * 2 * Q_BYTES;
          mbar_arrive_expect_tx(&q_full[slot], 2 * Q_BYTES);
          tma_load_4d(qd, &tmQ, &q_full[slot], 0, q0, h, b);
          tma_load_4d(qd + Q_BYTES, &tmQ, &q_full[slot], 0, q0 + FQ, h, b);
        }
        for (int j = 0; ok && j < nkv; ++j, ++gk) {
          const int s = gk % kKvStages;
          if (!(ok = mbar_wait(&kv_empty[s], ((gk / kKvStages) & 1) ^ 1, abort_flag, err))) break;
          mbar_arrive_expect_tx(&kv_full[s], 2 * KV_BYTES);
          const int key0 = kblock(slot, j, nkv) * FK;
          tma_load_4d(sm + L::K + s * KV_BYTES, &tmK, &kv_full[s], 0, key0, hk, b);
          tma_load_4d(sm + L::V + s * KV_BYTES, &tmV, &kv_full[s], 0, key0, hk, b);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
  };
  auto issue = [&]() {
    // One MMA thread per tile: S_x = Q_x K_j^T (128 x 128 fp32) for the next
    // block as soon as the softmax holds S_x in registers, O_x += P_x V_j
    // once P_x is in TMEM. The two tiles progress independently; each walks
    // every block of the item's list and releases the ones it does not use.
    const int x = warp == 1 ? 0 : 1;
    if (lane == 0) {
      constexpr uint32_t idS = umma_idesc_bf16(128, FK, 0, 0);
      constexpr uint32_t idO = umma_idesc_bf16(128, HD, 0, 1);  // A = P in TMEM, B = V MN-major
      bool ok = true;
      int gk = 0, jx = 0, ii = 0;  // ring block, this tile's running block, item
      for (; ok; ++ii) {
        const int slot = ii & 1;
        if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
        const FwdItem inf = items[slot];
        if (inf.nkv < 0) break;  // no more items
        const int nb = x == 0 ? inf.n0 : (inf.has1 ? inf.nkv : 0);
        // the tile's blocks are list entries [j0, j0 + nb)
        const int j0 = x == 0 ? inf.nkv - nb : 0;
        const uint32_t sQ = smem_u32(sm + L::Q + (slot * 2 + x) * Q_BYTES);
        auto issue_s = [&](int s) {
          const uint32_t sK = smem_u32(sm + L::K + s * KV_BYTES);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            umma_bf16(tS(x), umma_smem_desc(sQ + k * 32, 16, 1024),
                      umma_smem_desc(sK + k * 32, 16, 1024), idS, k > 0);
          umma_commit(&s_full[x]);
        };
        // a block this tile skips: release it once it has arrived
        auto skip = [&](int j) {
          const int s = (gk + j) % kKvStages;
          if (!mbar_wait(&kv_full[s], ((gk + j) / kKvStages) & 1, abort_flag, err)) return false;
          mbar_arrive(&kv_empty[s]);
          return true;
        };
        for (int j = 0; ok && j < j0; ++j) ok = skip(j);
        if (!ok) break;
        if (nb > 0) {
          // S of the item's first block: Q loaded, the block loaded, and the
          // previous item's last S taken out of TMEM by the softmax
          const int s0 = (gk + j0) % kKvStages;
          ok = mbar_wait(&q_full[slot], (ii >> 1) & 1, abort_flag, err) &&
               mbar_wait(&kv_full[s0], ((gk + j0) / kKvStages) & 1, abort_flag, err) &&
               (jx == 0 || mbar_wait(&s_free[x], (jx - 1) & 1, abort_flag, err));
          if (!ok) break;
          tc_fence_after();
          issue_s(s0);
        }
        for (int j = j0; ok && j < inf.nkv; ++j) {
          const int s = (gk + j) % kKvStages;
          if (j >= j0 + nb) {
            ok = skip(j);
            continue;
          }
          const int jj = jx + j - j0;  // running block index of this tile
          if (j + 1 < j0 + nb) {
            const int s1 = (gk + j + 1) % kKvStages;
            if (!(ok = mbar_wait(&kv_full[s1], ((gk + j + 1) / kKvStages) & 1, abort_flag, err)) ||
                !(ok = mbar_wait(&s_free[x], jj & 1, abort_flag, err)))
              break;
            tc_fence_after();
            issue_s(s1);
          }
          if (!(ok = mbar_wait(&p_full[x], jj & 1, abort_flag, err))) break;
          tc_fence_after();
          const uint32_t sV = smem_u32(sm + L::V + s * KV_BYTES);
          // O_x += P_x V_j, P read from TMEM (keys 16k..16k+15 at column 8k)
#pragma unroll
          for (int k = 0; k < FK / 16; ++k)
            umma_bf16_ts(tO(x), tP(x) + k * 8, umma_smem_desc(sV + k * 2048, KV_BYTES, 1024), idO,
                         (j > j0 || k > 0));
          umma_commit(&pv_done[x]);
          umma_commit(&kv_empty[s]);
        }
        if (!ok) break;
        // the item's Q tile is free once its last S MMA has completed
        if (nb > 0)
          umma_commit(&q_empty[slot]);
        else
          mbar_arrive(&q_empty[slot]);
        mbar_arrive(&item_empty[slot]);
        gk += inf.nkv;
        jx += nb;
      }
    }
  };
  // Softmax warpgroup x; thread = query row r of the tile (TMEM lane r). One streaming
  // pass per block against the reference that the rows have so far (Score::stream).
  // Blocks with masked places, a row whose scores outgrow its reference and scores past
  // the short form of tanh take steps instead, from the raw scores still in TMEM. The
  // pass is a loop over 32 keys and no longer code: all 128 keys unrolled (15 KB) or 64
  // take 268 to 283 us at 1 x 12 x 8192, this 259 (279 with TMEM loads that nothing
  // covers).
  auto softmax = [&]() {
    const int x = (warp - kSoftmaxWarp) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    bool ok = true;
    int jx = 0, ii = 0;
    for (; ok; ++ii) {
      const int slot = ii & 1;
      if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
      const FwdItem inf = items[slot];
      if (inf.nkv < 0) break;  // no more items
      const int nb = x == 0 ? inf.n0 : (inf.has1 ? inf.nkv : 0);
      const int j0 = x == 0 ? inf.nkv - nb : 0;
      const int bh = inf.bh, b = bh / p.H, h = bh - b * p.H;
      const int q0 = inf.pr * 2 * FQ;
      const int d0 = q0 / FK;
      const int qrow = q0 + x * FQ + r;
      const int* segrow = SEG ? p.seg + (int64_t)b * p.T : nullptr;
      const int2* segtab = SEG ? segtab_of(slot) : nullptr;
      // this row's segment id (rows past T take one no key has)
      const int sq = SEG ? (qrow < p.T ? seg_query_id(segrow[qrow]) : -2) : 0;
      const int2 qrng = SEG ? seg_range(segtab, inf.nch, 2 * (d0 + x), 2) : make_int2(0, 0);
      // the last key this row sees under the causal and the prefix mask
      const int last = max(qrow, inf.prefix - 1);
      const Score<MODE> score(p, (MODE & kBias) ? p.slopes[h] * kLog2e : 0.f);
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < nb && ok; ++j) {
        const int jj = jx + j;
        const int jb = kblock(slot, j0 + j, inf.nkv);
        int kid[4] = {0, 0, 0, 0};  // the block's key ids, lane l keys l + 32 w
        if constexpr (SEG) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int key = jb * FK + 32 * w + lane;
            kid[w] = key < p.T ? seg_key_id(segrow[key]) : -1;
          }
        }
        // keys past a query (and past T) are masked, keys of another id too
        const bool diag = jb * FK + FK - 1 > max(q0 + x * FQ, inf.prefix - 1);
        const bool segmask = SEG && !seg_single(seg_range(segtab, inf.nch, 2 * jb, 2), qrng);
        const bool ahead = (MODE & kBias) && jb * FK + FK - 1 > q0 + x * FQ;  // |i - j| either way
        if (!(ok = mbar_wait(&s_full[x], jj & 1, abort_flag, err))) break;
        tc_fence_after();
        // P and O of the previous block must have been consumed by its P.V MMA,
        // which may still run while this block's first scores are computed.
        auto previous_done = [&]() {
          if (j > 0) {
            ok = mbar_wait(&pv_done[x], (jj - 1) & 1, abort_flag, err);
            tc_fence_after();
          }
          return ok;
        };
        const uint32_t aS = tS(x) + lane_off, aP = tP(x) + lane_off;
        const float at0 = (float)(jb * FK - qrow);
        uint32_t v[32], pk[16];
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        float alpha = 1.f;
        bool rescale = false;
        bool steps = diag || segmask || ahead;
        if (!steps) {
          float far = 0.f;
          float2 k[Score<MODE>::TERMS], off[4];
          if constexpr ((MODE & kCap) != 0) score.stream_coefs(k);
          uint32_t va[16], vb[16];
          tmem_ld16_nw(aS, va);
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {
            score.stream_bias(at0 + (float)(32 * w), m_used, off);
            tmem_wait_ld();
            tmem_ld16_nw(aS + 32 * w + 16, vb);
            score.stream(va, k, off, pk, acc, far);
            tmem_wait_ld();
            if (w < 3) tmem_ld16_nw(aS + 32 * w + 32, va);
            score.stream(vb, k, off, pk + 8, acc, far);
            if (w == 0 && !previous_done()) break;
            tmem_st8_nw(aP + 16 * w, pk);
            tmem_st8_nw(aP + 16 * w + 8, pk + 8);
          }
          if (!ok) break;
          const float2 both = fadd2(acc[0], acc[1]);
          steps = score.discard(both.x + both.y, far);
        }
        if (steps) {
          // Masks, a new maximum or tanh's long form: modified scores go back
          // into S, then the maximum, then the probabilities. Words (32 keys)
          // hidden from the whole warp cost nothing but their zeros.
          uint32_t see[4];  // which keys this row sees
          causal_words(last - jb * FK, see);
          if (segmask) segment_words(kid, sq, see);
          float top = -INFINITY;
          unsigned hidden = 0;  // bit w: word w
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {
            const uint32_t sees = w < 2 ? (w == 0 ? see[0] : see[1]) : (w == 2 ? see[2] : see[3]);
            if (__all_sync(0xffffffffu, sees == 0u)) {
              hidden |= 1u << w;
              continue;
            }
            const bool full = __all_sync(0xffffffffu, sees == 0xffffffffu);
            tmem_ld32_nw(aS + 32 * w, v);
            tmem_wait_ld();
            top = fmaxf(top, score.modify(v, at0 + (float)(32 * w), sees, full));
            tmem_st32(aS + 32 * w, reinterpret_cast<const float*>(v));
          }
          // Decided per warp (the TMEM accesses of O are warp-collective); a row
          // whose max stays rescales by 1, one that has seen no key yet too.
          rescale = __any_sync(0xffffffffu, top > m_used + 8.0f);
          if (rescale) {
            const float m_new = top > m_used ? top + Score<MODE>::kRoom : m_used;
            alpha = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
            m_used = m_new;
          }
          if (!previous_done()) break;
          const float sub = m_used == -INFINITY ? 0.f : m_used;  // exp2(-inf - sub) = 0
          acc[0] = acc[1] = make_float2(0.f, 0.f);
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {
            if ((hidden >> w) & 1u) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0;
            } else {
              tmem_ld32_nw(aS + 32 * w, v);
              tmem_wait_ld();
              Score<MODE>::exponentials(v, sub, pk, acc);
            }
            tmem_st8_nw(aP + 16 * w, pk);
            tmem_st8_nw(aP + 16 * w + 8, pk + 8);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[x]);
        const float2 s2 = fadd2(acc[0], acc[1]);
        const float sum = s2.x + s2.y;
        l = l * alpha + sum;
        if (rescale && j > 0) {
          float o[32];
#pragma unroll
          for (int cc = 0; cc < HD / 32; ++cc) {
            tmem_ld32(tO(x) + lane_off + cc * 32, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(tO(x) + lane_off + cc * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (ok && nb > 0) {
        if (!(ok = mbar_wait(&pv_done[x], (jx + nb - 1) & 1, abort_flag, err))) break;
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key: zeros
        float o[32];
        bf16* orow = p.o + b * p.osb + h * p.osh + (int64_t)qrow * p.ost;
#pragma unroll
        for (int cc = 0; cc < HD / 32; ++cc) {
          tmem_ld32(tO(x) + lane_off + cc * 32, o);
          if (qrow < p.T && p.o32) {
            float* row = p.o32 + ((int64_t)bh * p.T + qrow) * HD + cc * 32;
#pragma unroll
            for (int g = 0; g < 8; ++g)
              reinterpret_cast<float4*>(row)[g] = make_float4(
                  o[4 * g] * inv, o[4 * g + 1] * inv, o[4 * g + 2] * inv, o[4 * g + 3] * inv);
          } else if (qrow < p.T) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint4 q;
              q.x = pack_bf16x2(o[8 * g] * inv, o[8 * g + 1] * inv);
              q.y = pack_bf16x2(o[8 * g + 2] * inv, o[8 * g + 3] * inv);
              q.z = pack_bf16x2(o[8 * g + 4] * inv, o[8 * g + 5] * inv);
              q.w = pack_bf16x2(o[8 * g + 6] * inv, o[8 * g + 7] * inv);
              *reinterpret_cast<uint4*>(orow + cc * 32 + 8 * g) = q;
            }
          }
        }
        if (qrow < p.T && !p.o32)
          p.lse[(int64_t)bh * p.T + qrow] = l == 0.f ? -INFINITY : (m_used + __log2f(l)) * kLn2;
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      jx += nb;
    }
  };
  if (warp < kSoftmaxWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwdRegsIssue));
    if (warp == 0) {
      produce();
    } else if (warp <= kMma1Warp) {
      issue();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFwdRegsSoftmax));
    softmax();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) sched_finish(p.sched);
}

// ------------------------------------------------------------------ backward
// Persistent: one CTA per SM walks work items (key tile kt, batch*head bh),
// item = bh * nkt + kt, handed out by next_item. Every role
// walks the same item list and keeps running tile / query-pair counters across
// items, so the rings (Q/dO stages, TMEM score buffers, dS^T slots, dQ pairs)
// flow from one item into the next without draining: while the last tiles of
// an item finish, the TMA warp already holds the next item's K/V (two K/V
// slots) and the scores MMA thread computes its first scores.
constexpr int BT = 128;                 // keys per item (TMEM lanes)
constexpr int BQ = 64;                  // queries per inner tile
constexpr int BT_BYTES = BT * 128;      // 128 rows x 64 bf16
constexpr int BQ_BYTES = BQ * 128;      // 64 rows x 64 bf16
constexpr int kBwdSmWarps = 16;         // softmax warps: four per TMEM lane quadrant
// The softmax warps form GROUPS groups (a kernel template parameter) that take
// alternate tiles; a warp of a group covers 64 / (group warps / 4) query
// columns of its tile. One group (every warp on every tile) has the shortest
// latency per tile and wins at T = 1024, where items are a few tiles long;
// two groups overlap consecutive tiles and win on long sequences.
constexpr int kBwdScoreWarp = 2 + kBwdSmWarps;  // issues the S^T / dP^T MMAs
constexpr int kBwdFlushWarp = kBwdScoreWarp + 1;  // first of four dQ read-out warps
constexpr int kBwdThreads = 32 * (kBwdFlushWarp + 4);
// Arrivals that release an item slot: both MMA threads, the softmax warps and
// the dQ warps.
constexpr int kBwdItemUsers = 2 + kBwdSmWarps + 4;

// Item slot written by the TMA warp: key tile, batch*head, number of 64-query
// tiles (always even: an odd count gets one tile past the sequence end, whose
// rows load as zeros and carry no probability, so query pairs never straddle
// two items).
// MODE > kClassic: bh counts key/value heads and the list is walked once per
// query head of the group, nq1 tiles each (nq = group * nq1); tile indexes
// count from position qb, 0 where the key tile reaches into the prefix.
struct BwdItem {
  int kt, bh, nq, nq1, qb, prefix, pad0, pad1;
};

template <bool SEG>
struct BwdSmem {
  static constexpr int kQStages = SEG ? 2 : 4;          // Q / dO tile ring
  static constexpr int kStatBytes = SEG ? 768 : 512;    // per stage: lse, delta (, segment ids)
  static constexpr int KV = 0;                          // 2 slots x (K, V)
  static constexpr int Q = KV + 4 * BT_BYTES;           // kQStages tiles
  static constexpr int DO = Q + kQStages * BQ_BYTES;    // kQStages tiles
  static constexpr int DST = DO + kQStages * BQ_BYTES;  // ring of 4 dS^T tiles [128 keys x 64 queries]
  static constexpr int DQS = DST + 4 * BT_BYTES;        // dQ staging: 4 warps x 2 x (32 x 32 fp32)
  // per Q/dO stage, the tile's query statistics copied in by the producer
  // warp: 64 x lse, 64 x delta, 64 segment ids (zeros past the sequence end)
  static constexpr int STAT = DQS + 8 * 4096;
  static constexpr int ITEM = STAT + kQStages * kStatBytes;  // 2 BwdItem slots
  // segment ids only: per slot, (min, max) id per 64-position chunk from k0
  // and the list of query tiles that can see the key tile
  static constexpr int SEGTAB = ITEM + 64;
  static constexpr int QLIST = SEGTAB + (SEG ? 2 * kMaxSegChunks * 8 : 0);
  static constexpr int BAR = QLIST + (SEG ? 2 * kMaxSegChunks * 4 : 0);
  // the dynamic shared memory base is 1024-byte aligned (checked at entry)
  static constexpr int TOTAL = BAR + 272;
};

// MODE > kClassic: whole warpgroups, so that registers can move from the one that
// loads and issues (warps 0-3: TMA, gradient MMAs, score MMAs, idle) to the one
// that reads dQ out (20-23); warps 4-19 are the softmax, in two groups on
// alternate tiles. Measured (us, 1 x 12 x 8192 capped and biased | 8 x 12 x 1024):
// 458 | 107 so, 494 | 116 with three groups of four warps, 513 | 116 with two
// groups of four and twice the registers: fewer warps leave more of the TMEM
// reads' latency in the open.
constexpr int kBwdGeneralThreads = 32 * 24;
constexpr int kBwdRegs = 80, kBwdRegsIssue = 48, kBwdRegsSoftmax = 80, kBwdRegsFlush = 112;
static_assert(kBwdRegsIssue + 4 * kBwdRegsSoftmax + kBwdRegsFlush == 6 * kBwdRegs,
              "register shares");

template <bool SEG, int GROUPS, int MODE>
__global__ void __launch_bounds__(MODE == kClassic ? kBwdThreads : kBwdGeneralThreads, 1)
    attn_bwd_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                const __grid_constant__ CUtensorMap tmDQ, const AttnParams p) {
  using L = BwdSmem<SEG>;
  constexpr bool GENERAL = MODE != kClassic;
  constexpr int kQS = L::kQStages;
  constexpr int kBwdSmGroups = GROUPS;
  constexpr int kSmWarps = kBwdSmWarps;
  constexpr int kSmWarp0 = GENERAL ? 4 : 2;  // first softmax warp
  constexpr int kScoreWarp = GENERAL ? 2 : kBwdScoreWarp;
  constexpr int kFlushWarp = GENERAL ? 20 : kBwdFlushWarp;
  constexpr int kBwdGroupWarps = kSmWarps / kBwdSmGroups;
  constexpr int kBwdWarpCols = 64 / (kBwdGroupWarps / 4);
  extern __shared__ __align__(1024) uint8_t smem_bwd[];
  uint8_t* sm = smem_bwd;
  if (smem_u32(sm) & 1023) {  // the layout needs 1024-byte aligned tiles: give up, flagged
    if (threadIdx.x == 0) {
      atomicCAS(&g_attn_error, 0, kErrSmemAlign);
      sched_finish(p.sched);
    }
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BAR);
  uint64_t* kv_full = bars + 0;       // [2] K/V slot loaded
  uint64_t* kv_empty = bars + 2;      // [2] every MMA of the slot's item has completed
  uint64_t* q_full = bars + 4;        // [4]
  uint64_t* q_empty = bars + 8;       // [4]
  uint64_t* s_full = bars + 12;       // [3]: S^T and dP^T of a tile are in TMEM buffer b
  uint64_t* p_full = bars + 15;       // [3]: P^T, dS^T of a tile written (TMEM buffer b, smem ring)
  uint64_t* done = bars + 18;         // [4]: every MMA issued up to the end of tile g has completed
  uint64_t* dq_full = bars + 22;      // [2]: dQ of query pair J is in TMEM
  uint64_t* dq_free = bars + 24;      // [2]: ... and has been read out
  uint64_t* fin = bars + 26;          // an item's dK / dV are complete in TMEM
  uint64_t* acc_free = bars + 27;     // ... and have been read out
  uint64_t* item_full = bars + 28;    // [2]
  uint64_t* item_empty = bars + 30;   // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  BwdItem* items = reinterpret_cast<BwdItem*>(sm + L::ITEM);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = GENERAL ? p.KVH : p.H;
  const int BH = p.B * heads;
  const int n_items = ((p.T + BT - 1) / BT) * BH;  // item = bh * nkt + kt
  int* err = &g_attn_error;
  // query tile (64-position index past k0) of list entry `it` of the item in `slot`
  auto qtile = [&](int slot, int it) -> int {
    if constexpr (SEG)
      return reinterpret_cast<const int*>(sm + L::QLIST)[slot * kMaxSegChunks + it];
    else
      return it;
  };
  auto segtab_of = [&](int slot) {
    return reinterpret_cast<int2*>(sm + L::SEGTAB) + slot * kMaxSegChunks;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], kBwdItemUsers - kBwdSmWarps + kSmWarps);
      mbar_init(&dq_full[s], 1);
      mbar_init(&dq_free[s], 4);
    }
    for (int s = 0; s < kQS; ++s) {
      mbar_init(&q_full[s], 33);  // the Q/dO TMA and the 32 lanes' statistics copies
      mbar_init(&q_empty[s], 2);  // the scores MMAs and the gradient MMAs of the tile
    }
    for (int s = 0; s < 3; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], kBwdGroupWarps);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&done[s], 1);
    mbar_init(fin, 1);
    mbar_init(acc_free, 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // TMEM columns: three tile buffers of 128 columns, then dV | dK. In buffer
  // b, columns [0, 64) receive S^T and [64, 128) dP^T (fp32, lane = key). The
  // softmax writes P^T and dS^T as bf16 pairs over the S^T half (query group
  // cg = 16 queries: columns 16 cg + [0, 8) for P^T, 16 cg + [8, 16) for
  // dS^T); the dP^T half then holds dQ when the tile closes a query pair.
  const uint32_t tmem = *tmem_slot;
  const uint32_t tDV = tmem + 384, tDK = tmem + 448;
  auto tBuf = [&](int bb) { return tmem + 128 * bb; };

  auto produce = [&]() {
    // Item producer: publishes each item's slot (and, with segment ids, its
    // chunk ranges and query-tile list), then loads its K/V and Q/dO tiles.
    bool ok = true;
    int g = 0;
    for (int ii = 0; ok; ++ii) {
      const int slot = ii & 1;
      const int item = next_item(p.sched, lane);
      if (!(ok = mbar_wait(&item_empty[slot], ((ii >> 1) & 1) ^ 1, abort_flag, err))) break;
      if (item >= n_items) {  // no more work: an empty slot ends every role's loop
        if (lane == 0) {
          items[slot].nq = -1;
          mbar_arrive(&item_full[slot]);
        }
        break;
      }
      const int nkt = (p.T + BT - 1) / BT;
      int bh = item / nkt, kt = item - bh * nkt;
      if (GENERAL && p.by_weight) {
        kt = item / BH;
        bh = item % BH;
      }
      const int b = bh / heads, h = bh - b * heads;
      const int k0 = kt * BT;
      int qb = k0, pf = 0;
      if constexpr (GENERAL) {
        if (p.prefix) {
          pf = min(max(p.prefix[b], 0), p.T);
          if (k0 < pf) qb = 0;  // queries before the diagonal see the prefix's keys
        }
      }
      const int nq_all = (p.T - qb + BQ - 1) / BQ;  // 64-query tiles from the diagonal on
      int nq = nq_all;
      if constexpr (SEG && GENERAL) {
        // as below, from position qb; without a visible tile two tiles past the
        // sequence end remain, which leave dK and dV zero
        const int* segrow = p.seg + (int64_t)b * p.T;
        int2* tab = segtab_of(slot);
        const int nch = (p.T + kSegChunk - 1) / kSegChunk - qb / kSegChunk;
        for (int c = 0; c < nch; ++c) {
          int mn = INT_MAX, mx = INT_MIN;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t = qb + c * kSegChunk + u * 32 + lane;
            if (t < p.T) {
              const int v = segrow[t];
              mn = min(mn, v);
              mx = max(mx, v);
            }
          }
          mn = __reduce_min_sync(0xffffffffu, mn);
          mx = __reduce_max_sync(0xffffffffu, mx);
          if (lane == 0) tab[c] = seg_chunk(mn, mx);
        }
        __syncwarp();
        if (lane == 0) {
          int* ql = reinterpret_cast<int*>(sm + L::QLIST) + slot * kMaxSegChunks;
          const int2 kr = seg_range(tab, nch, (k0 - qb) / kSegChunk, 2);
          int n = 0;
          for (int it = 0; it < nq_all; ++it)
            if (seg_meet(seg_range(tab, nch, it, 1), kr)) ql[n++] = it;
          while ((n & 1) || n == 0) ql[n++] = nq_all;
          nq = n;
        }
        nq = __shfl_sync(0xffffffffu, nq, 0);
      } else if constexpr (SEG) {
        // (min, max) segment id per 64-position chunk from k0, then the query
        // tiles whose ids can meet this key tile's, in order
        const int* segrow = p.seg + (int64_t)b * p.T;
        int2* tab = segtab_of(slot);
        const int nch = (p.T + kSegChunk - 1) / kSegChunk - 2 * kt;
        for (int c = 0; c < nch; ++c) {
          int mn = INT_MAX, mx = INT_MIN;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t = (2 * kt + c) * kSegChunk + u * 32 + lane;
            if (t < p.T) {
              const int v = segrow[t];
              mn = min(mn, v);
              mx = max(mx, v);
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          }
          if (lane == 0) tab[c] = make_int2(mn, mx);
        }
        __syncwarp();
        if (lane == 0) {
          int* ql = reinterpret_cast<int*>(sm + L::QLIST) + slot * kMaxSegChunks;
          const int2 kr = seg_range(tab, nch, 0, 2);
          int n = 0;
          for (int it = 0; it < nq_all; ++it)
            if (rng_meet(seg_range(tab, nch, it, 1), kr)) ql[n++] = it;
          if (n & 1) ql[n++] = nq_all;  // past the sequence end: no probability
          nq = n;
        }
        nq = __shfl_sync(0xffffffffu, nq, 0);
      } else {
        nq += nq & 1;
      }
      const int nq1 = nq;
      if constexpr (GENERAL) nq *= p.group;
      if (lane == 0) {
        items[slot] = BwdItem{kt, bh, nq, nq1, qb, pf, 0, 0};
        mbar_arrive(&item_full[slot]);
        const int kvs = ii & 1;
        ok = mbar_wait(&kv_empty[kvs], ((ii >> 1) & 1) ^ 1, abort_flag, err);
        if (ok) {
          uint8_t* kv = sm + L::KV + kvs * 2 * BT_BYTES;
          mbar_arrive_expect_tx(&kv_full[kvs], 2 * BT_BYTES);
          tma_load_4d(kv, &tmK, &kv_full[kvs], 0, k0, h, b);
          tma_load_4d(kv + BT_BYTES, &tmV, &kv_full[kvs], 0, k0, h, b);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      // query head: the key/value head's own, or the first of its group
      int hq = GENERAL ? h * p.group : h;
      // (GENERAL: -lse log2(e) and -delta, as the arithmetic uses them)
      const float* Lg = (GENERAL ? p.neg_lse2 : p.lse) + ((int64_t)b * p.H + hq) * p.T;
      const float* Dg = p.delta + ((int64_t)b * p.H + hq) * p.T;
      int ql = 0;  // entry of the head's list
      for (int it = 0; ok && it < nq; ++it, ++ql, ++g) {
        if (GENERAL && ql == nq1) {  // the group's next head
          ql = 0;
          ++hq;
          Lg += p.T;
          Dg += p.T;
        }
        const int s = g % kQS;
        const int qq = qb + qtile(slot, ql) * BQ;
        if (lane == 0) {
          ok = mbar_wait(&q_empty[s], ((g / kQS) & 1) ^ 1, abort_flag, err);
          if (ok) {
            mbar_arrive_expect_tx(&q_full[s], 2 * BQ_BYTES);
            tma_load_4d(sm + L::Q + s * BQ_BYTES, &tmQ, &q_full[s], 0, qq, hq, b);
            tma_load_4d(sm + L::DO + s * BQ_BYTES, &tmDO, &q_full[s], 0, qq, hq, b);
          }
        }
        if (!(ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0)) break;
        // the tile's statistics, copied asynchronously (each lane arrives on
        // the stage's barrier once its copies have landed)
        float* st = reinterpret_cast<float*>(sm + L::STAT + s * L::kStatBytes);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int cidx = lane + 32 * u, t = qq + cidx;
          const uint32_t nb = t < p.T ? 4u : 0u;
          const int tc = min(t, p.T - 1);
          cp_async_4(st + cidx, Lg + tc, nb);
          cp_async_4(st + 64 + cidx, Dg + tc, nb);
          if constexpr (SEG) cp_async_4(st + 128 + cidx, p.seg + (int64_t)b * p.T + tc, nb);
        }
        cp_async_mbar_arrive(&q_full[s]);
      }
    }
  };
  auto gradients = [&]() {
    // Gradient MMAs of tile g once its softmax is done. This thread and the
    // scores thread (warp 18) issue independently: a thread that stops at a
    // barrier leaves the tensor pipe to the other one.
    if (lane == 0) {
      constexpr uint32_t idKN = umma_idesc_bf16(128, 64, 0, 1);  // dV, dK: A in TMEM, B MN-major
      constexpr uint32_t idMN = umma_idesc_bf16(128, 64, 1, 1);  // dQ: A, B MN-major
      bool ok = true;
      int g = 0, ii = 0;
      for (; ok; ++ii) {
        const int slot = ii & 1, kvs = ii & 1;
        if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
        const int nq = items[slot].nq;
        if (nq < 0) break;  // no more items
        // dV / dK of the previous item have been read out of TMEM
        if (ii > 0 && !(ok = mbar_wait(acc_free, (ii - 1) & 1, abort_flag, err))) break;
        const uint32_t sK = smem_u32(sm + L::KV + kvs * 2 * BT_BYTES);
        for (int it = 0; it < nq; ++it, ++g) {
          const int bb = g % 3, s = g % kQS;
          if (!(ok = mbar_wait(&p_full[bb], (g / 3) & 1, abort_flag, err))) break;
          tc_fence_after();
          const uint32_t sQ = smem_u32(sm + L::Q + s * BQ_BYTES);
          const uint32_t sDO = smem_u32(sm + L::DO + s * BQ_BYTES);
          // dV += P^T dO and dK += dS^T Q with the A operands read from TMEM:
          // queries 16k..16k+15 sit at column 16k of the buffer (P^T, bf16
          // pairs), 8 further on for dS^T.
#pragma unroll
          for (int k = 0; k < BQ / 16; ++k) {
            const uint32_t acol = tBuf(bb) + k * 16;
            umma_bf16_ts(tDV, acol, umma_smem_desc(sDO + k * 2048, BQ_BYTES, 1024), idKN,
                         (it > 0 || k > 0));
            umma_bf16_ts(tDK, acol + 8, umma_smem_desc(sQ + k * 2048, BQ_BYTES, 1024), idKN,
                         (it > 0 || k > 0));
          }
          umma_commit(&q_empty[s]);
          if (it & 1) {
            // dQ of query pair J (tiles g-1, g) = dS K into the dP^T half of
            // this buffer: A = the pair's two dS^T tiles of the ring read
            // MN-major (M = 128 queries, 16 KB apart), B = K tile MN-major.
            const int J = g >> 1;
            const uint32_t sd = smem_u32(sm + L::DST + ((g - 1) & 3) * BT_BYTES);
#pragma unroll
            for (int k = 0; k < BT / 16; ++k)
              umma_bf16(tBuf(bb) + 64, umma_smem_desc(sd + k * 2048, BT_BYTES, 1024),
                        umma_smem_desc(sK + k * 2048, BT_BYTES, 1024), idMN, k > 0);
            umma_commit(&dq_full[J & 1]);
          }
          umma_commit(&done[g & 3]);
        }
        if (!ok) break;
        umma_commit(fin);
        umma_commit(&kv_empty[kvs]);
        mbar_arrive(&item_empty[slot]);
      }
    }
  };
  auto scores = [&]() {
    // S^T = K Q^T and dP^T = V dO^T of each tile into TMEM buffer g % 3, as
    // far ahead as the buffers allow. The buffer last served tile g-3: read by
    // that tile's dV / dK MMAs and, when g-3 closed a query pair, holding that
    // pair's dQ until the dQ warps have read it out.
    if (lane == 0) {
      constexpr uint32_t idS = umma_idesc_bf16(128, BQ, 0, 0);
      bool ok = true;
      int g = 0, ii = 0;
      for (; ok; ++ii) {
        const int slot = ii & 1, kvs = ii & 1;
        if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
        const int nq = items[slot].nq;
        if (nq < 0) break;  // no more items
        if (!(ok = mbar_wait(&kv_full[kvs], (ii >> 1) & 1, abort_flag, err))) break;
        const uint32_t sK = smem_u32(sm + L::KV + kvs * 2 * BT_BYTES), sV = sK + BT_BYTES;
        for (int it = 0; it < nq; ++it, ++g) {
          const int s = g % kQS;
          if (g >= 3) {
            const int o = g - 3;
            if (!(ok = mbar_wait(&done[o & 3], (o >> 2) & 1, abort_flag, err))) break;
            if ((o & 1) && !(ok = mbar_wait(&dq_free[(o >> 1) & 1], (o >> 2) & 1, abort_flag, err)))
              break;
          }
          if (!(ok = mbar_wait(&q_full[s], (g / kQS) & 1, abort_flag, err))) break;
          tc_fence_after();
          const uint32_t sQ = smem_u32(sm + L::Q + s * BQ_BYTES);
          const uint32_t sDO = smem_u32(sm + L::DO + s * BQ_BYTES);
          const uint32_t tb = tBuf(g % 3);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            umma_bf16(tb, umma_smem_desc(sK + k * 32, 16, 1024),
                      umma_smem_desc(sQ + k * 32, 16, 1024), idS, k > 0);
            umma_bf16(tb + 64, umma_smem_desc(sV + k * 32, 16, 1024),
                      umma_smem_desc(sDO + k * 32, 16, 1024), idS, k > 0);
          }
          umma_commit(&s_full[g % 3]);
          umma_commit(&q_empty[s]);
        }
        if (!ok) break;
        mbar_arrive(&item_empty[slot]);
      }
    }
  };
  auto softmax = [&]() {
    // Softmax group wg takes the tiles it = wg, wg + kBwdSmGroups, ... of
    // each item. Warp w reads TMEM lanes of quadrant w % 4 (key rows) and
    // kBwdWarpCols query columns of the tile, in 16-column groups cg, and
    // writes P^T and dS^T (bf16 pairs) over exactly those S^T columns, so no
    // warp overwrites scores another warp has yet to read. The tile's
    // statistics come from the shared memory of its Q/dO stage (cp.async).
    const int quad = warp & 3;
    const int wg = (warp - kSmWarp0) / kBwdGroupWarps;
    const int cg0 = (((warp - kSmWarp0) % kBwdGroupWarps) >> 2) * (kBwdWarpCols / 16);
    const int r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const float c = p.scale * kLog2e;
    bool ok = true;
    int g = 0, ii = 0;
    for (; ok; ++ii) {
      const int slot = ii & 1;
      if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
      const BwdItem inf = items[slot];
      if (inf.nq < 0) break;  // no more items
      const int nq = inf.nq;
      const int b = inf.bh / heads;
      const int k0 = inf.kt * BT;
      const int key = k0 + r;
      const int qoff = GENERAL ? inf.qb - k0 : 0;  // first query tile relative to the keys
      [[maybe_unused]] Score<MODE> score(p, 0.f);
      // this key's row is seen by every query of its sequence
      const bool open = GENERAL && key < inf.prefix;
      int ql = wg, hq = GENERAL ? (inf.bh - b * heads) * p.group : 0;
      const int* segrow = SEG ? p.seg + (int64_t)b * p.T : nullptr;
      const int2* segtab = SEG ? segtab_of(slot) : nullptr;
      const int nch = (p.T + kSegChunk - 1) / kSegChunk -
                      (GENERAL ? inf.qb / kSegChunk : 2 * inf.kt);
      // this key row's segment id (rows past T take an id no query has)
      int sk = segrow ? (key < p.T ? segrow[key] : INT_MAX) : 0;
      if (SEG && GENERAL) sk = key < p.T ? seg_key_id(sk) : -1;
      const int2 krng =
          segrow ? seg_range(segtab, nch, -qoff / kSegChunk, 2) : make_int2(0, 0);
      for (int it = wg; it < nq; it += kBwdSmGroups, ql += kBwdSmGroups) {
        if (GENERAL && ql >= inf.nq1) {  // the group's next head
          ql -= inf.nq1;
          ++hq;
        }
        const int gt = g + it;  // running tile index
        const int bb = gt % 3;
        const uint32_t tb = tBuf(bb);
        const int qt = qtile(slot, GENERAL ? ql : it);  // query tile index (64 positions) past k0
        if constexpr ((MODE & kBias) != 0) score.slope2 = p.slopes[hq] * kLog2e;
        if (!(ok = mbar_wait(&s_full[bb], (gt / 3) & 1, abort_flag, err))) break;
        if (!(ok = mbar_wait(&q_full[gt % kQS], (gt / kQS) & 1, abort_flag, err))) break;
        // The dS^T ring slot of this tile was last read by the dQ MMA of the
        // pair closed by tile gt-3.
        if (gt >= 4 && !(ok = mbar_wait(&done[(gt - 3) & 3], ((gt - 3) >> 2) & 1, abort_flag, err)))
          break;
        tc_fence_after();
        uint8_t* sd = sm + L::DST + (gt & 3) * BT_BYTES;
        if constexpr (GENERAL) {
          const int q0 = qoff + qt * BQ;  // the tile's first query relative to the keys
          // per-element segment test unless this key tile and query tile share one id
          const bool segmask = SEG && !seg_single(seg_range(segtab, nch, qt, 1), krng);
          const bool diag = q0 < BT;  // some key may be past some query
          const float* stat =
              reinterpret_cast<const float*>(sm + L::STAT + (gt % kQS) * L::kStatBytes);
          const uint32_t ts = tb + lane_off;
          auto fetch = [&](int cg, uint32_t (&sv)[16], uint32_t (&dp)[16]) {
            tmem_ld16_nw(ts + cg * 16, sv);
            tmem_ld16_nw(ts + 64 + cg * 16, dp);
          };
          auto put = [&](int cg, const uint32_t (&pk)[8], const uint32_t (&dk)[8]) {
            tmem_st8_nw(ts + cg * 16, pk);
            tmem_st8_nw(ts + cg * 16 + 8, dk);
            *reinterpret_cast<uint4*>(sd + swz128(r, cg * 2)) = make_uint4(dk[0], dk[1], dk[2], dk[3]);
            *reinterpret_cast<uint4*>(sd + swz128(r, cg * 2 + 1)) =
                make_uint4(dk[4], dk[5], dk[6], dk[7]);
          };
          uint32_t pk[8], dk[8];
          if (!diag && !segmask && k0 + q0 + BQ <= p.T) {
            // every query sees every key
#pragma unroll 1
            for (int cg = cg0; cg < cg0 + kBwdWarpCols / 16; ++cg) {
              uint32_t sv[16], dp[16];
              fetch(cg, sv, dp);
              tmem_wait_ld();
              score.template gradients<false>(sv, dp, stat + cg * 16, (float)(r - q0 - cg * 16), 0,
                                              pk, dk);
              put(cg, pk, dk);
            }
          } else {
#pragma unroll 1
            for (int cg = cg0; cg < cg0 + kBwdWarpCols / 16; ++cg) {
              uint32_t sv[16], dp[16];
              fetch(cg, sv, dp);
              const int rel = r - q0 - cg * 16;            // key - query of column 0
              const int tail = p.T - k0 - q0 - cg * 16;    // columns from here lie past the end
              // which of the 16 queries see this key
              uint32_t see = 0xffffu;
              if (diag && !open) see = rel <= 0 ? see : rel >= 16 ? 0u : see << rel & 0xffffu;
              if (tail < 16) see &= tail <= 0 ? 0u : (1u << tail) - 1u;
              if (segmask) {
                const int id = reinterpret_cast<const int*>(stat)[128 + cg * 16 + (lane & 15)];
                see &= segment_columns(seg_query_id(id), sk);
              }
              tmem_wait_ld();
              if (__all_sync(0xffffffffu, see == 0u)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) pk[i] = dk[i] = 0;
              } else {
                score.template gradients<true>(sv, dp, stat + cg * 16, (float)rel, see, pk, dk);
              }
              put(cg, pk, dk);
            }
          }
        } else {
#pragma unroll
        for (int sub = 0; sub < kBwdWarpCols / 16; ++sub) {
        const int cg = cg0 + sub;
        // this 16-column group's statistics; the scores of the tile exist only
        // after its Q/dO stage (statistics included) was full
        const float* stat =
            reinterpret_cast<const float*>(sm + L::STAT + (gt % kQS) * L::kStatBytes) + cg * 16;
        const int* stat_seg = reinterpret_cast<const int*>(stat) + 128;
        uint32_t sraw[16], draw[16];
        tmem_ld16_nw(tb + lane_off + cg * 16, sraw);
        tmem_ld16_nw(tb + 64 + lane_off + cg * 16, draw);
        tmem_wait_ld();
        const int qbase = qt * BQ + cg * 16;  // query index relative to k0
        const bool diag = (qt < 2);           // key r > query masks only near the diagonal
        const int tail = p.T - k0 - qbase;    // columns j >= tail lie past the sequence end
        const bool mask = diag || tail < 16;
        // per-element segment test unless this key tile and query tile share one id
        const bool segmask = segrow && !rng_single(seg_range(segtab, nch, qt, 1), krng);
        // P^T = exp2(S^T c - lse log2e) and dS^T = P^T (dP^T - delta), two
        // columns per packed f32x2 instruction; the causal and end-of-sequence
        // tests run only on tiles that need them and the segment test only
        // when the tiles' ids differ.
        uint32_t pk[8], dk[8];
        auto softmax_cols = [&](auto mask_tag) {
          constexpr bool kMask = decltype(mask_tag)::value;
          const float2 c2 = make_float2(c, c);
          const float2 nlog2e = make_float2(-kLog2e, -kLog2e);
          const float2 m1 = make_float2(-1.f, -1.f);
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4) {
            const float4 l4 = reinterpret_cast<const float4*>(stat)[j4];
            const float4 d4 = reinterpret_cast<const float4*>(stat + 64)[j4];
            const float2 x01 = ffma2(make_float2(__uint_as_float(sraw[4 * j4]),
                                                 __uint_as_float(sraw[4 * j4 + 1])),
                                     c2, fmul2(make_float2(l4.x, l4.y), nlog2e));
            const float2 x23 = ffma2(make_float2(__uint_as_float(sraw[4 * j4 + 2]),
                                                 __uint_as_float(sraw[4 * j4 + 3])),
                                     c2, fmul2(make_float2(l4.z, l4.w), nlog2e));
            float pv[4] = {ex2(x01.x), ex2(x01.y), ex2(x23.x), ex2(x23.y)};
            // dP^T - delta as fma(delta, -1, dP^T): one rounding, as a subtraction
            const float2 g01 = ffma2(make_float2(d4.x, d4.y), m1,
                                     make_float2(__uint_as_float(draw[4 * j4]),
                                                 __uint_as_float(draw[4 * j4 + 1])));
            const float2 g23 = ffma2(make_float2(d4.z, d4.w), m1,
                                     make_float2(__uint_as_float(draw[4 * j4 + 2]),
                                                 __uint_as_float(draw[4 * j4 + 3])));
            float2 dv01 = fmul2(make_float2(pv[0], pv[1]), g01);
            float2 dv23 = fmul2(make_float2(pv[2], pv[3]), g23);
            float dvs[4] = {dv01.x, dv01.y, dv23.x, dv23.y};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int j = 4 * j4 + u;
              bool off = false;
              if (kMask) off = (diag && r > qbase + j) || j >= tail;
              if (SEG && segmask && stat_seg[j] != sk) off = true;
              if (off) pv[u] = dvs[u] = 0.f;
            }
            dv01 = make_float2(dvs[0], dvs[1]);
            dv23 = make_float2(dvs[2], dvs[3]);
            pk[2 * j4] = pack_bf16x2(pv[0], pv[1]);
            pk[2 * j4 + 1] = pack_bf16x2(pv[2], pv[3]);
            dk[2 * j4] = pack_bf16x2(dv01.x, dv01.y);
            dk[2 * j4 + 1] = pack_bf16x2(dv23.x, dv23.y);
          }
        };
        if (mask)
          softmax_cols(std::integral_constant<bool, true>());
        else
          softmax_cols(std::integral_constant<bool, false>());
        tmem_st8_nw(tb + lane_off + cg * 16, pk);
        tmem_st8_nw(tb + lane_off + cg * 16 + 8, dk);
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2)
          *reinterpret_cast<uint4*>(sd + swz128(r, cg * 2 + q2)) =
              make_uint4(dk[4 * q2], dk[4 * q2 + 1], dk[4 * q2 + 2], dk[4 * q2 + 3]);
        }
        }
        tmem_wait_st();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[bb]);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      g += nq;
    }
  };
  auto flush = [&]() {
    // dQ read-out: warp kFlushWarp + i serves TMEM lane quadrant
    // (kFlushWarp + i) % 4. For each query pair (list entries 2j, 2j+1 of
    // an item; TMEM lane m is row m of the pair, quadrants 0-1 the first tile,
    // 2-3 the second) it loads its 32 rows x 64 fp32 columns as soon as the
    // pair's dQ MMA has completed, releases the TMEM buffer, stages the rows
    // in two 128-byte swizzled [32 x 32] boxes of its own and reduces them
    // into dq_acc with TMA reduce-adds (rows past the sequence end are clipped
    // by the map; a box that starts past it is skipped). At the end of an
    // item the same warps write dK and dV. The softmax warps never wait for
    // this.
    const int quad = warp & 3;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    uint8_t* stage = sm + L::DQS + (warp - kFlushWarp) * 8192;
    bool ok = true;
    int g = 0, ii = 0;
    for (; ok; ++ii) {
      const int slot = ii & 1;
      if (!(ok = mbar_wait(&item_full[slot], (ii >> 1) & 1, abort_flag, err))) break;
      const BwdItem inf = items[slot];
      if (inf.nq < 0) break;  // no more items
      const int k0 = inf.kt * BT;
      int ql = 0, bhq = inf.bh;  // the pair's list entry and its row block of dq_acc
      if constexpr (GENERAL) bhq = inf.bh / heads * p.H + inf.bh % heads * p.group;
      for (int j = 0; j < inf.nq / 2; ++j, ql += 2) {
        if (GENERAL && ql == inf.nq1) {
          ql = 0;
          ++bhq;
        }
        const int J = (g >> 1) + j;  // running pair index
        if (!(ok = mbar_wait(&dq_full[J & 1], (J >> 1) & 1, abort_flag, err))) break;
        tc_fence_after();
        const int bb = (g + 2 * j + 1) % 3;  // buffer of the pair's closing tile
        float v[64];
        tmem_ld32(tBuf(bb) + 64 + lane_off, v);
        tmem_ld32(tBuf(bb) + 96 + lane_off, v + 32);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dq_free[J & 1]);
        const int row0 = (GENERAL ? inf.qb : k0) + qtile(slot, ql + (quad >> 1)) * BQ +
                         (quad & 1) * 32;
        if (row0 < p.T) {  // warp-uniform
          if (lane == 0) bulk_wait_read();  // the previous reduce has read the staging boxes
          __syncwarp();
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int ch = 0; ch < 8; ++ch)
              *reinterpret_cast<float4*>(stage + hh * 4096 + swz128(lane, ch)) =
                  make_float4(v[32 * hh + 4 * ch], v[32 * hh + 4 * ch + 1],
                              v[32 * hh + 4 * ch + 2], v[32 * hh + 4 * ch + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_reduce_add_3d(&tmDQ, stage, 0, row0, bhq);
            tma_reduce_add_3d(&tmDQ, stage + 4096, 32, row0, bhq);
            bulk_commit();
          }
        }
      }
      if (!ok) break;
      // dK (times the softmax scale, rotated back by RoPE) and dV of the
      // item's 128 keys, this warp's 32 rows. All four 32-column chunks leave
      // TMEM first (dK parked in this warp's staging area, dV in registers) so
      // the next item's gradient MMAs can start; then the rows are written.
      if (!(ok = mbar_wait(fin, ii & 1, abort_flag, err))) break;
      tc_fence_after();
      {
        const int key = k0 + quad * 32 + lane;
        const int bi = inf.bh / heads, hi = inf.bh - bi * heads;
        if (lane == 0) bulk_wait_read();  // the last dQ reduce has read the staging area
        __syncwarp();
        float* park = reinterpret_cast<float*>(stage);  // [32 rows][64] fp32, 16-byte chunks xor-swizzled
        auto park_at = [&](int chunk) { return park + lane * 64 + ((chunk ^ (lane & 15)) << 2); };
        {
          float t64[64];
          tmem_ld32_nw(tDK + lane_off, reinterpret_cast<uint32_t*>(t64));
          tmem_ld32_nw(tDK + lane_off + 32, reinterpret_cast<uint32_t*>(t64) + 32);
          tmem_wait_ld();
#pragma unroll
          for (int c4 = 0; c4 < 16; ++c4)
            *reinterpret_cast<float4*>(park_at(c4)) =
                make_float4(t64[4 * c4], t64[4 * c4 + 1], t64[4 * c4 + 2], t64[4 * c4 + 3]);
        }
        float dvv[64];
        tmem_ld32_nw(tDV + lane_off, reinterpret_cast<uint32_t*>(dvv));
        tmem_ld32_nw(tDV + lane_off + 32, reinterpret_cast<uint32_t*>(dvv) + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_free);
        if (key < p.T) {
          bf16* vrow = p.dv + bi * p.sb + hi * p.sh + (int64_t)key * p.st;
          bf16* krow = p.dk + bi * p.sb + hi * p.sh + (int64_t)key * p.st;
#pragma unroll
          for (int q8 = 0; q8 < 8; ++q8) {
            const float* gv = dvv + 8 * q8;
            uint4 o;
            o.x = pack_bf16x2(gv[0], gv[1]);
            o.y = pack_bf16x2(gv[2], gv[3]);
            o.z = pack_bf16x2(gv[4], gv[5]);
            o.w = pack_bf16x2(gv[6], gv[7]);
            *reinterpret_cast<uint4*>(vrow + 8 * q8) = o;
          }
#pragma unroll 2
          for (int q8 = 0; q8 < 8; ++q8) {
            const float4 a4 = *reinterpret_cast<const float4*>(park_at(2 * q8));
            const float4 b4 = *reinterpret_cast<const float4*>(park_at(2 * q8 + 1));
            float gv[8] = {a4.x, a4.y, a4.z, a4.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) gv[i] *= p.scale;
            if (p.rcos) rope_back(gv, p.rcos, p.rsin, key, q8);
            uint4 o;
            o.x = pack_bf16x2(gv[0], gv[1]);
            o.y = pack_bf16x2(gv[2], gv[3]);
            o.z = pack_bf16x2(gv[4], gv[5]);
            o.w = pack_bf16x2(gv[6], gv[7]);
            *reinterpret_cast<uint4*>(krow + 8 * q8) = o;
          }
        }
        __syncwarp();  // the park area is read before the next dQ staging writes
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      g += inf.nq;
    }
    if (lane == 0) bulk_wait_all();
  };
  if constexpr (GENERAL) {
    if (warp < kSmWarp0) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBwdRegsIssue));
      if (warp == 0) {
        produce();
      } else if (warp == 1) {
        gradients();
      } else if (warp == kScoreWarp) {
        scores();
      }
    } else if (warp < kFlushWarp) {
      softmax();
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBwdRegsFlush));
      flush();
    }
  } else if (warp == 0) {
    produce();
  } else if (warp == 1) {
    gradients();
  } else if (warp == kScoreWarp) {
    scores();
  } else if (warp < kSmWarp0 + kSmWarps) {
    softmax();
  } else {
    flush();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) sched_finish(p.sched);
}

// delta[bh, t] = sum_e dO * O, and zero the dQ accumulator row. With neg_lse2
// the statistics as the score-modified backward takes them: -delta, -lse log2(e). Eight lanes
// per row (16-byte loads), four rows per warp.
__global__ void attn_delta_kernel(const bf16* __restrict__ o, const bf16* __restrict__ dout,
                                  int64_t osb, int64_t osh, int64_t ost, int64_t gsb, int64_t gsh,
                                  int64_t gst, int B, int H, int T, float* __restrict__ delta,
                                  float* __restrict__ dq_acc, const float* __restrict__ lse,
                                  float* __restrict__ neg_lse2, bool o_in_acc) {
  const int64_t rows = (int64_t)B * H * T;
  const int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  const int seg = threadIdx.x & 7;
  const bool valid = r < rows;  // no early return: the 8-lane shuffles below span the warp
  const int64_t rr = valid ? r : 0;
  const int64_t bh = rr / T;
  const int t = (int)(rr - bh * T);
  const int b = (int)(bh / H), h = (int)(bh - (int64_t)b * H);
  const int64_t off = b * osb + h * osh + (int64_t)t * ost + seg * 8;
  const int64_t goff = b * gsb + h * gsh + (int64_t)t * gst + seg * 8;
  const uint4 qg = *reinterpret_cast<const uint4*>(dout + goff);
  const uint32_t* wg = &qg.x;
  float s = 0.f;
  if (o_in_acc) {  // fp32 rows in the accumulator's place; this thread clears what it reads
    const float4* src = reinterpret_cast<const float4*>(dq_acc + rr * HD + seg * 8);
    const float4 a = src[0], c = src[1];
    const float ov[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float g0, g1;
      unpack_bf16x2(wg[j], g0, g1);
      s += ov[2 * j] * g0 + ov[2 * j + 1] * g1;
    }
  } else {
    const uint4 qo = *reinterpret_cast<const uint4*>(o + off);
    const uint32_t* wo = &qo.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float o0, o1, g0, g1;
      unpack_bf16x2(wo[j], o0, o1);
      unpack_bf16x2(wg[j], g0, g1);
      s += o0 * g0 + o1 * g1;
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  if (!valid) return;
  if (seg == 0) {
    delta[r] = neg_lse2 ? -s : s;
    if (neg_lse2) neg_lse2[r] = -kLog2e * lse[r];
  }
  float4* z = reinterpret_cast<float4*>(dq_acc + r * HD + seg * 8);
  z[0] = make_float4(0.f, 0.f, 0.f, 0.f);
  z[1] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// dq = bf16(scale * dq_acc), rotated back by RoPE when tables are given.
__global__ void attn_dq_store_kernel(const float* __restrict__ dq_acc, bf16* __restrict__ dq,
                                     int64_t sb, int64_t sh, int64_t st, int B, int H, int T,
                                     float scale, const bf16* rcos, const bf16* rsin) {
  const int64_t chunks = (int64_t)B * H * T * (HD / 8);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < chunks;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i >> 3;
    const int c = (int)(i & 7);
    const int64_t bh = row / T;
    const int t = (int)(row - bh * T);
    const int b = (int)(bh / H), h = (int)(bh - (int64_t)b * H);
    const float4* src = reinterpret_cast<const float4*>(dq_acc + row * HD + c * 8);
    float4 a = src[0], e = src[1];
    float v[8] = {a.x * scale, a.y * scale, a.z * scale, a.w * scale,
                  e.x * scale, e.y * scale, e.z * scale, e.w * scale};
    if (rcos) rope_back(v, rcos, rsin, t, c);
    uint4 q;
    q.x = pack_bf16x2(v[0], v[1]);
    q.y = pack_bf16x2(v[2], v[3]);
    q.z = pack_bf16x2(v[4], v[5]);
    q.w = pack_bf16x2(v[6], v[7]);
    *reinterpret_cast<uint4*>(dq + b * sb + h * sh + (int64_t)t * st + c * 8) = q;
  }
}

int attention_read_error(int clear) {
  int hv = 0;
  cudaMemcpyFromSymbol(&hv, g_attn_error, sizeof(int));
  if (clear) {
    int z = 0;
    cudaMemcpyToSymbol(g_attn_error, &z, sizeof(int));
  }
  return hv;
}

// ------------------------------------------------------------------ host
// The counter slots of one device. Launches on a stream run one after the other,
// so a stream keeps one slot for all of its launches; streams go by their ids,
// which no two of a process have in common. A captured launch runs wherever its
// graph is launched, beside any stream's launches and beside other branches of the
// graph, so each has a slot to itself until the graph and everything instantiated
// from it are gone (a graph does not run beside itself).
struct SchedSlots {
  std::shared_mutex launching;  // shared: from the choice of a slot to the launch
  std::mutex mu;                // the fields below
  unsigned* base = nullptr;
  int used = 0;                                // slots [0, used) have been handed out
  std::vector<int> free;                       // of these, those that nothing holds
  std::unordered_map<unsigned long long, int> of_stream;

  int take() {  // -1: none is left
    if (!free.empty()) {
      const int k = free.back();
      free.pop_back();
      return k;
    }
    return used < kSchedSlots ? used++ : -1;
  }
  // A program that has used as many streams as there are slots: once the device is
  // idle, and no thread between its choice and its launch, no stream needs its slot.
  cudaError_t forget_streams() {
    std::unique_lock<std::shared_mutex> none(launching);
    const cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    for (const auto& s : of_stream) free.push_back(s.second);
    of_stream.clear();
    return cudaSuccess;
  }
};
struct GraphSlot {
  SchedSlots* owner;
  int slot;
};
static void CUDART_CB return_slot(void* p) {  // a graph's last reference has gone
  GraphSlot* g = reinterpret_cast<GraphSlot*>(p);
  {
    std::lock_guard<std::mutex> lock(g->owner->mu);
    g->owner->free.push_back(g->slot);
  }
  delete g;
}

// The counter slot of a launch on `st`; kept until the launch has been made. status:
// 0, or an error (65,536 captured launches at a time leave no slot).
struct SchedSlot {
  int status;
  unsigned* counter = nullptr;
  explicit SchedSlot(cudaStream_t st) {
    try {
      status = choose(st);
    } catch (const std::bad_alloc&) {
      status = -static_cast<int>(cudaErrorMemoryAllocation);
    }
  }

 private:
  std::shared_lock<std::shared_mutex> launching_;

  int choose(cudaStream_t st) {
    static SchedSlots* const devices = new SchedSlots[64];  // graphs may outlive static objects
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64) return GPTB200_EUNSUPPORTED;
    SchedSlots& d = devices[dev];
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaGraph_t graph = nullptr;
    unsigned long long id = 0;
    cudaError_t e = cudaStreamGetCaptureInfo(st, &capture, &id, &graph);
    const bool captured = capture == cudaStreamCaptureStatusActive;
    if (e == cudaSuccess && !captured) e = cudaStreamGetId(st, &id);
    if (e != cudaSuccess) return -static_cast<int>(e);
    int k = -1;
    for (int tries = 0; k < 0; ++tries) {
      launching_ = std::shared_lock<std::shared_mutex>(d.launching);
      {
        std::lock_guard<std::mutex> lock(d.mu);
        if (!d.base) {
          void* ptr = nullptr;
          e = cudaGetSymbolAddress(&ptr, g_attn_sched);
          if (e != cudaSuccess) return -static_cast<int>(e);
          d.free.reserve(kSchedSlots);  // return_slot has no way to report a failure
          d.base = reinterpret_cast<unsigned*>(ptr);
        }
        const auto known = captured ? d.of_stream.end() : d.of_stream.find(id);
        k = known != d.of_stream.end() ? known->second : d.take();
        if (!captured && k >= 0) d.of_stream.emplace(id, k);
      }
      if (k >= 0) break;
      launching_.unlock();
      if (captured || tries) return GPTB200_EUNSUPPORTED;
      e = d.forget_streams();
      if (e != cudaSuccess) return -static_cast<int>(e);
    }
    if (captured) {
      GraphSlot* g = new GraphSlot{&d, k};
      cudaUserObject_t kept;
      e = cudaUserObjectCreate(&kept, g, return_slot, 1, cudaUserObjectNoDestructorSync);
      if (e != cudaSuccess) {
        return_slot(g);
        return -static_cast<int>(e);
      }
      e = cudaGraphRetainUserObject(graph, kept, 1, cudaGraphUserObjectMove);
      if (e != cudaSuccess) {
        cudaUserObjectRelease(kept, 1);  // the last reference: returns the slot
        return -static_cast<int>(e);
      }
    }
    counter = d.base + 2 * (size_t)k;
    return 0;
  }
};
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// 4-D map over a [b, t, h, e] tensor with element strides (sb, st, sh), box
// 64 (e) x box_rows (t), 128-byte swizzle.
static bool make_map4(CUtensorMap* m, const void* base, int B, int H, int T, int64_t sb,
                      int64_t sh, int64_t st, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[4] = {HD, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)st * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {HD, (cuuint32_t)box_rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  auto encode = [&] {
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // a thread that has not used the device yet (autograd's): bind its context
    cudaFree(nullptr);
    r = encode();
  }
  return r == CUDA_SUCCESS;
}

}  // namespace gptb200

using namespace gptb200;

// 3-D fp32 map over dq_acc [B*H, T, 64], box 32 x 32 x 1, 128-byte swizzle
// (the bwd kernel's TMA reduce-add target).
static bool make_dq_map(CUtensorMap* m, float* base, int BH, int T) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {HD, (cuuint64_t)T, (cuuint64_t)BH};
  cuuint64_t strides[2] = {(cuuint64_t)HD * 4, (cuuint64_t)T * HD * 4};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int check_attn(const void* q, const void* k, const void* v, int64_t sb, int64_t sh,
                      int64_t st, int64_t osb, int64_t osh, int64_t ost, int64_t batch,
                      int64_t heads, int64_t seq, int64_t hd) {
  if (!q || !k || !v) return GPTB200_EINVAL;
  if (batch <= 0 || heads <= 0 || seq <= 0) return GPTB200_EINVAL;
  if (hd != HD) return GPTB200_EUNSUPPORTED;
  if (batch * heads > 65535 || seq > (1 << 24)) return GPTB200_ESHAPE;
  if ((sb | sh | st | osb | osh | ost) % 8) return GPTB200_ESHAPE;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
       reinterpret_cast<uintptr_t>(v)) & 15)
    return GPTB200_ESHAPE;
  return 0;
}

extern "C" int gptb200_attention_fwd(const void* q, const void* k, const void* v, int64_t stride_b,
                                     int64_t stride_h, int64_t stride_t, void* o,
                                     int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_t,
                                     float* lse, int64_t batch, int64_t heads, int64_t seq,
                                     int64_t head_dim, float softmax_scale,
                                     const int32_t* segment_ids, void* stream) {
  int s = check_attn(q, k, v, stride_b, stride_h, stride_t, o_stride_b, o_stride_h, o_stride_t,
                     batch, heads, seq, head_dim);
  if (s) return s;
  if (!o || !lse || !(softmax_scale > 0.f)) return GPTB200_EINVAL;
  if (segment_ids && seq > (int64_t)kMaxSegChunks * kSegChunk) return GPTB200_EUNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(segment_ids) & 3) return GPTB200_ESHAPE;
  if (reinterpret_cast<uintptr_t>(o) & 15) return GPTB200_ESHAPE;
  CUtensorMap mq, mk, mv;
  if (!make_map4(&mq, q, (int)batch, (int)heads, (int)seq, stride_b, stride_h, stride_t, FQ) ||
      !make_map4(&mk, k, (int)batch, (int)heads, (int)seq, stride_b, stride_h, stride_t, FK) ||
      !make_map4(&mv, v, (int)batch, (int)heads, (int)seq, stride_b, stride_h, stride_t, FK))
    return GPTB200_ESHAPE;
  AttnParams p = {};
  p.B = (int)batch;
  p.H = (int)heads;
  p.T = (int)seq;
  p.scale = softmax_scale;
  p.o = reinterpret_cast<bf16*>(o);
  p.osb = o_stride_b;
  p.osh = o_stride_h;
  p.ost = o_stride_t;
  p.lse = lse;
  p.seg = segment_ids;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const SchedSlot slot(st);
  if (slot.status) return slot.status;
  p.sched = slot.counter;
  static bool cfg[64][2] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int seg = segment_ids != nullptr;
  auto kern = seg ? attn_fwd_tc<true> : attn_fwd_tc<false>;
  const int smem = seg ? FwdSmem<true>::TOTAL : FwdSmem<false>::TOTAL;
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 64 || !cfg[dev][seg]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 64) cfg[dev][seg] = true;
  }
  // persistent: one CTA per SM (or per item, when there are fewer items)
  const int64_t items = (seq + 2 * FQ - 1) / (2 * FQ) * batch * heads;
  const unsigned grid = (unsigned)std::min<int64_t>(items, sms);
  kern<<<grid, kFwdThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(mq, mk, mv, p);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

extern "C" size_t gptb200_attention_bwd_workspace_size(int64_t batch, int64_t heads, int64_t seq) {
  if (batch <= 0 || heads <= 0 || seq <= 0) return 0;
  const int64_t rows = batch * heads * seq;
  return (size_t)((rows * 4 + 255) / 256 * 256 + rows * HD * 4);
}

extern "C" int gptb200_attention_bwd(const void* q, const void* k, const void* v, int64_t stride_b,
                                     int64_t stride_h, int64_t stride_t, const void* o,
                                     const void* dout, int64_t o_stride_b, int64_t o_stride_h,
                                     int64_t o_stride_t, const float* lse, void* dq, void* dk,
                                     void* dv, int64_t batch, int64_t heads, int64_t seq,
                                     int64_t head_dim, float softmax_scale, const void* rope_cos,
                                     const void* rope_sin, const int32_t* segment_ids,
                                     void* workspace, void* stream) {
  int s = check_attn(q, k, v, stride_b, stride_h, stride_t, o_stride_b, o_stride_h, o_stride_t,
                     batch, heads, seq, head_dim);
  if (s) return s;
  if (!o || !dout || !lse || !dq || !dk || !dv || !workspace || !(softmax_scale > 0.f))
    return GPTB200_EINVAL;
  if (segment_ids && seq > (int64_t)kMaxSegChunks * kSegChunk) return GPTB200_EUNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(segment_ids) & 3) return GPTB200_ESHAPE;
  if ((rope_cos == nullptr) != (rope_sin == nullptr)) return GPTB200_EINVAL;
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
       reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return GPTB200_ESHAPE;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const int B = (int)batch, H = (int)heads, T = (int)seq;
  CUtensorMap mq, mk, mv, mdo;
  if (!make_map4(&mq, q, B, H, T, stride_b, stride_h, stride_t, BQ) ||
      !make_map4(&mk, k, B, H, T, stride_b, stride_h, stride_t, BT) ||
      !make_map4(&mv, v, B, H, T, stride_b, stride_h, stride_t, BT) ||
      !make_map4(&mdo, dout, B, H, T, o_stride_b, o_stride_h, o_stride_t, BQ))
    return GPTB200_ESHAPE;
  const int64_t rows = batch * heads * seq;
  float* delta = reinterpret_cast<float*>(workspace);
  float* dq_acc = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) +
                                           (rows * 4 + 255) / 256 * 256);
  attn_delta_kernel<<<(unsigned)((rows * 8 + 255) / 256), 256, 0, st>>>(
      reinterpret_cast<const bf16*>(o), reinterpret_cast<const bf16*>(dout), o_stride_b,
      o_stride_h, o_stride_t, o_stride_b, o_stride_h, o_stride_t, B, H, T, delta, dq_acc, nullptr,
      nullptr, false);
  GPTB200_CHECK_LAUNCH();
  AttnParams p = {};
  p.B = B;
  p.H = H;
  p.T = T;
  p.scale = softmax_scale;
  p.lse = const_cast<float*>(lse);
  p.delta = delta;
  p.dq_acc = dq_acc;
  p.dk = reinterpret_cast<bf16*>(dk);
  p.dv = reinterpret_cast<bf16*>(dv);
  p.sb = stride_b;
  p.sh = stride_h;
  p.st = stride_t;
  p.rcos = reinterpret_cast<const bf16*>(rope_cos);
  p.rsin = reinterpret_cast<const bf16*>(rope_sin);
  p.seg = segment_ids;
  const SchedSlot slot(st);
  if (slot.status) return slot.status;
  p.sched = slot.counter;
  static bool cfg[64][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int seg = segment_ids != nullptr;
  const int groups = seq >= 2048 ? 2 : 1;
  auto kern = seg ? (groups == 2 ? attn_bwd_tc<true, 2, kClassic> : attn_bwd_tc<true, 1, kClassic>)
                  : (groups == 2 ? attn_bwd_tc<false, 2, kClassic>
                                 : attn_bwd_tc<false, 1, kClassic>);
  const int smem = seg ? BwdSmem<true>::TOTAL : BwdSmem<false>::TOTAL;
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int ci = seg * 2 + (groups - 1);
  if (dev >= 64 || !cfg[dev][ci]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 64) cfg[dev][ci] = true;
  }
  // persistent: one CTA per SM (or per item, when there are fewer items)
  const int64_t items = (seq + BT - 1) / BT * batch * heads;
  const unsigned grid = (unsigned)std::min<int64_t>(items, sms);
  CUtensorMap mdq;
  if (!make_dq_map(&mdq, dq_acc, B * H, T)) return GPTB200_ESHAPE;
  kern<<<grid, kBwdThreads, smem, st>>>(mq, mk, mv, mdo, mdq, p);
  GPTB200_CHECK_LAUNCH();
  const int64_t chunks = rows * (HD / 8);
  int blocks = (int)std::min<int64_t>((chunks + 255) / 256, (int64_t)sms * 8);
  attn_dq_store_kernel<<<blocks, 256, 0, st>>>(dq_acc, reinterpret_cast<bf16*>(dq), stride_b,
                                               stride_h, stride_t, B, H, T, softmax_scale,
                                               reinterpret_cast<const bf16*>(rope_cos),
                                               reinterpret_cast<const bf16*>(rope_sin));
  GPTB200_CHECK_LAUNCH();
  return 0;
}

// ------------------------------------------------------------------ score-modified attention
namespace gptb200 {

// Everything about a call that is checked or looked up before a launch.
static int score_check(const gptb200_score_attention* a) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->lse) return GPTB200_EINVAL;
  if (a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->seq <= 0) return GPTB200_EINVAL;
  if (!(a->softmax_scale > 0.f) || !(a->softcap >= 0.f) || isinf(a->softcap) ||
      isinf(a->softmax_scale))
    return GPTB200_EINVAL;
  if (a->head_dim != HD || a->heads % a->kv_heads) return GPTB200_EUNSUPPORTED;
  if (a->batch * a->heads > 65535 || a->seq > (1 << 24)) return GPTB200_ESHAPE;
  if (a->segment_ids && a->seq > (int64_t)kMaxSegChunks * kSegChunk) return GPTB200_EUNSUPPORTED;
  int64_t strides = 0;
  for (int i = 0; i < 3; ++i) strides |= a->q_stride[i] | a->kv_stride[i] | a->o_stride[i];
  if (strides % 8) return GPTB200_ESHAPE;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
       reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->o)) & 15)
    return GPTB200_ESHAPE;
  if ((reinterpret_cast<uintptr_t>(a->segment_ids) | reinterpret_cast<uintptr_t>(a->prefix_lens) |
       reinterpret_cast<uintptr_t>(a->slopes) | reinterpret_cast<uintptr_t>(a->lse)) & 3)
    return GPTB200_ESHAPE;
  return 0;
}

static AttnParams score_params(const gptb200_score_attention* a) {
  AttnParams p = {};
  p.B = (int)a->batch;
  p.H = (int)a->heads;
  p.T = (int)a->seq;
  p.KVH = (int)a->kv_heads;
  p.group = p.H / p.KVH;
  p.scale = a->softmax_scale;
  p.cap = a->softcap;
  p.slopes = a->slopes;
  p.prefix = a->prefix_lens;
  p.o = reinterpret_cast<bf16*>(a->o);
  p.osb = a->o_stride[0];
  p.osh = a->o_stride[1];
  p.ost = a->o_stride[2];
  p.lse = a->lse;
  p.seg = a->segment_ids;
  return p;
}

// Whether a launch walks the items of all heads by falling weight instead of
// head by head. By weight the last items are light and every SM ends at about
// the same time; head by head the tiles that the items of a head share stay in
// L2. So: by weight while the shared tiles of all heads (`bytes`) fit, and in the
// backward longer for capped scores, which compute more per byte. One limit cannot tell
// many short sequences from few long ones: the capped backward of 128 x 1024 is past it
// and 8% slower for that, 16 x 8192 20% faster. Measured at 12
// heads (us, by weight / head by head; MB of shared tiles), capped and biased |
// without either:
//   forward  25 MB (1 x 8192): 260 / 331 | 185 / 235;  101 MB (4 x 8192): 945 / 1011
//            | 690 / 718;  151 MB (48 x 1024): 257 / 259 | 206 / 192;  403 MB (128 x
//            1024): 707 / 662 | 559 / 477
//   backward 25 MB: 457 / 525 | 343 / 397;  101 MB: 1830 / 1834 | 1442 / 1390;
//            151 MB: 553 / 619 | 517 / 476;  403 MB: 1477 / 1596 | 1374 / 1238 at
//            128 x 1024, 8836 / 7381 | 7831 / 6131 at 16 x 8192
static int by_weight(int64_t bytes, int64_t limit) { return bytes <= limit << 20; }

// One persistent launch: the shared-memory attribute (set once per kernel and
// device) and one CTA per SM or item.
template <typename K, typename... Args>
static int launch_persistent(K kern, bool (&done)[64], int64_t items, int threads, int smem,
                             cudaStream_t st, Args... args) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 64 || !done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 64) done[dev] = true;
  }
  kern<<<(unsigned)std::min<int64_t>(items, sms), threads, smem, st>>>(args...);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

struct ScoreMaps {
  CUtensorMap q, k, v, g, dq;
};

template <bool SEG, int MODE>
static int score_fwd_launch(const AttnParams& p, const ScoreMaps& m, cudaStream_t st) {
  static bool done[64] = {};
  const int64_t items = (int64_t)((p.T + 2 * FQ - 1) / (2 * FQ)) * p.B * p.H;
  return launch_persistent(score_fwd_tc<SEG, MODE>, done, items, kFwdGeneralThreads,
                           FwdSmem<SEG>::TOTAL, st, m.q, m.k, m.v, p);
}

template <bool SEG, int MODE>
static int score_bwd_launch(const AttnParams& p, const ScoreMaps& m, cudaStream_t st) {
  static bool done[64] = {};
  const int64_t items = (int64_t)((p.T + BT - 1) / BT) * p.B * p.KVH;
  return launch_persistent(attn_bwd_tc<SEG, 2, MODE>, done, items, kBwdGeneralThreads,
                           BwdSmem<SEG>::TOTAL, st, m.q, m.k, m.v, m.g, m.dq, p);
}

// f<MODE>() for the call's cap and bias.
template <typename F>
static int score_mode(const gptb200_score_attention* a, F&& f) {
  if (a->softcap > kShortCap)
    return a->slopes ? f(std::integral_constant<int, kGeneral | kCap | kWide | kBias>())
                     : f(std::integral_constant<int, kGeneral | kCap | kWide>());
  if (a->softcap > 0.f)
    return a->slopes ? f(std::integral_constant<int, kGeneral | kCap | kBias>())
                     : f(std::integral_constant<int, kGeneral | kCap>());
  return a->slopes ? f(std::integral_constant<int, kGeneral | kBias>())
                   : f(std::integral_constant<int, kGeneral>());
}

// The forward of a checked call, with fp32 rows for o and no lse if o32.
static int score_forward(const gptb200_score_attention* a, float* o32, cudaStream_t st) {
  AttnParams p = score_params(a);
  p.o32 = o32;
  ScoreMaps m;
  const int64_t *qs = a->q_stride, *ks = a->kv_stride;
  if (!make_map4(&m.q, a->q, p.B, p.H, p.T, qs[0], qs[1], qs[2], FQ) ||
      !make_map4(&m.k, a->k, p.B, p.KVH, p.T, ks[0], ks[1], ks[2], FK) ||
      !make_map4(&m.v, a->v, p.B, p.KVH, p.T, ks[0], ks[1], ks[2], FK))
    return GPTB200_ESHAPE;
  const SchedSlot slot(st);
  if (slot.status) return slot.status;
  p.sched = slot.counter;
  // K and V of every head
  p.by_weight = by_weight(a->batch * a->kv_heads * a->seq * 2 * HD * 2, 128);
  return score_mode(a, [&](auto mode) {
    constexpr int MODE = decltype(mode)::value;
    return p.seg ? score_fwd_launch<true, MODE>(p, m, st) : score_fwd_launch<false, MODE>(p, m, st);
  });
}

}  // namespace gptb200

extern "C" int gptb200_score_attention_fwd(const gptb200_score_attention* a, void* stream) {
  const int s = score_check(a);
  return s ? s : score_forward(a, nullptr, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t gptb200_score_attention_bwd_workspace_size(int64_t batch, int64_t heads,
                                                             int64_t seq) {
  if (batch <= 0 || heads <= 0 || seq <= 0) return 0;
  const int64_t rows = batch * heads * seq;
  return (size_t)(2 * ((rows * 4 + 255) / 256 * 256) + rows * HD * 4);
}

extern "C" int gptb200_score_attention_bwd(const gptb200_score_attention* a, const void* dout,
                                           const int64_t* dout_stride, void* dq, void* dk, void* dv,
                                           const int64_t* dq_stride, const int64_t* dkv_stride,
                                           const void* rope_cos, const void* rope_sin,
                                           void* workspace, void* stream) {
  const int s = score_check(a);
  if (s) return s;
  if (!dout || !dout_stride || !dq || !dk || !dv || !dq_stride || !dkv_stride || !workspace)
    return GPTB200_EINVAL;
  if ((rope_cos == nullptr) != (rope_sin == nullptr)) return GPTB200_EINVAL;
  int64_t strides = 0;
  for (int i = 0; i < 3; ++i) strides |= dout_stride[i] | dq_stride[i] | dkv_stride[i];
  if (strides % 8) return GPTB200_ESHAPE;
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return GPTB200_ESHAPE;
  AttnParams p = score_params(a);
  const int64_t rows = a->batch * a->heads * a->seq;
  const int64_t stat_bytes = (rows * 4 + 255) / 256 * 256;
  float* delta = reinterpret_cast<float*>(workspace);
  float* neg_lse2 = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + stat_bytes);
  float* dq_acc = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 2 * stat_bytes);
  ScoreMaps m;
  const int64_t *qs = a->q_stride, *ks = a->kv_stride;
  if (!make_map4(&m.q, a->q, p.B, p.H, p.T, qs[0], qs[1], qs[2], BQ) ||
      !make_map4(&m.k, a->k, p.B, p.KVH, p.T, ks[0], ks[1], ks[2], BT) ||
      !make_map4(&m.v, a->v, p.B, p.KVH, p.T, ks[0], ks[1], ks[2], BT) ||
      !make_map4(&m.g, dout, p.B, p.H, p.T, dout_stride[0], dout_stride[1], dout_stride[2], BQ) ||
      !make_dq_map(&m.dq, dq_acc, p.B * p.H, p.T))
    return GPTB200_ESHAPE;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  // delta = sum dO O from the stored O carries its rounding to bf16 (2^-9 |dO| |O|)
  // into dS = P (dP - delta) of the whole row. Where a row has few keys, one of
  // them tends to hold most of P, dP - delta is small for it and the rounding
  // weighs more. Off by (dq, relative): rows of up to 8 keys 0.0046, 16 0.0041, 33
  // 0.0038, 64 0.0036, 300 0.0035, 1,024 0.0034; with an exact delta 0.0025 at any
  // length. So sequences of one key tile compute O again, in fp32 and into the
  // accumulator that delta's kernel clears (O as stored is not read then): one more
  // launch of one block a tile, 3 us. Longer ones would pay a whole forward (1 x 12 x
  // 8192: 454 us and 259 more), so short documents in them keep the errors above, as
  // they have them in the plain attention.
  const bool short_rows = p.T <= FK;
  if (short_rows) {
    const int f = score_forward(a, dq_acc, st);
    if (f) return f;
  }
  attn_delta_kernel<<<(unsigned)((rows * 8 + 255) / 256), 256, 0, st>>>(
      p.o, reinterpret_cast<const bf16*>(dout), p.osb, p.osh, p.ost, dout_stride[0], dout_stride[1],
      dout_stride[2], p.B, p.H, p.T, delta, dq_acc, a->lse, neg_lse2, short_rows);
  GPTB200_CHECK_LAUNCH();
  const SchedSlot slot(st);
  if (slot.status) return slot.status;
  p.sched = slot.counter;
  p.delta = delta;
  p.neg_lse2 = neg_lse2;
  p.dq_acc = dq_acc;
  p.dk = reinterpret_cast<bf16*>(dk);
  p.dv = reinterpret_cast<bf16*>(dv);
  p.sb = dkv_stride[0];
  p.sh = dkv_stride[1];
  p.st = dkv_stride[2];
  p.rcos = reinterpret_cast<const bf16*>(rope_cos);
  p.rsin = reinterpret_cast<const bf16*>(rope_sin);
  // Q and dO of every head
  p.by_weight = by_weight(rows * 2 * HD * 2, a->softcap > 0.f ? 256 : 64);
  const int e = score_mode(a, [&](auto mode) {
    constexpr int MODE = decltype(mode)::value;
    return p.seg ? score_bwd_launch<true, MODE>(p, m, st) : score_bwd_launch<false, MODE>(p, m, st);
  });
  if (e) return e;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t chunks = rows * (HD / 8);
  const int blocks = (int)std::min<int64_t>((chunks + 255) / 256, (int64_t)sms * 8);
  attn_dq_store_kernel<<<blocks, 256, 0, st>>>(dq_acc, reinterpret_cast<bf16*>(dq), dq_stride[0],
                                               dq_stride[1], dq_stride[2], p.B, p.H, p.T, p.scale,
                                               p.rcos, p.rsin);
  GPTB200_CHECK_LAUNCH();
  return 0;
}
