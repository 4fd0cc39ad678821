// CompleteP AdamW over one flat fp32 parameter buffer (three launches):
//   1. sqnorm_partial : per-block partial sums of grad^2 (fixed grid, deterministic)
//   2. adamw_scalars  : one block -> global grad norm, step+1, learning rate
//                       (warmup + cosine, train.py:1219-1236), bias
//                       corrections, clip scale, history row
//   3. adamw_update   : the element-wise m/v/param update with per-tensor
//                       lr/eps/decay multipliers looked up from the group
//                       table, plus the bf16 compute copy of the new params.
// The step counter lives on the device, so a captured CUDA graph of the whole
// step replays correctly.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace gptb200 {

constexpr int kNormBlocks = 1184;  // 8 x 148
constexpr int kNormThreads = 512;

struct AdamScalars {
  float lr;
  float bc1;
  float bc2;
  float gscale;     // grad_scale * clip scale
  float grad_norm;
  int step;
};

__global__ void __launch_bounds__(kNormThreads) sqnorm_partial_kernel(const float* __restrict__ g,
                                                                      int64_t n,
                                                                      double* __restrict__ part) {
  __shared__ double red[kNormThreads / 32];
  double acc = 0.0;
  float accf = 0.f;
  const int64_t n4 = n >> 2;
  int cnt = 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4;
       i += (int64_t)gridDim.x * blockDim.x) {
    float4 v = reinterpret_cast<const float4*>(g)[i];
    accf += v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
    if (++cnt == 64) {
      acc += accf;
      accf = 0.f;
      cnt = 0;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
    float t = g[(n4 << 2) + threadIdx.x];
    accf += t * t;
  }
  acc += accf;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < kNormThreads / 32; ++w) s += red[w];
    part[blockIdx.x] = s;
  }
}

static __device__ int g_optim_error;

__global__ void adamw_scalars_kernel(const double* __restrict__ part, int nparts,
                                     const gptb200_adamw_config cfg, int32_t* step_io,
                                     const float* loss, float* history, AdamScalars* out) {
  __shared__ double red[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += blockDim.x) s += part[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double tot = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) tot += red[w];
  // Gradients are scaled by grad_scale before the norm (1.0 for the reference step).
  const float gs = cfg.grad_scale;
  const float grad_norm = (float)sqrt(tot) * gs;
  float clip = 1.0f;
  if (cfg.grad_clip > 0.f) clip = fminf(1.0f, cfg.grad_clip / (grad_norm + 1.0e-6f));
  const int step = *step_io + 1;
  const float stepf = (float)step;
  float warm = 1.0f;
  if (cfg.warmup_steps > 0) warm = fminf(1.0f, stepf / (float)cfg.warmup_steps);
  const int span = max(1, cfg.total_steps - cfg.warmup_steps);
  float prog = (stepf - (float)cfg.warmup_steps) / (float)span;
  prog = fminf(fmaxf(prog, 0.0f), 1.0f);
  const float cosine = 0.5f * (1.0f + cosf(3.14159265358979323846f * prog));
  const float mult = cfg.min_lr_ratio + (1.0f - cfg.min_lr_ratio) * cosine;
  const float lr = (cfg.learning_rate * cfg.horizon_lr_scale) * warm * mult;
  AdamScalars a;
  a.lr = lr;
  a.bc1 = 1.0f - powf(cfg.beta1, stepf);
  a.bc2 = 1.0f - powf(cfg.beta2, stepf);
  a.gscale = gs * clip;
  a.grad_norm = grad_norm;
  a.step = step;
  *out = a;
  *step_io = step;
  // A non-finite loss or gradient norm is the reference's FloatingPointError
  // (rig/mesh.py finite_metric); record it for gptb200_device_error().
  if (!isfinite(grad_norm) || (loss && !isfinite(*loss))) g_optim_error = kErrNonFinite;
  if (history && step >= 1 && step <= cfg.total_steps) {
    float* row = history + (int64_t)(step - 1) * 3;
    row[0] = loss ? *loss : 0.f;
    row[1] = lr;
    row[2] = grad_norm;
  }
}

// Finds the tensor group holding element e (offsets increasing); -1 for the
// padding between tensors. `gi` is the caller's cached guess.
__device__ __forceinline__ int find_group(const gptb200_tensor_group* sg, int ngroups, int gi,
                                          int64_t e) {
  if (gi >= 0 && gi < ngroups && e >= sg[gi].offset && e < sg[gi].offset + sg[gi].size) return gi;
  int lo = 0, hi = ngroups - 1, f = -1;
  while (lo <= hi) {
    const int mid = (lo + hi) >> 1;
    if (sg[mid].offset <= e) {
      f = mid;
      lo = mid + 1;
    } else {
      hi = mid - 1;
    }
  }
  return (f < 0 || e >= sg[f].offset + sg[f].size) ? -1 : f;
}

// AdamW on the float4 at element e0 (elements [e0, min(e0 + 4, lim))) of
// tensor group G; returns the sum of squares of the (unscaled) gradients.
__device__ __forceinline__ float adamw_quad(float* __restrict__ p, float* __restrict__ m,
                                            float* __restrict__ v, const float* __restrict__ g,
                                            bf16* __restrict__ pbf, int64_t e0, int64_t lim,
                                            const gptb200_tensor_group& G,
                                            const gptb200_adamw_config& cfg,
                                            const AdamScalars& s) {
  const float b1 = cfg.beta1, b2 = cfg.beta2;
  const float omb1 = 1.0f - b1, omb2 = 1.0f - b2;
  const float lr = s.lr * G.lr_mult;
  const float eps = cfg.eps * cfg.eps_horizon_scale * G.eps_mult;
  const float wd = G.decay ? cfg.weight_decay * cfg.wd_horizon_scale * G.wd_mult : 0.f;
  const int cnt = (int)((lim - e0) < 4 ? (lim - e0) : 4);
  float sq = 0.f;
  if (cnt == 4) {
    const int64_t q = e0 >> 2;
    float4 P = reinterpret_cast<float4*>(p)[q];
    float4 M = reinterpret_cast<float4*>(m)[q];
    float4 V = reinterpret_cast<float4*>(v)[q];
    const float4 Gr = reinterpret_cast<const float4*>(g)[q];
    float* pp = &P.x;
    float* mm = &M.x;
    float* vv = &V.x;
    const float* gg = &Gr.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sq += gg[j] * gg[j];
      const float gr = gg[j] * s.gscale;
      mm[j] = b1 * mm[j] + omb1 * gr;
      vv[j] = b2 * vv[j] + omb2 * (gr * gr);
      const float adam = (mm[j] / s.bc1) / (sqrtf(vv[j] / s.bc2) + eps);
      pp[j] = pp[j] - lr * (adam + wd * pp[j]);
    }
    reinterpret_cast<float4*>(p)[q] = P;
    reinterpret_cast<float4*>(m)[q] = M;
    reinterpret_cast<float4*>(v)[q] = V;
    if (pbf) {
      uint2 o;
      o.x = pack_bf16x2(P.x, P.y);
      o.y = pack_bf16x2(P.z, P.w);
      reinterpret_cast<uint2*>(pbf)[q] = o;
    }
  } else {
    for (int j = 0; j < cnt; ++j) {
      const int64_t e = e0 + j;
      sq += g[e] * g[e];
      const float gr = g[e] * s.gscale;
      const float mj = b1 * m[e] + omb1 * gr;
      const float vj = b2 * v[e] + omb2 * (gr * gr);
      const float adam = (mj / s.bc1) / (sqrtf(vj / s.bc2) + eps);
      const float pj = p[e] - lr * (adam + wd * p[e]);
      m[e] = mj;
      v[e] = vj;
      p[e] = pj;
      if (pbf) pbf[e] = __float2bfloat16(pj);
    }
  }
  return sq;
}

__global__ void __launch_bounds__(256) adamw_update_kernel(
    float* __restrict__ p, float* __restrict__ m, float* __restrict__ v,
    const float* __restrict__ g, int64_t n, const gptb200_tensor_group* __restrict__ groups,
    int ngroups, const gptb200_adamw_config cfg, const AdamScalars* __restrict__ sc,
    bf16* __restrict__ pbf) {
  extern __shared__ gptb200_tensor_group sg[];
  for (int i = threadIdx.x; i < ngroups; i += blockDim.x) sg[i] = groups[i];
  __syncthreads();
  const AdamScalars s = *sc;
  const int64_t n4 = (n + 3) >> 2;
  int gi = 0;
  for (int64_t q = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; q < n4;
       q += (int64_t)gridDim.x * blockDim.x) {
    // Groups start on multiples of 4 elements, so a float4 never straddles two.
    const int64_t e0 = q << 2;
    gi = find_group(sg, ngroups, gi, e0);
    if (gi < 0) {
      gi = 0;
      continue;  // padding between tensors
    }
    const gptb200_tensor_group G = sg[gi];
    adamw_quad(p, m, v, g, pbf, e0, min(n, G.offset + G.size), G, cfg, s);
  }
}

// ------------------------------------------------------------------ bucketed update
// The same update split into ranges that can run as soon as their gradients
// are final (each bucket right after its all-reduce), possible when the step
// does not clip: the learning rate and bias corrections do not depend on the
// global gradient norm then. adamw_begin advances the step and computes the
// scalars; each range's update also stores, per block, the sum of squares of
// its gradients in slot `slot`; adamw_end adds every slot in order (slot,
// block: deterministic) into the logged gradient norm.
constexpr int kRangeBlocks = 1184;  // fixed grid of the ranged update (8 x 148)
constexpr int kMaxSlots = 256;

__global__ void adamw_begin_kernel(const gptb200_adamw_config cfg, int32_t* step_io,
                                   AdamScalars* out) {
  const int step = *step_io + 1;
  const float stepf = (float)step;
  float warm = 1.0f;
  if (cfg.warmup_steps > 0) warm = fminf(1.0f, stepf / (float)cfg.warmup_steps);
  const int span = max(1, cfg.total_steps - cfg.warmup_steps);
  float prog = (stepf - (float)cfg.warmup_steps) / (float)span;
  prog = fminf(fmaxf(prog, 0.0f), 1.0f);
  const float cosine = 0.5f * (1.0f + cosf(3.14159265358979323846f * prog));
  const float mult = cfg.min_lr_ratio + (1.0f - cfg.min_lr_ratio) * cosine;
  AdamScalars a;
  a.lr = (cfg.learning_rate * cfg.horizon_lr_scale) * warm * mult;
  a.bc1 = 1.0f - powf(cfg.beta1, stepf);
  a.bc2 = 1.0f - powf(cfg.beta2, stepf);
  a.gscale = cfg.grad_scale;
  a.grad_norm = 0.f;
  a.step = step;
  *out = a;
  *step_io = step;
}

__global__ void __launch_bounds__(256) adamw_range_kernel(
    float* __restrict__ p, float* __restrict__ m, float* __restrict__ v,
    const float* __restrict__ g, int64_t begin, int64_t end,
    const gptb200_tensor_group* __restrict__ groups, int ngroups, const gptb200_adamw_config cfg,
    const AdamScalars* __restrict__ sc, bf16* __restrict__ pbf, double* __restrict__ part) {
  extern __shared__ gptb200_tensor_group sg[];
  __shared__ double red[8];
  for (int i = threadIdx.x; i < ngroups; i += blockDim.x) sg[i] = groups[i];
  __syncthreads();
  const AdamScalars s = *sc;
  double acc = 0.0;
  float accf = 0.f;
  int cnt = 0, gi = 0;
  for (int64_t q = (begin >> 2) + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; (q << 2) < end;
       q += (int64_t)gridDim.x * blockDim.x) {
    const int64_t e0 = q << 2;
    gi = find_group(sg, ngroups, gi, e0);
    if (gi < 0) {
      gi = 0;
      continue;
    }
    const gptb200_tensor_group G = sg[gi];
    accf += adamw_quad(p, m, v, g, pbf, e0, min(end, G.offset + G.size), G, cfg, s);
    if (++cnt == 64) {
      acc += accf;
      accf = 0.f;
      cnt = 0;
    }
  }
  acc += accf;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += red[w];
    part[blockIdx.x] = t;
  }
}

__global__ void __launch_bounds__(1024) adamw_end_kernel(const double* __restrict__ part,
                                                         int nparts, const int32_t* step_io,
                                                         const gptb200_adamw_config cfg,
                                                         const float* loss, float* history) {
  __shared__ double red[32];
  // fixed association: thread t adds parts t, t + 1024, ...; then warps, then the 32 sums
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += blockDim.x) s += part[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double tot = 0.0;
  for (int w = 0; w < 32; ++w) tot += red[w];
  const float grad_norm = (float)sqrt(tot) * cfg.grad_scale;
  const int step = *step_io;
  if (history && step >= 1 && step <= cfg.total_steps) {
    float* row = history + (int64_t)(step - 1) * 3;
    row[0] = loss ? *loss : 0.f;
    // the learning rate of this step, recomputed as adamw_begin did
    const float stepf = (float)step;
    float warm = 1.0f;
    if (cfg.warmup_steps > 0) warm = fminf(1.0f, stepf / (float)cfg.warmup_steps);
    const int span = max(1, cfg.total_steps - cfg.warmup_steps);
    float prog = (stepf - (float)cfg.warmup_steps) / (float)span;
    prog = fminf(fmaxf(prog, 0.0f), 1.0f);
    const float cosine = 0.5f * (1.0f + cosf(3.14159265358979323846f * prog));
    row[1] = (cfg.learning_rate * cfg.horizon_lr_scale) * warm *
             (cfg.min_lr_ratio + (1.0f - cfg.min_lr_ratio) * cosine);
    row[2] = grad_norm;
  }
  if (!isfinite(grad_norm) || (loss && !isfinite(*loss))) g_optim_error = kErrNonFinite;
}

// ------------------------------------------------------------------ 8-bit moments
// The same update with both moments in 8 bits. 64 consecutive elements (a
// block) share one exponent byte E per moment, the largest magnitude's; a
// magnitude code holds its exponent relative to E in 4 bits and the mantissa's
// leading bits below it:
//   m: sign, 4 exponent bits, 3 mantissa bits;  r = sqrt(v): 4 + 4 bits,
//   value = 2^(E - 127 - 15 + exponent) (1 + mantissa / 8 or / 16), code 0 = 0,
//   E = 255 marks a block that held a NaN or an infinity (it decodes to NaN).
// Floating codes, because the update is m / r element by element: with a step
// size common to a block, elements far below its largest would get moments off
// by many times their size. r and not v, because r's range is half as wide and
// r is what the update divides by. An m below the range becomes 0 and an r
// below it the smallest code, so rounding never enlarges |m / r| without bound.
// The bits below a code are rounded by adding random bits and cutting: with
// beta2 = 0.95 an r whose gradients vanish falls by 2.5% a step, less than half
// a unit of the code, and rounding to nearest would hold it up for ever. The
// random bits are a hash of (seed, step, element), so a step is a function of
// its inputs. Moments enter the update unrounded; every operation up to the
// codes is rounded by itself (no contraction), so that a restatement with
// separate operations yields the same codes.
// Parameters, gradient, codes and the bf16 copy move 18.06 bytes per parameter,
// where fp32 moments need 30: 344 us of HBM at 124.7 M parameters, of 507 measured
// (685 with fp32 moments). The instructions (below) take 375 us at every issue slot; a
// pass's loads stand at its head, so memory and issue wait for each other in part.
constexpr int kQBlock = 64;

// The finalizer of MurmurHash3 (32 bits; Appleby, public domain).
__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}
// 32 random bits of element e: mix32(e * 0x9E3779B1 + (e >> 32) * 0x85EBCA77 + key).

// Magnitude of a code with M mantissa bits under block exponent E < 255, given
// `bits`, the code shifted to the mantissa's top.
template <int M>
__device__ __forceinline__ float q8_decode(uint32_t bits, int E) {
  return bits == 0 ? 0.f : __uint_as_float(bits + ((uint32_t)(E - 15) << 23));
}
// Block exponent for a largest magnitude with these bits: the one above if the
// top code would not reach it. At least 16, so that the smallest code is a
// normal number.
template <int M>
__device__ __forceinline__ int q8_exponent(uint32_t top_bits) {
  const int e = (int)((top_bits + ((1u << (23 - M)) - 1u)) >> 23);
  return e >= 255 ? 255 : max(e, 16);
}
// Code of a magnitude's bits; at least `low`. Below 16 << M without a test, as
// q8_exponent leaves room for any dither below a unit (and where it could not,
// in a block with E = 255, codes do not matter).
template <int M>
__device__ __forceinline__ uint32_t q8_encode(uint32_t bits, uint32_t dither, int E, int low) {
  return (uint32_t)max((int)(bits + dither - ((uint32_t)(E - 15) << 23)) >> (23 - M), low);
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t bytes4(const uint32_t* c) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// Eight lanes share a block, eight elements each: what a lane does once (group
// lookup, addresses, exponents, shuffles) is spread over eight updates, since
// the arithmetic, 106 instructions an element, half of them integer, fills three
// quarters of the issue slots of the whole run. The quotient m / r is the only
// operation that is not rounded to nearest (its error, 2^-22 of the update, is
// far below half a unit of the parameter).
constexpr int kQLane = 8;

// The group whose elements a lane's quad belongs to, and its multipliers.
struct QuadGroup {
  int64_t lo, hi;  // elements [lo, hi)
  float lr, eps, wd;
};

// Four blocks of 256 threads on an SM (64 registers): 507 us at 124.7 M parameters,
// 4.4 TB/s; three blocks (80) and five (48, with spills) take 530 both.
__global__ void __launch_bounds__(256, 4) adamw8_kernel(
    float* __restrict__ p, uint8_t* __restrict__ mq, uint8_t* __restrict__ me,
    uint8_t* __restrict__ vq, uint8_t* __restrict__ ve, const float* __restrict__ g, int64_t begin,
    int64_t end, const gptb200_tensor_group* __restrict__ groups, int ngroups,
    const gptb200_adamw_config cfg, const AdamScalars* __restrict__ sc, uint32_t seed,
    bf16* __restrict__ pbf, double* __restrict__ part) {
  extern __shared__ gptb200_tensor_group sg[];
  __shared__ double red[8];
  for (int i = threadIdx.x; i < ngroups; i += blockDim.x) sg[i] = groups[i];
  __syncthreads();
  const AdamScalars s = *sc;
  const uint32_t key = mix32(mix32((uint32_t)s.step) ^ seed);
  const float b1 = cfg.beta1, b2 = cfg.beta2;
  const float omb1 = 1.0f - b1, omb2 = 1.0f - b2;
  const float inv1 = 1.0f / s.bc1, inv2 = 1.0f / sqrtf(s.bc2);
  double acc = 0.0;
  float accf = 0.f;
  int cnt = 0;
  QuadGroup q = {0, 0, 0.f, 0.f, 0.f};  // of the last element looked up
  int gi = 0;
  auto look_up = [&](int64_t e) {  // the elements of q from e on, at most 4
    if (e < q.lo || e >= q.hi) {
      gi = e < end ? find_group(sg, ngroups, gi, e) : -1;
      if (gi < 0) {  // padding between tensors, or past the end
        gi = 0;
        return 0;
      }
      const gptb200_tensor_group& G = sg[gi];
      q.lo = G.offset;
      q.hi = min(end, G.offset + G.size);
      q.lr = s.lr * G.lr_mult;
      q.eps = cfg.eps * cfg.eps_horizon_scale * G.eps_mult;
      q.wd = G.decay ? cfg.weight_decay * cfg.wd_horizon_scale * G.wd_mult : 0.f;
    }
    return (int)min((int64_t)4, q.hi - e);
  };
  // Elements e0..e0 + 7, of which n0 of the first four and n1 of the others are live.
  auto update = [&](int64_t e0, int n0, int n1, const QuadGroup& ga, const QuadGroup& gb,
                    auto whole) {
    const bool all = decltype(whole)::value || n0 + n1 == 8;
    const bool any = decltype(whole)::value || n0 + n1 > 0;
    float P[8], Gr[8];
    uint32_t mc[2] = {0, 0}, vc[2] = {0, 0};
    int em = 16, ev = 16;
    if (all) {
      const float4 a0 = *reinterpret_cast<const float4*>(p + e0);
      const float4 a1 = *reinterpret_cast<const float4*>(p + e0 + 4);
      const float4 g0 = *reinterpret_cast<const float4*>(g + e0);
      const float4 g1 = *reinterpret_cast<const float4*>(g + e0 + 4);
      P[0] = a0.x, P[1] = a0.y, P[2] = a0.z, P[3] = a0.w;
      P[4] = a1.x, P[5] = a1.y, P[6] = a1.z, P[7] = a1.w;
      Gr[0] = g0.x, Gr[1] = g0.y, Gr[2] = g0.z, Gr[3] = g0.w;
      Gr[4] = g1.x, Gr[5] = g1.y, Gr[6] = g1.z, Gr[7] = g1.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = (j & 3) < (j < 4 ? n0 : n1);
        P[j] = in ? p[e0 + j] : 0.f;
        Gr[j] = in ? g[e0 + j] : 0.f;
      }
    }
    if (any) {
      const uint2 a = *reinterpret_cast<const uint2*>(mq + e0);
      const uint2 b = *reinterpret_cast<const uint2*>(vq + e0);
      mc[0] = a.x, mc[1] = a.y, vc[0] = b.x, vc[1] = b.y;
      em = me[e0 / kQBlock];
      ev = ve[e0 / kQBlock];
    }
    // a block that held a NaN or an infinity stays NaN
    const float b1n = em == 255 ? __int_as_float(0x7fffffff) : b1;
    const float b2n = ev == 255 ? __int_as_float(0x7fffffff) : b2;
    em = min(em, 254);
    ev = min(ev, 254);
    float M[8], R[8];
    uint32_t mtop = 0, vtop = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int w = j >> 2, sh = 8 * (j & 3);
      accf += Gr[j] * Gr[j];
      const float gr = __fmul_rn(Gr[j], s.gscale);
      // code (and its sign) to the top of the mantissa
      const uint32_t mb = sh < 20 ? mc[w] << (20 - sh) : mc[w] >> (sh - 20);
      const uint32_t vb = sh < 19 ? vc[w] << (19 - sh) : vc[w] >> (sh - 19);
      const float mag = q8_decode<3>(mb & 0x07f00000u, em);
      const float r = q8_decode<4>(vb & 0x07f80000u, ev);
      const float m0 = __uint_as_float(__float_as_uint(mag) ^ (mb << 4 & 0x80000000u));
      M[j] = __fadd_rn(__fmul_rn(b1n, m0), __fmul_rn(omb1, gr));
      R[j] = __fsqrt_rn(
          __fadd_rn(__fmul_rn(b2n, __fmul_rn(r, r)), __fmul_rn(omb2, __fmul_rn(gr, gr))));
      if (!all && (j & 3) >= (j < 4 ? n0 : n1)) M[j] = R[j] = 0.f;
      mtop = max(mtop, __float_as_uint(M[j]) & 0x7fffffffu);
      vtop = max(vtop, __float_as_uint(R[j]));  // >= 0 or NaN
      const QuadGroup& G = j < 4 ? ga : gb;
      const float adam = __fdividef(M[j] * inv1, R[j] * inv2 + G.eps);
      P[j] = P[j] - G.lr * (adam + G.wd * P[j]);
    }
    if (all) {
      *reinterpret_cast<float4*>(p + e0) = make_float4(P[0], P[1], P[2], P[3]);
      *reinterpret_cast<float4*>(p + e0 + 4) = make_float4(P[4], P[5], P[6], P[7]);
      if (pbf) {
        *reinterpret_cast<uint2*>(pbf + e0) =
            make_uint2(pack_bf16x2(P[0], P[1]), pack_bf16x2(P[2], P[3]));
        *reinterpret_cast<uint2*>(pbf + e0 + 4) =
            make_uint2(pack_bf16x2(P[4], P[5]), pack_bf16x2(P[6], P[7]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if ((j & 3) < (j < 4 ? n0 : n1)) {
          p[e0 + j] = P[j];
          if (pbf) pbf[e0 + j] = __float2bfloat16(P[j]);
        }
      }
    }
    // the block's exponents: the eight lanes' largest magnitudes (as integers, so
    // that a NaN or an infinity is larger than every number)
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      mtop = max(mtop, __shfl_xor_sync(0xffffffffu, mtop, o));
      vtop = max(vtop, __shfl_xor_sync(0xffffffffu, vtop, o));
    }
    em = q8_exponent<3>(mtop);
    ev = q8_exponent<4>(vtop);
    const uint32_t h0 =
        (uint32_t)e0 * 0x9E3779B1u + (uint32_t)(e0 >> 32) * 0x85EBCA77u + key;  // e0 + j: no carry
    uint32_t bm[8], bv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = mix32(h0 + (uint32_t)j * 0x9E3779B1u);
      const uint32_t mb = __float_as_uint(M[j]), rb = __float_as_uint(R[j]);
      const uint32_t c = q8_encode<3>(mb & 0x7fffffffu, h >> 12 & 0xffff0u, em, 0);
      bm[j] = c | ((c + 127u) & (mb >> 24) & 0x80u);  // the sign of a code that is not 0
      bv[j] = q8_encode<4>(rb, h << 3 & 0x7fff8u, ev, (int)min(rb, 1u));
    }
    const uint32_t cm[2] = {bytes4(bm), bytes4(bm + 4)}, cv[2] = {bytes4(bv), bytes4(bv + 4)};
    // Codes are written wherever an element of the quad is live; dead quads of a
    // live block belong to no tensor and stay as they are.
    if (all) {
      *reinterpret_cast<uint2*>(mq + e0) = make_uint2(cm[0], cm[1]);
      *reinterpret_cast<uint2*>(vq + e0) = make_uint2(cv[0], cv[1]);
    } else {
      if (n0) {
        *reinterpret_cast<uint32_t*>(mq + e0) = cm[0];
        *reinterpret_cast<uint32_t*>(vq + e0) = cv[0];
      }
      if (n1) {
        *reinterpret_cast<uint32_t*>(mq + e0 + 4) = cm[1];
        *reinterpret_cast<uint32_t*>(vq + e0 + 4) = cv[1];
      }
    }
    // one lane of each block writes its exponents: the first that holds a tensor's element
    const unsigned holds = __ballot_sync(0xffffffffu, any) >> (threadIdx.x & 24) & 0xff;
    if (any && (threadIdx.x & 7) == __ffs(holds) - 1) {
      me[e0 / kQBlock] = (uint8_t)em;
      ve[e0 / kQBlock] = (uint8_t)ev;
    }
  };
  const int64_t stride = (int64_t)gridDim.x * blockDim.x * kQLane;
  const int64_t stop = (end + kQBlock - 1) / kQBlock * kQBlock;  // whole blocks: shuffles below
  for (int64_t e0 = begin + ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * kQLane;
       e0 - kQLane * (threadIdx.x & 31) < stop; e0 += stride) {
    // One group holds all eight elements of every lane, mostly: then without the
    // tests that a tensor's end needs (issued, predicated off, in every pass).
    if (__all_sync(0xffffffffu, e0 >= q.lo && e0 + kQLane <= q.hi))
      update(e0, 4, 4, q, q, std::true_type());
    else {
      const int n0 = look_up(e0);
      const QuadGroup qa = q;
      const int n1 = look_up(e0 + 4);
      update(e0, n0, n1, qa, q, std::false_type());
    }
    if (++cnt == 8) {
      acc += accf;
      accf = 0.f;
      cnt = 0;
    }
  }
  if (!part) return;
  acc += accf;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += red[w];
    part[blockIdx.x] = t;
    for (int b = blockIdx.x + gridDim.x; b < kRangeBlocks; b += gridDim.x) part[b] = 0.0;
  }
}

// The values that codes stand for (each fits bf16 exactly).
__global__ void __launch_bounds__(256) adamw8_values_kernel(
    const uint8_t* __restrict__ mq, const uint8_t* __restrict__ me,
    const uint8_t* __restrict__ vq, const uint8_t* __restrict__ ve, int64_t n,
    bf16* __restrict__ m, bf16* __restrict__ r) {
  for (int64_t e = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; e < n;
       e += (int64_t)gridDim.x * blockDim.x * 8) {
    const uint2 mc = *reinterpret_cast<const uint2*>(mq + e);
    const uint2 vc = *reinterpret_cast<const uint2*>(vq + e);
    const int em = me[e / kQBlock], ev = ve[e / kQBlock];
    // NaN blocks: one factor for the whole lane
    const float fm = em == 255 ? __int_as_float(0x7fffffff) : 1.f;
    const float fv = ev == 255 ? __int_as_float(0x7fffffff) : 1.f;
    const int emc = min(em, 254), evc = min(ev, 254);
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int sh = 8 * (j & 3);
      const uint32_t mw = j < 4 ? mc.x : mc.y, vw = j < 4 ? vc.x : vc.y;
      const uint32_t mb = sh < 20 ? mw << (20 - sh) : mw >> (sh - 20);
      const uint32_t vb = sh < 19 ? vw << (19 - sh) : vw >> (sh - 19);
      const float mag = q8_decode<3>(mb & 0x07f00000u, emc);
      a[j] = fm * __uint_as_float(__float_as_uint(mag) ^ (mb << 4 & 0x80000000u));
      b[j] = fv * q8_decode<4>(vb & 0x07f80000u, evc);
    }
    *reinterpret_cast<uint4*>(m + e) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]),
                                                  pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
    *reinterpret_cast<uint4*>(r + e) = make_uint4(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]),
                                                  pack_bf16x2(b[4], b[5]), pack_bf16x2(b[6], b[7]));
  }
}

}  // namespace gptb200

using namespace gptb200;

// Workspace: [kNormBlocks] doubles of the one-shot norm, the AdamScalars
// (256 bytes), then kMaxSlots x kRangeBlocks doubles of the ranged update.
constexpr size_t kScalarsOffset = kNormBlocks * sizeof(double);
constexpr size_t kSlotsOffset = kScalarsOffset + 256;

extern "C" size_t gptb200_adamw_workspace_size(int64_t n) {
  (void)n;
  return kSlotsOffset + (size_t)kMaxSlots * kRangeBlocks * sizeof(double);
}

extern "C" int gptb200_adamw_step(float* params, float* m, float* v, const float* grads, int64_t n,
                                  const gptb200_tensor_group* groups, int32_t n_groups,
                                  const gptb200_adamw_config* cfg, int32_t* step, const float* loss,
                                  float* history, void* params_bf16, void* workspace,
                                  void* stream) {
  if (!params || !m || !v || !grads || !groups || !cfg || !step || !workspace || n <= 0 ||
      n_groups <= 0)
    return GPTB200_EINVAL;
  if (n_groups > 4096) return GPTB200_EUNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(params) | reinterpret_cast<uintptr_t>(m) |
        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(grads) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (params_bf16 && (reinterpret_cast<uintptr_t>(params_bf16) & 7)))
    return GPTB200_ESHAPE;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  double* part = reinterpret_cast<double*>(workspace);
  AdamScalars* sc = reinterpret_cast<AdamScalars*>(reinterpret_cast<char*>(workspace) +
                                                   kScalarsOffset);
  sqnorm_partial_kernel<<<kNormBlocks, kNormThreads, 0, st>>>(grads, n, part);
  GPTB200_CHECK_LAUNCH();
  adamw_scalars_kernel<<<1, 1024, 0, st>>>(part, kNormBlocks, *cfg, step, loss, history, sc);
  GPTB200_CHECK_LAUNCH();
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int64_t n4 = (n + 3) / 4;
  int blocks = (int)std::min<int64_t>((n4 + 255) / 256, (int64_t)sms * 8);
  size_t smem = (size_t)n_groups * sizeof(gptb200_tensor_group);
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(adamw_update_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
  }
  adamw_update_kernel<<<blocks, 256, smem, st>>>(params, m, v, grads, n, groups, n_groups, *cfg, sc,
                                                 reinterpret_cast<bf16*>(params_bf16));
  GPTB200_CHECK_LAUNCH();
  return 0;
}

namespace gptb200 {
int optim_read_error(int clear) {
  int h = 0;
  cudaMemcpyFromSymbol(&h, g_optim_error, sizeof(int));
  if (clear) {
    int z = 0;
    cudaMemcpyToSymbol(g_optim_error, &z, sizeof(int));
  }
  return h;
}
}  // namespace gptb200

extern "C" int gptb200_adamw_begin(const gptb200_adamw_config* cfg, int32_t* step, void* workspace,
                                   void* stream) {
  if (!cfg || !step || !workspace) return GPTB200_EINVAL;
  if (cfg->grad_clip > 0.f) return GPTB200_EUNSUPPORTED;  // clipping needs the norm first
  auto sc = reinterpret_cast<AdamScalars*>(reinterpret_cast<char*>(workspace) + kScalarsOffset);
  adamw_begin_kernel<<<1, 1, 0, reinterpret_cast<cudaStream_t>(stream)>>>(*cfg, step, sc);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

extern "C" int gptb200_adamw_update_range(float* params, float* m, float* v, const float* grads,
                                          int64_t begin, int64_t end,
                                          const gptb200_tensor_group* groups, int32_t n_groups,
                                          const gptb200_adamw_config* cfg, int32_t slot,
                                          void* params_bf16, void* workspace, void* stream) {
  if (!params || !m || !v || !grads || !groups || !cfg || !workspace || n_groups <= 0)
    return GPTB200_EINVAL;
  if (begin < 0 || end <= begin || (begin & 3) || slot < 0 || slot >= kMaxSlots)
    return GPTB200_EINVAL;
  if (n_groups > 4096 || cfg->grad_clip > 0.f) return GPTB200_EUNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(params) | reinterpret_cast<uintptr_t>(m) |
        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(grads) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (params_bf16 && (reinterpret_cast<uintptr_t>(params_bf16) & 7)))
    return GPTB200_ESHAPE;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  auto sc = reinterpret_cast<const AdamScalars*>(ws + kScalarsOffset);
  auto part = reinterpret_cast<double*>(ws + kSlotsOffset) + (int64_t)slot * kRangeBlocks;
  size_t smem = (size_t)n_groups * sizeof(gptb200_tensor_group);
  if (smem > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(adamw_range_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
  }
  adamw_range_kernel<<<kRangeBlocks, 256, smem, st>>>(params, m, v, grads, begin, end, groups,
                                                      n_groups, *cfg, sc,
                                                      reinterpret_cast<bf16*>(params_bf16), part);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

extern "C" int gptb200_adamw_end(int32_t n_slots, const gptb200_adamw_config* cfg,
                                 const int32_t* step, const float* loss, float* history,
                                 void* workspace, void* stream) {
  if (!cfg || !step || !workspace || n_slots <= 0 || n_slots > kMaxSlots) return GPTB200_EINVAL;
  auto part = reinterpret_cast<const double*>(reinterpret_cast<char*>(workspace) + kSlotsOffset);
  adamw_end_kernel<<<1, 1024, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      part, n_slots * kRangeBlocks, step, *cfg, loss, history);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

// ------------------------------------------------------------------ 8-bit moments (entry points)
static int adamw8_check(const gptb200_adamw8_state* state, const void* params, const void* grads,
                        const gptb200_tensor_group* groups, int32_t n_groups,
                        const gptb200_adamw_config* cfg, const void* params_bf16,
                        const void* workspace) {
  if (!state || !state->m || !state->m_exp || !state->v || !state->v_exp || !params || !grads ||
      !groups || !cfg || !workspace || n_groups <= 0)
    return GPTB200_EINVAL;
  if (n_groups > 4096) return GPTB200_EUNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(params) | reinterpret_cast<uintptr_t>(grads) |
        reinterpret_cast<uintptr_t>(state->m) | reinterpret_cast<uintptr_t>(state->v) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (params_bf16 && (reinterpret_cast<uintptr_t>(params_bf16) & 7)))
    return GPTB200_ESHAPE;
  return 0;
}

// Updates elements [begin, end); part: kRangeBlocks sums of squared gradients, or null.
static int adamw8_launch(float* params, const gptb200_adamw8_state& q, const float* grads,
                         int64_t begin, int64_t end, const gptb200_tensor_group* groups,
                         int32_t n_groups, const gptb200_adamw_config& cfg, const AdamScalars* sc,
                         uint32_t seed, void* params_bf16, double* part, cudaStream_t st) {
  const size_t smem = (size_t)n_groups * sizeof(gptb200_tensor_group);
  if (smem > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(adamw8_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -static_cast<int>(e);
  }
  const int64_t wanted = (end - begin + 256 * kQLane - 1) / (256 * kQLane);
  const int blocks = (int)std::min<int64_t>(wanted, kRangeBlocks);
  adamw8_kernel<<<blocks, 256, smem, st>>>(
      params, q.m, q.m_exp, q.v, q.v_exp, grads, begin, end, groups, n_groups, cfg, sc, seed,
      reinterpret_cast<bf16*>(params_bf16), part);
  GPTB200_CHECK_LAUNCH();
  return 0;
}

extern "C" int gptb200_adamw8_step(float* params, const gptb200_adamw8_state* state,
                                   const float* grads, int64_t n,
                                   const gptb200_tensor_group* groups, int32_t n_groups,
                                   const gptb200_adamw_config* cfg, int32_t* step,
                                   const float* loss, float* history, void* params_bf16,
                                   uint32_t seed, void* workspace, void* stream) {
  const int s = adamw8_check(state, params, grads, groups, n_groups, cfg, params_bf16, workspace);
  if (s) return s;
  if (!step || n <= 0) return GPTB200_EINVAL;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  AdamScalars* sc = reinterpret_cast<AdamScalars*>(ws + kScalarsOffset);
  if (cfg->grad_clip > 0.f) {  // clipping needs the global norm first
    double* part = reinterpret_cast<double*>(ws);
    sqnorm_partial_kernel<<<kNormBlocks, kNormThreads, 0, st>>>(grads, n, part);
    GPTB200_CHECK_LAUNCH();
    adamw_scalars_kernel<<<1, 1024, 0, st>>>(part, kNormBlocks, *cfg, step, loss, history, sc);
    GPTB200_CHECK_LAUNCH();
    return adamw8_launch(params, *state, grads, 0, n, groups, n_groups, *cfg, sc, seed,
                         params_bf16, nullptr, st);
  }
  // without clipping the gradients are read once: the update also sums their squares
  int e = gptb200_adamw_begin(cfg, step, workspace, stream);
  if (e) return e;
  e = adamw8_launch(params, *state, grads, 0, n, groups, n_groups, *cfg, sc, seed, params_bf16,
                    reinterpret_cast<double*>(ws + kSlotsOffset), st);
  if (e) return e;
  return gptb200_adamw_end(1, cfg, step, loss, history, workspace, stream);
}

extern "C" int gptb200_adamw8_update_range(float* params, const gptb200_adamw8_state* state,
                                           const float* grads, int64_t begin, int64_t end,
                                           const gptb200_tensor_group* groups, int32_t n_groups,
                                           const gptb200_adamw_config* cfg, int32_t slot,
                                           void* params_bf16, uint32_t seed, void* workspace,
                                           void* stream) {
  const int s = adamw8_check(state, params, grads, groups, n_groups, cfg, params_bf16, workspace);
  if (s) return s;
  if (begin < 0 || end <= begin || begin % kQBlock || end % kQBlock || slot < 0 ||
      slot >= kMaxSlots)
    return GPTB200_EINVAL;
  if (cfg->grad_clip > 0.f) return GPTB200_EUNSUPPORTED;
  char* ws = reinterpret_cast<char*>(workspace);
  return adamw8_launch(params, *state, grads, begin, end, groups, n_groups, *cfg,
                       reinterpret_cast<const AdamScalars*>(ws + kScalarsOffset), seed,
                       params_bf16,
                       reinterpret_cast<double*>(ws + kSlotsOffset) + (int64_t)slot * kRangeBlocks,
                       reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int gptb200_adamw8_values(const gptb200_adamw8_state* state, int64_t n, void* m,
                                     void* v_root, void* stream) {
  if (!state || !state->m || !state->m_exp || !state->v || !state->v_exp || !m || !v_root ||
      n <= 0)
    return GPTB200_EINVAL;
  if (n % kQBlock || ((reinterpret_cast<uintptr_t>(state->m) | reinterpret_cast<uintptr_t>(state->v) |
                       reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v_root)) & 15))
    return GPTB200_ESHAPE;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int blocks = (int)std::min<int64_t>((n / 8 + 255) / 256, (int64_t)sms * 8);
  adamw8_values_kernel<<<blocks, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      state->m, state->m_exp, state->v, state->v_exp, n, reinterpret_cast<bf16*>(m),
      reinterpret_cast<bf16*>(v_root));
  GPTB200_CHECK_LAUNCH();
  return 0;
}
