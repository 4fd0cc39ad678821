// Layer norm, forward and backward.
//
//   y  = (x - mean) rstd scale + bias,   rstd = 1 / sqrt(var + eps)
//   dn = dy scale, hat = (x - mean) rstd
//   dx = rstd (dn - mean(dn) - hat mean(dn hat))  (+ dx_in, the residual stream's gradient)
//   dscale += sum dy hat, dbias += sum dy, dx_colsum += alpha sum dx   (sums over the rows)
//
// Both passes are bound by HBM: the row stays in registers between the
// statistics and the output, so x is read once in the forward and x, dy, dx_in
// once in the backward. W warps share a row (W grows with the width so that a
// lane keeps at most four 8-element chunks), the next row's loads are issued
// before this row's reductions, and the three column sums of the backward live
// in the lanes' registers over the whole grid-stride loop: a lane owns the same
// columns of every row. Each block then writes one row of partials and a second
// launch adds the partials in a fixed order, so results repeat bit for bit.
// Statistics are fp32 and the variance is taken about the mean, not from
// sum(x^2): rows far from zero lose nothing. Outputs are rounded once.
#include <algorithm>

#include "common.cuh"

namespace gptb200 {

constexpr int kLnMaxWidth = 16384;
// Rows a block of one-warp rows works on at a time. The backward's lanes hold
// three column sums, so its blocks are one to an SM and as wide as registers allow.
constexpr int kLnRows = 8, kLnBwdRows = 8;

// VEC elements as loaded. stay(): keeps a loop from holding the elements of a
// loop-invariant vector unpacked, at twice the registers.
template <typename T, int VEC>
struct LnRaw;
template <>
struct LnRaw<bf16, 8> {
  uint4 q;
  GPTB200_DEV void load(const bf16* p) { q = *reinterpret_cast<const uint4*>(p); }
  GPTB200_DEV void zero() { q = make_uint4(0, 0, 0, 0); }
  GPTB200_DEV void stay() { asm volatile("" : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w)); }
  GPTB200_DEV void get(float* v) const {
    unpack_bf16x2(q.x, v[0], v[1]);
    unpack_bf16x2(q.y, v[2], v[3]);
    unpack_bf16x2(q.z, v[4], v[5]);
    unpack_bf16x2(q.w, v[6], v[7]);
  }
  static GPTB200_DEV void store(bf16* p, const float* v) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                   pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct LnRaw<float, 8> {
  float4 a, b;
  GPTB200_DEV void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  GPTB200_DEV void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  GPTB200_DEV void stay() {}
  GPTB200_DEV void get(float* v) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static GPTB200_DEV void store(float* p, const float* v) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <>
struct LnRaw<bf16, 1> {
  bf16 q;
  GPTB200_DEV void load(const bf16* p) { q = *p; }
  GPTB200_DEV void zero() { q = __float2bfloat16(0.f); }
  GPTB200_DEV void stay() {}
  GPTB200_DEV void get(float* v) const { v[0] = __bfloat162float(q); }
  static GPTB200_DEV void store(bf16* p, const float* v) { *p = __float2bfloat16(v[0]); }
};
template <>
struct LnRaw<float, 1> {
  float q;
  GPTB200_DEV void load(const float* p) { q = *p; }
  GPTB200_DEV void zero() { q = 0.f; }
  GPTB200_DEV void stay() {}
  GPTB200_DEV void get(float* v) const { v[0] = q; }
  static GPTB200_DEV void store(float* p, const float* v) { *p = v[0]; }
};

// Sums of a and b over the W warps of a row, in every thread. With W > 1 the
// block is one row's group; `red` has two halves that calls use in turn, so one
// barrier a call suffices (a half is written again only after every thread has
// passed the other half's barrier, hence has read this one).
template <int W>
GPTB200_DEV void ln_row_sums(float& a, float& b, float2 (*red)[W], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += red[turn][w].x;
      b += red[turn][w].y;
    }
    turn ^= 1;
  }
}

struct LnSums {  // the backward's column sums: scale, bias, columns of dx
  float* out[3];
  float alpha[3];
};

struct LnParams {
  const void *x, *scale, *bias, *dy, *dx_in;
  void *y, *dx_out;
  float *mean, *rstd, *part;
  int64_t rows, ldx, ldy, lddx;  // ldy: of y (forward) or dy (backward)
  int d;
  float eps;
  LnSums to;
};

constexpr int ln_rows_per_block(int w, bool bwd) { return w > 1 ? 1 : bwd ? kLnBwdRows : kLnRows; }
constexpr int ln_threads(int w, bool bwd) { return 32 * w * ln_rows_per_block(w, bwd); }

template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(ln_threads(W, false)) ln_fwd_kernel(const LnParams p) {
  constexpr bool AHEAD = true, BWD = false;
  using Raw = LnRaw<T, VEC>;
  __shared__ float2 red[2][W];
  int turn = 0;
  const int g = W == 1 ? threadIdx.x >> 5 : 0;
  const int t = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * ln_rows_per_block(W, BWD);
  const T* x = reinterpret_cast<const T*>(p.x);
  T* y = reinterpret_cast<T*>(p.y);
  auto col = [&](int i) { return (i * 32 * W + t) * VEC; };
  auto fetch = [&](Raw* to, int64_t r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      to[i].zero();
      if (col(i) < p.d) to[i].load(x + r * p.ldx + col(i));
    }
  };
  Raw w[NV], c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    w[i].zero();
    c[i].zero();
    if (col(i) < p.d) {
      w[i].load(reinterpret_cast<const T*>(p.scale) + col(i));
      if (p.bias) c[i].load(reinterpret_cast<const T*>(p.bias) + col(i));
    }
  }
  const float inv_d = 1.f / (float)p.d;
  Raw now[NV], next[NV];
  int64_t r = (int64_t)blockIdx.x * ln_rows_per_block(W, BWD) + g;
  if (r < p.rows) fetch(now, r);
  for (; r < p.rows; r += step) {
    if constexpr (AHEAD) {
      if (r + step < p.rows) fetch(next, r + step);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      w[i].stay();
      c[i].stay();
    }
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[VEC];
      now[i].get(v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += v[j];
    }
    ln_row_sums<W>(sum, none, red, turn);
    const float mean = sum * inv_d;
    float var = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[VEC];
      now[i].get(v);
      if (col(i) < p.d) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) var = fmaf(v[j] - mean, v[j] - mean, var);
      }
    }
    ln_row_sums<W>(var, none, red, turn);
    const float rstd = rsqrtf(var * inv_d + p.eps);
    if (t == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
        float v[VEC], a[VEC], b[VEC];
        now[i].get(v);
        w[i].get(a);
        c[i].get(b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = fmaf((v[j] - mean) * rstd, a[j], b[j]);
        Raw::store(y + r * p.ldy + col(i), v);
      }
    }
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < NV; ++i) now[i] = next[i];
    } else {
      if (r + step < p.rows) fetch(now, r + step);
    }
  }
}

// RES: dx_in is added. COL: the column sums of dx are wanted too.
template <typename T, int VEC, int W, int NV, bool RES, bool COL>
__global__ void __launch_bounds__(ln_threads(W, true)) ln_bwd_kernel(const LnParams p) {
  using Raw = LnRaw<T, VEC>;
  // 32-bit rows have twice the bytes in flight already
  constexpr bool AHEAD = sizeof(T) == 2, BWD = true;
  __shared__ float2 red[2][W];
  extern __shared__ float fold[];  // W == 1: one warp's columns for each row of the block
  int turn = 0;
  const int g = W == 1 ? threadIdx.x >> 5 : 0;
  const int t = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * ln_rows_per_block(W, BWD);
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* dy = reinterpret_cast<const T*>(p.dy);
  const T* res = reinterpret_cast<const T*>(p.dx_in);
  T* dx = reinterpret_cast<T*>(p.dx_out);
  auto col = [&](int i) { return (i * 32 * W + t) * VEC; };
  struct Row {
    Raw x[NV], g[NV], r[RES ? NV : 1];
    float mean, rstd;
  };
  auto fetch = [&](Row& to, int64_t r) {
    to.mean = p.mean[r];
    to.rstd = p.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      to.x[i].zero();
      to.g[i].zero();
      if constexpr (RES) to.r[i].zero();
      if (col(i) < p.d) {
        to.x[i].load(x + r * p.ldx + col(i));
        to.g[i].load(dy + r * p.ldy + col(i));
        if constexpr (RES) to.r[i].load(res + r * p.lddx + col(i));
      }
    }
  };
  Raw w[NV];
  float ds[NV][VEC], db[NV][VEC], dc[COL ? NV : 1][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    w[i].zero();
    if (col(i) < p.d) w[i].load(reinterpret_cast<const T*>(p.scale) + col(i));
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ds[i][j] = db[i][j] = 0.f;
      if constexpr (COL) dc[i][j] = 0.f;
    }
  }
  const float inv_d = 1.f / (float)p.d;
  Row now, next;
  int64_t r = (int64_t)blockIdx.x * ln_rows_per_block(W, BWD) + g;
  if (r < p.rows) fetch(now, r);
  for (; r < p.rows; r += step) {
    if constexpr (AHEAD) {
      if (r + step < p.rows) fetch(next, r + step);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i].stay();
    const float mean = now.mean, rstd = now.rstd;
    const float shift = -mean * rstd;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[VEC], gy[VEC], a[VEC];
      now.x[i].get(v);
      now.g[i].get(gy);
      w[i].get(a);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {  // columns past the width have dy = 0
        const float hat = fmaf(v[j], rstd, shift);
        ds[i][j] = fmaf(gy[j], hat, ds[i][j]);
        db[i][j] += gy[j];
        const float dn = gy[j] * a[j];
        s0 += dn;
        s1 = fmaf(dn, hat, s1);
      }
    }
    ln_row_sums<W>(s0, s1, red, turn);
    s0 *= inv_d;
    s1 *= inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
        float v[VEC], gy[VEC], a[VEC], add[VEC];
        now.x[i].get(v);
        now.g[i].get(gy);
        w[i].get(a);
        if constexpr (RES) now.r[i].get(add);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float hat = fmaf(v[j], rstd, shift);
          float o = rstd * (fmaf(gy[j], a[j], -s0) - hat * s1);
          if constexpr (RES) o += add[j];
          if constexpr (COL) dc[i][j] += o;  // before the rounding to T
          v[j] = o;
        }
        Raw::store(dx + r * p.lddx + col(i), v);
      }
    }
    if constexpr (AHEAD) {
      now = next;
    } else {
      if (r + step < p.rows) fetch(now, r + step);
    }
  }
  // part[q][block][d]: the block's sums of quantity q (scale, bias, columns); a
  // single block adds its sums to the results itself.
  const bool last = gridDim.x == 1;
  auto put = [&](int q, int c, float* out, float v) {
    if (!last)
      out[c] = v;
    else if (p.to.out[q])
      p.to.out[q][c] += p.to.alpha[q] * v;
  };
#pragma unroll
  for (int q = 0; q < (COL ? 3 : 2); ++q) {
    float* out = p.part + ((int64_t)q * gridDim.x + blockIdx.x) * p.d;
    if constexpr (W == 1) __syncthreads();  // the previous quantity has been read
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float s = q == 0 ? ds[i][j] : db[i][j];
          if constexpr (COL) {
            if (q == 2) s = dc[i][j];
          }
          if constexpr (W == 1)
            fold[g * p.d + col(i) + j] = s;
          else
            put(q, col(i) + j, out, s);
        }
      }
    }
    if constexpr (W == 1) {
      __syncthreads();
      for (int k = threadIdx.x; k < p.d; k += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < kLnBwdRows; ++u) s += fold[u * p.d + k];
        put(q, k, out, s);
      }
    }
  }
}

// out[q][c] += alpha[q] sum over the blocks of part[q][block][c], in block order
// within each of 16 interleaved chains and then in chain order.
__global__ void __launch_bounds__(512) ln_sums_kernel(const float* __restrict__ part, int blocks,
                                                      int d, const LnSums to) {
  __shared__ float red[16][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int q = blockIdx.y;
  float s = 0.f;
  if (c < d) {
    const float* src = part + (int64_t)q * blocks * d + c;
#pragma unroll 8
    for (int b = threadIdx.y; b < blocks; b += 16) s += src[(int64_t)b * d];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < d && to.out[q]) {
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < 16; ++u) v += red[u][threadIdx.x];
    to.out[q][c] += to.alpha[q] * v;
  }
}

static int ln_sms() {  // of the current device, asked once
  static int known[64] = {};
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  if (dev < 64 && known[dev]) return known[dev];
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < 64) known[dev] = n;
  return n;
}

// Warps that share a row: as few as keep a lane's elements in registers, four
// 8-element chunks at most, or for element accesses eight (up to 4096) or 32.
static int ln_warps(int64_t d, bool vec) {
  if (vec) return d <= 1024 ? 1 : d <= 8192 ? 8 : 16;
  return d <= 256 ? 1 : d <= 1024 ? 4 : 16;
}
// A grid of what can be resident, or one pass over the rows. The backward's
// blocks leave one row of partials each: `warps` on an SM.
constexpr int kLnFwdWarps = 32, kLnBwdWarps = 16;
// A backward of few rows has one block, which needs no second launch for its sums:
// 33 and 64 rows of 256 take 3.9 and 5.0 us on the device so, 72 rows in nine
// blocks with the sums' launch 4.5 us, and the host saves 5 us.
constexpr int kLnSmall = 64;
static int64_t ln_blocks(int64_t rows, int w, bool bwd) {
  const int64_t per = ln_rows_per_block(w, bwd);
  if (bwd && rows <= kLnSmall / 8 * per) return 1;
  const int block_warps = ln_threads(w, bwd) / 32;
  const int64_t fit = (int64_t)ln_sms() * std::max(1, (bwd ? kLnBwdWarps : kLnFwdWarps) / block_warps);
  return std::min((rows + per - 1) / per, fit);
}

// Calls f with <VEC, W, NV> for the width: 8-element chunks where the rows
// allow 16-byte accesses, single elements otherwise.
template <typename F>
static int ln_dispatch(int64_t d, bool vec, F&& f) {
  const int w = ln_warps(d, vec);
  const int n = (int)((d + 32 * w - 1) / (32 * w));  // elements of a lane
#define GPTB200_LN(V, W, N) return f.template operator()<V, W, N>()
  if (vec && w == 1) {
    if (n <= 8) GPTB200_LN(8, 1, 1);
    if (n <= 16) GPTB200_LN(8, 1, 2);
    if (n <= 24) GPTB200_LN(8, 1, 3);
    GPTB200_LN(8, 1, 4);
  }
  if (vec && w == 8) {
    if (n <= 8) GPTB200_LN(8, 8, 1);
    if (n <= 16) GPTB200_LN(8, 8, 2);
    GPTB200_LN(8, 8, 4);
  }
  if (vec) GPTB200_LN(8, 16, 4);
  if (w == 1) GPTB200_LN(1, 1, 8);
  if (w == 4) GPTB200_LN(1, 4, 8);
  if (n <= 8) GPTB200_LN(1, 16, 8);
  GPTB200_LN(1, 16, 32);
#undef GPTB200_LN
}

template <typename T>
struct LnForward {
  const LnParams& p;
  cudaStream_t st;
  template <int VEC, int W, int NV>
  int operator()() const {
    const unsigned blocks = (unsigned)ln_blocks(p.rows, W, false);
    ln_fwd_kernel<T, VEC, W, NV><<<blocks, ln_threads(W, false), 0, st>>>(p);
    GPTB200_CHECK_LAUNCH();
    return 0;
  }
};

template <typename T>
struct LnBackward {
  const LnParams& p;
  bool col;
  cudaStream_t st;
  template <int VEC, int W, int NV>
  int operator()() const {
    if (p.dx_in) return col ? launch<VEC, W, NV, true, true>() : launch<VEC, W, NV, true, false>();
    return col ? launch<VEC, W, NV, false, true>() : launch<VEC, W, NV, false, false>();
  }
  template <int VEC, int W, int NV, bool RES, bool COL>
  int launch() const {
    const unsigned blocks = (unsigned)ln_blocks(p.rows, W, true);
    const size_t smem = W == 1 ? sizeof(float) * kLnBwdRows * (size_t)p.d : 0;  // <= 48 KB
    ln_bwd_kernel<T, VEC, W, NV, RES, COL><<<blocks, ln_threads(W, true), smem, st>>>(p);
    GPTB200_CHECK_LAUNCH();
    return 0;
  }
};

static bool ln_vec(const LnParams& p, int dtype, std::initializer_list<const void*> ptrs) {
  const int per16 = dtype == GPTB200_DTYPE_BF16 ? 8 : 4;
  uintptr_t any = 0;
  for (const void* q : ptrs) any |= reinterpret_cast<uintptr_t>(q);
  return p.d % 8 == 0 && (p.ldx | p.ldy | p.lddx) % per16 == 0 && (any & 15) == 0;
}

static int ln_check(int64_t rows, int64_t d, int dtype, float eps,
                    std::initializer_list<const void*> ptrs) {
  if (rows <= 0 || d <= 0 || !(eps >= 0.f)) return GPTB200_EINVAL;
  for (const void* q : ptrs)
    if (!q) return GPTB200_EINVAL;
  if (dtype != GPTB200_DTYPE_BF16 && dtype != GPTB200_DTYPE_F32) return GPTB200_EUNSUPPORTED;
  if (d > kLnMaxWidth) return GPTB200_ESHAPE;
  return 0;
}

}  // namespace gptb200

using namespace gptb200;

extern "C" int gptb200_layer_norm_fwd(const void* x, const void* scale, const void* bias, void* y,
                                      float* mean, float* rstd, int64_t rows, int64_t d,
                                      int64_t x_stride, int64_t y_stride, float eps, int dtype,
                                      void* stream) {
  const int s = ln_check(rows, d, dtype, eps, {x, scale, y, mean, rstd});
  if (s) return s;
  if (x_stride < d || y_stride < d) return GPTB200_ESHAPE;
  LnParams p = {};
  p.x = x;
  p.scale = scale;
  p.bias = bias;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.rows = rows;
  p.ldx = x_stride;
  p.ldy = y_stride;
  p.d = (int)d;
  p.eps = eps;
  const bool vec = ln_vec(p, dtype, {x, scale, bias, y});
  auto st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GPTB200_DTYPE_BF16) return ln_dispatch(d, vec, LnForward<bf16>{p, st});
  return ln_dispatch(d, vec, LnForward<float>{p, st});
}

extern "C" size_t gptb200_layer_norm_bwd_workspace_size(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0 || d > kLnMaxWidth) return 0;
  // for either access, which the pointers decide
  const int64_t blocks = std::max(ln_blocks(rows, ln_warps(d, true), true),
                                  ln_blocks(rows, ln_warps(d, false), true));
  return (size_t)blocks * 3 * (size_t)d * sizeof(float);
}

extern "C" int gptb200_layer_norm_bwd(const void* x, const void* scale, const float* mean,
                                      const float* rstd, const void* dy, const void* dx_in,
                                      void* dx_out, float* dscale, float* dbias, float* dx_colsum,
                                      float colsum_alpha, int64_t rows, int64_t d, int64_t x_stride,
                                      int64_t dy_stride, int64_t dx_stride, int dtype,
                                      void* workspace, void* stream) {
  const int s = ln_check(rows, d, dtype, 0.f, {x, scale, mean, rstd, dy, dx_out, dscale, workspace});
  if (s) return s;
  if (x_stride < d || dy_stride < d || dx_stride < d ||
      (reinterpret_cast<uintptr_t>(workspace) & 15))
    return GPTB200_ESHAPE;
  LnParams p = {};
  p.x = x;
  p.scale = scale;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.dy = dy;
  p.dx_in = dx_in;
  p.dx_out = dx_out;
  p.part = reinterpret_cast<float*>(workspace);
  p.rows = rows;
  p.ldx = x_stride;
  p.ldy = dy_stride;
  p.lddx = dx_stride;
  p.d = (int)d;
  const bool vec = ln_vec(p, dtype, {x, scale, dy, dx_in, dx_out});
  auto st = reinterpret_cast<cudaStream_t>(stream);
  const bool col = dx_colsum != nullptr;
  p.to = {{dscale, dbias, dx_colsum}, {1.f, 1.f, colsum_alpha}};
  const int e = dtype == GPTB200_DTYPE_BF16 ? ln_dispatch(d, vec, LnBackward<bf16>{p, col, st})
                                            : ln_dispatch(d, vec, LnBackward<float>{p, col, st});
  const int blocks = (int)ln_blocks(rows, ln_warps(d, vec), true);
  if (e || blocks == 1) return e;
  const dim3 grid((unsigned)((d + 31) / 32), col ? 3 : 2);
  ln_sums_kernel<<<grid, dim3(32, 16), 0, st>>>(p.part, blocks, (int)d, p.to);
  GPTB200_CHECK_LAUNCH();
  return 0;
}
