// Layer norm, forward and backward.
//
//   y  = (x - mean) rstd scale + bias,   rstd = 1 / sqrt(var + eps)
//   dn = dy scale, hat = (x - mean) rstd
//   dx = rstd (dn - mean(dn) - hat mean(dn hat))  (+ dx_in, the residual stream's gradient)
//   dscale += sum dy hat, dbias += sum dy, dx_colsum += alpha sum dx   (sums over the rows)
//
// Both passes are bound by HBM: x is read once in the forward, x, dy and dx_in once
// in the backward. W warps form a row's group and take the grid's rows in turn.
//
// Forward: the row stays in registers between the statistics and the output, the
// next row's loads are issued before this row's reductions, and the blocks are as
// many as are resident at once (one wave more left a third of the SMs idle at
// 8192 x 4096: 35 us, now 27).
//
// Backward: the three column sums live in the lanes' registers over the whole
// loop, as a lane owns the same columns of every row. They are 24 registers for
// eight columns, so bf16 rows stay out of the registers and pass through shared
// memory (below); held there as well, eight warps of 255 registers were all that
// fitted. Each block writes one row of partials and a second launch adds them in a
// fixed order: results repeat bit for bit. The arithmetic is two elements wide.
//
// Statistics are fp32, the variance is taken about the mean, and the mean is half a
// unit of its last place off where the row lies far from zero: bf16 numbers of a size
// have exact sums (8 bits, at most 2^14 of them), and the sum is divided by d, not just
// multiplied by a rounded 1 / d; fp32 rows correct the mean by the sum of the distances
// from it. So a constant row gives the bias, and as both passes form x - mean before
// anything else, hat is off by |mean| rstd 2^-25 and no more. Outputs are rounded once.
//
// Measured (us and TB/s of the bytes named above; a copy moves 6.55): bf16
// 131072 x 768 forward 67 and 6.0, backward with dx_in and all sums 130 and 6.2;
// 8192 x 4096 forward 27 and 4.9 (a grid of 592 rows at a time: 14 turns); 65536 x
// 768 fp32 66 and 6.1, 128 and 6.3. Rows without 16-byte accesses are bound by the
// number of loads: bf16 65536 x 771 69 and 2.9, 132 and 3.1. Above 8192 the backward's
// lanes hold 32 elements and spill: 8192 x 12288 81 and 5.0, 298 and 2.7 (bf16, with
// dx_in and all sums), 216 and 3.7, 681 and 2.4 (fp32).
#include <algorithm>

#include "common.cuh"

namespace gptb200 {

constexpr int kLnMaxWidth = 16384;

// 32-bit registers of a lane's part of a row.
template <typename T, int VEC, int NV>
constexpr int ln_regs = VEC == 1 ? NV : NV * VEC * (int)sizeof(T) / 4;
// Rows that a block works on at a time. The backward's blocks are one to an SM.
template <int W>
constexpr int ln_fwd_rows = W == 1 ? 4 : 1;
template <int VEC, int W, int NV>
constexpr int ln_bwd_rows = (VEC == 8 && NV == 3 ? 12 : 16) / W;
// Warps of an SM in the forward, by the registers that its lanes then have.
template <typename T, int VEC, int NV>
constexpr int ln_fwd_warps = ln_regs<T, VEC, NV> <= 8 ? 32 : ln_regs<T, VEC, NV> <= 12 ? 24 : 16;
template <typename T, int VEC, int W, int NV>
constexpr int ln_fwd_fit = ln_fwd_warps<T, VEC, NV> / (W * ln_fwd_rows<W>);

// VEC elements as loaded. stay(): keeps a loop from holding the elements of a
// loop-invariant vector unpacked, at twice the registers.
template <typename T, int VEC>
struct LnRaw;
template <>
struct LnRaw<bf16, 8> {
  uint4 q;
  GPTB200_DEV void load(const bf16* p) { q = *reinterpret_cast<const uint4*>(p); }
  // From shared memory where the read stands: moved up, a row's reads would hold
  // some 40 registers more (and spill).
  GPTB200_DEV void stage(const void* p) {
    asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "r"(smem_u32(p))
                 : "memory");
  }
  GPTB200_DEV void zero() { q = make_uint4(0, 0, 0, 0); }
  GPTB200_DEV void stay() { asm volatile("" : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w)); }
  GPTB200_DEV float2 pair(int k) const {
    float2 v;
    unpack_bf16x2(k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w, v.x, v.y);
    return v;
  }
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
  GPTB200_DEV float2 pair(int k) const {
    return k == 0 ? make_float2(a.x, a.y) : k == 1 ? make_float2(a.z, a.w)
         : k == 2 ? make_float2(b.x, b.y) : make_float2(b.z, b.w);
  }
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

// Elements 2k and 2k + 1 of a lane's part of a row.
template <typename T, int VEC>
GPTB200_DEV float2 ln_pair(const LnRaw<T, VEC>* a, int k) {
  if constexpr (VEC == 8) {
    return a[k / 4].pair(k % 4);
  } else {
    float2 v;
    a[2 * k].get(&v.x);
    a[2 * k + 1].get(&v.y);
    return v;
  }
}

// Sums of N = 1, 2, 4 or 8 values over the W warps of a row's group, in every
// thread of it. The first steps each leave half of the values to half of the
// lanes, so eight values take nine exchanges, not forty. `red` has two halves that
// calls use in turn, so one barrier a call suffices (a half is written again only
// after every thread has passed the other half's barrier, hence has read this one).
template <int W, int N>
GPTB200_DEV void ln_group_sums(float (&v)[N], float (*red)[W][N], int& turn, int group) {
  constexpr int L = 32 / N;  // lanes k L and up get value k
  const int lane = threadIdx.x & 31;
  auto fold = [&](int o) { v[0] += __shfl_xor_sync(0xffffffffu, v[0], o); };
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2) {
    const int o = L * n;
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const float away = up ? v[k] : v[k + n];
      v[k] = (up ? v[k + n] : v[k]) + __shfl_xor_sync(0xffffffffu, away, o);
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) fold(o);
  if constexpr (W > 1) {
    if (lane % L == 0) red[turn][threadIdx.x / 32 % W][lane / L] = v[0];
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * W) : "memory");
    v[0] = 0.f;
    if constexpr (N == 1) {
#pragma unroll
      for (int w = 0; w < W; ++w) v[0] += red[turn][w][0];
    } else {
#pragma unroll
      for (int w = 0; w < W; w += L)
        if (w + lane % L < W) v[0] += red[turn][w + lane % L][lane / L];
#pragma unroll
      for (int o = L / 2; o > 0; o /= 2) fold(o);
    }
    turn ^= 1;
  }
  if constexpr (N > 1) {
    const float mine = v[0];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xffffffffu, mine, k * L);
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

template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(32 * W * ln_fwd_rows<W>, ln_fwd_fit<T, VEC, W, NV>)
    ln_fwd_kernel(const LnParams p) {
  using Raw = LnRaw<T, VEC>;
  // 128 bytes of a lane are enough in flight without the next row's
  constexpr bool AHEAD = ln_regs<T, VEC, NV> < 32;
  // fp32: the mean is corrected by the distances from it
  constexpr bool CORRECT = sizeof(T) == 4;
  __shared__ float red[2][W][1], red2[2][W][CORRECT ? 2 : 1];  // in turn: one barrier each
  int turn = 0;
  const int g = W == 1 ? threadIdx.x >> 5 : 0;
  const int t = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * ln_fwd_rows<W>;
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
  int64_t r = (int64_t)blockIdx.x * ln_fwd_rows<W> + g;
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
    // chunks two elements wide; single ones would have to be brought together first
    float2 add = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC == 1) {
        float v;
        now[i].get(&v);
        add.x += v;
      } else {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) add = fadd2(add, now[i].pair(k));
      }
    }
    float sum[1] = {add.x + add.y};
    ln_group_sums<W>(sum, red, turn, 0);
    float mean;
    if constexpr (VEC == 1) {  // the division costs these 78 us, this 69 (65536 x 771 bf16)
      mean = sum[0] * inv_d;
      mean = fmaf(fmaf(-mean, (float)p.d, sum[0]), inv_d, mean);  // and what that leaves of the sum
    } else {  // 67 us so, 72 the other way (131072 x 768 bf16)
      mean = sum[0] / (float)p.d;
    }
    float2 lean = make_float2(0.f, 0.f), square = lean;  // of the distances from it
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
        if constexpr (VEC == 1) {
          float z;
          now[i].get(&z);
          z -= mean;
          if constexpr (CORRECT) lean.x += z;
          square.x = fmaf(z, z, square.x);
        } else {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) {
            const float2 z = fadd2(now[i].pair(k), make_float2(-mean, -mean));
            if constexpr (CORRECT) lean = fadd2(lean, z);
            square = ffma2(z, z, square);
          }
        }
      }
    }
    float dev[CORRECT ? 2 : 1] = {square.x + square.y};
    if constexpr (CORRECT) dev[1] = lean.x + lean.y;
    ln_group_sums<W>(dev, red2, turn, 0);
    float var = dev[0] * inv_d;
    if constexpr (CORRECT) {
      const float off = dev[1] * inv_d;
      mean += off;
      var = fmaxf(fmaf(-off, off, var), 0.f);
    }
    const float rstd = rsqrtf(var + p.eps);
    if (t == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
        float v[VEC];
        if constexpr (VEC == 1) {
          float a, b;
          now[i].get(v);
          w[i].get(&a);
          c[i].get(&b);
          v[0] = fmaf((v[0] - mean) * rstd, a, b);
        } else {
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) {
            const float2 z = fmul2(fadd2(now[i].pair(k), make_float2(-mean, -mean)),
                                   make_float2(rstd, rstd));
            const float2 o = ffma2(z, w[i].pair(k), c[i].pair(k));
            v[2 * k] = o.x;
            v[2 * k + 1] = o.y;
          }
        }
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

// 16 bytes of global memory to shared memory, or zeros.
GPTB200_DEV void ln_copy16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

// Rows of packed chunks pass through shared memory: slots of a block's rows in work.
template <typename T, int VEC>
constexpr bool ln_staged = VEC == 8 && sizeof(T) == 2;
template <int W, int NV, bool RES>
constexpr int ln_slot = 32 * W * ln_bwd_rows<8, W, NV> * (RES ? 3 : 2) * NV * 16;
template <int W, int NV, bool RES>
constexpr int ln_slots = std::min(4, 220 * 1024 / ln_slot<W, NV, RES>);

// RES: dx_in is added. COL: the column sums of dx are wanted too.
//
// STAGED (bf16 chunks): each lane copies its own parts of the next rows to shared
// memory asynchronously and reads them back twice, for the statistics and for dx.
// No lane reads what another copied, so there is nothing to wait for but the
// lane's own copies. 131072 x 768 takes 130 us so, 157 us with the rows in
// registers. fp32 chunks are four to a slot's two and fit the slots only once:
// 65536 x 768 takes 222 us so, 128 us with two rows at a time in registers.
template <typename T, int VEC, int W, int NV, bool RES, bool COL>
__global__ void __launch_bounds__(32 * W * ln_bwd_rows<VEC, W, NV>, 1) ln_bwd_kernel(const LnParams p) {
  using Raw = LnRaw<T, VEC>;
  constexpr int ROWS = ln_bwd_rows<VEC, W, NV>;
  constexpr int THREADS = 32 * W * ROWS;
  constexpr bool STAGED = ln_staged<T, VEC>;
  constexpr int N = RES ? 3 : 2;
  constexpr int SLOTS = STAGED ? ln_slots<W, NV, RES> : 1;
  // single elements: rows that a group has in work, as many as the registers hold
  constexpr int R = !STAGED && NV * VEC <= 8 ? 2 : 1;
  constexpr int P = NV * VEC / 2;  // pairs of elements of a lane: the arithmetic is two wide
  // WIDE: a lane's part of the scales is read (from L1) for every row
  constexpr bool WIDE = VEC == 1 && NV > 8;
  __shared__ float red[ROWS][2][W][2 * R];
  // the slots; then, ROWS > 1, each group's columns of a quantity
  extern __shared__ __align__(16) uint8_t ln_smem[];
  float* fold = reinterpret_cast<float*>(ln_smem);
  int turn = 0;
  const int g = threadIdx.x / (32 * W);
  const int t = threadIdx.x % (32 * W);
  const int64_t step = (int64_t)gridDim.x * ROWS;
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* dy = reinterpret_cast<const T*>(p.dy);
  const T* res = reinterpret_cast<const T*>(p.dx_in);
  const T* scale = reinterpret_cast<const T*>(p.scale);
  T* dx = reinterpret_cast<T*>(p.dx_out);
  auto col = [&](int i) { return (i * 32 * W + t) * VEC; };
  // a lane's chunk i of array a; consecutive lanes have consecutive ones
  auto spot = [&](int slot, int a, int i) {
    return ln_smem + (((slot * N + a) * NV + i) * THREADS + threadIdx.x) * 16;
  };
  auto ask = [&](int slot, int64_t r) {
    if (r < p.rows) {
#pragma unroll
      for (int a = 0; a < N; ++a) {
        const T* src = a == 0 ? x + r * p.ldx : a == 1 ? dy + r * p.ldy : res + r * p.lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const bool in = col(i) < p.d;
          ln_copy16(spot(slot, a, i), in ? src + col(i) : src, in);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  struct Row {  // of single elements
    Raw x[NV], g[NV], r[RES ? NV : 1];
  };
  Row now[STAGED ? 1 : R];
  auto fetch = [&](int64_t first) {
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int64_t r = first + u * step;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        now[u].x[i].zero();
        now[u].g[i].zero();
        if constexpr (RES) now[u].r[i].zero();
        if (r < p.rows && col(i) < p.d) {  // a row past the end adds zeros
          now[u].x[i].load(x + r * p.ldx + col(i));
          now[u].g[i].load(dy + r * p.ldy + col(i));
          if constexpr (RES) now[u].r[i].load(res + r * p.lddx + col(i));
        }
      }
    }
  };
  Raw w[WIDE ? 1 : NV];
  float2 ds[P], db[P], dc[COL ? P : 1];
#pragma unroll
  for (int i = 0; i < (WIDE ? 0 : NV); ++i) {
    w[i].zero();
    if (col(i) < p.d) w[i].load(scale + col(i));
  }
#pragma unroll
  for (int k = 0; k < P; ++k) {
    ds[k] = db[k] = make_float2(0.f, 0.f);
    if constexpr (COL) dc[k] = make_float2(0.f, 0.f);
  }
  const float inv_d = 1.f / (float)p.d;
  int64_t r = (int64_t)blockIdx.x * ROWS + g;
  if constexpr (STAGED) {
#pragma unroll
    for (int k = 0; k < SLOTS - 1; ++k) ask(k, r + k * step);
  }
  float mean[R], rstd[R], mean_next = 0.f, rstd_next = 0.f;
  if (STAGED && r < p.rows) mean_next = p.mean[r], rstd_next = p.rstd[r];
  int slot = 0;
  for (; r < p.rows; r += step * R) {
    if constexpr (STAGED) {
      // the slot of the row before, which this lane has read
      ask(slot == 0 ? SLOTS - 1 : slot - 1, r + (SLOTS - 1) * step);
      mean[0] = mean_next;
      rstd[0] = rstd_next;
      if (r + step < p.rows) mean_next = p.mean[r + step], rstd_next = p.rstd[r + step];
      asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
    } else {
      fetch(r);
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const bool in = r + u * step < p.rows;
        mean[u] = in ? p.mean[r + u * step] : 0.f;
        rstd[u] = in ? p.rstd[r + u * step] : 0.f;
      }
    }
    auto part = [&](int u, int a, int i) {  // chunk i of array a
      Raw q;
      if constexpr (STAGED) {
        q.stage(spot(slot, a, i));
      } else {
        q = a == 0 ? now[u].x[i] : a == 1 ? now[u].g[i] : now[u].r[RES ? i : 0];
      }
      return q;
    };
    auto scales = [&](int i) {
      if constexpr (WIDE) {
        Raw q;
        q.zero();
        if (col(i) < p.d) q.load(scale + col(i));
        return q;
      } else {
        return w[i];
      }
    };
    constexpr int C = VEC == 8 ? 1 : 2;  // chunks that make pairs
    constexpr int PAIRS = VEC * C / 2;
    float s[2 * R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const float2 m = make_float2(rstd[u], rstd[u]), b = make_float2(-mean[u], -mean[u]);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int i = 0; i < NV; i += C) {
        Raw xs[C], gs[C], ws[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          xs[c] = part(u, 0, i + c);
          gs[c] = part(u, 1, i + c);
          ws[c] = scales(i + c);
        }
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {  // columns past the width have dy = 0
          const int k = i * VEC / 2 + j;
          const float2 gy = ln_pair<T, VEC>(gs, j);
          const float2 hat = fmul2(fadd2(ln_pair<T, VEC>(xs, j), b), m);
          const float2 dn = fmul2(gy, ln_pair<T, VEC>(ws, j));
          ds[k] = ffma2(gy, hat, ds[k]);
          db[k] = fadd2(db[k], gy);
          s0 = fadd2(s0, dn);
          s1 = ffma2(dn, hat, s1);
        }
      }
      s[2 * u] = s0.x + s0.y;
      s[2 * u + 1] = s1.x + s1.y;
    }
    ln_group_sums<W>(s, red[g], turn, g);
#pragma unroll
    for (int i = 0; i < (WIDE ? 0 : NV); ++i) w[i].stay();  // packed between the passes
#pragma unroll
    for (int u = 0; u < R; ++u) {
      // per x - mean, not per hat: one operation less
      const float s0 = -s[2 * u] * inv_d, s1 = -s[2 * u + 1] * inv_d * rstd[u];
      const float2 m = make_float2(rstd[u], rstd[u]), b = make_float2(-mean[u], -mean[u]);
      const float2 m0 = make_float2(s0, s0), m1 = make_float2(s1, s1);
      T* to = dx + (r + u * step) * p.lddx;
      const bool in = R == 1 || r + u * step < p.rows;
#pragma unroll
      for (int i = 0; i < NV; i += C) {
        Raw xs[C], gs[C], as[C], ws[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          xs[c] = part(u, 0, i + c);
          gs[c] = part(u, 1, i + c);
          if constexpr (RES) as[c] = part(u, 2, i + c);
          ws[c] = scales(i + c);
        }
        float v[C * VEC];
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {  // past the width or the last row: not stored
          const float2 away = fadd2(ln_pair<T, VEC>(xs, j), b);
          const float2 dn = ffma2(ln_pair<T, VEC>(gs, j), ln_pair<T, VEC>(ws, j), m0);
          float2 o = ffma2(away, m1, dn);
          if constexpr (RES)
            o = ffma2(o, m, ln_pair<T, VEC>(as, j));
          else
            o = fmul2(o, m);
          if constexpr (COL) {  // before the rounding to T
            const int k = i * VEC / 2 + j;
            dc[k] = fadd2(dc[k], o);
          }
          v[2 * j] = o.x;
          v[2 * j + 1] = o.y;
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (in && col(i + c) < p.d) Raw::store(to + col(i + c), v + c * VEC);
      }
    }
    if constexpr (STAGED) slot = slot == SLOTS - 1 ? 0 : slot + 1;
  }
  if constexpr (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
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
    if constexpr (ROWS > 1) __syncthreads();  // the previous quantity has been read
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col(i) < p.d) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int k = (i * VEC + j) / 2;
          float2 both = q == 0 ? ds[k] : db[k];
          if constexpr (COL) {
            if (q == 2) both = dc[k];
          }
          const float s = (i * VEC + j) % 2 ? both.y : both.x;
          if constexpr (ROWS > 1)
            fold[g * p.d + col(i) + j] = s;
          else
            put(q, col(i) + j, out, s);
        }
      }
    }
    if constexpr (ROWS > 1) {
      __syncthreads();
      for (int k = threadIdx.x; k < p.d; k += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < ROWS; ++u) s += fold[u * p.d + k];
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

// Blocks of the backward, each of which leaves a row of partials. Few rows have one
// block, which needs no second launch for its sums: 33 rows of 256 take 4.6 us on
// the device, 72 rows in five blocks 5.4, and the host saves a launch of 5 us.
static int64_t ln_bwd_blocks(int64_t rows, int per) {
  if (rows <= 4 * per) return 1;
  return std::min((rows + per - 1) / per, (int64_t)ln_sms());
}

// Calls f with <VEC, W, NV> for the width: 8-element chunks where the rows allow
// 16-byte accesses, single elements otherwise, W warps to a row and NV of either to
// a lane: as few warps as a lane's registers allow, since a row's reductions and
// barriers cost the same for any width. The backward holds three sums for every
// element of a lane, so it takes two chunks (three where they fill the width), and
// for fp32, which holds the rows too, one.
template <bool BWD, typename F>
static int ln_dispatch(int64_t d, bool vec, const F& f) {
#define GPTB200_LN(MAX, V, W, N) \
  if (d <= MAX) return f.template operator()<V, W, N>()
  if (vec) {
    GPTB200_LN(256, 8, 1, 1);
    if constexpr (BWD) {
      if constexpr (F::kBytes == 2) {
        GPTB200_LN(512, 8, 1, 2);
        GPTB200_LN(768, 8, 1, 3);
        GPTB200_LN(1024, 8, 2, 2);
        GPTB200_LN(2048, 8, 4, 2);
        GPTB200_LN(4096, 8, 8, 2);
      } else {
        GPTB200_LN(512, 8, 2, 1);
        GPTB200_LN(768, 8, 3, 1);
        GPTB200_LN(1024, 8, 4, 1);
        GPTB200_LN(2048, 8, 8, 1);
        GPTB200_LN(4096, 8, 16, 1);
      }
      GPTB200_LN(8192, 8, 16, 2);
    } else {
      GPTB200_LN(512, 8, 1, 2);
      GPTB200_LN(768, 8, 1, 3);
      GPTB200_LN(1024, 8, 1, 4);
      GPTB200_LN(2048, 8, 8, 1);
      GPTB200_LN(4096, 8, 8, 2);
      GPTB200_LN(8192, 8, 8, 4);
    }
    GPTB200_LN(kLnMaxWidth, 8, 16, 4);
  }
  GPTB200_LN(256, 1, 1, 8);
  GPTB200_LN(1024, 1, 4, 8);
  GPTB200_LN(2048, 1, 8, 8);
  GPTB200_LN(4096, 1, 16, 8);
  GPTB200_LN(8192, 1, 16, 16);
  GPTB200_LN(kLnMaxWidth, 1, 16, 32);
#undef GPTB200_LN
  return GPTB200_ESHAPE;
}

template <typename T>
struct LnForward {
  static constexpr int kBytes = sizeof(T);
  const LnParams& p;
  cudaStream_t st;
  template <int VEC, int W, int NV>
  int operator()() const {  // a grid of what is resident, or one pass over the rows
    constexpr int rows = ln_fwd_rows<W>;
    const int64_t blocks = std::min((p.rows + rows - 1) / rows,
                                    (int64_t)ln_sms() * ln_fwd_fit<T, VEC, W, NV>);
    ln_fwd_kernel<T, VEC, W, NV><<<(unsigned)blocks, 32 * W * rows, 0, st>>>(p);
    GPTB200_CHECK_LAUNCH();
    return 0;
  }
};

template <typename T>
struct LnBackward {
  static constexpr int kBytes = sizeof(T);
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
    constexpr int rows = ln_bwd_rows<VEC, W, NV>;
    const int blocks = (int)ln_bwd_blocks(p.rows, rows);
    // 36 KB at most (12 rows of 768), which the slots of a staged variant cover
    size_t smem = rows > 1 ? sizeof(float) * rows * (size_t)p.d : 0;
    auto kern = ln_bwd_kernel<T, VEC, W, NV, RES, COL>;
    if constexpr (ln_staged<T, VEC>) {
      constexpr int slots = ln_slots<W, NV, RES> * ln_slot<W, NV, RES>;
      smem = std::max<size_t>(smem, slots);
      static bool known[64] = {};
      int dev = 0;
      cudaGetDevice(&dev);
      if (dev >= 64 || !known[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 std::max(slots, 16 * 1024));
        if (e != cudaSuccess) return -static_cast<int>(e);
        if (dev < 64) known[dev] = true;
      }
    }
    kern<<<blocks, 32 * W * rows, smem, st>>>(p);
    GPTB200_CHECK_LAUNCH();
    if (blocks == 1) return 0;
    const dim3 grid((unsigned)((p.d + 31) / 32), COL ? 3 : 2);
    ln_sums_kernel<<<grid, dim3(32, 16), 0, st>>>(p.part, blocks, p.d, p.to);
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
  if (dtype == GPTB200_DTYPE_BF16) return ln_dispatch<false>(d, vec, LnForward<bf16>{p, st});
  return ln_dispatch<false>(d, vec, LnForward<float>{p, st});
}

extern "C" size_t gptb200_layer_norm_bwd_workspace_size(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0 || d > kLnMaxWidth) return 0;
  // the most blocks that any access (the pointers decide) takes: one row at a time
  const int64_t blocks = std::min(rows, (int64_t)ln_sms());
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
  if (dtype == GPTB200_DTYPE_BF16) return ln_dispatch<true>(d, vec, LnBackward<bf16>{p, col, st});
  return ln_dispatch<true>(d, vec, LnBackward<float>{p, col, st});
}
