// The seam between two blocks of the attention bottleneck in one pass over its tokens:
//   y = x + s o sigmoid(g) o N_post(f),   h = N_pre(y)
// N is a root-mean-square norm (v rsqrt(mean v^2 + eps) w) or a layer norm ((v - mean) rsqrt(var + eps) w + b) over the channels; g (the
// block's gate, logits for each token and channel), s (residual scale for each channel), b and either side may be absent.
// Backward, with N's backward L(u) = rstd (u [- mean u] - z mean(u z)), z the normalised row:
//   du = dy + L_pre(dh w_pre),  dx = du,  dn = du s a,  df = L_post(dn w_post),  dg = du s n a (1 - a),
//   ds = sum du a n,  dw_post = sum dn z_f,  db_post = sum dn,  dw_pre = sum dh z_y,  db_pre = sum dh        (a = sigmoid(g), n = N_post(f))
// Bound by HBM: forward reads x, f, g and writes y, h; backward reads x, f, g, dy, dh (the rows' statistics and y itself in 32 bits are
// computed again: cheaper than reading them) and writes dx, df, dg.  A row stays in the registers of TPR threads.
// 31200 x 512 bf16: forward 29 us (5.5 TB/s), backward 62 to 70 us (256 MB at 3.7 to 4.1 TB/s; its few workgroups, which keep the weights' sums in
// registers, have half the forward's waves) and 6 us for the joined sums.
#include "common.h"
#include "dtypes.h"
#include <cmath>

namespace im2im {

struct NormArgs {
  const void *x, *f, *g;
  int64_t xs, fs, gs;                 // row strides in elements
  const float *s, *wp, *bp, *wq, *bq; // [C] each or null (absent)
  void *y, *h;                        // [rows][C]; y may be null
  const void *dy, *dh;                // [rows][C] or null (zero)
  void *dx, *df, *dg;                 // [rows][C] or null
  float* part;                        // [blocks][5][C]: ds, dwp, dbp, dwq, dbq
  int64_t rows;
  int C;
  float eps;
};

// A thread's VPL channels: groups of 8 consecutive ones, group i of thread t at (t + i TPR) * 8, in 16-byte accesses.  Rows need not start at
// 16 bytes (an odd C): global memory takes such accesses at any element, and element by element a wave would touch each line eight times
// (19 us instead of 8 for 4097 rows of 333 floats, forward).
template <typename T> struct Row16;
template <> struct Row16<float> {
  static constexpr int N = 4;
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ void load(float* v, const float* p) {
    const Vec x = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e];
  }
  static __device__ __forceinline__ void store(float* p, const float* v) { *reinterpret_cast<Vec*>(p) = Vec{v[0], v[1], v[2], v[3]}; }
};
template <> struct Row16<bf16_t> {
  static constexpr int N = 8;
  typedef unsigned Vec __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ void load(float* v, const bf16_t* p) {
    const Vec x = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(x[e] << 16);
      v[2 * e + 1] = __uint_as_float(x[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float* v) {
    bf16x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (__bf16)v[e];
    *reinterpret_cast<Vec*>(p) = __builtin_bit_cast(u32x4, x);
  }
};
template <typename T, int TPR, int VPL> struct RowIo {
  static __device__ __forceinline__ int channel(int t, int e) { return (t + (e >> 3) * TPR) * 8 + (e & 7); }
  static __device__ __forceinline__ void load(float* v, const T* row, int t, int C) {
#pragma unroll
    for (int g = 0; g < VPL / 8; ++g) {
      const int c = channel(t, g * 8);
      if (c + 8 <= C) {
#pragma unroll
        for (int e = 0; e < 8; e += Row16<T>::N) Row16<T>::load(v + g * 8 + e, row + c + e);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[g * 8 + e] = c + e < C ? to_float(row[c + e]) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(T* row, const float* v, int t, int C) {
#pragma unroll
    for (int g = 0; g < VPL / 8; ++g) {
      const int c = channel(t, g * 8);
      if (c + 8 <= C) {
#pragma unroll
        for (int e = 0; e < 8; e += Row16<T>::N) Row16<T>::store(row + c + e, v + g * 8 + e);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < C) row[c + e] = from_float<T>(v[g * 8 + e]);
      }
    }
  }
};

// sums of N values over the TPR threads of a row (all get them); TPR > 64: through LDS, in the order of the waves
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* lds) {
#pragma unroll
  for (int s = (TPR < 64 ? TPR : 64) / 2; s >= 1; s >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], s);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) lds[(threadIdx.x >> 6) * N + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) v[n] += lds[w * N + n];
    }
  }
}

// z = the normalised row (zeros behind its C channels), the return value its reciprocal deviation.  The variance is taken around the mean,
// in a second sum over registers: a one-pass E[v^2] - mean^2 loses it where the mean is large.
template <int TPR, int VPL, bool LAYER> __device__ __forceinline__ float normalise(float* z, const float* v, int t, int C, float eps, float* lds) {
  float mean = 0.f;
  if (LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < VPL; ++e) s[0] += v[e];
    row_sums<TPR>(s, lds);
    mean = s[0] / C;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    z[e] = v[e] - mean;
    if (LAYER && RowIo<float, TPR, VPL>::channel(t, e) >= C) z[e] = 0.f;
    q[0] = fmaf(z[e], z[e], q[0]);
  }
  row_sums<TPR>(q, lds);
  const float rstd = 1.f / sqrtf(q[0] / C + eps);
#pragma unroll
  for (int e = 0; e < VPL; ++e) z[e] *= rstd;
  return rstd;
}

// N's backward: u -> rstd (u - mean u - z mean(u z)); u is zero behind the row
template <int TPR, int VPL, bool LAYER> __device__ __forceinline__ void norm_back(float* u, const float* z, float rstd, int t, int C, float* lds) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    s[0] = fmaf(u[e], z[e], s[0]);
    if (LAYER) s[1] += u[e];
  }
  row_sums<TPR>(s, lds);
  const float along = s[0] / C, mean = LAYER ? s[1] / C : 0.f;
#pragma unroll
  for (int e = 0; e < VPL; ++e) u[e] = rstd * (u[e] - mean - z[e] * along);
}

__device__ __forceinline__ float sigmoid_(float g) { return 1.f / (1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g)); }

template <typename T, int TPR, int VPL, bool LAYER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_gate_fwd_kernel(const NormArgs a) {
  using Io = RowIo<T, TPR, VPL>;
  using Wt = RowIo<float, TPR, VPL>;
  constexpr int RPB = (TPR > 256 ? TPR : 256) / TPR;
  __shared__ float lds[32];
  const int t = threadIdx.x % TPR;
  // every thread of the block runs every round (the rows' sums meet at barriers where TPR > 64)
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool mine = row < a.rows;
    const int64_t at = mine ? row : a.rows - 1;
    float y[VPL];
    Io::load(y, static_cast<const T*>(a.x) + at * a.xs, t, a.C);
    if (a.f) {
      float f[VPL], z[VPL], w[VPL];
      Io::load(f, static_cast<const T*>(a.f) + at * a.fs, t, a.C);
      normalise<TPR, VPL, LAYER>(z, f, t, a.C, a.eps, lds);
      Wt::load(w, a.wp, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) z[e] *= w[e];
      if (LAYER && a.bp) {
        Wt::load(w, a.bp, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) z[e] += w[e];
      }
      if (a.s) {
        Wt::load(w, a.s, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) z[e] *= w[e];
      }
      if (a.g) {
        Io::load(f, static_cast<const T*>(a.g) + at * a.gs, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) z[e] *= sigmoid_(f[e]);
      }
#pragma unroll
      for (int e = 0; e < VPL; ++e) y[e] += z[e];
    }
    if (a.y && mine) Io::store(static_cast<T*>(a.y) + row * a.C, y, t, a.C);
    if (a.h) {
      float z[VPL], w[VPL];
      normalise<TPR, VPL, LAYER>(z, y, t, a.C, a.eps, lds);
      Wt::load(w, a.wq, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) z[e] *= w[e];
      if (LAYER && a.bq) {
        Wt::load(w, a.bq, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) z[e] += w[e];
      }
      if (mine) Io::store(static_cast<T*>(a.h) + row * a.C, z, t, a.C);
    }
  }
}

template <typename T, int TPR, int VPL, bool LAYER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_gate_bwd_kernel(const NormArgs a) {
  using Io = RowIo<T, TPR, VPL>;
  using Wt = RowIo<float, TPR, VPL>;
  constexpr int RPB = (TPR > 256 ? TPR : 256) / TPR;
  __shared__ float lds[32];
  __shared__ float acc_lds[RPB > 1 ? RPB * TPR * VPL : 1];
  const int t = threadIdx.x % TPR;
  float sums[5][VPL];                                             // ds, dwp, dbp, dwq, dbq of this thread's channels and rows
#pragma unroll
  for (int n = 0; n < 5; ++n)
#pragma unroll
    for (int e = 0; e < VPL; ++e) sums[n][e] = 0.f;

  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool mine = row < a.rows;
    const int64_t at = mine ? row : a.rows - 1;
    float du[VPL], zf[VPL], n[VPL], ga[VPL];
    float rf = 0.f;
    Io::load(du, static_cast<const T*>(a.x) + at * a.xs, t, a.C);          // y, for now
    if (a.f) {
      float w[VPL];
      Io::load(n, static_cast<const T*>(a.f) + at * a.fs, t, a.C);
      rf = normalise<TPR, VPL, LAYER>(zf, n, t, a.C, a.eps, lds);
      Wt::load(w, a.wp, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) n[e] = zf[e] * w[e];
      if (LAYER && a.bp) {
        Wt::load(w, a.bp, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) n[e] += w[e];
      }
      if (a.g) {
        Io::load(ga, static_cast<const T*>(a.g) + at * a.gs, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) ga[e] = sigmoid_(ga[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VPL; ++e) ga[e] = 1.f;
      }
      if (a.h) {
        if (a.s) Wt::load(w, a.s, t, a.C);
#pragma unroll
        for (int e = 0; e < VPL; ++e) du[e] += (a.s ? n[e] * w[e] : n[e]) * ga[e];
      }
    }
    if (a.dh) {
      float zy[VPL], u[VPL], w[VPL];
      const float ry = normalise<TPR, VPL, LAYER>(zy, du, t, a.C, a.eps, lds);
      Io::load(u, static_cast<const T*>(a.dh) + at * a.C, t, a.C);
      Wt::load(w, a.wq, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) {
        if (mine) {
          sums[3][e] = fmaf(u[e], zy[e], sums[3][e]);
          if (LAYER) sums[4][e] += u[e];
        }
        u[e] *= w[e];
      }
      norm_back<TPR, VPL, LAYER>(u, zy, ry, t, a.C, lds);
#pragma unroll
      for (int e = 0; e < VPL; ++e) du[e] = u[e];
    } else {
#pragma unroll
      for (int e = 0; e < VPL; ++e) du[e] = 0.f;
    }
    if (a.dy) {
      float u[VPL];
      Io::load(u, static_cast<const T*>(a.dy) + at * a.C, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) du[e] += u[e];
    }
    if (a.dx && mine) Io::store(static_cast<T*>(a.dx) + row * a.C, du, t, a.C);
    if (a.f) {
      float w[VPL];
      if (a.s) Wt::load(w, a.s, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) {
        const float ug = du[e] * ga[e];
        if (mine) sums[0][e] = fmaf(ug, n[e], sums[0][e]);
        const float dn = a.s ? ug * w[e] : ug;
        n[e] = dn * n[e] * (1.f - ga[e]);                         // dg
        du[e] = dn;
        if (mine) {
          sums[1][e] = fmaf(dn, zf[e], sums[1][e]);
          if (LAYER) sums[2][e] += dn;
        }
      }
      if (a.dg && mine) Io::store(static_cast<T*>(a.dg) + row * a.C, n, t, a.C);
      Wt::load(w, a.wp, t, a.C);
#pragma unroll
      for (int e = 0; e < VPL; ++e) du[e] *= w[e];
      norm_back<TPR, VPL, LAYER>(du, zf, rf, t, a.C, lds);
      if (a.df && mine) Io::store(static_cast<T*>(a.df) + row * a.C, du, t, a.C);
    }
  }
  // the block's sums: over its rows, in order
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if ((k < 3 && !a.f) || (k >= 3 && !a.dh) || (!LAYER && (k == 2 || k == 4))) continue;      // the same for every thread
    float* out = a.part + ((int64_t)blockIdx.x * 5 + k) * a.C;
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VPL; ++e) acc_lds[((threadIdx.x / TPR) * VPL + e) * TPR + t] = sums[k][e];
      __syncthreads();
      for (int w = threadIdx.x; w < TPR * VPL; w += 256) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) s += acc_lds[r * VPL * TPR + w];
        const int c = Wt::channel(w % TPR, w / TPR);
        if (c < a.C) out[c] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < VPL; ++e) {
        const int c = Wt::channel(t, e);
        if (c < a.C) out[c] = sums[k][e];
      }
    }
  }
}

// [blocks][5][C] -> the weights' gradients: 64 channels a workgroup, the blocks dealt to its 16 waves (with four waves its chains of loads took
// 33 us at 512 blocks, more than the pass over the rows of a small call)
struct NormSumArgs { const float* part; float* out[5]; int blocks, C; };
__global__ __launch_bounds__(1024) void norm_gate_sum_kernel(const NormSumArgs a) {
  __shared__ double part[16][64];
  const int k = blockIdx.y, l = threadIdx.x & 63, c = blockIdx.x * 64 + l, wave = threadIdx.x >> 6;
  if (!a.out[k]) return;
  double acc = 0.0;
  if (c < a.C)
#pragma unroll 8
    for (int b = wave; b < a.blocks; b += 16) acc += (double)a.part[((int64_t)b * 5 + k) * a.C + c];
  part[wave][l] = acc;
  __syncthreads();
  if (wave == 0 && c < a.C) {
#pragma unroll
    for (int w = 1; w < 16; ++w) acc += part[w][l];
    a.out[k][c] = (float)acc;
  }
}

// -------------------------------------------------------------------------------------------------------------------- host
struct NormPlan { int tpr, vpl; };
static NormPlan norm_plan(int C) {
  if (C <= 64) return {8, 8};
  if (C <= 128) return {16, 8};
  if (C <= 256) return {32, 8};
  if (C <= 512) return {64, 8};
  if (C <= 1024) return {64, 16};
  if (C <= 2048) return {256, 8};
  if (C <= 4096) return {512, 8};
  return {1024, 8};
}
constexpr int NORM_MAX_C = 8192;
static int64_t norm_rows_per_block(int C) {
  const int tpr = norm_plan(C).tpr;
  return tpr > 256 ? 1 : 256 / tpr;
}
// two workgroups a CU, four where each still has seven rounds of rows: 101 -> 71 us at 31200 x 512 bf16; fewer rounds pay for the longer join
// (33 -> 35 us at 4097 x 333 fp32)
static int64_t bwd_blocks(int64_t rows, int C) {
  const int64_t rounds = cdiv(rows, norm_rows_per_block(C));
  return std::min<int64_t>(rounds, std::min<int64_t>(1024, std::max<int64_t>(512, rounds / 7)));
}

template <typename T, int TPR, int VPL, bool LAYER> static int launch_norm(const NormArgs& a, bool bwd, hipStream_t st) {
  constexpr int threads = TPR > 256 ? TPR : 256;
  const int64_t per = threads / TPR;
  if (bwd) {
    hipLaunchKernelGGL((norm_gate_bwd_kernel<T, TPR, VPL, LAYER>), dim3((unsigned)bwd_blocks(a.rows, a.C)), dim3(threads), 0, st, a);
    return check_launch("norm_gate_bwd_kernel");
  }
  hipLaunchKernelGGL((norm_gate_fwd_kernel<T, TPR, VPL, LAYER>), dim3((unsigned)std::min<int64_t>(cdiv(a.rows, per), 4096)), dim3(threads), 0, st, a);
  return check_launch("norm_gate_fwd_kernel");
}

template <typename T, bool LAYER> static int dispatch_plan(const NormArgs& a, bool bwd, hipStream_t st) {
  const NormPlan p = norm_plan(a.C);
  if (p.tpr == 8) return launch_norm<T, 8, 8, LAYER>(a, bwd, st);
  if (p.tpr == 16) return launch_norm<T, 16, 8, LAYER>(a, bwd, st);
  if (p.tpr == 32) return launch_norm<T, 32, 8, LAYER>(a, bwd, st);
  if (p.tpr == 64) return p.vpl == 8 ? launch_norm<T, 64, 8, LAYER>(a, bwd, st) : launch_norm<T, 64, 16, LAYER>(a, bwd, st);
  if (p.tpr == 256) return launch_norm<T, 256, 8, LAYER>(a, bwd, st);
  if (p.tpr == 512) return launch_norm<T, 512, 8, LAYER>(a, bwd, st);
  return launch_norm<T, 1024, 8, LAYER>(a, bwd, st);
}

static int dispatch_norm(const NormArgs& a, int dtype, bool layer, bool bwd, hipStream_t st) {
  if (dtype == IM2IM_BF16) return layer ? dispatch_plan<bf16_t, true>(a, bwd, st) : dispatch_plan<bf16_t, false>(a, bwd, st);
  return layer ? dispatch_plan<float, true>(a, bwd, st) : dispatch_plan<float, false>(a, bwd, st);
}

static int norm_check(const im2im_norm_gate_desc* p, NormArgs* a) {
  IM2IM_REQUIRE(p != nullptr);
  IM2IM_REQUIRE(p->x && p->rows >= 1 && p->C >= 1 && p->C <= NORM_MAX_C && p->rows < (1ll << 40));
  IM2IM_REQUIRE(p->dtype == IM2IM_F32 || p->dtype == IM2IM_BF16);
  IM2IM_REQUIRE(p->norm == IM2IM_NORM_RMS || p->norm == IM2IM_NORM_LAYER);
  IM2IM_REQUIRE(p->x_stride >= 0 && p->f_stride >= 0 && p->gate_stride >= 0);
  IM2IM_REQUIRE(p->f ? p->post_weight != nullptr : (!p->gate && !p->scale && !p->post_weight && !p->post_bias));
  IM2IM_REQUIRE(p->pre_weight || !p->pre_bias);
  IM2IM_REQUIRE(p->norm == IM2IM_NORM_LAYER || (!p->post_bias && !p->pre_bias));
  IM2IM_REQUIRE(p->f || p->pre_weight);
  IM2IM_REQUIRE(p->eps > 0.f && std::isfinite(p->eps));
  a->x = p->x; a->f = p->f; a->g = p->gate; a->xs = p->x_stride; a->fs = p->f_stride; a->gs = p->gate_stride;
  a->s = p->scale; a->wp = p->post_weight; a->bp = p->post_bias; a->wq = p->pre_weight; a->bq = p->pre_bias;
  a->rows = p->rows; a->C = p->C; a->eps = p->eps;
  return IM2IM_OK;
}

static bool weights_aligned(const NormArgs& a) {
  const float* p[] = {a.s, a.wp, a.bp, a.wq, a.bq};
  uintptr_t bits = 0;
  for (const float* q : p) bits |= reinterpret_cast<uintptr_t>(q);
  return (bits & 15) == 0;
}

}  // namespace im2im

using namespace im2im;

extern "C" int im2im_norm_gate_fwd(const im2im_norm_gate_desc* p, void* y, void* h, im2im_stream_t stream) {
  NormArgs a = {};
  if (int rc = norm_check(p, &a)) return rc;
  IM2IM_REQUIRE((p->f != nullptr) == (y != nullptr) && (p->pre_weight != nullptr) == (h != nullptr));
  a.y = y; a.h = h;
  IM2IM_REQUIRE(weights_aligned(a));
  return dispatch_norm(a, p->dtype, p->norm == IM2IM_NORM_LAYER, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t im2im_norm_gate_bwd_workspace_bytes(int64_t rows, int32_t C) {
  if (rows < 1 || C < 1 || C > NORM_MAX_C) return -1;
  return bwd_blocks(rows, C) * 5 * C * 4;
}

extern "C" int im2im_norm_gate_bwd(const im2im_norm_gate_desc* p, const void* dy, const void* dh, void* dx, void* df, void* dgate, float* dscale,
                                   float* dpost_weight, float* dpost_bias, float* dpre_weight, float* dpre_bias, void* ws, int64_t ws_bytes,
                                   im2im_stream_t stream) {
  NormArgs a = {};
  if (int rc = norm_check(p, &a)) return rc;
  IM2IM_REQUIRE(dy || dh);
  IM2IM_REQUIRE((!dy || p->f) && (!dh || p->pre_weight));
  IM2IM_REQUIRE((!df && !dscale && !dpost_weight && !dpost_bias) || p->f);
  IM2IM_REQUIRE((!dgate || p->gate) && (!dscale || p->scale) && (!dpost_bias || p->post_bias) && (!dpre_bias || (p->pre_bias && dh)) && (!dpre_weight || dh));
  IM2IM_REQUIRE(ws && ws_bytes >= bwd_blocks(a.rows, a.C) * 5 * a.C * 4);
  a.h = const_cast<void*>(dh);                                   // the kernel needs y where a gradient comes through its norm
  a.dy = dy; a.dh = dh; a.dx = dx; a.df = df; a.dg = dgate; a.part = static_cast<float*>(ws);
  IM2IM_REQUIRE(weights_aligned(a));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (int rc = dispatch_norm(a, p->dtype, p->norm == IM2IM_NORM_LAYER, true, st)) return rc;
  if (!dscale && !dpost_weight && !dpost_bias && !dpre_weight && !dpre_bias) return IM2IM_OK;
  NormSumArgs s = {};
  s.part = a.part; s.blocks = (int)bwd_blocks(a.rows, a.C); s.C = a.C;
  s.out[0] = dscale; s.out[1] = dpost_weight; s.out[2] = dpost_bias; s.out[3] = dpre_weight; s.out[4] = dpre_bias;
  hipLaunchKernelGGL(norm_gate_sum_kernel, dim3((unsigned)cdiv(a.C, 64), 5), dim3(1024), 0, st, s);
  return check_launch("norm_gate_sum_kernel");
}
