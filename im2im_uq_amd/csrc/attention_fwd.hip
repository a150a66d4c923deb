// Grid attention, forward: softmax attention over the pixels of a grid with a learned relative position bias, and its
// differential form (the difference of two softmax maps that share the values).
//   s_ij = scale q_i . k_j + bias(j - i),   o_i = sum_j softmax_j(s_i)_j v_j          (keys from lengths[b] on take no part)
//   two maps: o = o1 - lam o2
// One pass over the keys with a running maximum and sum; work split over the keys and joined when there are few queries.
#include "attention_common.h"
#include <cmath>
#include <mutex>
#include <unordered_map>

namespace im2im {

// ---------------------------------------------------------------------------------------------------------- bias table -> line
struct LineArgs {
  const float* table;    // [ny][nx][H]
  float* line;           // [H][line_len]
  int ny, nx, H, gh, gw, len;
  int thr_y[32], thr_x[32];   // smallest distance of bucket 1, 2, ...
};

__device__ __forceinline__ int axis_bucket(int delta, int n, const int* thr) {
  if (n == 1) return 0;
  const int side = n / 2, t = delta < 0 ? -delta : delta;
  int b = 0;
  for (int m = 0; m < side - 1; ++m) b += t >= thr[m];
  return b + (delta > 0 ? side : 0);
}

// a few thousand floats: bound by its launch (3 to 5 us)
__global__ __launch_bounds__(256) void relpos_line_kernel(const LineArgs a) {
  const int idx = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (idx >= a.len) return;
  const int w = 2 * a.gw - 1;
  const int b = axis_bucket(idx / w - (a.gh - 1), a.ny, a.thr_y) * a.nx + axis_bucket(idx % w - (a.gw - 1), a.nx, a.thr_x);
  a.line[(int64_t)h * a.len + idx] = bias_log2(a.table[(int64_t)b * a.H + h]);
}

// ------------------------------------------------------------------------------------------------------------------- forward
// One workgroup: 128 queries (a wave has 32 of them as its columns), keys in tiles of 64 through LDS, a wave takes 32 of them at a time.  KS = 2: 64
// queries, two waves share 32 and take one half of each tile's keys (joined at the end): for calls that would leave CUs without work.
// The running maximum follows the scores only where they pass it by more than 2^GROW: until then probabilities up to 2^GROW are as exact in
// 32 bits and in bf16 as those up to 1, and the accumulators need no rescaling (a handful of times a row).
// P enters the product as bf16 hi + lo, 16 bits of it: a result is a sum of terms that cancel, and with P rounded to 8 bits one lay 1.15 (one map) to 1.5
// (two) times as far from its value as its own rounding, many times that where it is small beside its terms.  Costs the matrix unit a second product
// (inference 78 x 20x20 x 8 x 64: 77 -> 90 us, 8 x 32x32 x 8 x 128: 57 -> 70; two maps, the second one's added, 16 x 40x40 x 4 x 2 x 64, ragged: 213 -> 246).
// SAVE (training): each map's result leaves in 32 bits too: the backward's row sums D = dO . O are taken from it.
// Measured (bf16): training 78 x 20x20 x 8 x 64 80 us (320 TFLOP/s; the vector unit issues in 51 % of the cycles, the matrix unit is busy in 20 %: the
// exponentials, maxima and packing of 64-wide heads bound it), 8 x 32x32 x 8 x 128 67 us (510 TFLOP/s); two maps at 16 x 40x40 x 4 x 2 x 64, half to full
// lengths, 246 us (510 TFLOP/s; 1.6 rounds of two workgroups a CU, all 256 registers); one query of 4 x 16384 keys x 8 x 2 x 32 32 us (4.2 TB/s).
constexpr float GROW = 8.f;

// what the backward takes a row's probabilities from: exp2(score - reference - logarithm).  No key at all: +infinity, they come out as zeros.
// A sum of NaN is none of these: its row's probabilities are NaN there as they are here.
__device__ __forceinline__ void save_row(const AttnArgs& a, int64_t at, float top, float sum) {
  a.top[at] = sum == 0.f ? 0.f : top;
  a.lsum[at] = sum == 0.f ? INFINITY : __builtin_amdgcn_logf(sum);
}

// TOKEN (one query, nothing saved): a key's bias is taken from the table itself, a launch and the line less; a tile's window is its keys in their order.
template <typename T, int DQ, int DV, int MAPS, bool SAVE, bool ROW4, int KS, bool TOKEN = false>
__global__ __launch_bounds__(64 * WAVES, DV * sizeof(T) >= 512 ? 1 : 2) void attn_fwd_kernel(const AttnArgs a) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr bool HILO = sizeof(T) == 2;
  constexpr int QR = ROWS / KS, NB = DV / 32, NBUF = buffers<T>(MAPS * DQ + DV);
  constexpr size_t KT = tile_bytes<T>(DQ), TILES = tile_bytes<T>(MAPS * DQ + DV);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const size_t buffer = TILES + KEYS * 4 + (size_t)a.window * 4;           // tiles, codes, window

  const int lin = xcd_band(blockIdx.x, gridDim.x), sp = lin % a.splits, item = lin / a.splits;
  // all images of a head, then the next head: each XCD gets many images, whose lengths may differ (224 -> 215 us at 16 x 40x40 x 4 x 2 x 64, half to full)
  const int qt = item % a.nq, h = item / a.nq / a.B, b = item / a.nq % a.B, bh = b * a.H + h;
  const int wave = wave_index() / KS, kw = wave_index() % KS, lane = threadIdx.x & 63, half = lane >> 5;
  const int i0 = qt * QR, i_last = min(i0 + QR, a.Lq) - 1;
  const int i = i0 + wave * 32 + (lane & 31);
  const bool mine = i < a.Lq, busy = i0 + wave * 32 < a.Lq;
  const int code_last = grid_code(a.q_start + i_last, a.gw);
  const int aoff = code_last - grid_code(a.q_start + min(i, i_last), a.gw);
  const int qspan = code_last - grid_code(a.q_start + i0, a.gw);
  const float scale2 = a.scale * LOG2E;

  Frag qf[MAPS][DQ / M::KC];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    load_row_frags<T, DQ>(qf[m], static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)min(i, i_last) * a.qs[1] + (int64_t)(MAPS * h + m) * a.qs[2],
                          mine, a.d, half);
  float mx[MAPS], sum[MAPS];                                      // of this lane's keys (a row's other half is 32 lanes away)
  f32x16 o[MAPS][NB];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    mx[m] = -INFINITY;
    sum[m] = 0.f;
#pragma unroll
    for (int n = 0; n < NB; ++n) o[m][n] = zero16();
  }

  const int len = a.lengths ? max(0, min(a.lengths[b], a.Lk)) : a.Lk;
  const int t0 = sp * a.tiles_per_split, t1 = min(t0 + a.tiles_per_split, (len + KEYS - 1) / KEYS);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)(MAPS * h) * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)h * a.vs[2];
  const float* line = TOKEN ? a.table + h : a.line + (int64_t)h * a.line_len;
  const int thr = TOKEN ? a.thr[lane] : 0, q_row = TOKEN ? a.q_start / a.gw : 0, q_col = TOKEN ? a.q_start % a.gw : 0;

  TileFetch<T, DQ> kt;
  TileFetch<T, DV> vt;
  kt.prepare(a.ks[1]);
  vt.prepare(a.vs[1]);
  const bool full = a.d == DQ && a.dv == DV;
  Raster keys(t0 * KEYS, a.gw);
  // TOKEN: a wave without a query looks up its lanes' keys of the coming tile (behind the last one: any entry) while the others work on this one
  const bool spare = TOKEN && wave_index() == WAVES - 1;
  auto entry = [&] { return line[(int64_t)(lane_bucket(keys.row - q_row, a.ny, thr, 0) * a.nx + lane_bucket(keys.col - q_col, a.nx, thr, 32)) * a.H]; };
  float ahead = spare ? entry() : 0.f;
  auto fetch = [&](int t, char* to) {                             // tiles in their order
    if (spare) {
      int* codes = reinterpret_cast<int*>(to + TILES);
      reinterpret_cast<float*>(codes + KEYS)[lane] = bias_log2(ahead);
      codes[lane] = 4 * lane;
      keys.next();
    }
    const int j0 = t * KEYS, valid = min(len - j0, KEYS);
    const T *k = kp + (int64_t)j0 * a.ks[1], *v = vp + (int64_t)j0 * a.vs[1];
    if (full && valid == KEYS) {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) kt.whole(to + m * KT, k + m * a.ks[2]);
      vt.whole(to + MAPS * KT, v);
    } else {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) kt.part(to + m * KT, k + m * a.ks[2], a.ks[1], valid, a.d);
      vt.part(to + MAPS * KT, v, a.vs[1], valid, a.dv);
    }
    if (TOKEN) {
      if (spare) ahead = entry();
      return;
    }
    const int code = keys.code(), first = __builtin_amdgcn_readfirstlane(code), last = __builtin_amdgcn_readlane(code, valid - 1);
    keys.next();
    int* codes = reinterpret_cast<int*>(to + TILES);
    fetch_window(reinterpret_cast<float*>(codes + KEYS), line, a.line_len, first - code_last + a.line_off, last - first + qspan + 1);
    if (threadIdx.x < KEYS) codes[threadIdx.x] = 4 * (min(code, last) - first);
  };
  if (t0 < t1) fetch(t0, smem);
  for (int t = t0; t < t1; ++t) {
    char* at = smem + (NBUF == 2 && ((t - t0) & 1) ? buffer : 0);
    lds_loads_done();
    __syncthreads();
    if (NBUF == 2 && t + 1 < t1) fetch(t + 1, (t - t0) & 1 ? smem : smem + buffer);
    const char *Ks = at, *Vs = at + MAPS * KT;
    const int* kc = reinterpret_cast<const int*>(at + TILES);
    const unsigned win = window_place(reinterpret_cast<const float*>(kc + KEYS), aoff);
    const int valid = min(len - t * KEYS, KEYS);
    if (busy)
#pragma unroll 1
    for (int sub = kw; sub < 2; sub += KS) {
      if (sub * 32 >= valid) break;
      float bias[16];
      window_bias<ROW4>(bias, win, kc + sub * 32, half);
      f32x16 s[MAPS];
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        f32x16 acc = zero16();
#pragma unroll
        for (int c = 0; c < DQ / M::KC; ++c)
          acc = M::mma(tile_frag<T, DQ>(Ks + m * KT, sub * 32, c), qf[m][c], acc);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[m][r] = fmaf(acc[r], scale2, bias[r]);
      }
      if (valid < sub * 32 + 32) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (sub * 32 + mfma_row(r, half) >= valid)
#pragma unroll
            for (int m = 0; m < MAPS; ++m) s[m][r] = -INFINITY;
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        float top = s[m][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[m][r]);
        if (__any(top > mx[m] + GROW)) {
          top = fmaxf(mx[m], fmaxf(top, __shfl_xor(top, 32)));
          const float shrink = top == -INFINITY ? 1.f : exp2_(mx[m] - top);
          mx[m] = top;
          sum[m] *= shrink;
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[m][n][r] *= shrink;
        }
        const float ref = mx[m] == -INFINITY ? 0.f : mx[m];      // nothing but masks so far
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[m][r] = exp2_(s[m][r] - ref);
          sum[m] += s[m][r];
        }
      }
#pragma unroll
      for (int ks = 0; ks < 32 / M::KC; ++ks) {
        Frag pf[MAPS], pr[MAPS];
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          pf[m] = M::pack(s[m], ks);
          if (HILO) pr[m] = M::pack_rest(s[m], pf[m], ks);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const Frag vf = M::template load_t<DV>(Vs, sub * 32, ks, n);
#pragma unroll
          for (int m = 0; m < MAPS; ++m) {
            o[m][n] = M::mma(vf, pf[m], o[m][n]);
            if (HILO) o[m][n] = M::mma(vf, pr[m], o[m][n]);
          }
        }
      }
    }
    if (NBUF == 1 && t + 1 < t1) {
      __syncthreads();
      fetch(t + 1, smem);
    }
  }

  if (KS == 2) {                                                  // the two waves of 32 queries, through LDS
    float* box = reinterpret_cast<float*>(smem) + wave * (MAPS * (NB * 16 + 2) * 64) + lane;
    __syncthreads();
    if (kw == 1) {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        float* to = box + m * (NB * 16 + 2) * 64;
        to[0] = mx[m];
        to[64] = sum[m];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) to[(2 + n * 16 + r) * 64] = o[m][n][r];
      }
    }
    __syncthreads();
    if (kw == 1) return;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const float* from = box + m * (NB * 16 + 2) * 64;
      const float top = fmaxf(mx[m], from[0]), ref = top == -INFINITY ? 0.f : top, w0 = exp2_(mx[m] - ref), w1 = exp2_(from[0] - ref);
      mx[m] = top;
      sum[m] = sum[m] * w0 + from[64] * w1;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[m][n][r] = o[m][n][r] * w0 + from[(2 + n * 16 + r) * 64] * w1;
    }
  }
  if (!busy) return;
  const int64_t row = (int64_t)bh * a.Lq + i;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) sum[m] += __shfl_xor(sum[m], 32);
  if (!mine) return;
  if (a.splits > 1) {                                             // joined by attn_combine_kernel
    const int64_t rows = (int64_t)a.B * a.H * a.Lq;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const int64_t at = ((int64_t)sp * rows + row) * MAPS + m;
      if (half == 0) {
        a.part_ml[at * 2] = mx[m];
        a.part_ml[at * 2 + 1] = sum[m];
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = n * 32 + 8 * g + 4 * half;
          if (c < a.dv) store4(a.part + at * a.dv + c, o[m][n][4 * g], o[m][n][4 * g + 1], o[m][n][4 * g + 2], o[m][n][4 * g + 3]);
        }
    }
    return;
  }
  float inv[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    inv[m] = sum[m] == 0.f ? 0.f : 1.f / sum[m];                  // no key at all: a row of zeros
    if (SAVE && half == 0) save_row(a, ((int64_t)bh * MAPS + m) * a.Lq + i, mx[m], sum[m]);
  }
  const float lam = MAPS == 2 ? a.lam[h] : 0.f;
  T* out = static_cast<T*>(a.out) + (((int64_t)b * a.Lq + i) * a.H + h) * a.dv;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = n * 32 + 8 * g + 4 * half;
      if (c >= a.dv) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = o[0][n][4 * g + e] * inv[0];
        if (MAPS == 2) v[e] -= lam * (o[MAPS - 1][n][4 * g + e] * inv[MAPS - 1]);
      }
      store4(out + c, v[0], v[1], v[2], v[3]);
      if (SAVE)
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
          store4(a.osave + (row * MAPS + m) * a.dv + c, o[m][n][4 * g] * inv[m], o[m][n][4 * g + 1] * inv[m], o[m][n][4 * g + 2] * inv[m],
                 o[m][n][4 * g + 3] * inv[m]);
    }
}

// joins the parts of a row: 32 lanes (four channels each) times G groups, which take the parts in turn.  Bound by the latency of its loads:
// one group needs 40 us for 64 parts, eight need 5.
template <typename T, int MAPS, int G> __global__ __launch_bounds__(256) void attn_combine_kernel(const AttnArgs a) {
  __shared__ float tops[8][MAPS], sums[8][MAPS];
  __shared__ f32x4 parts[8][MAPS][32];
  const int64_t rows = (int64_t)a.B * a.H * a.Lq, row = (int64_t)blockIdx.x * (8 / G) + (threadIdx.x >> 5) / G;
  const int group = (threadIdx.x >> 5) % G, slot = (threadIdx.x >> 5) / G * G, l = threadIdx.x & 31, c = l * 4;
  const bool mine = row < rows;
  float top[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    top[m] = -INFINITY;
    if (mine)
      for (int s = group * 32 + l; s < a.splits; s += 32 * G) top[m] = fmaxf(top[m], a.part_ml[((s * rows + row) * MAPS + m) * 2]);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) top[m] = fmaxf(top[m], __shfl_xor(top[m], x));
    if (G > 1 && l == 0) tops[slot + group][m] = top[m];
  }
  if (G > 1) {
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int g = 0; g < G; ++g) top[m] = fmaxf(top[m], tops[slot + g][m]);
  }
  float sum[MAPS];
  f32x4 o[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float ref = top[m] == -INFINITY ? 0.f : top[m];
    sum[m] = 0.f;
    o[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (mine)
#pragma unroll 4
      for (int s = group; s < a.splits; s += G) {
        const int64_t at = (s * rows + row) * MAPS + m;
        const float w = exp2_(a.part_ml[at * 2] - ref);
        sum[m] += w * a.part_ml[at * 2 + 1];
        if (c < a.dv) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + at * a.dv + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][e] = fmaf(w, x[e], o[m][e]);
        }
      }
    if (G > 1) {
      if (l == 0) sums[slot + group][m] = sum[m];
      parts[slot + group][m][l] = o[m];
    }
  }
  if (G > 1) {
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int g = 1; g < G; ++g) {
        sum[m] += sums[slot + g][m];
        const f32x4 x = parts[slot + g][m][l];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][e] += x[e];
      }
  }
  if (!mine) return;
  const int i = (int)(row % a.Lq), bh = (int)(row / a.Lq), h = bh % a.H, b = bh / a.H;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float inv = sum[m] == 0.f ? 0.f : 1.f / sum[m];
    if (a.top && l == 0) save_row(a, ((int64_t)bh * MAPS + m) * a.Lq + i, top[m], sum[m]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[m][e] *= inv;
      v[e] += m == 0 ? o[m][e] : -a.lam[h] * o[m][e];
    }
    if (a.osave && c < a.dv) store4(a.osave + (row * MAPS + m) * a.dv + c, o[m][0], o[m][1], o[m][2], o[m][3]);
  }
  if (c < a.dv) store4(static_cast<T*>(a.out) + (((int64_t)b * a.Lq + i) * a.H + h) * a.dv + c, v[0], v[1], v[2], v[3]);
}

// -------------------------------------------------------------------------------------------------------------------- host
int attn_allow_lds(const void* kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return IM2IM_OK;
  static std::mutex mu;
  static std::unordered_map<const void*, size_t> set[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return fail_invalid("attention: device index");
  std::lock_guard<std::mutex> lock(mu);
  size_t& have = set[dev][kernel];
  if (bytes > have) {
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
      (void)hipGetLastError();
      return fail_invalid("attention: the device refuses the kernel's LDS size");
    }
    have = bytes;
  }
  return IM2IM_OK;
}

bool attn_buckets_ok(int32_t ny, int32_t nx, const int32_t* thr_y, const int32_t* thr_x) {
  return ny >= 1 && ny <= 64 && (ny == 1 || ny % 2 == 0) && nx >= 1 && nx <= 64 && (nx == 1 || nx % 2 == 0) && (ny <= 2 || thr_y) && (nx <= 2 || thr_x);
}

int attn_check(const im2im_attention_desc* p, AttnArgs* a) {
  IM2IM_REQUIRE(p != nullptr);
  IM2IM_REQUIRE(p->q && p->k && p->v);
  IM2IM_REQUIRE(p->line || (p->Lq == 1 && p->table && attn_buckets_ok(p->ny, p->nx, p->thr_y, p->thr_x)));
  IM2IM_REQUIRE(p->dtype == IM2IM_F32 || p->dtype == IM2IM_BF16);
  IM2IM_REQUIRE(p->maps == 1 || p->maps == 2);
  IM2IM_REQUIRE(p->maps == 1 || p->lam != nullptr);
  IM2IM_REQUIRE(p->B >= 1 && p->Lq >= 1 && p->Lk >= 1 && p->H >= 1);
  IM2IM_REQUIRE(p->D >= 8 && p->D % 8 == 0 && p->D * p->maps <= 128);
  IM2IM_REQUIRE(p->gh >= 1 && p->gw >= 1 && (p->gh == 1 || p->gw <= 512));
  IM2IM_REQUIRE((int64_t)p->gh * p->gw <= (1 << 24));
  IM2IM_REQUIRE(p->Lk <= p->gh * p->gw);
  IM2IM_REQUIRE(p->q_start >= 0 && p->q_start <= p->gh * p->gw - p->Lq);
  IM2IM_REQUIRE(std::isfinite(p->scale));
  const int64_t e = p->dtype == IM2IM_BF16 ? 2 : 4;
  const void* ptr[3] = {p->q, p->k, p->v};
  const int64_t* st[3] = {p->q_stride, p->k_stride, p->v_stride};
  for (int t = 0; t < 3; ++t) {
    IM2IM_REQUIRE((reinterpret_cast<uintptr_t>(ptr[t]) & 15) == 0);
    IM2IM_REQUIRE(st[t][1] * e * KEYS < (1ll << 31));
    for (int x = 0; x < 3; ++x) IM2IM_REQUIRE(st[t][x] >= 0 && (st[t][x] * e) % 16 == 0);
  }
  a->q = p->q; a->k = p->k; a->v = p->v;
  for (int x = 0; x < 3; ++x) { a->qs[x] = p->q_stride[x]; a->ks[x] = p->k_stride[x]; a->vs[x] = p->v_stride[x]; }
  a->line = p->line; a->lengths = p->lengths; a->lam = p->lam;
  a->B = p->B; a->Lq = p->Lq; a->Lk = p->Lk; a->H = p->H; a->d = p->D; a->dv = p->D * p->maps;
  a->gw = p->gh == 1 ? 1 << 25 : p->gw;
  a->line_len = (2 * p->gh - 1) * (2 * p->gw - 1);
  a->line_off = (p->gh - 1) * (2 * p->gw - 1) + p->gw - 1;
  a->q_start = p->q_start;
  a->row4 = p->gh == 1 || p->gw % 4 == 0;
  a->row4q = a->row4 && p->q_start % 4 == 0;
  a->nk = (int)cdiv(p->Lk, ROWS);
  a->scale = p->scale;
  a->window = round64(window_floats(p->gh, p->gw) + 4);            // a run of four may reach three over the end
  IM2IM_REQUIRE((int64_t)p->B * p->H * p->Lq < (1ll << 31));
  IM2IM_REQUIRE((int64_t)p->B * p->H * std::max(cdiv(p->Lq, ROWS), cdiv(p->Lk, ROWS)) < (1ll << 32) / (64 * WAVES));      // work-items of a launch
  return IM2IM_OK;
}

// Half as many queries for each workgroup where there would be fewer than two workgroups a CU (23 -> 20.5 us for 320 of them: 10 x 20x20 x 8 x 64),
// or one query has the workgroup for itself
static void set_queries(AttnArgs* a) {
  a->ks_q = a->Lq == 1 || (int64_t)a->B * a->H * cdiv(a->Lq, ROWS) < 512 ? 2 : 1;
  a->nq = (int)cdiv(a->Lq, ROWS / a->ks_q);
}

// Parts of the keys: with fewer workgroups than two for each of the 256 CUs the rest of the chip takes key tiles (a single token against
// 4096 keys: 8 workgroups without).
static int key_splits(const AttnArgs& a) {
  const int64_t items = (int64_t)a.B * a.H * a.nq, tiles = cdiv(a.Lk, KEYS);
  if (items >= 256 || tiles < 2) return 1;
  int64_t n = cdiv(512, items);
  if (n > tiles) n = tiles;
  return (int)cdiv(tiles, cdiv(tiles, n));
}

template <typename T, int DQ, int DV, int MAPS, bool SAVE, bool ROW4> static int launch_fwd(const AttnArgs& a, hipStream_t st) {
  auto kern = a.ks_q == 2 ? attn_fwd_kernel<T, DQ, DV, MAPS, SAVE, ROW4, 2> : attn_fwd_kernel<T, DQ, DV, MAPS, SAVE, ROW4, 1>;
  if constexpr (!SAVE && ROW4)
    if (!a.line) kern = attn_fwd_kernel<T, DQ, DV, MAPS, false, true, 2, true>;
  size_t smem = buffers<T>(MAPS * DQ + DV) * (tile_bytes<T>(MAPS * DQ + DV) + KEYS * 4 + (size_t)a.window * 4);
  if (a.ks_q == 2) smem = std::max<size_t>(smem, 2 * MAPS * (DV / 2 + 2) * 64 * 4);
  if (int rc = attn_allow_lds(reinterpret_cast<const void*>(kern), smem)) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)a.B * a.H * a.nq * a.splits)), dim3(64 * WAVES), smem, st, a);
  if (int rc = check_launch("attn_fwd_kernel")) return rc;
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.Lq;
    if (a.splits >= 8) hipLaunchKernelGGL((attn_combine_kernel<T, MAPS, 8>), dim3((unsigned)rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_combine_kernel<T, MAPS, 1>), dim3((unsigned)cdiv(rows, 8)), dim3(256), 0, st, a);
    return check_launch("attn_combine_kernel");
  }
  return IM2IM_OK;
}

template <typename T, int DQ, int DV, int MAPS, bool SAVE> static int launch_fwd(const AttnArgs& a, hipStream_t st) {
  return a.row4 || !a.line ? launch_fwd<T, DQ, DV, MAPS, SAVE, true>(a, st) : launch_fwd<T, DQ, DV, MAPS, SAVE, false>(a, st);
}

template <typename T, bool SAVE> static int dispatch_fwd(const AttnArgs& a, int maps, hipStream_t st) {
  if (maps == 2) return a.d <= 32 ? launch_fwd<T, 32, 64, 2, SAVE>(a, st) : launch_fwd<T, 64, 128, 2, SAVE>(a, st);
  if (a.d <= 32) return launch_fwd<T, 32, 32, 1, SAVE>(a, st);
  if (a.d <= 64) return launch_fwd<T, 64, 64, 1, SAVE>(a, st);
  return launch_fwd<T, 128, 128, 1, SAVE>(a, st);
}

}  // namespace im2im

using namespace im2im;

extern "C" int64_t im2im_relpos_line_len(int32_t gh, int32_t gw) {
  if (gh < 1 || gw < 1 || (int64_t)gh * gw > (1 << 24)) return -1;
  return (int64_t)(2 * gh - 1) * (2 * gw - 1);
}

extern "C" int im2im_relpos_line(const float* table, int32_t ny, int32_t nx, int32_t H, const int32_t* thr_y, const int32_t* thr_x, int32_t gh,
                                 int32_t gw, float* line, im2im_stream_t stream) {
  IM2IM_REQUIRE(table && line && H >= 1 && H <= 65535);
  IM2IM_REQUIRE(attn_buckets_ok(ny, nx, thr_y, thr_x));
  IM2IM_REQUIRE(gh >= 1 && gw >= 1 && (int64_t)gh * gw <= (1 << 24));
  LineArgs a = {};
  a.table = table; a.line = line; a.ny = ny; a.nx = nx; a.H = H; a.gh = gh; a.gw = gw; a.len = (2 * gh - 1) * (2 * gw - 1);
  for (int m = 0; m + 1 < ny / 2; ++m) a.thr_y[m] = thr_y[m];
  for (int m = 0; m + 1 < nx / 2; ++m) a.thr_x[m] = thr_x[m];
  hipLaunchKernelGGL(relpos_line_kernel, dim3((unsigned)cdiv(a.len, 256), (unsigned)H), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch("relpos_line_kernel");
}

extern "C" int64_t im2im_attention_fwd_workspace_bytes(const im2im_attention_desc* p) {
  AttnArgs a = {};
  if (attn_check(p, &a)) return -1;
  set_queries(&a);
  const int n = key_splits(a);
  return n < 2 ? 0 : (int64_t)n * a.B * a.H * a.Lq * p->maps * (a.dv + 2) * 4;
}

extern "C" int im2im_attention_fwd(const im2im_attention_desc* p, void* out, float* lse, float* map_out, void* ws, int64_t ws_bytes,
                                   im2im_stream_t stream) {
  AttnArgs a = {};
  if (int rc = attn_check(p, &a)) return rc;
  IM2IM_REQUIRE(out && (lse != nullptr) == (map_out != nullptr));
  IM2IM_REQUIRE(p->line || !lse);
  a.out = out; a.osave = map_out;
  if (lse) { a.top = lse; a.lsum = lse + saved_rows(p); }
  if (!p->line) {
    a.table = p->table; a.ny = p->ny; a.nx = p->nx; a.window = KEYS;
    for (int m = 0; m + 1 < p->ny / 2; ++m) a.thr[m] = p->thr_y[m];
    for (int m = 0; m + 1 < p->nx / 2; ++m) a.thr[32 + m] = p->thr_x[m];
  }
  set_queries(&a);
  a.splits = key_splits(a);
  a.tiles_per_split = (int)cdiv(cdiv(a.Lk, KEYS), a.splits);
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.splits * a.B * a.H * a.Lq * p->maps;
    IM2IM_REQUIRE(ws && ws_bytes >= rows * (a.dv + 2) * 4);
    a.part = static_cast<float*>(ws);
    a.part_ml = a.part + rows * a.dv;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == IM2IM_BF16) return lse ? dispatch_fwd<bf16_t, true>(a, p->maps, st) : dispatch_fwd<bf16_t, false>(a, p->maps, st);
  return lse ? dispatch_fwd<float, true>(a, p->maps, st) : dispatch_fwd<float, false>(a, p->maps, st);
}
