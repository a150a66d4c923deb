// Grid attention, backward.  With P_m the softmax maps, A = P_1 (- lam P_2) and dP = dO V^T:
//   dV = A^T dO,   dS_1 = P_1 o (dP - D_1),   dS_2 = P_2 o (-lam dP - D_2),   D_m = rowsum(P_m o dP_m) = dO . O_m (times -lam for m = 2),
//   dQ_m = scale dS_m K_m,   dK_m = scale dS_m^T Q_m,   dbias(j - i) = sum of dS_1 + dS_2,   dlam = -sum P_2 o dP.
// Two passes, each with its own tile of the scores (computed again from Q, K and the rows' saved references and log-sums): D, the queries' gradients and the bias
// in one, the keys' and values' gradients in the other.  No global atomics: every sum has one order.
// bf16: dS and P enter the products of dQ, dK and dV as bf16 hi + lo.  A row of dS sums to zero, so of dQ only what the keys differ by is left while the
// roundings of dS to 8 bits kept all of them: 1.41 to 1.54 times as far from its value as by its own rounding alone, at every head size.  Costs a product
// more each: 78 x 20x20 x 8 x 64 queries' gradients 159 -> 172 us, keys' 121 -> 145; 8 x 32x32 x 8 x 128 136 -> 149 and 114 -> 140.
#include "attention_common.h"

namespace im2im {

// a place of the ring, summed over its copies in their order, and zeros in its place
template <bool ROW4> __device__ __forceinline__ double take_place(double* ring, unsigned place, unsigned size) {
  double s = 0.0, *at = ring + place;
#pragma unroll
  for (int c = 0; c < 2 * WAVES; ++c, at += size + 4) {
    s += at[0];
    at[0] = 0.0;
    if (ROW4 && place < 3) {                                      // what ran over the end
      s += at[size];
      at[size] = 0.0;
    }
  }
  return s;
}

// ... and into the workgroup's line (places in front of it belong to queries that are not there)
__device__ __forceinline__ void put_place(float* line, int at, double s, bool first) {
  if (at >= 0) line[at] = first ? (float)s : line[at] + (float)s;
}

// a neighbour's value, zero over the ends of 16 lanes
__device__ __forceinline__ float from_lane_before(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x111, 0xf, 0xf, true));                 // row_shr:1
}
template <int N> __device__ __forceinline__ float from_lane_behind(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x100 + N, 0xf, 0xf, true));             // row_shl:N
}

// accumulators of two waves that share their columns: the second puts its own into LDS, the first adds them
template <int N> __device__ __forceinline__ void join_halves(f32x16* acc, float* box, int kw, bool put) {
  if (put != (kw == 1)) return;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (put) box[(n * 16 + r) * 64] = acc[n][r];
      else acc[n][r] += box[(n * 16 + r) * 64];
    }
}

// -------------------------------------------------------------------------------------- queries' gradients, bias and lam
// One workgroup: 128 queries of one head, of `group_images` images in turn, against their keys in tiles of 64.
// Bias gradient: a pair's place in the line is code(j) - code(i) + off.  Within one instruction 32 lanes have 32 different queries and the
// same key, so their places differ; the other 32 lanes have another key and add to a copy of their own; each wave has its own pair
// of copies and its additions are in program order: no order is left open.  A copy is a ring over the line's index: the places
// that the following tiles cannot reach any more are summed over the copies and written, each once.  The copies are 64-bit:
// ds_add_f32 takes 193 cycles for a wave on this part, ds_add_f64 10.5 (ds_read_b32 7 to 10): 833 -> 226 us at 78 x 20x20 x 8 x 64.  ROW4: four
// queries' terms of a diagonal are summed from lane to lane first; with that and the tiles' asynchronous loads 226 -> 152 us.
// Bound by the latency of a wave's own chain (scores, probabilities, dP, dS, diagonals) at two waves a SIMD, which is what the registers allow: there the
// vector unit issues in 41 % of the cycles, the matrix unit is busy in 13 %, LDS in 26 %: 172 us at 78 x 20x20 x 8 x 64 by now.  Heads of 128 channels leave one
// wave a SIMD: 8 x 32x32 x 8 x 128 145 us.
template <typename T, int DQ, int DV, int MAPS, bool BIAS, bool ROW4, int KS>
__global__ __launch_bounds__(64 * WAVES, MAPS * DV * sizeof(T) >= 512 || (sizeof(T) == 2 && DV == 128) ? 1 : 2) void attn_bwd_q_kernel(const AttnArgs a) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr bool HILO = sizeof(T) == 2;
  constexpr int QR = ROWS / KS, NBUF = buffers<T>(MAPS * DQ + DV);
  constexpr size_t QT = tile_bytes<T>(DQ), TILES = tile_bytes<T>(MAPS * DQ + DV);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const size_t buffer = TILES + KEYS * 4 + (size_t)a.window * 4;       // tiles, codes, window
  double* ring = reinterpret_cast<double*>(smem + NBUF * buffer);          // [2 * WAVES][a.ring + 4]: four places in a row may run over the end by three
  __shared__ float red[WAVES];

  const int lin = xcd_band(blockIdx.x, gridDim.x), sp = lin % a.q_splits, item = lin / a.q_splits;
  const int qt = a.qt0 + item % a.q_here, h = item / a.q_here / a.groups, group = item / a.q_here % a.groups, slot = group * a.q_splits + sp;
  const int wave = wave_index() / KS, kw = wave_index() % KS, lane = threadIdx.x & 63, half = lane >> 5;
  const int i0 = qt * QR, i_last = min(i0 + QR, a.Lq) - 1;
  const int i = i0 + wave * 32 + (lane & 31), ic = min(i, i_last);
  const bool mine = i < a.Lq, busy = i0 + wave * 32 < a.Lq;
  const bool behind = i0 + wave * 32 + 32 > a.Lq;                      // some columns have no query: their bias, of pairs that are not there, may be NaN
  const int code_last = grid_code(a.q_start + i0 + QR - 1, a.gw);      // of 32 columns for each wave, on behind the last query
  const int aoff = code_last - grid_code(a.q_start + i, a.gw);
  const int qspan = code_last - grid_code(a.q_start + i0, a.gw);
  const float scale2 = a.scale * LOG2E, lam = MAPS == 2 ? a.lam[h] : 0.f;
  const float* line = a.line + (int64_t)h * a.line_len;
  const unsigned size = a.ring, copy = size + 4;
  double* my_ring = ring + (wave_index() * 2 + half) * copy;
  float* line_out = BIAS ? a.line_part + (((int64_t)slot * a.q_here + item % a.q_here) * a.H + h) * a.line_len : nullptr;
  const int line_shift = a.line_off - code_last, places = grid_code(a.Lk - 1, a.gw) + qspan + 1;
  // the last lane of a run: of queries side by side within 16 lanes
  const bool run_end = (lane & 15) == 15 || (a.q_start + i + 1) % a.gw == 0;
  const bool run_tail = run_end || (lane & 15) >= 13 || (a.q_start + i + 2) % a.gw == 0 || (a.q_start + i + 3) % a.gw == 0;
  float dlam = 0.f;

  if (BIAS)
    for (int w = threadIdx.x; w < 2 * WAVES * (int)copy; w += 64 * WAVES) ring[w] = 0.0;

  TileFetch<T, DQ> kt;
  TileFetch<T, DV> vt;
  kt.prepare(a.ks[1]);
  vt.prepare(a.vs[1]);
  const bool full = a.d == DQ && a.dv == DV;
  const int b0 = group * a.group_images, b1 = min(b0 + a.group_images, a.B);
  for (int b = b0; b < b1; ++b) {
    const int64_t bh = (int64_t)b * a.H + h;
    Frag qf[MAPS][DQ / M::KC], gf[DV / M::KC];
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
      load_row_frags<T, DQ>(qf[m], static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)ic * a.qs[1] + (int64_t)(MAPS * h + m) * a.qs[2], mine,
                            a.d, half);
    load_row_frags<T, DV>(gf, static_cast<const T*>(a.dout) + (((int64_t)b * a.Lq + ic) * a.H + h) * a.dv, mine, a.dv, half);
    float top[MAPS], lsum[MAPS], del[MAPS];
    f32x16 acc[MAPS][DQ / 32];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      top[m] = mine ? a.top[(bh * MAPS + m) * a.Lq + ic] : 0.f;
      lsum[m] = mine ? a.lsum[(bh * MAPS + m) * a.Lq + ic] : INFINITY;
      // D of this lane's query from dO and the saved map result, half a row in each of its two lanes; kept for the other pass
      const float* o = a.osave + ((bh * a.Lq + ic) * MAPS + m) * a.dv;
      float d = 0.f;
#pragma unroll
      for (int c = 0; c < DV / M::KC; ++c) {
        const int at = c * M::KC + half * M::NE;
        if (at < a.dv) d = M::dot(gf[c], o + at, d);
      }
      d += __shfl_xor(d, 32);
      del[m] = !mine ? 0.f : m == 0 ? d : -lam * d;
      if (mine && half == 0 && kw == 0 && sp == 0) a.delta[(bh * MAPS + m) * a.Lq + ic] = del[m];
#pragma unroll
      for (int n = 0; n < DQ / 32; ++n) acc[m][n] = zero16();
    }
    const int len = a.lengths ? max(0, min(a.lengths[b], a.Lk)) : a.Lk;
    const int t0 = sp * a.q_tiles, t1 = min(t0 + a.q_tiles, (len + KEYS - 1) / KEYS);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)(MAPS * h) * a.ks[2];
    const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)h * a.vs[2];
    int done = 0;                                                // places (line places from line_shift on) that are written

    Raster keys(t0 * KEYS, a.gw);
    auto fetch = [&](int t, char* to) {                          // tiles in their order
      const int j0 = t * KEYS, valid = min(len - j0, KEYS);
      const T *k = kp + (int64_t)j0 * a.ks[1], *v = vp + (int64_t)j0 * a.vs[1];
      if (full && valid == KEYS) {
#pragma unroll
        for (int m = 0; m < MAPS; ++m) kt.whole(to + m * QT, k + m * a.ks[2]);
        vt.whole(to + MAPS * QT, v);
      } else {
#pragma unroll
        for (int m = 0; m < MAPS; ++m) kt.part(to + m * QT, k + m * a.ks[2], a.ks[1], valid, a.d);
        vt.part(to + MAPS * QT, v, a.vs[1], valid, a.dv);
      }
      const int code = keys.code(), first = __builtin_amdgcn_readfirstlane(code), last = __builtin_amdgcn_readlane(code, valid - 1);
      keys.next();
      int* codes = reinterpret_cast<int*>(to + TILES);
      fetch_window(reinterpret_cast<float*>(codes + KEYS), line, a.line_len, first - code_last + a.line_off, last - first + qspan + 1);
      if (threadIdx.x < KEYS) codes[threadIdx.x] = 4 * (min(code, last) - first);
    };
    __syncthreads();                                             // the image before this one is done with the buffers
    if (t0 < t1) fetch(t0, smem);
    if (BIAS && t0 < t1) {                                       // places in front of this part's keys
      done = grid_code(t0 * KEYS, a.gw);
      for (int w = threadIdx.x; w < done; w += 64 * WAVES) put_place(line_out, w + line_shift, 0.0, b == b0);
    }
    for (int t = t0; t < t1; ++t) {
      const int base = grid_code(t * KEYS, a.gw), valid = min(len - t * KEYS, KEYS);
      char* at = smem + (NBUF == 2 && ((t - t0) & 1) ? buffer : 0);
      lds_loads_done();
      __syncthreads();
      if (BIAS && done < base) {                                 // a place's thread is the same for every image
        for (int w = done + ((int)threadIdx.x - done & 255); w < base; w += 64 * WAVES) {
          const double s = take_place<ROW4>(ring, (unsigned)w % size, size);
          put_place(line_out, w + line_shift, s, b == b0);
        }
        done = base;
        if (!a.ring_wide) __syncthreads();                       // else the places that this tile adds to are others
      }
      if (NBUF == 2 && t + 1 < t1) fetch(t + 1, (t - t0) & 1 ? smem : smem + buffer);
      const unsigned ring_base = (unsigned)base % size;
      const char *Ks = at, *Vs = at + MAPS * QT;
      const int* kc = reinterpret_cast<const int*>(at + TILES);
      const unsigned win = window_place(reinterpret_cast<const float*>(kc + KEYS), aoff);
      if (busy)
#pragma unroll 1
      for (int sub = kw; sub < 2; sub += KS) {
        if (sub * 32 >= valid) break;
        float bias[16];
        window_bias<ROW4>(bias, win, kc + sub * 32, half);
        // one map: the accumulators start at -D, the product ends at dP - D
        f32x16 dp = splat16(MAPS == 1 ? -del[0] : 0.f), s[MAPS];
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          s[m] = zero16();
#pragma unroll
          for (int c = 0; c < DQ / M::KC; ++c)
            s[m] = M::mma(tile_frag<T, DQ>(Ks + m * QT, sub * 32, c), qf[m][c], s[m]);
        }
#pragma unroll
        for (int c = 0; c < DV / M::KC; ++c)
          dp = M::mma(tile_frag<T, DV>(Vs, sub * 32, c), gf[c], dp);
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[m][r] = exp2_(fmaf(s[m][r], scale2, bias[r]) - top[m] - lsum[m]);
        if (valid < sub * 32 + 32) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (sub * 32 + mfma_row(r, half) >= valid)
#pragma unroll
              for (int m = 0; m < MAPS; ++m) s[m][r] = 0.f;
        }
        if (behind && !mine) {
          dp = zero16();
#pragma unroll
          for (int m = 0; m < MAPS; ++m) s[m] = zero16();
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (MAPS == 1) {
            s[0][r] *= dp[r];
            bias[r] = s[0][r];
          } else {
            dlam = fmaf(s[1][r], dp[r], dlam);
            s[0][r] *= dp[r] - del[0];
            s[1][r] *= fmaf(-lam, dp[r], -del[1]);
            bias[r] = s[0][r] + s[1][r];
          }
        }
        if (BIAS) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int* code = kc + sub * 32 + 8 * g + 4 * half;
            if constexpr (ROW4) {
              // Four keys side by side: the pairs (i, j + e) and (i + 1, j + e + 1) share a place, so they are summed from lane to lane first, and
              // four additions to LDS become one and, at the end of a run, where the sums that have no next lane lie, another.
              const float d0 = bias[4 * g], d1 = bias[4 * g + 1] + from_lane_before(run_end ? 0.f : d0);
              const float d2 = bias[4 * g + 2] + from_lane_before(run_end ? 0.f : d1);
              const float d3 = bias[4 * g + 3] + from_lane_before(run_end ? 0.f : d2);
              const float tail = (run_end ? d0 : 0.f) + from_lane_behind<1>(run_end ? d1 : 0.f) + from_lane_behind<2>(run_end ? d2 : 0.f);
              const unsigned at = ring_base + (unsigned)code[0] / 4 + aoff;                                        // < 2 size
              double* to = my_ring + min(at, at - size);
              __hip_atomic_fetch_add(to + 3, (double)d3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
              if (run_tail) __hip_atomic_fetch_add(to, (double)tail, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const unsigned at = ring_base + (unsigned)code[e] / 4 + aoff;
                __hip_atomic_fetch_add(my_ring + min(at, at - size), (double)bias[4 * g + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
              }
            }
          }
        }
#pragma unroll
        for (int ks = 0; ks < 32 / M::KC; ++ks)
#pragma unroll
          for (int m = 0; m < MAPS; ++m) {
            const Frag df = M::pack(s[m], ks), dr = M::pack_rest(s[m], df, ks);
#pragma unroll
            for (int n = 0; n < DQ / 32; ++n) {
              const Frag kf = M::template load_t<DQ>(Ks + m * QT, sub * 32, ks, n);
              acc[m][n] = M::mma(kf, df, acc[m][n]);
              if (HILO) acc[m][n] = M::mma(kf, dr, acc[m][n]);
            }
          }
      }
      if (NBUF == 1 && t + 1 < t1) {
        __syncthreads();
        fetch(t + 1, smem);
      }
    }

    if (BIAS) {
      __syncthreads();
      for (int w = done + ((int)threadIdx.x - done & 255); w < places; w += 64 * WAVES) {
        const double s = w - done < a.ring ? take_place<ROW4>(ring, (unsigned)w % size, size) : 0.0;
        put_place(line_out, w + line_shift, s, b == b0);
      }
    }
    if (KS == 2) {
      float* box = reinterpret_cast<float*>(smem) + wave * (MAPS * DQ / 2 * 64) + lane;
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MAPS; ++m) join_halves<DQ / 32>(acc[m], box + m * (DQ / 2 * 64), kw, true);
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MAPS; ++m) join_halves<DQ / 32>(acc[m], box + m * (DQ / 2 * 64), kw, false);
    }
    if (mine && kw == 0) {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        float* part = a.dq_part + ((((int64_t)sp * a.B + b) * a.Lq + i) * a.H * MAPS + MAPS * h + m) * a.d;
        T* dst = static_cast<T*>(a.dq) + b * a.dqs[0] + (int64_t)i * a.dqs[1] + (int64_t)(MAPS * h + m) * a.dqs[2];
#pragma unroll
        for (int n = 0; n < DQ / 32; ++n)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int c = n * 32 + 8 * g + 4 * half;
            if (c >= a.d) continue;
            if (KS == 2 && a.q_splits > 1)
              store4(part + c, acc[m][n][4 * g] * a.scale, acc[m][n][4 * g + 1] * a.scale, acc[m][n][4 * g + 2] * a.scale, acc[m][n][4 * g + 3] * a.scale);
            else
              store4(dst + c, acc[m][n][4 * g] * a.scale, acc[m][n][4 * g + 1] * a.scale, acc[m][n][4 * g + 2] * a.scale, acc[m][n][4 * g + 3] * a.scale);
          }
      }
    }
  }
  if (MAPS == 2) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) dlam += __shfl_xor(dlam, s);
    __syncthreads();
    if (lane == 0) red[wave_index()] = dlam;
    __syncthreads();
    if (threadIdx.x == 0) a.dlam_part[((int64_t)slot * a.nq + qt) * a.H + h] = -(red[0] + red[1] + red[2] + red[3]);
  }
}

// ---------------------------------------------------------------------------------------------- keys' and values' gradients
// One workgroup: 128 keys of one image and head (a wave has 32 of them as its columns), the queries in tiles of 64.  Scores and dP are computed
// once more (two of its four products): cheaper than writing and reading them.  78 x 20x20 x 8 x 64: 143 us, 355 TFLOP/s with them; at three workgroups a
// CU it spills and loses what the third gains.
template <typename T, int DQ, int DV, int MAPS, bool ROW4, int KS>
__global__ __launch_bounds__(64 * WAVES, DV >= 128 ? 1 : 2) void attn_bwd_kv_kernel(const AttnArgs a) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr bool HILO = sizeof(T) == 2;
  constexpr int QR = ROWS / KS, NBUF = buffers<T>(MAPS * DQ + DV);
  constexpr size_t QT = tile_bytes<T>(DQ), TILES = tile_bytes<T>(MAPS * DQ + DV);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const size_t buffer = TILES + (KEYS + 3 * MAPS * KEYS + (size_t)a.window) * 4;      // tiles, codes, [3][MAPS][KEYS] references, log-sums and D, window

  const int lin = xcd_band(blockIdx.x, gridDim.x), sp = lin % a.k_splits, item = lin / a.k_splits;
  const int kt = item % a.nk, h = item / a.nk / a.B, b = item / a.nk % a.B, bh = b * a.H + h;
  const int wave = wave_index() / KS, kw = wave_index() % KS, lane = threadIdx.x & 63, half = lane >> 5;
  const int len = a.lengths ? max(0, min(a.lengths[b], a.Lk)) : a.Lk;
  const int k0 = kt * QR, k_last = min(k0 + QR, a.Lk) - 1;
  const int j = k0 + wave * 32 + (lane & 31), jc = min(j, k_last);
  const bool mine = j < len, busy = k0 + wave * 32 < len;
  const int code_first = grid_code(k0, a.gw), koff = grid_code(jc, a.gw) - code_first, kspan = grid_code(k_last, a.gw) - code_first;
  const float scale2 = a.scale * LOG2E, lam = MAPS == 2 ? a.lam[h] : 0.f;
  const float* line = a.line + (int64_t)h * a.line_len;

  Frag kf[MAPS][DQ / M::KC], vf[DV / M::KC];
  f32x16 dk[MAPS][DQ / 32], dv[DV / 32];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    load_row_frags<T, DQ>(kf[m], static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)jc * a.ks[1] + (int64_t)(MAPS * h + m) * a.ks[2], mine, a.d,
                          half);
#pragma unroll
    for (int n = 0; n < DQ / 32; ++n) dk[m][n] = zero16();
  }
  load_row_frags<T, DV>(vf, static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)jc * a.vs[1] + (int64_t)h * a.vs[2], mine, a.dv, half);
#pragma unroll
  for (int n = 0; n < DV / 32; ++n) dv[n] = zero16();

  const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)(MAPS * h) * a.qs[2];
  const T* gp = static_cast<const T*>(a.dout) + ((int64_t)b * a.Lq * a.H + h) * a.dv;
  const int t0 = sp * a.k_tiles, t1 = k0 < len ? min(t0 + a.k_tiles, (a.Lq + KEYS - 1) / KEYS) : 0;
  const int64_t gstride = (int64_t)a.H * a.dv;
  TileFetch<T, DQ> qt;
  TileFetch<T, DV> gt;
  qt.prepare(a.qs[1]);
  gt.prepare(gstride);
  const bool full = a.d == DQ && a.dv == DV;
  Raster queries(a.q_start + t0 * KEYS, a.gw);
  auto fetch = [&](int t, char* to) {                             // tiles in their order
    const int i0 = t * KEYS, valid = min(a.Lq - i0, KEYS);
    const T *q = qp + (int64_t)i0 * a.qs[1], *g = gp + (int64_t)i0 * gstride;
    if (full && valid == KEYS) {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) qt.whole(to + m * QT, q + m * a.qs[2]);
      gt.whole(to + MAPS * QT, g);
    } else {
#pragma unroll
      for (int m = 0; m < MAPS; ++m) qt.part(to + m * QT, q + m * a.qs[2], a.qs[1], valid, a.d);
      gt.part(to + MAPS * QT, g, gstride, valid, a.dv);
    }
    int* codes = reinterpret_cast<int*>(to + TILES);
    float* rows = reinterpret_cast<float*>(codes + KEYS);
    for (int which = wave_index(); which < 3 * MAPS; which += WAVES) {          // a wave fetches one of them of a map (behind the last query P = 0)
      const float* from = which < MAPS ? a.top : which < 2 * MAPS ? a.lsum : a.delta;
      load4_to_lds(lane < valid ? from + ((int64_t)bh * MAPS + which % MAPS) * a.Lq + i0 + lane : attn_fill + (which / MAPS == 1 ? 4 : 0), rows + which * KEYS);
    }
    const int code = queries.code(), first = __builtin_amdgcn_readfirstlane(code), last = __builtin_amdgcn_readlane(code, valid - 1);
    queries.next();
    fetch_window(rows + 3 * MAPS * KEYS, line, a.line_len, code_first - last + a.line_off, last - first + kspan + 1);
    // falls along the row.  Rows without a query read the last one's bias (ROW4: the last four's): that of a pair which is not there may be NaN.
    if (threadIdx.x < KEYS) codes[threadIdx.x] = (int)threadIdx.x < valid ? 4 * (last - code) : ROW4 ? 12 : 0;
  };
  if (t0 < t1) fetch(t0, smem);
  for (int t = t0; t < t1; ++t) {
    char* at = smem + (NBUF == 2 && ((t - t0) & 1) ? buffer : 0);
    lds_loads_done();
    __syncthreads();
    if (NBUF == 2 && t + 1 < t1) fetch(t + 1, (t - t0) & 1 ? smem : smem + buffer);
    const char *Qs = at, *Gs = at + MAPS * QT;
    const int* qc = reinterpret_cast<const int*>(at + TILES);
    const float* rows = reinterpret_cast<const float*>(qc + KEYS);
    const unsigned win = window_place(rows + 3 * MAPS * KEYS, koff);
    const int valid = min(a.Lq - t * KEYS, KEYS);
    if (busy)
#pragma unroll 1
    for (int sub = kw; sub < 2; sub += KS) {
      if (sub * 32 >= valid) break;
      float bias[16];
      window_bias<ROW4, -1>(bias, win, qc + sub * 32, half);
      f32x16 dp = zero16(), s[MAPS], mix;
      constexpr bool START = MAPS == 1 && DV <= 64;              // at -D, then the product ends at dP - D (wider heads lose 5 % with it)
      if (START) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 del = *reinterpret_cast<const f32x4*>(rows + 2 * KEYS + sub * 32 + 8 * g + 4 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * g + e] = -del[e];
        }
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int c = 0; c < DQ / M::KC; ++c)
          s[m] = M::mma(tile_frag<T, DQ>(Qs + m * QT, sub * 32, c), kf[m][c], s[m]);
      }
#pragma unroll
      for (int c = 0; c < DV / M::KC; ++c)
        dp = M::mma(tile_frag<T, DV>(Gs, sub * 32, c), vf[c], dp);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          const int i = m * KEYS + sub * 32 + 8 * g + 4 * half;
          const f32x4 top = *reinterpret_cast<const f32x4*>(rows + i), lsum = *reinterpret_cast<const f32x4*>(rows + MAPS * KEYS + i);
          f32x4 del = {0.f, 0.f, 0.f, 0.f};
          if (!START) del = *reinterpret_cast<const f32x4*>(rows + 2 * MAPS * KEYS + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            const float p = exp2_(fmaf(s[m][r], scale2, bias[r]) - top[e] - lsum[e]);
            mix[r] = m == 0 ? p : fmaf(-lam, p, mix[r]);
            s[m][r] = p * (START ? dp[r] : m == 0 ? dp[r] - del[e] : fmaf(-lam, dp[r], -del[e]));
          }
        }
#pragma unroll
      for (int ks = 0; ks < 32 / M::KC; ++ks) {
        const Frag pf = M::pack(mix, ks), pr = M::pack_rest(mix, pf, ks);
#pragma unroll
        for (int n = 0; n < DV / 32; ++n) {
          const Frag gf = M::template load_t<DV>(Gs, sub * 32, ks, n);
          dv[n] = M::mma(gf, pf, dv[n]);
          if (HILO) dv[n] = M::mma(gf, pr, dv[n]);
        }
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          const Frag df = M::pack(s[m], ks), dr = M::pack_rest(s[m], df, ks);
#pragma unroll
          for (int n = 0; n < DQ / 32; ++n) {
            const Frag qf = M::template load_t<DQ>(Qs + m * QT, sub * 32, ks, n);
            dk[m][n] = M::mma(qf, df, dk[m][n]);
            if (HILO) dk[m][n] = M::mma(qf, dr, dk[m][n]);
          }
        }
      }
    }
    if (NBUF == 1 && t + 1 < t1) {
      __syncthreads();
      fetch(t + 1, smem);
    }
  }
  if (KS == 2) {
    float* box = reinterpret_cast<float*>(smem) + wave * ((MAPS * DQ + DV) / 2 * 64) + lane;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) join_halves<DQ / 32>(dk[m], box + m * (DQ / 2 * 64), kw, true);
    join_halves<DV / 32>(dv, box + MAPS * (DQ / 2 * 64), kw, true);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) join_halves<DQ / 32>(dk[m], box + m * (DQ / 2 * 64), kw, false);
    join_halves<DV / 32>(dv, box + MAPS * (DQ / 2 * 64), kw, false);
    if (kw == 1) return;
  }
  if (j >= a.Lk) return;
  if (!mine) {                                                   // a key from lengths[b] on: zeros (its column has whatever its clamped place gave)
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int n = 0; n < DQ / 32; ++n) dk[m][n] = zero16();
#pragma unroll
    for (int n = 0; n < DV / 32; ++n) dv[n] = zero16();
  }
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    float* part = a.dk_part + ((((int64_t)sp * a.B + b) * a.Lk + j) * a.H * MAPS + MAPS * h + m) * a.d;
    T* dst = static_cast<T*>(a.dk) + b * a.dks[0] + (int64_t)j * a.dks[1] + (int64_t)(MAPS * h + m) * a.dks[2];
#pragma unroll
    for (int n = 0; n < DQ / 32; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = n * 32 + 8 * g + 4 * half;
        if (c >= a.d) continue;
        if (KS == 2 && a.k_splits > 1)
          store4(part + c, dk[m][n][4 * g] * a.scale, dk[m][n][4 * g + 1] * a.scale, dk[m][n][4 * g + 2] * a.scale, dk[m][n][4 * g + 3] * a.scale);
        else
          store4(dst + c, dk[m][n][4 * g] * a.scale, dk[m][n][4 * g + 1] * a.scale, dk[m][n][4 * g + 2] * a.scale, dk[m][n][4 * g + 3] * a.scale);
      }
  }
  float* part = a.dv_part + ((((int64_t)sp * a.B + b) * a.Lk + j) * a.H + h) * a.dv;
  T* dst = static_cast<T*>(a.dvv) + b * a.dvs[0] + (int64_t)j * a.dvs[1] + (int64_t)h * a.dvs[2];
#pragma unroll
  for (int n = 0; n < DV / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = n * 32 + 8 * g + 4 * half;
      if (c >= a.dv) continue;
      if (KS == 2 && a.k_splits > 1) store4(part + c, dv[n][4 * g], dv[n][4 * g + 1], dv[n][4 * g + 2], dv[n][4 * g + 3]);
      else store4(dst + c, dv[n][4 * g], dv[n][4 * g + 1], dv[n][4 * g + 2], dv[n][4 * g + 3]);
    }
}

// ------------------------------------------------------------------------------------------------------ joining the parts
// dq, dk and dv of split calls: the parts summed in their order, four channels a thread
struct JoinArgs {
  const float* part[3];
  void* out[3];
  int64_t st[3][3], n[3];    // strides of batch, token and head; elements
  int splits[3], L[3], heads[3], d[3];
};
template <typename T> __global__ __launch_bounds__(256) void attn_join_kernel(const JoinArgs a) {
  const int w = blockIdx.y;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= a.n[w]) return;
  f32x4 s = *reinterpret_cast<const f32x4*>(a.part[w] + at);
  for (int p = 1; p < a.splits[w]; ++p) s += *reinterpret_cast<const f32x4*>(a.part[w] + p * a.n[w] + at);
  const int c = (int)(at % a.d[w]), head = (int)(at / a.d[w] % a.heads[w]);
  const int64_t token = at / a.d[w] / a.heads[w];
  store4(static_cast<T*>(a.out[w]) + token / a.L[w] * a.st[w][0] + token % a.L[w] * a.st[w][1] + head * a.st[w][2] + c, s[0], s[1], s[2], s[3]);
}

// line_sum[h][x] = sum over this launch's slots whose queries reach x, added to the launches' before it: 64 places a workgroup, the slots dealt to its 16 waves (bound by the latency of these loads:
// 10 us for 312 slots of 8 x 1521; with four waves 28)
__global__ __launch_bounds__(1024) void attn_line_sum_kernel(const AttnArgs a) {
  __shared__ double part[16][64];
  const int l = threadIdx.x & 63, x = blockIdx.x * 64 + l, h = blockIdx.y, wave = threadIdx.x >> 6;
  double acc = 0.0, *sum = a.line_sum + (int64_t)h * a.line_len + x;
  if (x < a.line_len)
    for (int qt = 0; qt < a.q_here; ++qt) {
      const int i0 = (a.qt0 + qt) * (ROWS / a.ks_q);
      const int first = grid_code(a.q_start + i0, a.gw), last = grid_code(a.q_start + min(i0 + ROWS / a.ks_q, a.Lq) - 1, a.gw);
      if (x < a.line_off - last || x > grid_code(a.Lk - 1, a.gw) - first + a.line_off) continue;
#pragma unroll 8
      for (int g = wave; g < a.groups * a.q_splits; g += 16) acc += (double)a.line_part[(((int64_t)g * a.q_here + qt) * a.H + h) * a.line_len + x];
    }
  part[wave][l] = acc;
  __syncthreads();
  if (wave == 0 && x < a.line_len) {
#pragma unroll
    for (int w = 1; w < 16; ++w) acc += part[w][l];
    *sum = a.qt0 == 0 ? acc : *sum + acc;
  }
}

struct BucketArgs {
  const double* line;    // [H][line_len] or null
  const float* dlam_part;
  float *dtable, *dlam;
  int ny, nx, H, gh, gw, slots;
  int thr_y[32], thr_x[32];
};

// distances key - query of a bucket: they are consecutive, [lo, hi) clipped to the grid
__device__ __forceinline__ void bucket_range(int b, int n, int size, const int* thr, int& lo, int& hi) {
  const int far = size - 1;
  if (n == 1) { lo = -far; hi = far + 1; return; }
  const int side = n / 2, m = b % side;
  const int from = m == 0 ? 0 : thr[m - 1], to = m + 1 < side ? thr[m] : size;      // distances [from, to)
  if (b >= side) { lo = from < 1 ? 1 : from; hi = to < size ? to : size; }
  else { lo = -(to < size ? to : size) + 1; hi = -from + 1; }
}

// one wave for each entry of the table (a bucket is a rectangle of distances), one more for each head's lam
__global__ __launch_bounds__(64) void attn_bucket_sum_kernel(const BucketArgs a) {
  const int h = blockIdx.y, b = blockIdx.x, lane = threadIdx.x;
  double acc = 0.0;
  if (b < a.ny * a.nx) {
    if (!a.line) return;
    int y0, y1, x0, x1;
    bucket_range(b / a.nx, a.ny, a.gh, a.thr_y, y0, y1);
    bucket_range(b % a.nx, a.nx, a.gw, a.thr_x, x0, x1);
    const int w = max(x1 - x0, 0), n = max(y1 - y0, 0) * w;
    const double* p = a.line + (int64_t)h * (2 * a.gh - 1) * (2 * a.gw - 1);
    for (int e = lane; e < n; e += 64) acc += p[(int64_t)(y0 + e / w + a.gh - 1) * (2 * a.gw - 1) + x0 + e % w + a.gw - 1];
  } else {
    for (int s = lane; s < a.slots; s += 64) acc += (double)a.dlam_part[(int64_t)s * a.H + h];
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) acc += __shfl_xor(acc, s);
  if (lane == 0) {
    if (b < a.ny * a.nx) a.dtable[(int64_t)b * a.H + h] = (float)acc;
    else a.dlam[h] = (float)acc;
  }
}

// -------------------------------------------------------------------------------------------------------------------- host

// Parts of the tiles that a workgroup would take in turn, at least two tiles each, for as many workgroups as the CUs hold at once, where there would be
// less than one a CU all the same (fp32: 4 x 24x24 x 4 x 2 x 32, 144 workgroups, keys' gradients 57 -> 42 us; 3 x 17x23 x 5 x 40, 105 of them, 39 -> 33 and
// 44 -> 35 us; 1 x 28x28 x 2 x 128, 26 of them, a whole training call 295 -> 145 us; joining the parts takes 5 to 6)
static int split(bool small, int64_t items, int64_t tiles, int per_cu) {
  const int64_t n = std::min<int64_t>(256 * per_cu / items, tiles / 2);
  return small && n > 1 ? (int)cdiv(tiles, cdiv(tiles, n)) : 1;
}

static void set_tiles(AttnArgs* a, const im2im_attention_desc* p) {
  // half as many queries (keys) for each workgroup where there would be less than one workgroup a CU (fp32, 3 x 17x23 x 5 x 40: 66 -> 46 and
  // 69 -> 44 us with 60 of them, 39 and 44 by now; with 320, 10 x 20x20 x 8 x 64 bf16, it costs: 39 -> 51 and 26 -> 27 us)
  a->ks_q = (int64_t)a->B * a->H * cdiv(a->Lq, ROWS) < 256 ? 2 : 1;
  a->ks_k = (int64_t)a->B * a->H * cdiv(a->Lk, ROWS) < 256 ? 2 : 1;
  a->nq = (int)cdiv(a->Lq, ROWS / a->ks_q);
  a->nk = (int)cdiv(a->Lk, ROWS / a->ks_k);
  const bool wide = a->dv > 64;                                   // as the kernels' launch bounds
  a->q_splits = split(a->ks_q == 2, (int64_t)a->B * a->H * a->nq, cdiv(a->Lk, KEYS), wide || (p->dtype == IM2IM_F32 && p->maps == 2) ? 1 : 2);
  a->k_splits = split(a->ks_k == 2, (int64_t)a->B * a->H * a->nk, cdiv(a->Lq, KEYS), wide ? 1 : 2);
}

struct BwdLayout { int64_t delta, part, line, dlam, dq, dk, dv, bytes; };
static BwdLayout bwd_layout(const AttnArgs& a, int maps, bool table) {
  const auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  BwdLayout l;
  l.delta = 0;
  l.line = up((int64_t)a.B * a.H * maps * a.Lq * 4);
  l.part = l.line + (table ? up((int64_t)a.H * a.line_len * 8) : 0);
  l.dlam = l.part + (table ? up((int64_t)a.groups * a.q_splits * a.q_chunk * a.H * a.line_len * 4) : 0);
  l.dq = l.dlam + up((int64_t)a.groups * a.q_splits * a.nq * a.H * 4);
  l.dk = l.dq + (a.q_splits > 1 ? up((int64_t)a.q_splits * a.B * a.Lq * a.H * maps * a.d * 4) : 0);
  l.dv = l.dk + (a.k_splits > 1 ? up((int64_t)a.k_splits * a.B * a.Lk * a.H * maps * a.d * 4) : 0);
  l.bytes = l.dv + (a.k_splits > 1 ? up((int64_t)a.k_splits * a.B * a.Lk * a.H * a.dv * 4) : 0);
  return l;
}

// Each workgroup of the queries' gradients writes a line of its own, which is as long as four times the tokens: what has to be bounded.  One image a
// workgroup where that takes at most 256 MiB and the workspace holds it; else several in turn (they add to their line in memory, a read and a wait
// a tile).  Where one group of all images takes more than 1 GiB, or than the workspace holds, the pass is cut into launches of as many query
// tiles as fit, whose lines are summed one launch after the other (8 heads: 256x256 tokens in four launches of 1024 workgroups).
static BwdLayout set_groups(AttnArgs* a, int maps, bool table, int64_t ws_bytes) {
  int64_t groups = a->B;
  a->q_chunk = a->nq;
  if (a->q_splits > 1 || a->k_splits > 1) {                       // parts, if the workspace holds them
    a->groups = a->B;
    a->group_images = 1;
    const BwdLayout l = bwd_layout(*a, maps, table);
    if (l.bytes <= ws_bytes && l.bytes <= 256ll << 20) return l;
    a->q_splits = a->k_splits = 1;
  }
  if (table) groups = std::max<int64_t>(1, std::min<int64_t>(groups, (256ll << 20) / ((int64_t)a->H * a->nq * a->line_len * 4)));
  for (a->group_images = (int)cdiv(a->B, groups);; ++a->group_images) {
    a->groups = (int)cdiv(a->B, a->group_images);
    const BwdLayout l = bwd_layout(*a, maps, table);
    if (l.bytes <= ws_bytes && l.dlam - l.part <= 1ll << 30) return l;
    if (a->groups == 1 && !table) return l;
    if (a->groups == 1) break;
  }
  const int64_t tile = (int64_t)a->H * a->line_len * 4;
  a->q_chunk = 0;
  const int64_t room = std::min<int64_t>(1ll << 30, ws_bytes - bwd_layout(*a, maps, table).bytes);
  a->q_chunk = (int)std::max<int64_t>(1, std::min<int64_t>(a->nq, room / 256 * 256 / tile));
  a->q_chunk = (int)cdiv(a->nq, cdiv(a->nq, a->q_chunk));
  return bwd_layout(*a, maps, table);
}

template <typename T, int DQ, int DV, int MAPS, bool BIAS, bool ROW4> static int launch_bwd_q(const AttnArgs& a, hipStream_t st) {
  auto kern = a.ks_q == 2 ? attn_bwd_q_kernel<T, DQ, DV, MAPS, BIAS, ROW4, 2> : attn_bwd_q_kernel<T, DQ, DV, MAPS, BIAS, ROW4, 1>;
  const size_t smem = buffers<T>(MAPS * DQ + DV) * (tile_bytes<T>(MAPS * DQ + DV) + KEYS * 4 + (size_t)a.window * 4) +
                      (size_t)(BIAS ? 2 * WAVES * (a.ring + 4) : 0) * 8;
  if (int rc = attn_allow_lds(reinterpret_cast<const void*>(kern), smem)) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.groups * a.H * a.q_here * a.q_splits)), dim3(64 * WAVES), smem, st, a);
  return check_launch("attn_bwd_q_kernel");
}

template <typename T, int DQ, int DV, int MAPS, bool ROW4> static int launch_bwd_kv(const AttnArgs& a, hipStream_t st) {
  auto kern = a.ks_k == 2 ? attn_bwd_kv_kernel<T, DQ, DV, MAPS, ROW4, 2> : attn_bwd_kv_kernel<T, DQ, DV, MAPS, ROW4, 1>;
  size_t smem = buffers<T>(MAPS * DQ + DV) * (tile_bytes<T>(MAPS * DQ + DV) + (KEYS + 3 * MAPS * KEYS + (size_t)a.window) * 4);
  if (a.ks_k == 2) smem = std::max<size_t>(smem, (size_t)(MAPS * DQ + DV) * 64 * 4);
  if (int rc = attn_allow_lds(reinterpret_cast<const void*>(kern), smem)) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)a.B * a.H * a.nk * a.k_splits)), dim3(64 * WAVES), smem, st, a);
  return check_launch("attn_bwd_kv_kernel");
}

template <typename T, int DQ, int DV, int MAPS> static int launch_bwd(const AttnArgs& a, hipStream_t st) {
  int rc = IM2IM_OK;
  for (AttnArgs c = a; c.qt0 < a.nq; c.qt0 += a.q_chunk) {
    c.q_here = std::min(a.q_chunk, a.nq - c.qt0);
    if (a.line_part) rc = a.row4q ? launch_bwd_q<T, DQ, DV, MAPS, true, true>(c, st) : launch_bwd_q<T, DQ, DV, MAPS, true, false>(c, st);
    else rc = a.row4q ? launch_bwd_q<T, DQ, DV, MAPS, false, true>(c, st) : launch_bwd_q<T, DQ, DV, MAPS, false, false>(c, st);
    if (rc) return rc;
    if (!a.line_part) continue;
    hipLaunchKernelGGL(attn_line_sum_kernel, dim3((unsigned)cdiv(a.line_len, 64), (unsigned)a.H), dim3(1024), 0, st, c);
    if ((rc = check_launch("attn_line_sum_kernel"))) return rc;
  }
  // queries four by four: whole runs of four only (a band may end within one)
  rc = a.row4q && a.Lq % 4 == 0 ? launch_bwd_kv<T, DQ, DV, MAPS, true>(a, st) : launch_bwd_kv<T, DQ, DV, MAPS, false>(a, st);
  if (rc || (a.q_splits == 1 && a.k_splits == 1)) return rc;
  JoinArgs j = {};
  int n = 0;
  const auto add = [&](const float* part, void* out, const int64_t* stride, int splits, int L, int heads, int d) {
    if (splits == 1) return;
    j.part[n] = part; j.out[n] = out; j.splits[n] = splits; j.L[n] = L; j.heads[n] = heads; j.d[n] = d;
    j.n[n] = (int64_t)a.B * L * heads * d;
    for (int x = 0; x < 3; ++x) j.st[n][x] = stride[x];
    ++n;
  };
  add(a.dq_part, a.dq, a.dqs, a.q_splits, a.Lq, a.H * MAPS, a.d);
  add(a.dk_part, a.dk, a.dks, a.k_splits, a.Lk, a.H * MAPS, a.d);
  add(a.dv_part, a.dvv, a.dvs, a.k_splits, a.Lk, a.H, a.dv);
  hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)cdiv(std::max(j.n[0], std::max(j.n[1], j.n[2])), 1024), (unsigned)n), dim3(256), 0, st, j);
  return check_launch("attn_join_kernel");
}

template <typename T> static int dispatch_bwd(const AttnArgs& a, int maps, hipStream_t st) {
  if (maps == 2) return a.d <= 32 ? launch_bwd<T, 32, 64, 2>(a, st) : launch_bwd<T, 64, 128, 2>(a, st);
  if (a.d <= 32) return launch_bwd<T, 32, 32, 1>(a, st);
  if (a.d <= 64) return launch_bwd<T, 64, 64, 1>(a, st);
  return launch_bwd<T, 128, 128, 1>(a, st);
}

}  // namespace im2im

using namespace im2im;

extern "C" int64_t im2im_attention_bwd_workspace_bytes(const im2im_attention_desc* p, int32_t want_table) {
  AttnArgs a = {};
  if (attn_check(p, &a)) return -1;
  set_tiles(&a, p);
  return set_groups(&a, p->maps, want_table != 0, INT64_MAX).bytes;
}

extern "C" int im2im_attention_bwd(const im2im_attention_desc* p, const im2im_attention_grads* g, void* ws, int64_t ws_bytes,
                                   im2im_stream_t stream) {
  AttnArgs a = {};
  if (int rc = attn_check(p, &a)) return rc;
  IM2IM_REQUIRE(g != nullptr);
  IM2IM_REQUIRE(g->dout && g->lse && g->map_out && g->dq && g->dk && g->dv);
  IM2IM_REQUIRE(p->maps == 1 || g->dlam);
  IM2IM_REQUIRE((reinterpret_cast<uintptr_t>(g->dout) & 15) == 0);
  const int64_t e = p->dtype == IM2IM_BF16 ? 2 : 4;
  const void* ptr[3] = {g->dq, g->dk, g->dv};
  const int64_t* stride[3] = {g->dq_stride, g->dk_stride, g->dv_stride};
  for (int t = 0; t < 3; ++t) {
    IM2IM_REQUIRE((reinterpret_cast<uintptr_t>(ptr[t]) & 15) == 0);
    for (int x = 0; x < 3; ++x) IM2IM_REQUIRE(stride[t][x] > 0 && (stride[t][x] * e) % 16 == 0);
  }
  const bool table = g->dtable != nullptr;
  IM2IM_REQUIRE(p->line && (!table || attn_buckets_ok(p->ny, p->nx, p->thr_y, p->thr_x)));
  IM2IM_REQUIRE((int64_t)a.H * a.dv * e * KEYS < (1ll << 31));
  set_tiles(&a, p);
  const BwdLayout l = set_groups(&a, p->maps, table, ws_bytes);
  IM2IM_REQUIRE(ws && ws_bytes >= l.bytes && (reinterpret_cast<uintptr_t>(ws) & 15) == 0);
  char* w = static_cast<char*>(ws);
  a.dout = g->dout; a.top = const_cast<float*>(g->lse); a.lsum = a.top + saved_rows(p); a.osave = const_cast<float*>(g->map_out); a.delta = reinterpret_cast<float*>(w + l.delta);
  a.dq = g->dq; a.dk = g->dk; a.dvv = g->dv;
  for (int x = 0; x < 3; ++x) { a.dqs[x] = g->dq_stride[x]; a.dks[x] = g->dk_stride[x]; a.dvs[x] = g->dv_stride[x]; }
  a.line_part = table ? reinterpret_cast<float*>(w + l.part) : nullptr;
  a.line_sum = reinterpret_cast<double*>(w + l.line);
  a.dlam_part = reinterpret_cast<float*>(w + l.dlam);
  a.dq_part = reinterpret_cast<float*>(w + l.dq); a.dk_part = reinterpret_cast<float*>(w + l.dk); a.dv_part = reinterpret_cast<float*>(w + l.dv);
  a.q_tiles = (int)cdiv(cdiv(p->Lk, KEYS), a.q_splits); a.k_tiles = (int)cdiv(cdiv(p->Lq, KEYS), a.k_splits);
  // a ring of the window and one tile's advance: a tile's places are then none of those that are being written, and one barrier a tile will do.
  // Where LDS does not hold that (grids over 278 wide), the window alone, and a second barrier.
  a.ring = round64(window_floats(p->gh, p->gw) + code_span(KEYS + 1, p->gh, p->gw));
  a.ring_wide = a.ring <= 1088;
  if (!a.ring_wide) a.ring = round64(window_floats(p->gh, p->gw));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (int rc = p->dtype == IM2IM_BF16 ? dispatch_bwd<bf16_t>(a, p->maps, st) : dispatch_bwd<float>(a, p->maps, st)) return rc;
  if (!table && p->maps == 1) return IM2IM_OK;
  BucketArgs s = {};
  s.line = table ? a.line_sum : nullptr;
  s.dlam_part = a.dlam_part; s.dtable = g->dtable; s.dlam = g->dlam;
  s.ny = table ? p->ny : 0; s.nx = table ? p->nx : 0; s.H = a.H; s.gh = p->gh; s.gw = p->gw; s.slots = a.groups * a.q_splits * a.nq;
  for (int m = 0; m + 1 < s.ny / 2; ++m) s.thr_y[m] = p->thr_y[m];
  for (int m = 0; m + 1 < s.nx / 2; ++m) s.thr_x[m] = p->thr_x[m];
  hipLaunchKernelGGL(attn_bucket_sum_kernel, dim3((unsigned)(s.ny * s.nx + (p->maps == 2)), (unsigned)a.H), dim3(64), 0, st, s);
  return check_launch("attn_bucket_sum_kernel");
}
