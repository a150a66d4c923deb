// Shared pieces of the grid-attention kernels (attention_fwd.hip, attention_bwd.hip).
//
// Tokens are the pixels of a gh x gw grid in raster order.  With code(t) = (t / gw) * (2 gw - 1) + t % gw the learned bias of a
// (query i, key j) pair is line[code(j) - code(i) + off], off = code(gh gw - 1): one vector per head, expanded from the bucket table
// (im2im_relpos_line; a single row counts as one of endless width: code(t) = t), so a pair's bias is one subtraction and one LDS read, and its gradient one LDS add.
//
// MFMA shape: v_mfma_f32_32x32x16_bf16 (fp32: four v_mfma_f32_32x32x2_f32 per 16-byte fragment).  In the 32 x 32 result lane l holds column
// l % 32 and rows row(r) = 8 (r / 4) + 4 (l / 32) + r % 4, r = 0..15.  Scores are computed TRANSPOSED (keys as rows, queries as
// columns; the key gradients the other way round): a softmax row then lives in one lane pair, its running maximum and sum are plain
// per-lane registers, and the probabilities are already in the layout of the next product's right operand -- they never go through
// LDS.  That product needs its left operand transposed: ds_read_b64_tr_b16 (fp32: scalar reads).
#pragma once
#include "common.h"
#include "dtypes.h"

namespace im2im {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

struct AttnArgs {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];        // element strides: batch, token, head
  const float* line;                  // [H][line_len], in units of log2
  const float* table;                 // [ny][nx][H]: a single query's bias, when there is no line
  int ny, nx, thr[64];                // smallest distance of bucket 1, 2, ...: down from 0 on, across from 32 on
  const int32_t* lengths;             // [B] or null
  const float* lam;                   // [H] (two maps)
  int B, Lq, Lk, H, d, dv, gw, line_len, line_off, q_start, nq, nk;
  int ks_q, ks_k;                     // waves that share 32 queries (keys): 1 or 2
  int window;                         // floats of LDS for the window of `line` that a tile reaches
  int row4, row4q;                    // four keys (and queries) from a multiple of four on lie side by side in the grid
  float scale;                        // of the scores
  // forward
  void* out;                          // [B][Lq][H][dv]
  // a row's reference (its maximum, or up to 2^8 less) and the log2 of its probabilities' sum over that, [B*H][MAPS][Lq] each, or null.  Apart: a
  // bias of 1e7 is 2^24 times the sum's logarithm, of which one float for both would keep nothing.
  float *top, *lsum;
  float* osave;                       // [B*H][Lq][MAPS][dv] or null: each map's own result in 32 bits
  float* part;                        // split keys: [splits][B*H*Lq][MAPS][dv]
  float* part_ml;                     //             [splits][B*H*Lq][MAPS][2]
  int splits, tiles_per_split;
  // backward
  const void* dout;                   // [B][Lq][H][dv]
  float* delta;                       // [B*H][MAPS][Lq]: D
  void *dq, *dk, *dvv;
  int64_t dqs[3], dks[3], dvs[3];
  float* line_part;                   // [groups * q_splits * q_chunk][H][line_len] or null
  double* line_sum;                   // [H][line_len]
  float* dlam_part;                   // [groups * q_splits * nq][H]
  int q_chunk, qt0, q_here;           // query tiles of a launch of the queries' pass at most; this launch's first and how many
  int groups, group_images, ring, ring_wide;   // ring: places in one copy of the LDS accumulator
  int q_splits, q_tiles, k_splits, k_tiles;    // parts of the keys (queries) for the queries' (keys') gradients, tiles in each
  float *dq_part, *dk_part, *dv_part;          // [splits][B][tokens][heads][channels]
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEYS = 64;              // keys (queries in the key-gradient kernel) of one LDS tile
constexpr int WAVES = 4, ROWS = 32 * WAVES;   // queries (keys) of a workgroup: 32 columns for each wave

// Where 16-byte piece `slot` of row r (0..15, and on in steps of 16 rows) of an LDS tile with BYTES a row lies: rows are dense, their pieces
// permuted so that both ways of reading a tile meet all 64 banks: 16 rows' piece of the same place, and 4 rows' 64-byte stretch (transposed).
template <int BYTES> __device__ __forceinline__ int place(int r, int slot) {
  const int s = BYTES == 64 ? (r >> 2) & 3 : BYTES == 128 ? (r & 2) << 1 | (r & 4) >> 1 | (r & 8) >> 3 : (r & 3) << 2 | (r >> 2 & 3);
  return r * BYTES + ((slot ^ s) << 4);
}

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  static constexpr int KC = 16, NE = 8;          // reduction length of a fragment, elements of it in a lane
  using Frag = short8;
  static __device__ __forceinline__ Frag zero() { return short8{0, 0, 0, 0, 0, 0, 0, 0}; }
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
  }
  // result registers NE t .. NE t + NE - 1 as a right operand (the reduction order matches load_t's)
  static __device__ __forceinline__ Frag pack(const f32x16& s, int t) {
    bf16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (__bf16)s[8 * t + e];
    return __builtin_bit_cast(short8, r);
  }
  static __device__ __forceinline__ Frag pack_rest(const f32x16& s, Frag hi, int t) {   // what pack() rounded away
    const u32x4 h = __builtin_bit_cast(u32x4, hi);
    bf16x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[2 * e] = (__bf16)(s[8 * t + 2 * e] - __uint_as_float(h[e] << 16));
      r[2 * e + 1] = (__bf16)(s[8 * t + 2 * e + 1] - __uint_as_float(h[e] & 0xffff0000u));
    }
    return __builtin_bit_cast(short8, r);
  }
  static __device__ __forceinline__ float dot(Frag f, const float* x, float acc) {
    const bf16x8 v = as_bf16x8(f);
    const f32x4 lo = *reinterpret_cast<const f32x4*>(x), hi = *reinterpret_cast<const f32x4*>(x + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = fmaf((float)v[e], lo[e], acc);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = fmaf((float)v[4 + e], hi[e], acc);
    return acc;
  }
  // left operand taken transposed from an LDS tile: lane = column 32 n + l % 32, reduction = rows row0 + row(NE t + e)
  template <int D> static __device__ __forceinline__ Frag load_t(const char* tile, int row0, int t, int n) {
    const int lane = threadIdx.x & 63, q = lane & 15, r = 4 * (lane >> 5) + (q >> 2), slot = n * 4 + 2 * ((lane >> 4) & 1) + ((q & 3) >> 1);
    const char* p = tile + (row0 + 16 * t) * (2 * D) + (q & 1) * 8;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(p + place<D * 2>(r, slot)));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(p + place<D * 2>(r + 8, slot)));
    return short8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};
template <> struct Mma<float> {
  static constexpr int KC = 8, NE = 4;
  using Frag = f32x4;
  static __device__ __forceinline__ Frag zero() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag pack(const f32x16& s, int t) { return f32x4{s[4 * t], s[4 * t + 1], s[4 * t + 2], s[4 * t + 3]}; }
  static __device__ __forceinline__ Frag pack_rest(const f32x16&, Frag, int) { return zero(); }
  static __device__ __forceinline__ float dot(Frag f, const float* x, float acc) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(x);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = fmaf(f[e], v[e], acc);
    return acc;
  }
  template <int D> static __device__ __forceinline__ Frag load_t(const char* tile, int row0, int t, int n) {
    const int lane = threadIdx.x & 63, slot = n * 8 + ((lane & 31) >> 2);
    const char* p = tile + (row0 + 8 * (t & ~1)) * (4 * D) + (lane & 3) * 4;
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = *reinterpret_cast<const float*>(p + place<D * 4>(8 * (t & 1) + 4 * (lane >> 5) + e, slot));
    return f;
  }
};

template <typename T> __device__ __forceinline__ typename Mma<T>::Frag load_frag(const T* p) { return *reinterpret_cast<const typename Mma<T>::Frag*>(p); }
// left operand: fragment c of the 32 rows from row0 on
template <typename T, int D> __device__ __forceinline__ typename Mma<T>::Frag tile_frag(const char* tile, int row0, int c) {
  const int lane = threadIdx.x & 63;
  constexpr int BYTES = D * (int)sizeof(T);
  return *reinterpret_cast<const typename Mma<T>::Frag*>(tile + (row0 + (lane & 16)) * BYTES + place<BYTES>(lane & 15, 2 * c + (lane >> 5)));
}

__device__ __forceinline__ f32x16 zero16() { return f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ f32x16 splat16(float v) { return f32x16{v, v, v, v, v, v, v, v, v, v, v, v, v, v, v, v}; }
__device__ __forceinline__ int mfma_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }
__device__ __forceinline__ int grid_code(int t, int gw) { return (t / gw) * (2 * gw - 1) + t % gw; }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// a lane's right-operand fragments of one row (queries: columns of the transposed scores), zero behind the row's d elements
template <typename T, int D> __device__ __forceinline__ void load_row_frags(typename Mma<T>::Frag* f, const T* row, bool valid, int d, int half) {
#pragma unroll
  for (int c = 0; c < D / Mma<T>::KC; ++c) {
    const int at = c * Mma<T>::KC + half * Mma<T>::NE;
    f[c] = valid && at < d ? load_frag<T>(row + at) : Mma<T>::zero();
  }
}

// Loads straight into LDS (global_load_lds): 64 lanes' 16 or 4 bytes, each from its own address, to consecutive places.  What has to be zero (rows
// behind the last, elements behind a row) or infinite comes from here.  A masked row may hold anything, infinities and NaN too: a zero
// probability does not silence them in a product, a zero operand does.
static __device__ const float attn_fill[8] = {0.f, 0.f, 0.f, 0.f, INFINITY, INFINITY, INFINITY, INFINITY};
// Written as assembly: behind the builtin the compiler waits for every such load before the next transposed LDS read, which is the prefetch
// lost (the instructions have no result in registers; lds_loads_done() is their wait).  A load into LDS may follow the scalar write of M0 that it reads
// only after one wait state, which the compiler does not put into inline assembly: the s_nop.  (Five after a vector instruction's write of a base in scalar
// registers, v_readfirstlane among them: the s_mov and an s_nop of four.)  M0 is reserved, so it is no clobber that could be named:
// nothing else in the files that include this may use it (tests/test_lds_dma_cpu.py reads the built library for both).
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ void load16_to_lds(const void* from, const void* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_address(to)), "v"(from) : "memory");
}
__device__ __forceinline__ void load4_to_lds(const void* from, const void* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_address(to)), "v"(from) : "memory");
}
// every load of this wave into LDS is there; before the barrier behind which others read it
__device__ __forceinline__ void lds_loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt 0
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ __forceinline__ void load16_to_lds(const void* base, unsigned offset, const void* to) {       // uniform base, bytes of the lane from there
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %2, %1" ::"s"(lds_address(to)), "s"(base), "v"(offset) : "memory");
}

// KEYS rows of a tile, by the whole workgroup.  A lane's places are the same for every tile: their offsets are kept (64 rows of a tensor are
// within 2 GiB, attn_check).  Tiles with rows or elements to be zeroed choose an address for each piece.
template <typename T, int D> struct TileFetch {
  static constexpr int BYTES = D * (int)sizeof(T), PR = BYTES / 16, V = 16 / (int)sizeof(T), N = KEYS * PR / (64 * WAVES);
  unsigned offset[N];
  __device__ __forceinline__ static int piece_row(int n) { return ((n * WAVES + wave_index()) * 64 + ((int)threadIdx.x & 63)) / PR; }
  __device__ __forceinline__ static int piece_column(int n) {                                  // the piece that lies there
    const int r = piece_row(n) & 15;
    return ((place<BYTES>(r, (threadIdx.x & 63) % PR) - r * BYTES) >> 4) * V;
  }
  __device__ __forceinline__ void prepare(int64_t stride) {
#pragma unroll
    for (int n = 0; n < N; ++n) offset[n] = (unsigned)(piece_row(n) * stride + piece_column(n)) * (unsigned)sizeof(T);
  }
  __device__ __forceinline__ void whole(char* to, const T* src) const {
#pragma unroll
    for (int n = 0; n < N; ++n) load16_to_lds(src, offset[n], to + (n * WAVES + wave_index()) * 1024);
  }
  __device__ __forceinline__ static void part(char* to, const T* src, int64_t stride, int valid, int d) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = piece_row(n), c = piece_column(n);
      load16_to_lds(r < valid && c < d ? static_cast<const void*>(src + r * stride + c) : attn_fill, to + (n * WAVES + wave_index()) * 1024);
    }
  }
};

// the code of the token at lane l of a tile of 64, tile after tile without a division
struct Raster {
  int row, col, step_row, step_col, gw;
  __device__ __forceinline__ Raster(int first, int gw_) : gw(gw_) {
    const int t = first + (threadIdx.x & 63);
    row = t / gw;
    col = t % gw;
    step_row = KEYS / gw;
    step_col = KEYS % gw;
  }
  __device__ __forceinline__ int code() const { return row * (2 * gw - 1) + col; }
  __device__ __forceinline__ void next() {
    row += step_row;
    col += step_col;
    if (col >= gw) {
      col -= gw;
      ++row;
    }
  }
};

// `n` floats of the line from place `first` on, in whole runs of 64 (the window's size in LDS is a multiple of that).  The places of queries behind the
// last one may lie in front of the line: any value will do there.
__device__ __forceinline__ void fetch_window(float* to, const float* line, int line_len, int first, int n) {
  const int lane = threadIdx.x & 63;
  for (int w = wave_index() * 64; w < n; w += 64 * WAVES) load4_to_lds(line + max(0, min(first + w + lane, line_len - 1)), to + w);
}

// bucket of a signed distance; `thr`: lane `from` + m holds the smallest distance of bucket m + 1, searched by halves (all lanes take part)
__device__ __forceinline__ int lane_bucket(int delta, int n, int thr, int from) {
  if (n == 1) return 0;
  const int side = n / 2, t = delta < 0 ? -delta : delta;
  int b = 0;
#pragma unroll
  for (int step = 16; step >= 1; step >>= 1) {
    if (step >= side) continue;
    const int bound = __shfl(thr, from + b + step - 1);
    if (b + step < side && t >= bound) b += step;
  }
  return delta > 0 ? b + side : b;
}

// A table's entry in units of log2.  Entries over 2^126 in size would leave the range: from there on they rise half a unit for one, to 2.5e38 at most, which leaves
// them in their order and room for a score.  (Any two of them are so far apart that the larger takes all, so by how much does not matter.)
__device__ __forceinline__ float bias_log2(float t) {
  constexpr float END = 0x1p126f;
  const float size = fabsf(t);
  return size <= END || size == INFINITY ? t * LOG2E : copysignf(fmaf(size - END, 0.5f, END * LOG2E), t);
}

// LDS buffers of tiles: two (the next tile's loads run behind this tile's work, one barrier a tile), one for the widest heads in 32 bits
template <typename T> __host__ __device__ constexpr int buffers(int elements) { return elements * (int)sizeof(T) <= 512 ? 2 : 1; }
template <typename T> __host__ __device__ constexpr size_t tile_bytes(int elements) { return (size_t)KEYS * elements * sizeof(T); }

// the bias of a lane's 16 scores: at bytes codes[row] from the lane's own place in the window.  ROW4: four rows' codes are consecutive (rising or
// falling), one place serves them; behind the last valid row that may reach three places over the window's end, values that the callers mask.
typedef const __attribute__((address_space(3))) float* lds_floats;
__device__ __forceinline__ unsigned window_place(const float* win, int off) {
  unsigned p = lds_address(win) + 4 * off;
  asm("" : "+v"(p));                                             // one register, not the window's place added again to each read
  return p;
}
template <bool ROW4, int STEP = 1> __device__ __forceinline__ void window_bias(float* bias, unsigned place, const int* codes, int half) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ROW4) bias[4 * g + e] = ((lds_floats)(uintptr_t)(place + codes[8 * g + 4 * half]))[STEP * e];
      else bias[4 * g + e] = *(lds_floats)(uintptr_t)(place + codes[8 * g + 4 * half + e]);
    }
}

// four consecutive elements (16 bytes of fp32, 8 bytes of bf16)
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d}; }
__device__ __forceinline__ void store4(bf16_t* p, float a, float b, float c, float d) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<bf16x4*>(p) = bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
}

// a contiguous band of the work list for each of the 8 XCDs (workgroups are dealt to them round-robin), so that the workgroups that share
// an image and head share an L2
__device__ __forceinline__ int xcd_band(int id, int total) {
  const int each = total >> 3, more = total & 7, x = id & 7;
  return x * each + (x < more ? x : more) + (id >> 3);
}

// distance in the line that n consecutive tokens span at most (also on behind the grid's last row)
inline int code_span(int64_t n, int gh, int gw) { return (int)(gh == 1 ? n - 1 : n - 1 + (n - 1 + gw - 1) / gw * (gw - 1)); }
inline int window_floats(int gh, int gw) { return code_span(ROWS, gh, gw) + code_span(KEYS, gh, gw) + 1; }
inline int round64(int n) { return (n + 63) / 64 * 64; }

inline int64_t saved_rows(const im2im_attention_desc* p) { return (int64_t)p->B * p->H * p->maps * p->Lq; }

bool attn_buckets_ok(int32_t ny, int32_t nx, const int32_t* thr_y, const int32_t* thr_x);
int attn_check(const im2im_attention_desc* p, AttnArgs* a);      // validates the description, fills the common fields
int attn_allow_lds(const void* kernel, size_t bytes);            // raises the kernel's dynamic LDS limit on the current device

}  // namespace im2im
