// rope_kernels.hip — per-head RMS norm of queries and keys and their rotation by positions, one pass each way, for gfx950.
//
//   forward   z = x * r * w,  r = (mean(x^2) + eps)^-1/2 over the d values of a head;   y = R(angle) z
//   backward  dz = R(angle)^T dy;  dw = sum dz * (x r);  dx = r (dz w - (x r) mean(dz w * (x r)))
// with R the rotation of pair i (dims (i, i + d/2), or (2i, 2i + 1) interleaved) by angle = position[axis(i)] * inv_freq[i]: `sections`
// gives each axis (time, height, width, ...) its run of pairs.
//
// The pass is bound by memory: d values in and out per head, a few operations each.  Layout: a thread owns 8 pairs = 16 values of one
// head (two 16-byte pieces in 16-bit types), a group of 1, 2, 4, 8 or 16 lanes one head, so the mean of squares is at most four lane
// exchanges and nothing of a head leaves its group.  The angles belong to a token, not to a head: a workgroup takes a few tokens of - where the
// samples share their positions - several samples, computes the cosines and sines once into LDS, and all heads read them there; the next
// head's pieces are in flight while one is worked on.  Angles are products in 64 bits brought to (-1/2, 1/2] turns before they are rounded to
// 32 (a position of 10^6 at frequency 1 would be off by 0.03 rad in 32 bits).  x r is computed again in the backward instead of kept: it is in
// registers anyway and would cost as much memory as x.
// Sums (mean of squares, weight gradients) in 32 bits; one rounding to the output's type at the end.
// Measured: 32 x 1025 tokens, 12 + 12 heads of 64, bf16: forward 38 us (201 MB, 5.3 TB/s), backward 69 us (302 MB, 4.4 TB/s) + 4 us for the
// weights' sums; 2 x 1571 tokens, 16 + 4 heads of 128, fp32, interleaved: forward 13 us (64 MB, 4.9 TB/s; 19 us before the threads of a head took
// its 16-byte pieces in turn).  A copy of 2 GiB reaches 4.9 TB/s.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "apgd_hip.h"
#include "convnext_hip.h"
#include "rope_internal.h"

namespace {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline int launch_status() { return static_cast<int>(hipGetLastError()); }

constexpr int kMaxAxes = 4;
constexpr int kMaxHead = 256;
constexpr int kHeads = 4096;
constexpr int kFwdGrid = 1 << 20;               // workgroups (a side) of the forward at most: they step over the rest
constexpr int kBwdGrid = 1024;                  // workgroups (a side) of the backward at most: each leaves one row of partial weight gradients

struct View {                                   // [B, N, H, d] with unit stride in d
  int64_t b, n, h;
};

struct Side {                                   // the queries' or the keys' tensors
  const void *x, *dy;                           // input; backward: the output's gradient
  void* o;                                      // forward: y; backward: dx
  const void* w;                                // [d] or NULL
  View vx, vdy, vo;
  int32_t heads;
  uint32_t magic;                               // ceil(2^32 / heads): i / heads = mulhi(i, magic) for i * heads < 2^32
};

struct RopeArgs {
  Side q, k;
  const void* pos;                              // [(B,) N, axes] or NULL
  const float* inv_freq;                        // [d / 2]
  float* part;                                  // backward: [2][gridDim.x][d] partial weight gradients or NULL
  int64_t pos_b;                                // elements between the samples' positions (0: shared)
  int64_t B, N, tiles;                          // tiles: of `tile` tokens x `samples` samples
  int32_t first1, first2, first3;               // first pair of the second, third and fourth axis (d / 2 where there is none)
  int32_t axes, d, tile, log_tile, samples, sample_tiles, w_dtype, pos_dtype, norm;
  float eps;
};

struct bf16_t { uint16_t u; };

// 8 consecutive values as loaded and as 32-bit numbers
template <typename T> struct Io;
template <> struct Io<float> {
  struct Raw { float4 a, b; };
  static __device__ __forceinline__ void widen(const Raw& r, float* x) {
    x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w; x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
  }
};
template <> struct Io<bf16_t> {
  typedef __attribute__((ext_vector_type(8))) __bf16 v8;
  using Raw = uint4;
  static __device__ __forceinline__ Raw raw8(const bf16_t* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void widen(const Raw& a, float* x) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store8(bf16_t* p, const float* x) {
    v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<__bf16>(x[i]);
    *reinterpret_cast<v8*>(p) = v;
  }
};
template <> struct Io<__half> {
  typedef __attribute__((ext_vector_type(8))) _Float16 v8;
  using Raw = v8;
  static __device__ __forceinline__ Raw raw8(const __half* p) { return *reinterpret_cast<const v8*>(p); }
  static __device__ __forceinline__ void widen(const Raw& v, float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
  }
  static __device__ __forceinline__ void store8(__half* p, const float* x) {
    v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<_Float16>(x[i]);
    *reinterpret_cast<v8*>(p) = v;
  }
};

// The 16 values of a thread: a = first members of its 8 pairs, b = second members, in 16-byte pieces that the threads of a head take in turn, so
// that each load or store covers a head's bytes without gaps.  A piece holds kPer pairs (interleaved) or their first or second members.
template <bool IL, typename T> constexpr int kPer = (IL ? 8 : 16) / static_cast<int>(sizeof(T));
template <bool IL, typename T> __device__ __forceinline__ int pair_of(int i, int j, int tph) { return kPer<IL, T> * (j + i / kPer<IL, T> * tph) + i % kPer<IL, T>; }
template <typename T> struct Pairs { typename Io<T>::Raw lo, hi; };
template <bool IL, typename T>
__device__ __forceinline__ Pairs<T> raw_pairs(const T* head, int j, int tph, int d2) {
  if constexpr (sizeof(T) == 4) {
    const float4* p = reinterpret_cast<const float4*>(head) + j;
    return Pairs<T>{{p[0], p[tph]}, {p[2 * tph], p[3 * tph]}};         // (the second members begin at d / 2 = 2 tph pieces)
  } else {
    return Pairs<T>{Io<T>::raw8(head + 8 * j), Io<T>::raw8(head + (IL ? 8 * (j + tph) : 8 * j + d2))};
  }
}
template <bool IL, typename T>
__device__ __forceinline__ void widen(const Pairs<T>& r, float* a, float* b) {
  if constexpr (IL) {
    float t[16];
    Io<T>::widen(r.lo, t);
    Io<T>::widen(r.hi, t + 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) { a[i] = t[2 * i]; b[i] = t[2 * i + 1]; }
  } else {
    Io<T>::widen(r.lo, a);
    Io<T>::widen(r.hi, b);
  }
}
template <bool IL, typename T>
__device__ __forceinline__ void store_pairs(T* head, int j, int tph, int d2, const float* a, const float* b) {
  float t[16];
  if constexpr (IL) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { t[2 * i] = a[i]; t[2 * i + 1] = b[i]; }
    a = t;
    b = t + 8;
  }
  if constexpr (sizeof(T) == 4) {
    float4* p = reinterpret_cast<float4*>(head) + j;
    p[0] = make_float4(a[0], a[1], a[2], a[3]);
    p[tph] = make_float4(a[4], a[5], a[6], a[7]);
    p[2 * tph] = make_float4(b[0], b[1], b[2], b[3]);
    p[3 * tph] = make_float4(b[4], b[5], b[6], b[7]);
  } else {
    Io<T>::store8(head + 8 * j, a);
    Io<T>::store8(head + (IL ? 8 * (j + tph) : 8 * j + d2), b);
  }
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float(static_cast<uint32_t>(x.u) << 16); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int dtype, int at) {
  if (!w) return 1.f;
  if (dtype == APGD_F32) return static_cast<const float*>(w)[at];
  return to_f32(static_cast<const T*>(w)[at]);
}

// sum over the lanes of a group (a power of two; every lane of the wavefront is here)
__device__ __forceinline__ float group_sum(float v, int group) {
  for (int m = 1; m < group; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// cosine and sine of pair i of token n of sample b
__device__ __forceinline__ float2 cos_sin(const RopeArgs& a, int64_t b, int64_t n, int i) {
  const int axis = (i >= a.first1) + (i >= a.first2) + (i >= a.first3);
  const int64_t at = b * a.pos_b + n * a.axes + axis;
  double p;
  if (a.pos_dtype == CNX_POS_F32) p = static_cast<const float*>(a.pos)[at];
  else if (a.pos_dtype == CNX_POS_I32) p = static_cast<const int32_t*>(a.pos)[at];
  else p = static_cast<double>(static_cast<const int64_t*>(a.pos)[at]);
  const double turns = p * static_cast<double>(a.inv_freq[i]) * 0.15915494309189535;        // 1 / (2 pi)
  const float f = static_cast<float>(turns - rint(turns));
  return make_float2(cospif(2.f * f), sinpif(2.f * f));
}
// those of tokens n0 .. n0 + nt - 1 of sample b: cs[t][pair]
__device__ __forceinline__ void tile_angles(const RopeArgs& a, int64_t b, int64_t n0, int nt, float2* cs) {
  const int pairs = a.d >> 1;
  for (int e = threadIdx.x; e < nt * pairs; e += blockDim.x) {
    const int t = e / pairs, i = e - t * pairs;
    cs[t * pairs + i] = cos_sin(a, b, n0 + t, i);
  }
}
__global__ __launch_bounds__(256) void rope_table_kernel(const RopeArgs a, float2* __restrict__ cs, int64_t rows) {
  const int pairs = a.d >> 1;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < rows * pairs; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / pairs, b = a.pos_b ? row / a.N : 0;
    cs[e] = cos_sin(a, b, row - b * a.N, static_cast<int>(e - row * pairs));
  }
}

// blockIdx.y: 0 = queries, 1 = keys (so that a thread holds one side's sums)
// TO: type of the results (T, or fp16 for the attention's own copy of normalised bf16 heads)
template <typename T, typename TO, bool BWD, bool IL>
__global__ __launch_bounds__(256, BWD ? 3 : 4) void qk_norm_rope_kernel(const RopeArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  float* wl = reinterpret_cast<float*>(lds_raw);                      // [2][d / 2] weights of the pairs' first and second members
  float2* cs = reinterpret_cast<float2*>(wl + a.d);                   // [tile][d / 2] cosines, sines
  const Side z = blockIdx.y ? a.k : a.q;
  const int d = a.d, pairs = d >> 1, tph = d >> 4;                    // tph: threads that hold a head
  int group = 1;
  while (group < tph) group <<= 1;
  const int j = threadIdx.x & (group - 1), g0 = threadIdx.x / group, ngroups = 256 / group;
  const bool here = j < tph;                                          // d / 16 is no power of two: the group's last lanes idle
  const int jj = here ? j : 0;
  const float rd = 1.f / static_cast<float>(d);
  if (a.norm) {
    for (int e = threadIdx.x; e < d; e += 256) {
      const int member = IL ? e & 1 : e >= pairs, pair = IL ? e >> 1 : member ? e - pairs : e;
      wl[member * pairs + pair] = weight_at<T>(z.w, a.w_dtype, e);
    }
  }
  __syncthreads();
  float sa[8], sb[8];                                                 // BWD: weight gradients of this thread's dims
#pragma unroll
  for (int i = 0; i < 8; ++i) sa[i] = sb[i] = 0.f;

  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t nt0 = tile / a.sample_tiles, n0 = nt0 * a.tile, b0 = (tile - nt0 * a.sample_tiles) * a.samples;
    const int nt = static_cast<int>(a.N - n0 < a.tile ? a.N - n0 : a.tile), ns = static_cast<int>(a.B - b0 < a.samples ? a.B - b0 : a.samples);
    const T* px = static_cast<const T*>(z.x) + b0 * z.vx.b + n0 * z.vx.n;
    const T* pg = static_cast<const T*>(z.dy) + b0 * z.vdy.b + n0 * z.vdy.n;
    TO* po = static_cast<TO*>(z.o) + b0 * z.vo.b + n0 * z.vo.n;
    // item = (sample, token, head): places past the tile's last token are passed over
    const int items = (ns << a.log_tile) * z.heads;
    struct Item { int s, t, h; bool live; };
    auto item = [&](int it) {
      const int i = it < items ? it : items - 1;
      const int q = z.heads == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), z.magic));
      Item r = {q >> a.log_tile, q & (a.tile - 1), i - q * z.heads, it < items};
      if (r.t >= nt) { r.t = nt - 1; r.live = false; }
      return r;
    };
    Item cur = item(g0);
    Pairs<T> rx, rg;
    auto load = [&](const Item& i) {
      if (!BWD || a.norm) rx = raw_pairs<IL>(px + i.s * z.vx.b + i.t * z.vx.n + i.h * z.vx.h, jj, tph, d / 2);
      if constexpr (BWD) rg = raw_pairs<IL>(pg + i.s * z.vdy.b + i.t * z.vdy.n + i.h * z.vdy.h, jj, tph, d / 2);
    };
    if (items > 0) load(cur);
    if (a.pos) {
      __syncthreads();                                                // the last tile's readers are done
      tile_angles(a, b0, n0, nt, cs);
      __syncthreads();
    }
#pragma unroll 1
    for (int it0 = 0; it0 < items; it0 += ngroups) {                  // (uniform trip count: the lane exchanges need whole wavefronts)
      float xa[8], xb[8], ga[8], gb[8], c[8], s[8];
      if (!BWD || a.norm) widen<IL, T>(rx, xa, xb);
      if constexpr (BWD) widen<IL, T>(rg, ga, gb);
      const Item now = cur;
      if (it0 + ngroups < items) {                                    // the next item's pieces
        cur = item(it0 + ngroups + g0);
        load(cur);
      }
      const bool live = here && now.live;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = a.pos ? cs[now.t * pairs + pair_of<IL, T>(i, jj, tph)] : make_float2(1.f, 0.f);
        c[i] = v.x; s[i] = v.y;
      }
      if (a.norm) {                                                   // x -> x r
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
        ss = group_sum(here ? ss : 0.f, group);
        const float r = 1.f / sqrtf(ss * rd + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) { xa[i] *= r; xb[i] *= r; }
        if constexpr (BWD) {
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {                               // the rotation's transpose, then the norm's
            const float u = fmaf(ga[i], c[i], gb[i] * s[i]), v = fmaf(gb[i], c[i], -ga[i] * s[i]);
            const float ta = u * xa[i], tb = v * xb[i];
            const int at = pair_of<IL, T>(i, jj, tph);
            const float wa = wl[at], wb = wl[pairs + at];
            sa[i] += live ? ta : 0.f;
            sb[i] += live ? tb : 0.f;
            dot = fmaf(ta, wa, fmaf(tb, wb, dot));
            ga[i] = u * wa;
            gb[i] = v * wb;
          }
          dot = group_sum(here ? dot : 0.f, group) * rd;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ga[i] = r * fmaf(-xa[i], dot, ga[i]);
            gb[i] = r * fmaf(-xb[i], dot, gb[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = pair_of<IL, T>(i, jj, tph);
            xa[i] *= wl[at];
            xb[i] *= wl[pairs + at];
          }
        }
      } else if constexpr (BWD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = fmaf(ga[i], c[i], gb[i] * s[i]);
          gb[i] = fmaf(gb[i], c[i], -ga[i] * s[i]);
          ga[i] = u;
        }
      }
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ga[i] = fmaf(xa[i], c[i], -xb[i] * s[i]);
          gb[i] = fmaf(xb[i], c[i], xa[i] * s[i]);
        }
      }
      if constexpr (!std::is_same_v<T, TO>) {                         // (a NaN stays one)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ga[i] = ga[i] > 65504.f ? 65504.f : ga[i] < -65504.f ? -65504.f : ga[i];
          gb[i] = gb[i] > 65504.f ? 65504.f : gb[i] < -65504.f ? -65504.f : gb[i];
        }
      }
      if (live) store_pairs<IL>(po + now.s * z.vo.b + now.t * z.vo.n + now.h * z.vo.h, j, tph, d / 2, ga, gb);
    }
  }
  if constexpr (BWD) {
    if (a.part) {                                                     // (uniform) the workgroup's sums, in the order of its wavefronts
      float* red = reinterpret_cast<float*>(lds_raw);                 // [4 wavefronts][d]
      __syncthreads();
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        for (int m = group; m < 64; m <<= 1) {
          sa[i] += __shfl_xor(sa[i], m, 64);
          sb[i] += __shfl_xor(sb[i], m, 64);
        }
        if (lane < group && here) {
          const int at = pair_of<IL, T>(i, j, tph), ia = IL ? 2 * at : at, ib = IL ? ia + 1 : ia + pairs;
          red[wave * d + ia] = sa[i];
          red[wave * d + ib] = sb[i];
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < d; e += 256)
        a.part[(static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * d + e] = ((red[e] + red[d + e]) + red[2 * d + e]) + red[3 * d + e];
    }
  }
}

// dw[e] = sum over the workgroups' rows, in a fixed order: 16 columns x 64 row lanes, every lane its rows one after the other
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* __restrict__ pq, int nq, const float* __restrict__ pk, int nk, int d,
                                                       float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float red[64][17];
  float* dw = blockIdx.y ? dwk : dwq;
  const float* part = blockIdx.y ? pk : pq;
  const int rows = blockIdx.y ? nk : nq;
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, e = blockIdx.x * 16 + col;        // d is a multiple of 16
  float s = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 512) {                            // eight loads at a time
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int r = r0 + u * 64 + row;
      v[u] = r < rows ? part[static_cast<int64_t>(r) * d + e] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  red[row][col] = s;
  __syncthreads();
  if (row == 0 && dw) {
    s = 0.f;
#pragma unroll
    for (int r = 0; r < 64; ++r) s += red[r][col];
    dw[e] = s;
  }
}

int check_args(RopeArgs& a, int dtype, const int32_t* sections, int64_t B, int64_t N, int32_t Hq, int32_t Hk, int32_t d) {
  if (B < 0 || N < 0 || Hq < 0 || Hk < 0 || Hq > kHeads || Hk > kHeads) return APGD_ERR_SIZE;
  if (!cnx_qk_norm_rope_supported(d)) return APGD_ERR_ARG;
  if (dtype != APGD_F32 && dtype != APGD_BF16 && dtype != APGD_F16) return APGD_ERR_DTYPE;
  if ((a.q.w || a.k.w) && a.w_dtype != APGD_F32 && a.w_dtype != dtype) return APGD_ERR_DTYPE;
  if (N > 0 && B > INT64_MAX / N) return APGD_ERR_SIZE;
  if (a.pos) {
    if (!a.inv_freq || !sections) return APGD_ERR_NULL;
    if (a.pos_dtype != CNX_POS_F32 && a.pos_dtype != CNX_POS_I32 && a.pos_dtype != CNX_POS_I64) return APGD_ERR_DTYPE;
    if (a.axes < 1 || a.axes > kMaxAxes) return APGD_ERR_ARG;
    int32_t first[kMaxAxes + 1] = {0, d / 2, d / 2, d / 2, d / 2};
    for (int i = 0; i < a.axes; ++i) {
      if (sections[i] < 0 || sections[i] > d) return APGD_ERR_ARG;
      first[i + 1] = first[i] + sections[i];
    }
    if (first[a.axes] != d / 2) return APGD_ERR_ARG;
    a.first1 = first[1]; a.first2 = first[2]; a.first3 = first[3];
  }
  a.B = B;
  a.N = N;
  a.q.heads = Hq; a.k.heads = Hk; a.d = d;
  a.q.magic = Hq > 1 ? static_cast<uint32_t>((0x100000000ULL + Hq - 1) / Hq) : 0;
  a.k.magic = Hk > 1 ? static_cast<uint32_t>((0x100000000ULL + Hk - 1) / Hk) : 0;
  return APGD_OK;
}

// Tiles: up to 8 tokens of one sample, or - where the samples share their positions - of up to 8 samples, as long as that leaves the
// chip 512 workgroups a side (fewer tokens for the smallest calls, whose time is one pass through the kernel).
void cut(RopeArgs& a) {
  a.log_tile = 3;
  while (a.log_tile > 0 && ((a.N + (1 << a.log_tile) - 1) >> a.log_tile) * a.B < 512) --a.log_tile;
  a.tile = 1 << a.log_tile;
  const int64_t token_tiles = (a.N + a.tile - 1) / a.tile;
  a.samples = 1;
  while (a.pos_b == 0 && a.samples < 8 && a.samples < a.B && token_tiles * ((a.B + 2 * a.samples - 1) / (2 * a.samples)) >= 512) a.samples *= 2;
  a.sample_tiles = static_cast<int32_t>((a.B + a.samples - 1) / a.samples);
  a.tiles = token_tiles * a.sample_tiles;
}

template <bool BWD, bool IL>
void launch(const RopeArgs& a, int dtype, bool half, unsigned grid, hipStream_t s) {
  const size_t lds = static_cast<size_t>(BWD && a.tile < 3 ? 4 : a.tile + 1) * a.d * 4;     // d weights and tile x d / 2 (cos, sin); BWD: 4 x d sums
  const dim3 blocks(grid, 2);
  if constexpr (!BWD) {
    if (half) {
      hipLaunchKernelGGL((qk_norm_rope_kernel<bf16_t, __half, false, IL>), blocks, dim3(256), lds, s, a);
      return;
    }
  }
  if (dtype == APGD_F32) hipLaunchKernelGGL((qk_norm_rope_kernel<float, float, BWD, IL>), blocks, dim3(256), lds, s, a);
  else if (dtype == APGD_BF16) hipLaunchKernelGGL((qk_norm_rope_kernel<bf16_t, bf16_t, BWD, IL>), blocks, dim3(256), lds, s, a);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<__half, __half, BWD, IL>), blocks, dim3(256), lds, s, a);
}
template <bool BWD>
void launch(const RopeArgs& a, int dtype, bool half, bool interleaved, unsigned grid, hipStream_t s) {
  if (interleaved) launch<BWD, true>(a, dtype, half, grid, s);
  else launch<BWD, false>(a, dtype, half, grid, s);
}

View view_of(const int64_t* s) { return View{s[0], s[1], s[2]}; }

}  // namespace

int rope_table(const void* positions, int pos_dtype, int64_t pos_b, int32_t axes, const int32_t* sections, const float* inv_freq, int64_t B,
               int64_t N, int32_t d, float2* cs, hipStream_t s) {
  RopeArgs a = {};
  a.pos = positions; a.pos_dtype = pos_dtype; a.pos_b = pos_b; a.axes = axes; a.inv_freq = inv_freq;
  if (const int rc = check_args(a, APGD_F32, sections, B, N, 0, 0, d)) return rc;
  const int64_t rows = pos_b ? B * N : N, blocks = (rows * (d / 2) + 255) / 256;
  hipLaunchKernelGGL(rope_table_kernel, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, a, cs, rows);
  return launch_status();
}
int rope_forward(const void* q, const void* k, void* yq, void* yk, int dtype, bool half, const int64_t* strides, const void* wq, const void* wk,
                 int w_dtype, const void* positions, int pos_dtype, int64_t pos_batch_stride, int32_t axes, const int32_t* sections,
                 const float* inv_freq, int64_t B, int64_t N, int32_t Hq, int32_t Hk, int32_t d, float eps, int32_t norm, int32_t interleaved,
                 hipStream_t s) {
  RopeArgs a = {};
  a.q.x = q; a.k.x = k; a.q.o = yq; a.k.o = yk;
  a.q.w = wq; a.k.w = wk; a.w_dtype = w_dtype;
  a.pos = positions; a.pos_dtype = pos_dtype; a.pos_b = pos_batch_stride; a.axes = axes; a.inv_freq = inv_freq;
  a.norm = norm != 0; a.eps = eps;
  if (const int rc = check_args(a, dtype, sections, B, N, Hq, Hk, d)) return rc;
  if (B == 0 || N == 0 || Hq + Hk == 0) return APGD_OK;
  if (!strides || (Hq && (!q || !yq)) || (Hk && (!k || !yk))) return APGD_ERR_NULL;
  a.q.vx = view_of(strides); a.k.vx = view_of(strides + 3); a.q.vo = view_of(strides + 6); a.k.vo = view_of(strides + 9);
  cut(a);
  launch<false>(a, dtype, half, interleaved != 0, static_cast<unsigned>(a.tiles < kFwdGrid ? a.tiles : kFwdGrid), s);
  return launch_status();
}
int rope_dw(const float* pq, int nq, const float* pk, int nk, int32_t d, float* dwq, float* dwk, hipStream_t s) {
  hipLaunchKernelGGL(rope_dw_kernel, dim3(static_cast<unsigned>(d / 16), 2), dim3(1024), 0, s, pq, nq, pk, nk, d, dwq, dwk);
  return launch_status();
}

extern "C" {

int cnx_qk_norm_rope_supported(int32_t d) { return d >= 16 && d <= kMaxHead && d % 16 == 0; }

int64_t cnx_qk_norm_rope_ws_floats(int32_t d) { return cnx_qk_norm_rope_supported(d) ? static_cast<int64_t>(kBwdGrid) * 2 * d : 0; }

int cnx_qk_norm_rope_fwd(const void* q, const void* k, void* yq, void* yk, int dtype, const int64_t* strides, const void* wq, const void* wk,
                         int w_dtype, const void* positions, int pos_dtype, int64_t pos_batch_stride, int32_t axes, const int32_t* sections,
                         const float* inv_freq, int64_t B, int64_t N, int32_t Hq, int32_t Hk, int32_t d, float eps, int32_t norm,
                         int32_t interleaved, void* stream) {
  return rope_forward(q, k, yq, yk, dtype, false, strides, wq, wk, w_dtype, positions, pos_dtype, pos_batch_stride, axes, sections, inv_freq, B, N, Hq,
                      Hk, d, eps, norm, interleaved, as_stream(stream));
}

int cnx_qk_norm_rope_bwd(const void* dyq, const void* dyk, const void* q, const void* k, void* dq, void* dk, float* dwq, float* dwk, float* ws,
                         int dtype, const int64_t* strides, const void* wq, const void* wk, int w_dtype, const void* positions, int pos_dtype,
                         int64_t pos_batch_stride, int32_t axes, const int32_t* sections, const float* inv_freq, int64_t B, int64_t N,
                         int32_t Hq, int32_t Hk, int32_t d, float eps, int32_t norm, int32_t interleaved, void* stream) {
  RopeArgs a = {};
  a.q.x = q; a.k.x = k; a.q.dy = dyq; a.k.dy = dyk; a.q.o = dq; a.k.o = dk;
  a.q.w = wq; a.k.w = wk; a.w_dtype = w_dtype;
  a.pos = positions; a.pos_dtype = pos_dtype; a.pos_b = pos_batch_stride; a.axes = axes; a.inv_freq = inv_freq;
  a.norm = norm != 0; a.eps = eps;
  if (const int rc = check_args(a, dtype, sections, B, N, Hq, Hk, d)) return rc;
  const bool want_w = a.norm && (dwq || dwk);
  if (want_w && !ws) return APGD_ERR_NULL;
  unsigned grid = 0;
  if (B == 0 || N == 0 || Hq + Hk == 0) {
    if (!want_w) return APGD_OK;                                      // else: the weights' gradients are zeros
  } else {
    if (!strides || (Hq && (!dyq || !dq || (norm && !q))) || (Hk && (!dyk || !dk || (norm && !k)))) return APGD_ERR_NULL;
    a.q.vdy = view_of(strides); a.k.vdy = view_of(strides + 3); a.q.vx = view_of(strides + 6); a.k.vx = view_of(strides + 9);
    a.q.vo = view_of(strides + 12); a.k.vo = view_of(strides + 15);
    a.part = want_w ? ws : nullptr;
    cut(a);
    grid = static_cast<unsigned>(a.tiles < kBwdGrid ? a.tiles : kBwdGrid);
    launch<true>(a, dtype, false, interleaved != 0, grid, as_stream(stream));
  }
  return want_w ? rope_dw(ws, static_cast<int>(grid), ws + static_cast<int64_t>(grid) * d, static_cast<int>(grid), d, dwq, dwk, as_stream(stream)) : launch_status();
}

}  // extern "C"
