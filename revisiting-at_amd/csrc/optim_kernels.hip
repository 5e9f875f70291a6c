// optim_kernels.hip — the AdamW update of many tensors in one launch, with moments in 32 or in 8 bits, for gfx950.
//
//   p <- p (1 - lr wd);  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2
//   p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Element-wise and bound by memory: 28 bytes per fp32 parameter with 32-bit moments (p, m, v in and out, g in), 16.06 with 8-bit ones.
// Measured: 152 tensors, 21.8 M parameters, 32 bits: 101 us (6.0 TB/s); 152 M parameters, 8 bits: 427 - 500 us (5.7 - 4.9 TB/s; about 60
// instructions per element, a quarter of them for the two codes); a copy of 2 GiB reaches 4.9 TB/s.
//
// Layout.  The moments of all tensors lie in flat buffers, each tensor from a multiple of 256 elements on.  A workgroup takes a chunk of 4096
// elements of one tensor (a table of chunks, made once, says which), 16 per thread in four 16-byte pieces, so all its loads are in flight at
// once whatever the tensors' sizes; tensors too small for a chunk cost one workgroup each.  What differs from step to step - where the
// gradients are - travels in the kernel's arguments; t, the bias corrections and a learning rate in device memory are read on the device by a
// one-workgroup launch in front (adamw_prepare_kernel), so a captured step counts on by itself.
//
// 8 bits.  A block of 256 elements shares one fp32 scale, its largest magnitude; a code is the top of the scaled value's fp32 pattern:
//   m: sign, and 7 bits counting down from 1.0 in steps of 1/8 binade (3 mantissa bits): 2^-15.75 .. 1, and zero
//   v: its ROOT in 8 bits, 4 mantissa bits: 2^-15.9 .. 1, so v spans 2^-31; a root other than zero keeps at least the smallest code, because
//      the update divides by it (rounded to zero it would make m / eps)
// Rounding is to nearest, ties to even, by an integer addition - as long as a step of a moment can reach another code at all.  A root changes by
// (1 - b2) / 2 of itself in a step, a first moment by 1 - b1, and the finest half step of a code is 1/64 (1/32): above beta = 31/32 (kDither) what a step
// changes would be rounded away again, and a moment whose gradients have fallen would stay where it was.  There it is rounded up or down with the
// probability that keeps its mean, by a hash of the element and the step (the same every time).  Simulated, three quarters of a block falling tenfold,
// stored root over the true one, 5 - 95 %: normal gradients, b2 0.95: nearest 0.93 - 1.07, hashed 0.90 - 1.11; 0.98: 0.94 - 1.15, 0.86 - 1.14; 0.999:
// 7.4 - 12, 0.82 - 1.21.  (Nearest needs gradients that vary: where nothing else moves the block's scale, a constant tenth of a gradient leaves the
// root 1.4 times too large at 0.9, 6.2 times at 0.95.)  Scaling by the block's maximum lets a block decay as a whole: the largest
// element is always exact, which a fixed grid would keep from shrinking when b v rounds back to v.  A wavefront holds a block (4 elements per
// lane): its maximum is six steps through the lanes' neighbours (DPP).  Maxima are taken of bit patterns, so that a NaN or infinite moment
// makes its block's scale (and with it the block) non-finite instead of vanishing.  The update uses the moments before they are rounded.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "apgd_hip.h"
#include "convnext_hip.h"

namespace {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline int launch_status() { return static_cast<int>(hipGetLastError()); }

constexpr int kBlock = CNX_ADAMW_BLOCK, kChunk = CNX_ADAMW_CHUNK, kTensors = CNX_ADAMW_TENSORS;
constexpr int kGroups = CNX_ADAMW_GROUPS;
constexpr float kDither = 31.f / 32.f;
static_assert(kBlock == 256 && kChunk == 4096, "four elements per lane, sixteen per thread");

struct Grads { const void* g[kTensors]; };       // 3.5 KB of kernel arguments

struct Hyper {                                   // per parameter group
  double lr, b1, b2, eps, wd;
  const float* lr_dev;                           // overrides lr
};
struct Hypers { Hyper h[kGroups]; };

struct Coef {                                    // per tensor and step
  float decay, b1, nb1, b2, nb2, eps, step_size, inv_root;
};

struct State {
  float *m, *v;                                  // 32 bits
  uint8_t *mc, *vc;                              // 8 bits: codes, one per element
  float *ms, *vs;                                // scales, one per block
};

// four consecutive elements from any address of their type (unaligned 16-byte accesses are whole on gfx950)
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4u __attribute__((aligned(2)));

__device__ __forceinline__ float bf16_up(uint16_t u) { return __uint_as_float(static_cast<uint32_t>(u) << 16); }
__device__ __forceinline__ uint16_t bf16_down(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }

__device__ __forceinline__ f32x4 load4(const void* p, int64_t at, int n, bool bf16) {        // n < 4: the tensor's last elements
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (bf16) {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    if (n >= 4) {
      const u16x4 v = *reinterpret_cast<const u16x4u*>(q);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = bf16_up(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i) if (i < n) r[i] = bf16_up(q[i]);
    }
  } else {
    const float* q = static_cast<const float*>(p) + at;
    if (n >= 4) r = *reinterpret_cast<const f32x4u*>(q);
    else {
#pragma unroll
      for (int i = 0; i < 3; ++i) if (i < n) r[i] = q[i];
    }
  }
  return r;
}
__device__ __forceinline__ void store4(void* p, int64_t at, int n, bool bf16, f32x4 x) {
  if (bf16) {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    if (n >= 4) {
      u16x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = bf16_down(x[i]);
      *reinterpret_cast<u16x4u*>(q) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i) if (i < n) q[i] = bf16_down(x[i]);
    }
  } else {
    float* q = static_cast<float*>(p) + at;
    if (n >= 4) *reinterpret_cast<f32x4u*>(q) = x;
    else {
#pragma unroll
      for (int i = 0; i < 3; ++i) if (i < n) q[i] = x[i];
    }
  }
}

// code c > 0 of `MANT` mantissa bits, 1.0 at code TOP
template <int MANT, int TOP>
__device__ __forceinline__ float code_value(uint32_t c) {
  constexpr uint32_t one = 0x3f800000u >> (23 - MANT);
  return c ? __uint_as_float((c + (one - TOP)) << (23 - MANT)) : 0.f;
}
template <int MANT, int TOP>
__device__ __forceinline__ uint32_t value_code(float x) {                                      // x >= 0
  constexpr int sh = 23 - MANT;
  constexpr int one = 0x3f800000 >> sh;
  int b = static_cast<int>(__float_as_uint(x) & 0x7fffffffu);
  b = (b + ((1 << (sh - 1)) - 1) + ((b >> sh) & 1)) >> sh;
  b -= one - TOP;
  return static_cast<uint32_t>(b < 0 ? 0 : b > TOP ? TOP : b);
}
// the same, up where the part of a step that is cut off and `part` (16 bits) make a whole one
template <int MANT, int TOP>
__device__ __forceinline__ uint32_t value_code(float x, uint32_t part) {
  constexpr int sh = 23 - MANT;
  constexpr int one = 0x3f800000 >> sh;
  const int b = (static_cast<int>((__float_as_uint(x) & 0x7fffffffu) + (part << (sh - 16))) >> sh) - (one - TOP);
  return static_cast<uint32_t>(b < 0 ? 0 : b > TOP ? TOP : b);
}
// 32 mixed bits of an element and a step (odd multipliers: 2^32 times the fractional parts of the golden ratio and of the roots of 2, 3 and 7)
__device__ __forceinline__ uint32_t mixed(uint32_t element, uint32_t step) {
  uint32_t h = element * 0x9e3779b9u ^ step * 0x6a09e667u;
  h = (h ^ (h >> 15)) * 0xbb67ae85u;
  h = (h ^ (h >> 13)) * 0xa54ff53bu;
  return h ^ (h >> 16);
}
// the wavefront's largest value, by shifts within rows of 16 lanes and two broadcasts across them (a lane exchange through LDS would cost more
// than the rest of the block's arithmetic); the last lane has it, and all get it as a scalar
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_shifted(uint32_t v) {
  const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
  return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_shifted<0x111, 0xf>(v);                // row_shr:1, 2, 4, 8
  v = max_shifted<0x112, 0xf>(v);
  v = max_shifted<0x114, 0xf>(v);
  v = max_shifted<0x118, 0xf>(v);
  v = max_shifted<0x142, 0xa>(v);                // row_bcast:15 into rows 1 and 3
  v = max_shifted<0x143, 0xc>(v);                // row_bcast:31 into rows 2 and 3
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
// a block's scale from the pattern of its largest magnitude: values too small to be divided by are no scale
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __uint_as_float(top);
  return s < 1.17549435e-38f ? 0.f : s;
}

// (the quotient by v_rcp_f32, off by at most 1 ulp: a division's twelve instructions per element made the 8-bit step bound by them)
__device__ __forceinline__ void update(const Coef& c, f32x4& p, f32x4 g, f32x4& m, f32x4& v, f32x4& root) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = p[i] * c.decay;
    m[i] = m[i] * c.b1 + g[i] * c.nb1;
    v[i] = v[i] * c.b2 + (g[i] * g[i]) * c.nb2;
    root[i] = sqrtf(v[i]);
    p[i] = p[i] - (m[i] * __builtin_amdgcn_rcpf(root[i] * c.inv_root + c.eps)) * c.step_size;
  }
}

__global__ void adamw_prepare_kernel(const cnx_adamw_tensor* __restrict__ table, const Grads grads, int n, const Hypers hy, float* __restrict__ steps,
                                     Coef* __restrict__ coef) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    if (!grads.g[i]) continue;
    const float t = steps[table[i].step] + 1.f;
    steps[table[i].step] = t;
    const Hyper h = hy.h[table[i].group];
    const double lr = h.lr_dev ? static_cast<double>(*h.lr_dev) : h.lr;
    Coef c;
    c.decay = static_cast<float>(1.0 - lr * h.wd);
    c.b1 = static_cast<float>(h.b1); c.nb1 = static_cast<float>(1.0 - h.b1);
    c.b2 = static_cast<float>(h.b2); c.nb2 = static_cast<float>(1.0 - h.b2);
    c.eps = h.eps > 0.0 ? fmaxf(static_cast<float>(h.eps), 1.17549435e-38f) : 0.f;             // (v_rcp_f32 takes no subnormals)
    c.step_size = static_cast<float>(lr / (1.0 - pow(h.b1, static_cast<double>(t))));
    c.inv_root = static_cast<float>(1.0 / sqrt(1.0 - pow(h.b2, static_cast<double>(t))));
    coef[i] = c;
  }
}

// DITHER: one of the groups' betas is above kDither (a branch in the other form cost it 3 %)
template <bool DITHER>
__global__ __launch_bounds__(256) void adamw_step_kernel(const cnx_adamw_tensor* __restrict__ table, const cnx_adamw_chunk* __restrict__ chunks,
                                                         const Grads grads, const Coef* __restrict__ coef, const float* __restrict__ steps,
                                                         const State st) {
  const cnx_adamw_chunk ch = chunks[blockIdx.x];
  const cnx_adamw_tensor ts = table[ch.tensor];
  const void* g = grads.g[ch.tensor];
  if (!g) return;                                // no gradient in this step
  const Coef c = coef[ch.tensor];
  const bool bf16 = ts.dtype == APGD_BF16;
  const int64_t base = static_cast<int64_t>(ch.part) * kChunk;
  const int64_t left = ts.numel - base;
  f32x4 p[4], gr[4];
  int n[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = u * 1024 + threadIdx.x * 4;
    n[u] = left - e > 4 ? 4 : static_cast<int>(left - e);
    p[u] = load4(ts.param, base + e, n[u], bf16);
    gr[u] = load4(g, base + e, n[u], bf16);
  }
  if (ts.bits == 32) {
    float* m = st.m + ts.state + base;
    float* v = st.v + ts.state + base;
    f32x4 mv[4], vv[4], root;
#pragma unroll
    for (int u = 0; u < 4; ++u) {                // (a tensor's moments are padded to whole blocks of zeros)
      const int e = u * 1024 + threadIdx.x * 4;
      mv[u] = vv[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (n[u] > 0) {
        mv[u] = *reinterpret_cast<const f32x4*>(m + e);
        vv[u] = *reinterpret_cast<const f32x4*>(v + e);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = u * 1024 + threadIdx.x * 4;
      update(c, p[u], gr[u], mv[u], vv[u], root);
      if (n[u] > 0) {
        *reinterpret_cast<f32x4*>(m + e) = mv[u];
        *reinterpret_cast<f32x4*>(v + e) = vv[u];
      }
      store4(ts.param, base + e, n[u], bf16, p[u]);
    }
  } else {
    const bool dither_m = DITHER && c.b1 > kDither, dither_v = DITHER && c.b2 > kDither;
    const int64_t b0 = (ts.state + base) / kBlock;
    const int wave = threadIdx.x >> 6;
    uint32_t mc[4], vc[4];
    float ms[4], vs[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = u * 1024 + threadIdx.x * 4;
      const bool whole = u * 1024 + wave * 256 < left;                // (uniform in the wavefront) the block exists
      mc[u] = vc[u] = 0;
      ms[u] = vs[u] = 0.f;
      if (whole) {
        mc[u] = *reinterpret_cast<const uint32_t*>(st.mc + ts.state + base + e);
        vc[u] = *reinterpret_cast<const uint32_t*>(st.vc + ts.state + base + e);
        ms[u] = st.ms[b0 + u * 4 + wave];
        vs[u] = st.vs[b0 + u * 4 + wave];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = u * 1024 + threadIdx.x * 4;
      if (u * 1024 + wave * 256 >= left) break;
      f32x4 m, v, root;
      uint32_t tm = 0, tv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = (mc[u] >> (8 * i)) & 0xffu, b = (vc[u] >> (8 * i)) & 0xffu;
        const float x = code_value<3, 127>(a & 127u);
        m[i] = (a & 128u ? -x : x) * ms[u];
        const float r = code_value<4, 255>(b) * vs[u];
        v[i] = r * r;
      }
      update(c, p[u], gr[u], m, v, root);
      store4(ts.param, base + e, n[u], bf16, p[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t am = __float_as_uint(m[i]) & 0x7fffffffu, ar = __float_as_uint(root[i]) & 0x7fffffffu;
        tm = am > tm ? am : tm;
        tv = ar > tv ? ar : tv;
      }
      const float sm = scale_of(wave_max(tm)), sv = scale_of(wave_max(tv));
      const float im = sm > 0.f ? 1.f / sm : 0.f, iv = sv > 0.f ? 1.f / sv : 0.f;
      uint32_t om = 0, ov = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a, b;
        if (dither_m || dither_v) {                                   // (uniform)
          const uint32_t h = mixed(static_cast<uint32_t>(ts.state + base + e + i), static_cast<uint32_t>(steps[ts.step]));
          a = dither_m ? value_code<3, 127>(fabsf(m[i]) * im, h & 0xffffu) : value_code<3, 127>(fabsf(m[i]) * im);
          b = dither_v ? value_code<4, 255>(root[i] * iv, h >> 16) : value_code<4, 255>(root[i] * iv);
        } else {
          a = value_code<3, 127>(fabsf(m[i]) * im);
          b = value_code<4, 255>(root[i] * iv);
        }
        a |= m[i] < 0.f ? 128u : 0u;
        if (root[i] > 0.f && sv > 0.f && b == 0) b = 1;
        om |= a << (8 * i);
        ov |= b << (8 * i);
      }
      *reinterpret_cast<uint32_t*>(st.mc + ts.state + base + e) = om;
      *reinterpret_cast<uint32_t*>(st.vc + ts.state + base + e) = ov;
      if ((threadIdx.x & 63) == 0) {
        st.ms[b0 + u * 4 + wave] = sm;
        st.vs[b0 + u * 4 + wave] = sv;
      }
    }
  }
}

// the numbers that 8-bit moments stand for, in bf16 (a code has 4 or 5 significant bits); 152 M: 158 us for 0.92 GB, 5.8 TB/s
__global__ __launch_bounds__(256) void adamw_values_kernel(const uint8_t* __restrict__ mc, const float* __restrict__ ms, const uint8_t* __restrict__ vc,
                                                           const float* __restrict__ vs, uint16_t* __restrict__ m, uint16_t* __restrict__ v,
                                                           int64_t n) {
  for (int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; e < n; e += static_cast<int64_t>(gridDim.x) * 2048) {
    const uint2 a = *reinterpret_cast<const uint2*>(mc + e), b = *reinterpret_cast<const uint2*>(vc + e);
    const float sm = ms[e / kBlock], sv = vs[e / kBlock];
    uint32_t om[4], ov[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t ca = ((i < 4 ? a.x : a.y) >> (8 * (i & 3))) & 0xffu, cb = ((i < 4 ? b.x : b.y) >> (8 * (i & 3))) & 0xffu;
      const float x = code_value<3, 127>(ca & 127u) * sm, r = code_value<4, 255>(cb) * sv;
      const uint32_t hm = bf16_down(ca & 128u ? -x : x), hv = bf16_down(r * r);
      if (i & 1) { om[i >> 1] |= hm << 16; ov[i >> 1] |= hv << 16; }
      else { om[i >> 1] = hm; ov[i >> 1] = hv; }
    }
    *reinterpret_cast<uint4*>(m + e) = make_uint4(om[0], om[1], om[2], om[3]);
    *reinterpret_cast<uint4*>(v + e) = make_uint4(ov[0], ov[1], ov[2], ov[3]);
  }
}

}  // namespace

extern "C" {

int cnx_adamw_step(const cnx_adamw_tensor* table, const cnx_adamw_chunk* chunks, int64_t n_chunks, const void* const* grads, int32_t n_tensors,
                   const double* hyper, const float* const* lr_dev, int32_t n_groups, float* steps, float* coef, float* m, float* v, uint8_t* m_codes,
                   float* m_scales, uint8_t* v_codes, float* v_scales, void* stream) {
  if (n_tensors < 0 || n_chunks < 0 || n_chunks > (1LL << 23)) return APGD_ERR_SIZE;
  if (n_tensors > kTensors || n_groups < 1 || n_groups > kGroups) return APGD_ERR_ARG;
  if (n_tensors == 0) return APGD_OK;
  if (!table || !grads || !hyper || !steps || !coef || (n_chunks > 0 && !chunks)) return APGD_ERR_NULL;
  if (!(m && v) && !(m_codes && m_scales && v_codes && v_scales)) return APGD_ERR_NULL;
  Grads g = {};
  Hypers h = {};
  bool dither = false;
  for (int i = 0; i < n_tensors; ++i) g.g[i] = grads[i];
  for (int i = 0; i < n_groups; ++i) {
    const double* x = hyper + 5 * i;
    if (!(x[1] >= 0.0 && x[1] < 1.0 && x[2] >= 0.0 && x[2] < 1.0 && x[3] >= 0.0)) return APGD_ERR_ARG;
    dither |= x[1] > kDither || x[2] > kDither;
    h.h[i] = Hyper{x[0], x[1], x[2], x[3], x[4], lr_dev ? lr_dev[i] : nullptr};
  }
  hipStream_t s = as_stream(stream);
  const State st = {m, v, m_codes, v_codes, m_scales, v_scales};
  hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(256), 0, s, table, g, n_tensors, h, steps, reinterpret_cast<Coef*>(coef));
  if (n_chunks)
    hipLaunchKernelGGL(dither ? adamw_step_kernel<true> : adamw_step_kernel<false>, dim3(static_cast<unsigned>(n_chunks)), dim3(256), 0, s, table, chunks, g,
                       reinterpret_cast<const Coef*>(coef), steps, st);
  return launch_status();
}

int cnx_adamw_values(const uint8_t* m_codes, const float* m_scales, const uint8_t* v_codes, const float* v_scales, void* m, void* v, int64_t n,
                     void* stream) {
  if (n < 0 || n % kBlock) return APGD_ERR_SIZE;
  if (n == 0) return APGD_OK;
  if (!m_codes || !m_scales || !v_codes || !v_scales || !m || !v) return APGD_ERR_NULL;
  const int64_t blocks = (n + 2047) / 2048;
  hipLaunchKernelGGL(adamw_values_kernel, dim3(static_cast<unsigned>(blocks < 16384 ? blocks : 16384)), dim3(256), 0, as_stream(stream), m_codes, m_scales,
                     v_codes, v_scales, static_cast<uint16_t*>(m), static_cast<uint16_t*>(v), n);
  return launch_status();
}

}  // extern "C"
