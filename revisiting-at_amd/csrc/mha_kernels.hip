// mha_kernels.hip — softmax attention over any number of tokens and its backward pass, on gfx950's matrix cores.
//
//   out = softmax(scale q k^T) v                                                      q [B, Nq, H, d], k, v [B, Nk, Hkv, d], H = G Hkv
//   D = rowsum(dout out),  P = exp(scale q k^T - lse),  dS = P (dout v^T - D)
//   dv = P^T dout,  dq = scale dS k,  dk = scale dS^T q                               (P and dS summed over the G heads that share a key head)
// The N x N scores never reach memory: the forward keeps a running maximum and sum per query and saves only lse = log sum exp, the
// backward forms P again from it.
//
// Rows.  The G query heads that share a key head are G rows of one matrix: row r of key head hk is token r / G, head hk G + r % G.  Shared
// heads then cost no extra reads of k and v, a single token still fills G rows of a tile, and dk / dv are sums inside one workgroup - no
// atomics, the same bits every time.
//
// Orientation.  mfma 32x32x16 leaves, per lane, one COLUMN of its result and 16 rows in registers.
//   forward, dq:  S^T = K Q^T puts a query on each lane: maxima, sums, lse and D are one register, and P (rounded in registers) is the B
//                 operand of  O^T = V^T P^T,  dQ^T = K^T dS^T  whose results again have a query per lane - rescaling is one multiply.
//   dk, dv:       S = Q K^T puts a key on each lane; P and dS are B operands of  dV^T = dO^T P,  dK^T = Q^T dS.
// Operand images in LDS are row-major as in memory; a product over d reads rows (ds_read_b128), a product over tokens reads columns
// through the transposing read (ds_read_b64_tr_b16).  16-byte chunk c of row r is stored at chunk c ^ swz(r), which spreads both kinds of
// read over all banks.
//
// Masks.  Each row has an end: keys at or beyond it are not seen (key lengths, causal order, padded queries: end 0).  A row that sees no
// key gives zeros and lse = -inf, and no gradient.  Rows at or beyond their sample's length are staged as zeros whatever memory holds.
//
// Roundings.  Scores, maxima, sums, lse and all accumulators are 32 bits.  P and dS are rounded to 16 bits because they are matrix
// operands; the results once, at the end.  D is a 32-bit sum, of dout and the rounded out (u |dout| |out| off), or - for rows that see no key
// behind the first tile - of P dP as the tile gives them (errors against 64 bits, 2 keys: 2.4 -> 1.5 times those of one rounding at the end; dq's
// kernel 1 % slower at 512 px).  attention_rope's q' and k' have to lie in memory between two kernels and are rounded there - to
// fp16 where the norm bounds them, since every score and gradient sees that rounding.
//
// Measured (us; TFLOP/s of the products a kernel forms; a library product of 8192^3: 1263 bf16, 1214 fp16):
//                                                       forward      dq           dk, dv
//   64 x 1025 tokens, 6 heads, d 64, bf16               151   685    198   780    282          730
//   2 x 4096, causal, 16 heads on 4, d 128, fp16        165   830    233   885    373 + 16     705
//   32 x 577, 12 heads, d 64, with norm and rotation     61   535    101   485    128          510
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "apgd_hip.h"
#include "convnext_hip.h"
#include "rope_internal.h"

namespace {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline int launch_status() { return static_cast<int>(hipGetLastError()); }

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4), aligned(4))) float f32x4u;   // at any address of a float

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kKT = 64;                          // keys (rows) of a staged tile
constexpr float kSlack = 8.f;                    // see mha_fwd_kernel

// Operand types.  Io: of the tensors; mfma, pack: products with v or dout (P, dP); mfma_s, pack_s: products with q or k (S, dS).
struct Bf16 {
  using Io = Bf16;
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  }
  static __device__ __forceinline__ f32x16 mfma_s(u32x4 a, u32x4 b, f32x16 c) { return mfma(a, b, c); }
  static __device__ __forceinline__ uint32_t pack_s(float lo, float hi) { return pack(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
struct Fp16 {
  using Io = Fp16;
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
  static __device__ __forceinline__ f32x16 mfma_s(u32x4 a, u32x4 b, f32x16 c) { return mfma(a, b, c); }
  static __device__ __forceinline__ uint32_t pack_s(float lo, float hi) { return pack(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return static_cast<float>(__builtin_bit_cast(f16x2, w)[0]); }
  static __device__ __forceinline__ float hi(uint32_t w) { return static_cast<float>(__builtin_bit_cast(f16x2, w)[1]); }
};

// attention_rope on bf16 tensors: q' and k', normalised and so of known size, are in fp16, and with them dS
struct Mixed : Bf16 {
  static constexpr bool kScaled = true;
  static __device__ __forceinline__ f32x16 mfma_s(u32x4 a, u32x4 b, f32x16 c) { return Fp16::mfma(a, b, c); }
  static __device__ __forceinline__ uint32_t pack_s(float lo, float hi) { return Fp16::pack(lo, hi); }
};

struct View {                                    // 16-bit [B, N, heads, d], unit stride in d
  int64_t b, n, h;
};

// attention_rope's backward: the way back from q' (k') to q (k), at the end of dq (dk/dv)
struct Turn {
  const uint16_t* x;                             // q (k) as it was
  View vx;
  const float* w;                                // [D] or NULL
  float* part;                                   // [workgroup][D] partial weight gradients or NULL
};

struct MhaArgs {
  const uint16_t *q, *k, *v, *out, *dout;        // out, dout: backward
  uint16_t *o, *dq, *dk, *dv;                    // o: forward
  float* lse;                                    // [B, H, Nq]; forward: may be NULL
  float* dvec;                                   // backward: [B, H, Nq]
  float* part;                                   // key splits: partial results
  const int32_t *q_lens, *kv_lens;               // [B] or NULL
  View vq, vk, vv, vo, vdo, vdq, vdk, vdv;
  int32_t Nq, Nk, H, Hkv, G, causal;
  int32_t tiles, splits;                         // row (or key) tiles of a key head, splits of the keys
  int32_t span;                                  // keys of one split, a multiple of the key tile
  int64_t B;
  float scale;
  Turn tq, tk;                                   // TURN: G = 1, no lengths
  const float2* cs;                              // cosines and sines [(B,) N][D / 2] or NULL
  int64_t cs_b;                                  // pairs between the samples' (0: shared)
  float eps;
  int32_t norm, il;
  const float2* range;                           // kScaled: [B][H][pieces] largest sizes (row_size) of v's and dout's rows
  int32_t pieces;
};

// what a sample allows
struct Limits {
  int q_len, kv_len, off;
  __device__ __forceinline__ Limits(const MhaArgs& a, int64_t b) {
    q_len = a.q_lens ? min(max(a.q_lens[b], 0), a.Nq) : a.Nq;
    kv_len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Nk) : a.Nk;
    off = kv_len - q_len;                        // causal: the last query sees the last key
  }
  // first key that token i does not see
  __device__ __forceinline__ int end(int i, int causal) const {
    if (i >= q_len) return 0;
    return causal ? min(kv_len, max(0, i + off + 1)) : kv_len;
  }
};

// Spreads both kinds of read over the 64 banks: the 16 lanes that a 16-byte read serves at a time (rows 0 - 15, or 0 - 3, 12 - 15, 20 - 27 and
// so on) fall on 16 different pieces of 256 bytes, and the four rows x 64 bytes of a transposing read on its four quarters.
template <int D> __device__ __forceinline__ int swz(int row) {
  const int b0 = row & 1, b1 = (row >> 1) & 1, b2 = (row >> 2) & 1, b3 = (row >> 3) & 1;
  if constexpr (D == 64) return (b1 << 2) | (b3 << 1) | b2;            // (rows of 128 bytes: b0 is the half already)
  else return (b1 << 3) | (b0 << 2) | (b3 << 1) | b2;
}

template <typename T>
__device__ __forceinline__ uint32_t lds_addr(const T* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}
__device__ __forceinline__ u32x4 lds_read16(uint32_t addr) {
  return *reinterpret_cast<const u32x4 __attribute__((address_space(3)))*>(static_cast<uintptr_t>(addr));
}
__device__ __forceinline__ u32x2 lds_read_tr(uint32_t addr) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      reinterpret_cast<s16x4 __attribute__((address_space(3)))*>(static_cast<uintptr_t>(addr)));
  return __builtin_bit_cast(u32x2, r);
}

// How one lane reads row-major images [rows][D] of 16-bit values in LDS.  Addresses are made once; what changes - image, buffer, block - is a
// constant that the read's own offset field takes.
template <int D>
struct Lane {
  static constexpr int ROWB = D * 2, KS = D / 16, DB = D / 32;
  uint32_t ra[KS];                               // row l32 of a 32-row block, chunk 2 ks + half
  uint32_t ca[2][DB];                            // column db * 32 + lane % 32, rows {0..3} + 4 half and {8..11} + 4 half of 16 rows
  __device__ __forceinline__ Lane(uint32_t base) {
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5, g = lane >> 4, i = lane & 15;
    const uint32_t r = base + l32 * ROWB + ((half ^ swz<D>(l32)) << 4);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ra[ks] = r ^ (ks << 5);           // (the base is a multiple of a row: only chunk bits change)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = 4 * (g >> 1) + (i >> 2) + 8 * n, chunk = 2 * (g & 1) + ((i & 3) >> 1);
      const uint32_t c = base + row * ROWB + ((chunk ^ swz<D>(row)) << 4) + 8 * (i & 1);
#pragma unroll
      for (int db = 0; db < DB; ++db) ca[n][db] = c ^ (db << 6);
    }
  }
  // operand of a product over d: rows of 32-row block blk
  __device__ __forceinline__ u32x4 row(uint32_t image, int blk, int ks) const { return lds_read16(ra[ks] + (image + blk * 32 * ROWB)); }
  // operand of a product over rows: a column of rows 16 t .. 16 t + 15 of block blk
  __device__ __forceinline__ u32x4 col(uint32_t image, int blk, int t, int db) const {
    const uint32_t at = image + (blk * 32 + t * 16) * ROWB;
    const u32x2 a = lds_read_tr(ca[0][db] + at), b = lds_read_tr(ca[1][db] + at);
    return u32x4{a.x, a.y, b.x, b.y};
  }
};

// Staging of a 64-row tile by 256 threads straight from memory to LDS (no registers in between): instruction p of a wavefront fills the
// 16-byte pieces e = (4 p + wave) * 64 + lane, row e / CHUNKS, chunk position e % CHUNKS, which holds chunk position ^ swz(row).  Rows that do
// not exist have an offset beyond the buffer's end and come out as zeros.
constexpr uint32_t kNoRow = 0xfffffff0u;
template <int D>
struct Stage {
  static constexpr int CHUNKS = D / 8, PER = kKT * CHUNKS / 256;
  static __device__ __forceinline__ int row(int p) { return ((4 * p + (threadIdx.x >> 6)) * 64 + (threadIdx.x & 63)) / CHUNKS; }
  static __device__ __forceinline__ uint32_t chunk(int p) { return ((threadIdx.x & (CHUNKS - 1)) ^ swz<D>(row(p))) << 4; }
  uint32_t off[PER];                             // byte offset of the thread's pieces from the tile's first row
  __device__ __forceinline__ void rows_apart(int64_t stride) {
#pragma unroll
    for (int p = 0; p < PER; ++p) off[p] = static_cast<uint32_t>(row(p) * stride * 2) + chunk(p);
  }
  // the tile at `base` (uniform), its first `rows` rows, to LDS address `dst`
  __device__ __forceinline__ void load(const uint16_t* base, int rows, uint32_t dst) const {
    const u32x4 rs = buffer(base);
    const uint32_t at = __builtin_amdgcn_readfirstlane(dst + (threadIdx.x >> 6) * 1024);
    if (rows >= kKT) {
#pragma unroll
      for (int p = 0; p < PER; ++p) piece(rs, at + p * 4096, off[p]);
    } else {
#pragma unroll
      for (int p = 0; p < PER; ++p) piece(rs, at + p * 4096, row(p) < rows ? off[p] : kNoRow);
    }
  }
  template <typename Live>                       // Live: number of the thread's piece -> whether its row exists
  __device__ __forceinline__ void load(const uint16_t* base, uint32_t dst, Live live) const {
    const u32x4 rs = buffer(base);
    const uint32_t at = __builtin_amdgcn_readfirstlane(dst + (threadIdx.x >> 6) * 1024);
#pragma unroll
    for (int p = 0; p < PER; ++p) piece(rs, at + p * 4096, live(p) ? off[p] : kNoRow);
  }
  static __device__ __forceinline__ u32x4 buffer(const uint16_t* base) {                       // raw buffer of 2 GiB
    const uint64_t p64 = reinterpret_cast<uint64_t>(base);
    u32x4 rs = {static_cast<uint32_t>(p64), static_cast<uint32_t>(p64 >> 32) & 0xffffu, 0x80000000u, 0x00020000u};
    asm volatile("s_nop 4" : "+s"(rs));          // a scalar register written by a vector instruction is read by a load 5 wait states later; the compiler
    return rs;                                   // sees to that for its own loads only
  }
  // 64 lanes x 16 bytes to LDS addresses dst + 16 lane.  Inline, because the compiler waits for the builtin's load before any LDS read that it
  // cannot tell apart - the other buffer's; tile_barrier() waits instead.  (No destination registers; m0 is a reserved register, which the compiler
  // writes in front of each use of its own and does not take in a clobber list.)
  static __device__ __forceinline__ void piece(u32x4 rs, uint32_t dst, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(dst), "v"(off), "s"(rs) : "memory");
  }
};
// This wavefront's pieces have landed, then everybody's.  (The builtin, so that the compiler knows of the wait: it would wait once more, for
// loads in front of the loop, behind the next tile's pieces.)
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);            // vmcnt(0)
  __syncthreads();
}

__device__ __forceinline__ f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
__device__ __forceinline__ float both_halves_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float both_halves_sum(float v) { return v + __shfl_xor(v, 32, 64); }

// Workgroups go round robin over the 8 XCDs, each with an L2 of its own: a contiguous run of the work per XCD keeps the tiles that read
// one key head's k and v (or q and dout) on one L2.  In that order the samples of a head follow each other, so that every XCD gets some of all
// lengths of a padded batch (16 samples of up to 777 tokens, 12 heads:
// 35 + 43 + 58 us; in the samples' order 48 + 62 + 82).
__device__ __forceinline__ int64_t xcd_order(int64_t bid, int64_t total) {
  const int64_t per = total >> 3, rest = total & 7, x = bid & 7, i = bid >> 3;
  return x * per + (x < rest ? x : rest) + i;
}

__device__ __forceinline__ int over(int r, int G) { return G == 1 ? r : static_cast<int>(static_cast<uint32_t>(r) / static_cast<uint32_t>(G)); }

// sum of a row's three bf16 terms (k-slots 0 .. 2 of its half) times ones: the product of four k-slots per half
__device__ __forceinline__ f32x16 first_terms(u32x2 terms, u32x2 ones) {
  return __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(__builtin_bit_cast(s16x4, terms), __builtin_bit_cast(s16x4, ones), zeros16(), 0, 0, 0);
}

// dS in fp16 (kScaled): |dS| <= 2 |dout| |v|, and a power of two, carried by dout or v (in bf16, exactly) and D, brings that bound to 2^13 .. 2^14:
// no dS overflows, and one 2^-27 of it still has all its bits.
// The size |x| of a row is the root of its sum of squares, which 32 bits hold for values of 2^-32 .. 2^32 only; beyond, the squares are formed behind
// a power of two that the row's largest value chooses.  Sizes are kept behind 2^-4: 2^128 sqrt(128) is a number then, and bf16's smallest one still is.
__device__ __forceinline__ float square_scale(float top) { return top >= 0x1p32f ? 0x1p-72f : top < 0x1p-32f ? 0x1p72f : 1.f; }
__device__ __forceinline__ float row_size(float top, float squares) {
  return sqrtf(squares) * (top >= 0x1p32f ? 0x1p68f : top < 0x1p-32f ? 0x1p-76f : 0x1p-4f);
}
// The exponent, from the exponents of the sizes (2 |x| |y| itself may be no number), for the power that x carries: it and its inverse are normal and
// x times it is finite.  Where that leaves the bound below 2^13, dS times it is still above 2^-13, or the gradient below bf16's numbers.  A size of zero,
// or one that is not finite, may give any power: dS is zero or not finite behind all of them.
__device__ __forceinline__ int scale_exponent(float x, float y) {
  const int ex = __builtin_amdgcn_frexp_expf(x), ey = __builtin_amdgcn_frexp_expf(y);
  const bool carry = __builtin_amdgcn_frexp_mantf(x) * __builtin_amdgcn_frexp_mantf(y) >= 0.5f;
  return max(min(13 - (ex + ey + (carry ? 8 : 7)), min(126, 123 - ex)), -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// largest sizes of v's and dout's rows of a head
__device__ __forceinline__ float2 range_of(const float2* range, int64_t bh, int pieces) {
  float2 r = range[bh * pieces];
  for (int p = 1; p < pieces; ++p) {
    const float2 x = range[bh * pieces + p];
    r.x = fmaxf(r.x, x.x);
    r.y = fmaxf(r.y, x.y);
  }
  return r;
}
template <int N>
__device__ __forceinline__ void scale_bf16(u32x4 (&f)[N], float s) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) f[i][j] = Bf16::pack(Bf16::lo(f[i][j]) * s, Bf16::hi(f[i][j]) * s);
}

template <typename T> __device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) { return make_uint2(T::pack(a, b), T::pack(c, d)); }

// A workgroup of the forward or of dq: 128 rows of one key head against the keys [k_begin, k_end), tile by tile.
template <int D>
struct Tile {
  static constexpr int IMG = kKT * D * 2;
  Stage<D> sk, sv;
  const uint16_t *kp, *vp;                       // the key head's first key
  Limits lim;
  int64_t b;
  int hk, split;
  int tok, hd, end;                              // this lane's row: token (Nq where there is none), head of the key head, first key it does not see
  int wave_end;                                  // the same of the wavefront's rows together
  int k_begin, k_end;
  bool few;                                      // (uniform) some rows see no key behind the first tile
  uint32_t base;

  __device__ __forceinline__ Tile(const MhaArgs& a, uint32_t lds) : Tile(a, lds, xcd_order(blockIdx.x, gridDim.x)) {}
  __device__ __forceinline__ Tile(const MhaArgs& a, uint32_t lds, int64_t w) : lim(a, w / (a.tiles * a.splits) % a.B) {
    const int per_h = a.tiles * a.splits;
    const int64_t head = w / per_h;
    hk = static_cast<int>(head / a.B);
    b = head - hk * a.B;
    const int rest = static_cast<int>(w - head * per_h);
    const int tile = a.tiles - 1 - rest / a.splits;                    // causal: the long tiles first
    split = rest % a.splits;
    base = lds;
    kp = a.k + b * a.vk.b + hk * a.vk.h;
    vp = a.v + b * a.vv.b + hk * a.vv.h;
    const int R = a.Nq * a.G, row0 = tile * 128, wave = threadIdx.x >> 6;                     // (31 bits: checked on the host)
    // what the rows from `first` to `last` see of the keys
    auto end_of = [&](int first, int last) {
      const int t0 = over(first, a.G), t1 = min(over(min(last, R - 1), a.G), lim.q_len - 1);
      return first < R && t0 <= t1 ? lim.end(t1, a.causal) : 0;
    };
    k_begin = split * a.span;
    k_end = min(end_of(row0, row0 + 127), k_begin + a.span);
    wave_end = __builtin_amdgcn_readfirstlane(min(end_of(row0 + wave * 32, row0 + wave * 32 + 31), k_end));
    const int r = row0 + wave * 32 + (threadIdx.x & 31);
    tok = r < R ? over(r, a.G) : a.Nq;
    hd = r < R ? r - tok * a.G : 0;
    end = lim.end(tok, a.causal);
    few = k_begin == 0 && k_end > 0 && lim.end(over(row0, a.G), a.causal) <= kKT;
    sk.rows_apart(a.vk.n);
    sv.rows_apart(a.vv.n);
    if (k_begin < k_end) fetch(a, k_begin, 0);
  }
  __device__ __forceinline__ void fetch(const MhaArgs& a, int k0, uint32_t buffer) const {
    sk.load(kp + k0 * a.vk.n, lim.kv_len - k0, base + buffer);
    sv.load(vp + k0 * a.vv.n, lim.kv_len - k0, base + buffer + IMG);
  }
  // compute(first key, image) for every tile that the wavefront's rows see a key of
  template <typename F>
  __device__ __forceinline__ void walk(const MhaArgs& a, F compute) const {
    auto step = [&](int k0, uint32_t image, uint32_t next) {
      tile_barrier();                            // the tile is there, and nobody reads the other buffer any more
      if (k0 + kKT < k_end) fetch(a, k0 + kKT, next);
      if (wave_end > k0) compute(k0, image);
    };
    for (int k0 = k_begin; k0 < k_end; k0 += 2 * kKT) {
      step(k0, 0, 2 * IMG);
      if (k0 + kKT < k_end) step(k0 + kKT, 2 * IMG, 0);
    }
  }
};

// ===================================================================================================================== forward
// Workgroup: 4 wavefronts x 32 rows of one key head, over the keys [split * span, + span).  A row is a lane.
// The running maximum of a row moves only when a tile exceeds it by more than 2^kSlack: until then P grows to at most 2^8, which costs
// neither type any accuracy (both are relative) and saves the rescaling of the result's registers.
// What bounds it: per 32 x 32 block 8 (d = 64) products of 32 cycles and about 75 other instructions, 16 exponentials among them; the two
// share the issue slots of a SIMD (a product takes about half its cycles from the others), at the clock that the power limit leaves.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void mha_fwd_kernel(const MhaArgs a) {
  constexpr int KS = D / 16, DB = D / 32, IMG = kKT * D * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * 2 * IMG];              // [buffer][k, v]
  const Tile<D> w(a, lds_addr(&lds[0]));
  const int half = (threadIdx.x >> 5) & 1;
  u32x4 qf[KS];
  {
    const bool live = w.tok < w.lim.q_len;
    const uint16_t* src = a.q + w.b * a.vq.b + (static_cast<int64_t>(w.hk) * a.G + w.hd) * a.vq.h + (live ? w.tok : 0) * a.vq.n;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = u32x4{0, 0, 0, 0};
      if (live) qf[ks] = *reinterpret_cast<const u32x4*>(src + ks * 16 + half * 8);
    }
  }
  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zeros16();
  const Lane<D> L(w.base);
  auto compute = [&](int k0, uint32_t kimg) {
    constexpr int NB = kKT / 32;
    const uint32_t vimg = kimg + IMG;
    f32x16 s[NB];
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
      s[blk] = zeros16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[blk] = T::mfma_s(L.row(kimg, blk, ks), qf[ks], s[blk]);
    }
    if (__any(w.end < k0 + kKT)) {
#pragma unroll
      for (int blk = 0; blk < NB; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + blk * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          s[blk][r] = key < w.end ? s[blk][r] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int blk = 0; blk < NB; ++blk)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[blk][r]);
    mx = both_halves_max(mx) * c2;               // (c2 > 0: checked on the host)
    if (__any(mx > m + kSlack)) {                // lanes below keep their maximum
      const bool up = mx > m + kSlack;
      const float al = up ? __builtin_amdgcn_exp2f(m - mx) : 1.f;      // m = -inf: 0
      m = up ? mx : m;
      l *= al;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= al;
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[blk][r] = __builtin_amdgcn_exp2f(fmaf(s[blk][r], c2, -mu));
        l += s[blk][r];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = T::pack(s[blk][t * 8 + 2 * j], s[blk][t * 8 + 2 * j + 1]);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = T::mfma(L.col(vimg, blk, t, db), p, o[db]);
      }
    }
  };
  w.walk(a, compute);

  // lane = row: results of the row in registers, d = db * 32 + (r & 3) + 8 (r >> 2) + 4 half
  const float sum = both_halves_sum(l);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (__any(sum == 0.f)) {                       // rows that see no key, beside others whose keys are not finite: 0 x inf is in their registers
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = sum == 0.f ? 0.f : o[db][r];
  }
  if (w.tok >= a.Nq) return;
  const int h = w.hk * a.G + w.hd;
  const int64_t at = (w.b * a.H + h) * a.Nq + w.tok;
  const float ls = sum == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * kLn2;
  if (a.splits > 1) {                            // this split's normalised result in 32 bits and its log sum exp
    const int64_t rows = a.B * a.H * a.Nq;
    float* po = a.part + (w.split * rows + at) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(po + db * 32 + 8 * g + 4 * half) =
            make_float4(o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
    if (half == 0) a.part[a.splits * rows * D + w.split * rows + at] = ls;
  } else {
    uint16_t* po = a.o + w.b * a.vo.b + w.tok * a.vo.n + h * a.vo.h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(po + db * 32 + 8 * g + 4 * half) =
            pack4<T>(o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
    if (a.lse && half == 0) a.lse[at] = ls;
  }
}

// Joins the splits of the keys (one query against 16384 keys, 8 x 16 heads on 4, d 128: forward 41 us and this 4 us for 268 MB, 5.9 TB/s; a
// copy of 2 GiB reaches 4.9): out = sum_s exp(lse_s - lse) out_s.  D / 4 threads per row; eight splits' values are in flight at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void mha_join_kernel(const MhaArgs a) {
  constexpr int TPR = D / 4;
  const int64_t rows = a.B * a.H * a.Nq, at = static_cast<int64_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (at >= rows) return;
  const int d4 = threadIdx.x % TPR;
  const float* ls = a.part + static_cast<int64_t>(a.splits) * rows * D;
  float m = -INFINITY, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float e[8];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t s = min(s0 + u, a.splits - 1);
      e[u] = ls[s * rows + at];
      v[u] = *reinterpret_cast<const float4*>(a.part + (s * rows + at) * D + d4 * 4);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u >= a.splits) e[u] = -INFINITY;
      mn = fmaxf(mn, e[u]);
    }
    const float mu = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f((m - mu) * kLog2e);
    m = mn;
    sum *= al;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= al;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float g = __builtin_amdgcn_exp2f((e[u] - mu) * kLog2e);
      sum += g;
      x[0] = fmaf(g, v[u].x, x[0]); x[1] = fmaf(g, v[u].y, x[1]); x[2] = fmaf(g, v[u].z, x[2]); x[3] = fmaf(g, v[u].w, x[3]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t bh = at / a.Nq, b = bh / a.H;
  const int i = static_cast<int>(at - bh * a.Nq), h = static_cast<int>(bh - b * a.H);
  *reinterpret_cast<uint2*>(a.o + b * a.vo.b + i * a.vo.n + h * a.vo.h + d4 * 4) = pack4<T>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  if (a.lse && d4 == 0) a.lse[at] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum) * kLn2;
}

// ===================================================================================================================== backward
// Sums of 32 values over the 32 lanes of a half: lane l32 gets the sum of value l32.  Every step halves the values that a lane still holds; lanes
// of opposite bit trade what the other one keeps, across rows of 16 lanes, then within them.
template <int CTRL>
__device__ __forceinline__ float traded(bool upper, float lo, float hi) {
  const float keep = upper ? hi : lo, give = upper ? lo : hi;
  return keep + __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(give)), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float rows_sum(float (&v)[32]) {
  const int lane = threadIdx.x;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[k]), __float_as_uint(v[k + 16]), false, false);
    v[k] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = traded<0x140>(lane & 8, v[k], v[k + 8]);                  // row_mirror: lane 15 - i
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = traded<0x141>(lane & 4, v[k], v[k + 4]);                  // row_half_mirror: lane 7 - i
#pragma unroll
  for (int k = 0; k < 2; ++k) v[k] = traded<0x1b>(lane & 2, v[k], v[k + 2]);                   // quad_perm: lane 3 - i
  return traded<0xb1>(lane & 1, v[0], v[1]);                                                   // quad_perm: lane i ^ 1
}

// The gradient g of a row of q' (k') becomes that of q (k) in the accumulators it is in: lane = row, d = db * 32 + (r & 3) + 8 (r >> 2) + 4 half,
// so both members of a pair are one lane's, and a row's sums need one exchange of the two halves (32 x 577 tokens, 12 heads: 14 us on dq and 18 on
// dk / dv, where a pass of its own over dq' and dk' took 48).  With z = x r w the normalised row, R its
// rotation:  dz = R^T g,  dw = sum over the rows of dz * (x r),  dx = r (dz w - (x r) mean(dz w * (x r))).  Nothing is rounded in between.
template <typename T, int D>
__device__ __forceinline__ void turn_back(const MhaArgs& a, const Turn& t, f32x16 (&g)[D / 32], int64_t b, int tok, int h, bool live) {
  constexpr int DB = D / 32;
  const int half = (threadIdx.x >> 5) & 1;
  const int64_t i = live ? tok : 0;
  if (a.cs) {
    const float2* cs = a.cs + b * a.cs_b + i * (D / 2);
    if (a.il) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 p = *reinterpret_cast<const float4*>(cs + db * 16 + 4 * q + 2 * half);  // (cos, sin) of two pairs
          const float g0 = g[db][4 * q], g1 = g[db][4 * q + 1], g2 = g[db][4 * q + 2], g3 = g[db][4 * q + 3];
          g[db][4 * q] = fmaf(g0, p.x, g1 * p.y);
          g[db][4 * q + 1] = fmaf(g1, p.x, -g0 * p.y);
          g[db][4 * q + 2] = fmaf(g2, p.z, g3 * p.w);
          g[db][4 * q + 3] = fmaf(g3, p.z, -g2 * p.w);
        }
    } else {
#pragma unroll
      for (int db = 0; db < DB / 2; ++db)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float4 p = *reinterpret_cast<const float4*>(cs + db * 32 + 8 * (r >> 2) + 4 * half + (r & 3));
          const float g0 = g[db][r], g1 = g[db][r + 1], e0 = g[db + DB / 2][r], e1 = g[db + DB / 2][r + 1];
          g[db][r] = fmaf(g0, p.x, e0 * p.y);
          g[db + DB / 2][r] = fmaf(e0, p.x, -g0 * p.y);
          g[db][r + 1] = fmaf(g1, p.z, e1 * p.w);
          g[db + DB / 2][r + 1] = fmaf(e1, p.z, -g1 * p.w);
        }
    }
  }
  if (!a.norm) return;
  const uint16_t* px = t.x + b * t.vx.b + i * t.vx.n + h * t.vx.h + 4 * half;
  float x[DB][16], ss = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint2 v = *reinterpret_cast<const uint2*>(px + db * 32 + 8 * q);
      x[db][4 * q] = T::lo(v.x); x[db][4 * q + 1] = T::hi(v.x); x[db][4 * q + 2] = T::lo(v.y); x[db][4 * q + 3] = T::hi(v.y);
#pragma unroll
      for (int u = 0; u < 4; ++u) ss = fmaf(x[db][4 * q + u], x[db][4 * q + u], ss);
    }
  const float rn = 1.f / sqrtf(both_halves_sum(ss) * (1.f / D) + a.eps);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[db][r] *= rn;
  if (t.part) {                                  // (uniform) over the workgroup's 128 rows
    __shared__ float red[4 * D];
    const int l32 = threadIdx.x & 31, wave = threadIdx.x >> 6;
#pragma unroll
    for (int db = 0; db < DB; db += 2) {
      float e[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) e[k] = live ? g[db + (k >> 4)][k & 15] * x[db + (k >> 4)][k & 15] : 0.f;
      const int r = l32 & 15;
      red[wave * D + (db + (l32 >> 4)) * 32 + (r & 3) + 8 * (r >> 2) + 4 * half] = rows_sum(e);
    }
    __syncthreads();
    if (threadIdx.x < D) {
      const int e = threadIdx.x;
      t.part[static_cast<int64_t>(blockIdx.x) * D + e] = ((red[e] + red[D + e]) + red[2 * D + e]) + red[3 * D + e];
    }
  }
  float dot = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4u w = {1.f, 1.f, 1.f, 1.f};
      if (t.w) w = *reinterpret_cast<const f32x4u*>(t.w + db * 32 + 8 * q + 4 * half);
      g[db][4 * q] *= w.x; g[db][4 * q + 1] *= w.y; g[db][4 * q + 2] *= w.z; g[db][4 * q + 3] *= w.w;
#pragma unroll
      for (int u = 0; u < 4; ++u) dot = fmaf(g[db][4 * q + u], x[db][4 * q + u], dot);
    }
  dot = both_halves_sum(dot) * (1.f / D);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) g[db][r] = rn * fmaf(-x[db][r], dot, g[db][r]);
}

// Largest sizes (row_size) of v's and dout's rows of a head, `pieces` workgroups each.  16 bytes per lane, D / 8 lanes a row; bound by memory (32 x 577 tokens,
// 12 heads: 57 MB in 11 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void mha_range_kernel(const MhaArgs a, float2* __restrict__ range) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const int64_t bh = blockIdx.x / a.pieces, b = bh / a.H, h = bh - b * a.H;
  const int piece = static_cast<int>(blockIdx.x - bh * a.pieces), c = threadIdx.x % LANES;
  float top[2] = {0.f, 0.f};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const View& view = which ? a.vdo : a.vv;
    const uint16_t* p = (which ? a.dout : a.v) + b * view.b + h * view.h + c * 8;
    for (int i = piece * ROWS + threadIdx.x / LANES; i < a.Nk; i += a.pieces * ROWS) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p + i * view.n);
      float largest = 1.f;
      auto squares = [&](float up) {                                   // (a row's lanes are here together)
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = T::lo(x[j]) * up, hi = T::hi(x[j]) * up;
          s = fmaf(lo, lo, fmaf(hi, hi, s));
        }
        for (int m = 1; m < LANES; m <<= 1) s += __shfl_xor(s, m, 64);
        return s;
      };
      float s = squares(1.f);
      if (__any(!(s >= 0x1p-60f && s <= 0x1p60f))) {                   // (rows of zeros, too)
        largest = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) largest = fmaxf(largest, fmaxf(fabsf(T::lo(x[j])), fabsf(T::hi(x[j]))));
        for (int m = 1; m < LANES; m <<= 1) largest = fmaxf(largest, __shfl_xor(largest, m, 64));
        s = squares(square_scale(largest));
      }
      s = row_size(largest, s);
      top[which] = s > top[which] || s != s ? s : top[which];
    }
    for (int m = LANES; m < 64; m <<= 1) top[which] = fmaxf(top[which], __shfl_xor(top[which], m, 64));
  }
  __shared__ float2 red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(top[0], top[1]);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 4; ++k) { top[0] = fmaxf(top[0], red[k].x); top[1] = fmaxf(top[1], red[k].y); }
    range[blockIdx.x] = make_float2(top[0], top[1]);
  }
}

// dq: workgroup = 4 wavefronts x 32 rows, over the keys [split * span, + span).  Also leaves D in dvec.
template <typename T, int D, bool TURN>
__global__ __launch_bounds__(256, 2) void mha_dq_kernel(const MhaArgs a) {
  constexpr int KS = D / 16, DB = D / 32, IMG = kKT * D * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * 2 * IMG];              // [buffer][k, v]
  const Tile<D> w(a, lds_addr(&lds[0]));
  const int half = (threadIdx.x >> 5) & 1, h = w.hk * a.G + w.hd;
  const int64_t at = (w.b * a.H + h) * a.Nq + w.tok;
  u32x4 qf[KS], gf[KS];
  float lse2, dd, mul = a.scale, dd_mul = 1.f;
  {
    const bool live = w.end > 0;                 // a row without keys has no gradient
    const int64_t i = live ? w.tok : 0;
    const uint16_t* pq = a.q + w.b * a.vq.b + h * a.vq.h + i * a.vq.n + half * 8;
    const uint16_t* pg = a.dout + w.b * a.vdo.b + h * a.vdo.h + i * a.vdo.n + half * 8;
    const uint16_t* po = a.out + w.b * a.vo.b + h * a.vo.h + i * a.vo.n + half * 8;
    float part = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = gf[ks] = u32x4{0, 0, 0, 0};
      if (live) {
        qf[ks] = *reinterpret_cast<const u32x4*>(pq + ks * 16);
        gf[ks] = *reinterpret_cast<const u32x4*>(pg + ks * 16);
        const u32x4 of = *reinterpret_cast<const u32x4*>(po + ks * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) part = fmaf(T::lo(gf[ks][j]), T::lo(of[j]), fmaf(T::hi(gf[ks][j]), T::hi(of[j]), part));
      }
    }
    dd = both_halves_sum(part);
    lse2 = live ? a.lse[at] * kLog2e : INFINITY;                       // exp2(s - inf) = 0
    if constexpr (T::kScaled) {                  // a row's own scale
      float largest = 0.f, squares = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) largest = fmaxf(largest, fmaxf(fabsf(T::lo(gf[ks][j])), fabsf(T::hi(gf[ks][j]))));
      largest = both_halves_max(largest);
      const float up = square_scale(largest);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = T::lo(gf[ks][j]) * up, hi = T::hi(gf[ks][j]) * up;
          squares = fmaf(lo, lo, fmaf(hi, hi, squares));
        }
      const int e = scale_exponent(row_size(largest, both_halves_sum(squares)), range_of(a.range, w.b * a.H + h, a.pieces).x);
      scale_bf16(gf, power_of_two(e));
      dd *= power_of_two(e);
      dd_mul = power_of_two(-e);
      mul *= dd_mul;
    }
  }
  const float c2 = a.scale * kLog2e;
  const Lane<D> L(w.base);
  // D of rows with few keys from the tile itself, sum P dP: out is rounded, and of two or three keys' dP little is left when D is taken away
  if (w.few) {
    tile_barrier();
    float sum = 0.f;
#pragma unroll
    for (int blk = 0; blk < kKT / 32; ++blk) {
      f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = T::mfma_s(L.row(0, blk, ks), qf[ks], s);
        dp = T::mfma(L.row(IMG, blk, ks), gf[ks], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = blk * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
        sum += key < w.end ? __builtin_amdgcn_exp2f(fmaf(s[r], c2, -lse2)) * dp[r] : 0.f;
      }
    }
    sum = both_halves_sum(sum);
    if (w.end <= kKT) dd = sum;
  }
  if (w.split == 0 && half == 0 && w.tok < a.Nq) a.dvec[at] = dd * dd_mul;
  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zeros16();
  auto compute = [&](int k0, uint32_t kimg) {
    const uint32_t vimg = kimg + IMG;
    const bool masked = __any(w.end < k0 + kKT);
#pragma unroll
    for (int blk = 0; blk < kKT / 32; ++blk) {
      f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = T::mfma_s(L.row(kimg, blk, ks), qf[ks], s);
        dp = T::mfma(L.row(vimg, blk, ks), gf[ks], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, -lse2)) * (dp[r] - dd);
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + blk * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          s[r] = key < w.end ? s[r] : 0.f;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = T::pack_s(s[t * 8 + 2 * j], s[t * 8 + 2 * j + 1]);
#pragma unroll
        for (int db = 0; db < DB; ++db) dq[db] = T::mfma_s(L.col(kimg, blk, t, db), p, dq[db]);
      }
    }
  };
  w.walk(a, compute);
  if (__any(w.end <= w.k_begin)) {               // (as in the forward)
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[db][r] = w.end <= w.k_begin ? 0.f : dq[db][r];
  }
  if constexpr (TURN) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[db][r] *= mul;
    mul = 1.f;
    if (a.splits == 1) turn_back<T, D>(a, a.tq, dq, w.b, w.tok, h, w.tok < a.Nq);
  }
  if (w.tok >= a.Nq) return;
  if (a.splits > 1) {
    float* po = a.part + (w.split * a.B * a.H * a.Nq + at) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(po + db * 32 + 8 * g + 4 * half) =
            make_float4(dq[db][4 * g], dq[db][4 * g + 1], dq[db][4 * g + 2], dq[db][4 * g + 3]);
  } else {
    uint16_t* po = a.dq + w.b * a.vdq.b + w.tok * a.vdq.n + h * a.vdq.h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(po + db * 32 + 8 * g + 4 * half) =
            pack4<T>(dq[db][4 * g] * mul, dq[db][4 * g + 1] * mul, dq[db][4 * g + 2] * mul, dq[db][4 * g + 3] * mul);
  }
}

// dq = scale * sum of the splits' partial sums, in their order
template <typename T, int D>
__global__ __launch_bounds__(256) void mha_dq_join_kernel(const MhaArgs a) {
  constexpr int TPR = D / 4;
  const int64_t rows = a.B * a.H * a.Nq, at = static_cast<int64_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (at >= rows) return;
  const int d4 = threadIdx.x % TPR;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const float4*>(a.part + (min(s0 + u, a.splits - 1) * rows + at) * D + d4 * 4);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (s0 + u < a.splits) { x[0] += v[u].x; x[1] += v[u].y; x[2] += v[u].z; x[3] += v[u].w; }
  }
  const int64_t bh = at / a.Nq, b = bh / a.H;
  const int i = static_cast<int>(at - bh * a.Nq), h = static_cast<int>(bh - b * a.H);
  *reinterpret_cast<uint2*>(a.dq + b * a.vdq.b + i * a.vdq.n + h * a.vdq.h + d4 * 4) =
      pack4<T>(x[0] * a.scale, x[1] * a.scale, x[2] * a.scale, x[3] * a.scale);
}

// dk, dv: workgroup = 4 wavefronts x 32 keys of one key head, over the rows that see them, a tile of up to 64 at a time: the 64 / G tokens
// that fill one (or, with more than 64 heads on a key head, 64 heads of a token), so that a row's place in its tile never changes.
// Here a lane is a key and lse and D belong to registers.  They enter as the products' initial values instead: lane l32 of the lower half
// holds -lse / scale of row l32, of the upper half -D, as three bf16 terms (24 bits) in its first three k-slots, and one product with
// ones in the lower (upper) half's slots leaves -lse / scale (-D) in the accumulators of S (of dout v^T): exp2 of S times scale log2(e) is P.
template <typename T, int D, bool TURN>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void mha_dkv_kernel(const MhaArgs a) {
  constexpr int KS = D / 16, DB = D / 32, KEYS = 128, RT = kKT, IMG = RT * D * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * 2 * IMG];              // [buffer][q, dout]
  __shared__ __attribute__((aligned(16))) int row_tok[RT];                               // token of a tile's row, from the tile's first
  const int wave = threadIdx.x >> 6, l32 = threadIdx.x & 31, half = (threadIdx.x >> 5) & 1;
  const int64_t per_h = static_cast<int64_t>(a.tiles) * a.splits;
  int64_t w = xcd_order(blockIdx.x, gridDim.x);
  const int64_t head = w / per_h;
  const int hk = static_cast<int>(head / a.B);
  const int64_t b = head - hk * a.B;
  w -= head * per_h;
  const int tile = static_cast<int>(w / a.splits), split = static_cast<int>(w - static_cast<int64_t>(tile) * a.splits);    // causal: long ones first
  const Limits lim(a, b);
  const uint16_t* qb = a.q + b * a.vq.b + static_cast<int64_t>(hk) * a.G * a.vq.h;
  const uint16_t* gb = a.dout + b * a.vdo.b + static_cast<int64_t>(hk) * a.G * a.vdo.h;
  const uint16_t* kb = a.k + b * a.vk.b + hk * a.vk.h;
  const uint16_t* vb = a.v + b * a.vv.b + hk * a.vv.h;
  const int key0 = tile * KEYS, key = key0 + wave * 32 + l32;

  const int gt = min(a.G, RT), tt = RT / gt;                           // heads and tokens of a row tile
  // first token that sees a key of this tile; every row from there on sees one.  The splits share these tokens equally.
  const int t_first = a.causal ? max(0, key0 - lim.off) : 0, t_last = key0 < lim.kv_len ? lim.q_len : 0;
  const int share = (max(0, t_last - t_first) + a.splits * tt - 1) / (a.splits * tt) * tt;
  const int t_begin = min(t_first + split * share, max(t_first, t_last)), t_end = min(t_begin + share, t_last);
  Stage<D> sq, sg;
#pragma unroll
  for (int p = 0; p < Stage<D>::PER; ++p) {
    const int row = Stage<D>::row(p), i = row / gt, j = row - i * gt;
    sq.off[p] = static_cast<uint32_t>((i * a.vq.n + j * a.vq.h) * 2) + Stage<D>::chunk(p);
    sg.off[p] = static_cast<uint32_t>((i * a.vdo.n + j * a.vdo.h) * 2) + Stage<D>::chunk(p);
  }
  if (threadIdx.x < RT) row_tok[threadIdx.x] = threadIdx.x / gt;
  // the lane's rows' lse (lower half) or D (upper half)
  int st_off[2];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    const int row = blk * 32 + l32, i = row / gt;
    st_off[blk] = (row - i * gt) * a.Nq + i;
  }
  const float* st_base = (half ? a.dvec : a.lse) + (b * a.H + static_cast<int64_t>(hk) * a.G) * a.Nq;
  float st[2] = {0.f, 0.f};                                            // as loaded: nothing waits for them before the next tile
  const uint32_t base = lds_addr(&lds[0]);
  int t0 = t_begin, h0 = 0;                                            // the tile that is fetched next
  int rows = 0;                                                        // its rows (tokens of all G heads, or heads of a token: always the first ones)
  auto fetch = [&](uint32_t buffer) {
    rows = min(tt, t_end - t0) * min(gt, a.G - h0);
    sq.load(qb + t0 * a.vq.n + h0 * a.vq.h, rows, base + buffer);
    sg.load(gb + t0 * a.vdo.n + h0 * a.vdo.h, rows, base + buffer + IMG);
    const float* ps = st_base + static_cast<int64_t>(h0) * a.Nq + t0;
    st[0] = ps[l32 < rows ? st_off[0] : 0];
    st[1] = ps[32 + l32 < rows ? st_off[1] : 0];
  };
  if (t0 < t_end) fetch(0);

  u32x4 kf[KS], vf[KS];
  f32x16 dk[DB], dv[DB];
  {
    const bool live = key < lim.kv_len;
    const int64_t j = live ? key : 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = vf[ks] = u32x4{0, 0, 0, 0};
      if (live) {
        kf[ks] = *reinterpret_cast<const u32x4*>(kb + j * a.vk.n + ks * 16 + half * 8);
        vf[ks] = *reinterpret_cast<const u32x4*>(vb + j * a.vv.n + ks * 16 + half * 8);
      }
    }
  }
#pragma unroll
  for (int db = 0; db < DB; ++db) { dk[db] = zeros16(); dv[db] = zeros16(); }
  float dk_mul = a.scale, d_mul = -1.f;
  if constexpr (T::kScaled) {                    // one scale for the head: a key's dk sums over rows
    const float2 r = range_of(a.range, b * a.H + hk, a.pieces);
    const int e = scale_exponent(r.x, r.y);
    scale_bf16(vf, power_of_two(e));
    d_mul = -power_of_two(e);
    dk_mul *= power_of_two(-e);
  }
  const float c2 = a.scale * kLog2e;
  const Lane<D> L(base);
  const u32x2 ones = {0x3f803f80u, 0x00003f80u};                       // bf16 (1, 1, 1, 0)
  const u32x2 ones_s = half ? u32x2{0, 0} : ones, ones_d = half ? ones : u32x2{0, 0};
  const float st_mul = half ? d_mul : -1.f / a.scale;
  const int last_tok[2] = {31 / gt, 63 / gt};                          // token in the tile of a block's last row
  const int wave_key = key0 + wave * 32, wave_last = min(wave_key + 32, lim.kv_len) - 1;       // the wavefront's keys
  auto step = [&](int buf) {
    const uint32_t qimg = buf * 2 * IMG, gimg = qimg + IMG;
    tile_barrier();
    const int t = t0, here = rows;
    u32x2 init[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const float x = blk * 32 + l32 < here ? st[blk] * st_mul : half ? 0.f : -3e38f;        // no row: P = exp2(-huge) = 0
      const uint32_t hi = __float_as_uint(x) & 0xffff0000u;            // truncated: the rest keeps its sign and 16 bits
      const float y = x - __uint_as_float(hi);
      const uint32_t mid = __float_as_uint(y) & 0xffff0000u;
      const float z = y - __uint_as_float(mid);
      init[blk] = u32x2{(hi >> 16) | mid, __float_as_uint(z) >> 16};
    }
    h0 += gt;
    if (h0 >= a.G) { h0 = 0; t0 += tt; }
    if (t0 < t_end) fetch((buf ^ 1) * 2 * IMG);
    if (wave_last < wave_key) return;                                  // all its keys are padding
    // a tile needs no mask if its first token sees the wavefront's last key; keys beyond kv_len are zeros whose dk, dv are not kept
    const bool masked = a.causal && t + lim.off < wave_last;
    const int lim_tok = key - t - lim.off;                             // masked: the row's token in the tile has to be at least this
#pragma unroll
    for (int blk = 0; blk < RT / 32; ++blk) {
      if (blk * 32 >= here || (a.causal && t + last_tok[blk] + lim.off < wave_key)) continue;    // no row, or none that sees a key
      u32x4 qr[KS], gr[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qr[ks] = L.row(qimg, blk, ks);
        gr[ks] = L.row(gimg, blk, ks);
      }
      f32x16 s = first_terms(init[blk], ones_s), dp = first_terms(init[blk], ones_d);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = T::mfma_s(qr[ks], kf[ks], s);
        dp = T::mfma(gr[ks], vf[ks], dp);
      }
      u32x4 gc[2][DB], qc[2][DB];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          gc[t][db] = L.col(gimg, blk, t, db);
          qc[t][db] = L.col(qimg, blk, t, db);
        }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] * c2);
        dp[r] = s[r] * dp[r];
      }
      if (masked) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 e4 = *reinterpret_cast<const int4*>(&row_tok[blk * 32 + 8 * g + 4 * half]);
          const int ev[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            s[4 * g + u] = ev[u] >= lim_tok ? s[4 * g + u] : 0.f;
            dp[4 * g + u] = ev[u] >= lim_tok ? dp[4 * g + u] : 0.f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 pf, df;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pf[j] = T::pack(s[t * 8 + 2 * j], s[t * 8 + 2 * j + 1]);
          df[j] = T::pack_s(dp[t * 8 + 2 * j], dp[t * 8 + 2 * j + 1]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          dv[db] = T::mfma(gc[t][db], pf, dv[db]);
          dk[db] = T::mfma_s(qc[t][db], df, dk[db]);
        }
      }
    }
  };
  while (t0 < t_end) {
    step(0);
    if (t0 < t_end) step(1);
  }
  if constexpr (TURN) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[db][r] *= dk_mul;
  }
  if (TURN && a.splits == 1) {
    const bool live = key < a.Nk;
    if (live) {
      uint16_t* pv = a.dv + b * a.vdv.b + key * a.vdv.n + hk * a.vdv.h;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(pv + db * 32 + 8 * g + 4 * half) = pack4<T>(dv[db][4 * g], dv[db][4 * g + 1], dv[db][4 * g + 2], dv[db][4 * g + 3]);
    }
    turn_back<T, D>(a, a.tk, dk, b, key, hk, live);
    if (!live) return;
    uint16_t* pk = a.dk + b * a.vdk.b + key * a.vdk.n + hk * a.vdk.h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(pk + db * 32 + 8 * g + 4 * half) = pack4<T>(dk[db][4 * g], dk[db][4 * g + 1], dk[db][4 * g + 2], dk[db][4 * g + 3]);
    return;
  }
  if (key >= a.Nk) return;
  const bool live = key < lim.kv_len;
  if (a.splits > 1) {                            // [split][dk, dv][sample, head, key][D] in 32 bits
    const int64_t keys = a.B * a.Hkv * a.Nk, at = (b * a.Hkv + hk) * a.Nk + key;
    float* pk = a.part + (2 * split * keys + at) * D + 4 * half;
    float* pv = pk + keys * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r = 4 * g, e = db * 32 + 8 * g;
        *reinterpret_cast<float4*>(pk + e) = live ? make_float4(dk[db][r], dk[db][r + 1], dk[db][r + 2], dk[db][r + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(pv + e) = live ? make_float4(dv[db][r], dv[db][r + 1], dv[db][r + 2], dv[db][r + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    return;
  }
  uint16_t* pk = a.dk + b * a.vdk.b + key * a.vdk.n + hk * a.vdk.h;
  uint16_t* pv = a.dv + b * a.vdv.b + key * a.vdv.n + hk * a.vdv.h;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] = live ? dk[db][4 * g + u] * a.scale : 0.f;
        y[u] = live ? dv[db][4 * g + u] : 0.f;
      }
      *reinterpret_cast<uint2*>(pk + db * 32 + 8 * g + 4 * half) = pack4<T>(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<uint2*>(pv + db * 32 + 8 * g + 4 * half) = pack4<T>(y[0], y[1], y[2], y[3]);
    }
}

// dk = scale * sum of the splits' partial sums, dv = their sum, in their order
template <typename T, int D>
__global__ __launch_bounds__(256) void mha_dkv_join_kernel(const MhaArgs a) {
  constexpr int TPR = D / 4;
  const int64_t keys = a.B * a.Hkv * a.Nk, at = static_cast<int64_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (at >= keys) return;
  const int d4 = threadIdx.x % TPR, is_v = blockIdx.y;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += 4) {
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = *reinterpret_cast<const float4*>(a.part + ((2 * static_cast<int64_t>(min(s0 + u, a.splits - 1)) + is_v) * keys + at) * D + d4 * 4);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u < a.splits) { x[0] += v[u].x; x[1] += v[u].y; x[2] += v[u].z; x[3] += v[u].w; }
  }
  const int64_t bh = at / a.Nk, b = bh / a.Hkv;
  const int j = static_cast<int>(at - bh * a.Nk), h = static_cast<int>(bh - b * a.Hkv);
  const float mul = is_v ? 1.f : a.scale;
  uint16_t* po = is_v ? a.dv + b * a.vdv.b + j * a.vdv.n + h * a.vdv.h : a.dk + b * a.vdk.b + j * a.vdk.n + h * a.vdk.h;
  *reinterpret_cast<uint2*>(po + d4 * 4) = pack4<T>(x[0] * mul, x[1] * mul, x[2] * mul, x[3] * mul);
}

// The splits' sums of rows of dq' (blockIdx.y = 0 of one), or of dk' and dv (of two), and of the former the way back to dq (dk): as turn_back, with
// D / 4 threads to a row, 4 consecutive values each.  (Layer forward + backward, host included: 2 x 626 tokens, 3 heads 125 -> 93 us, 3 x 530, 8 heads
// 127 -> 85 against workgroups that meet all keys or rows.)
template <typename T, int D>
__global__ __launch_bounds__(256) void mha_turn_join_kernel(const MhaArgs a) {
  constexpr int TPR = D / 4, ROWS = 256 / TPR;
  __shared__ float red[ROWS * D];
  const bool keys = gridDim.y == 2, is_v = blockIdx.y == 1;
  const int64_t rows = a.B * a.H * a.Nk, at = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR, row = at < rows ? at : rows - 1;
  const int d4 = threadIdx.x % TPR;
  const float* part = a.part + ((is_v ? rows : 0) + row) * D + d4 * 4;
  const int64_t step = (keys ? 2 : 1) * rows * D;
  float g[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += 4) {
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const float4*>(part + min(s0 + u, a.splits - 1) * step);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u < a.splits) { g[0] += v[u].x; g[1] += v[u].y; g[2] += v[u].z; g[3] += v[u].w; }
  }
  const int64_t bh = row / a.Nk, b = bh / a.H;
  const int tok = static_cast<int>(row - bh * a.Nk), h = static_cast<int>(bh - b * a.H);
  const Turn& t = keys ? a.tk : a.tq;
  if (!is_v) {                                   // (uniform)
    if (a.cs) {
      const float2* cs = a.cs + b * a.cs_b + static_cast<int64_t>(tok) * (D / 2);
      if (a.il) {
        const float4 p = *reinterpret_cast<const float4*>(cs + 2 * d4);
        const float g0 = g[0], g2 = g[2];
        g[0] = fmaf(g0, p.x, g[1] * p.y);
        g[1] = fmaf(g[1], p.x, -g0 * p.y);
        g[2] = fmaf(g2, p.z, g[3] * p.w);
        g[3] = fmaf(g[3], p.z, -g2 * p.w);
      } else {
        const bool second = d4 >= TPR / 2;
        const float4* p = reinterpret_cast<const float4*>(cs + 4 * (d4 & (TPR / 2 - 1)));
        const float4 p0 = p[0], p1 = p[1];
        const float c[4] = {p0.x, p0.z, p1.x, p1.z}, s[4] = {p0.y, p0.w, p1.y, p1.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float o = __shfl_xor(g[u], TPR / 2, 64);
          g[u] = fmaf(g[u], c[u], second ? -o * s[u] : o * s[u]);
        }
      }
    }
    if (a.norm) {
      const uint2 xp = *reinterpret_cast<const uint2*>(t.x + b * t.vx.b + tok * t.vx.n + h * t.vx.h + d4 * 4);
      float x[4] = {T::lo(xp.x), T::hi(xp.x), T::lo(xp.y), T::hi(xp.y)}, ss = 0.f, dot = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) ss = fmaf(x[u], x[u], ss);
      for (int m = 1; m < TPR; m <<= 1) ss += __shfl_xor(ss, m, 64);
      const float rn = 1.f / sqrtf(ss * (1.f / D) + a.eps);
      f32x4u w = {1.f, 1.f, 1.f, 1.f};
      if (t.w) w = *reinterpret_cast<const f32x4u*>(t.w + d4 * 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] *= rn;
        if (t.part) red[threadIdx.x * 4 + u] = at < rows ? g[u] * x[u] : 0.f;
        g[u] *= w[u];
        dot = fmaf(g[u], x[u], dot);
      }
      for (int m = 1; m < TPR; m <<= 1) dot += __shfl_xor(dot, m, 64);
      dot *= 1.f / D;
#pragma unroll
      for (int u = 0; u < 4; ++u) g[u] = rn * fmaf(-x[u], dot, g[u]);
      if (t.part) {                              // the weights' gradients of the workgroup's rows
        __syncthreads();
        if (threadIdx.x < D) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) s += red[r * D + threadIdx.x];
          t.part[static_cast<int64_t>(blockIdx.x) * D + threadIdx.x] = s;
        }
      }
    }
  }
  if (at >= rows) return;
  uint16_t* po = !keys ? a.dq + b * a.vdq.b + tok * a.vdq.n + h * a.vdq.h
                       : is_v ? a.dv + b * a.vdv.b + tok * a.vdv.n + h * a.vdv.h : a.dk + b * a.vdk.b + tok * a.vdk.n + h * a.vdk.h;
  *reinterpret_cast<uint2*>(po + d4 * 4) = pack4<T>(g[0], g[1], g[2], g[3]);
}
template <int D> int64_t join_groups(const MhaArgs& a) { return (a.B * a.H * a.Nk * (D / 4) + 255) / 256; }

// ===================================================================================================================== host
constexpr int kPieces = 8;                       // workgroups that look for a head's largest rows, at most

// Splits of the keys for `groups` workgroups over Nk keys: enough to give the chip two workgroups per CU, at least 256 keys each.
int splits_for(int64_t groups, int32_t Nk) {
  if (groups <= 0 || groups >= 256) return 1;
  int64_t s = (512 + groups - 1) / groups;
  const int64_t most = (Nk + 255) / 256;
  if (s > most) s = most;
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}
// Splits of the rows that a tile of 128 keys meets in dk/dv: the count, 1 to 8, whose estimated time is least.  A workgroup takes about 2.3 us
// per 64 rows, and the chip runs 512 of them at a time (256 at head dim 128); whole rounds of them are counted, causal ones as half the work
// (long ones go first) at the lower clock of a chip that is busy throughout.  Against that stand a launch more and the splits' sums in 32 bits,
// written and read.  Measured, us with the join: 2 x 4096 tokens, causal, 16 heads on 4, d = 128: 1 split 611, 2: 423, 3: 448, 4: 444, 6: 472;
// 32 x 577 tokens, 12 heads, d = 64: 106, 186, 231, 299.
int dkv_splits(int64_t B, int64_t Nq, int64_t Nk, int64_t Hkv, int64_t G, int d, bool causal) {
  const double tiles = static_cast<double>(Nk + 127) / 128 * B * Hkv, slots = d == 64 ? 512 : 256, rows = static_cast<double>(Nq) * G;
  if (tiles >= 8 * slots) return 1;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 8 && (s == 1 || rows >= 256.0 * s); ++s) {
    const double one = rows / 64 * 2.3 / s, groups = tiles * s;       // a workgroup that meets all its rows
    double t;
    if (causal) t = one * std::max(1.0, 0.625 * groups / slots);
    else t = one * static_cast<double>(static_cast<int64_t>((groups + slots - 1) / slots));
    if (s > 1) t += 5 + s * (static_cast<double>(B) * Nk * Hkv * d * 16) / 4e6;
    if (s == 1 || t < least) { best = s; least = t; }
  }
  return best;
}
int64_t row_tiles(int64_t Nq, int64_t G) { return (Nq * G + 127) / 128; }

int check_args(const MhaArgs& a, int dtype, int32_t head_dim) {
  if (a.B < 0 || a.Nq < 0 || a.Nk < 0 || a.H < 1 || a.Hkv < 1) return APGD_ERR_SIZE;
  if (a.H % a.Hkv) return APGD_ERR_ARG;
  if (!cnx_mha_supported(head_dim)) return APGD_ERR_ARG;
  if (dtype != APGD_BF16 && dtype != APGD_F16) return APGD_ERR_DTYPE;
  if (!(a.scale >= 1e-30f) || a.scale > 1e30f) return APGD_ERR_ARG;
  const int64_t G = a.H / a.Hkv;
  // row numbers in 31 bits, threads of a launch in 32
  if (a.Nq * G > 0x7fffffffLL - 1024 || a.Nk > 0x7fffffff - 1024) return APGD_ERR_SIZE;
  const int64_t tiles = row_tiles(a.Nq, G) > (a.Nk + 127) / 128 ? row_tiles(a.Nq, G) : (a.Nk + 127) / 128;
  if (a.B > 0 && tiles > 0 && a.B > (1LL << 23) / tiles / a.H) return APGD_ERR_SIZE;
  return APGD_OK;
}
void cut(MhaArgs& a, int64_t tiles) {
  a.tiles = static_cast<int32_t>(tiles);
  a.splits = splits_for(a.B * a.Hkv * tiles, a.Nk);
  const int64_t per = ((a.Nk + a.splits - 1) / a.splits + kKT - 1) / kKT * kKT;
  a.span = static_cast<int32_t>(per < kKT ? kKT : per);
}

template <typename T, int D>
int launch_fwd(MhaArgs& a, hipStream_t s) {
  cut(a, row_tiles(a.Nq, a.G));
  hipLaunchKernelGGL((mha_fwd_kernel<T, D>), dim3(static_cast<unsigned>(a.B * a.Hkv * a.tiles * a.splits)), dim3(256), 0, s, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((mha_join_kernel<typename T::Io, D>), dim3(static_cast<unsigned>((a.B * a.H * a.Nq * (D / 4) + 255) / 256)), dim3(256), 0, s, a);
  return launch_status();
}
template <typename T, int D, bool TURN>
int launch_bwd(MhaArgs& a, hipStream_t s) {
  if (a.Nq > 0) {
    cut(a, row_tiles(a.Nq, a.G));
    hipLaunchKernelGGL((mha_dq_kernel<T, D, TURN>), dim3(static_cast<unsigned>(a.B * a.Hkv * a.tiles * a.splits)), dim3(256), 0, s, a);
    if (a.splits > 1) {
      if constexpr (TURN) hipLaunchKernelGGL((mha_turn_join_kernel<typename T::Io, D>), dim3(static_cast<unsigned>(join_groups<D>(a)), 1), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((mha_dq_join_kernel<T, D>), dim3(static_cast<unsigned>((a.B * a.H * a.Nq * (D / 4) + 255) / 256)), dim3(256), 0, s, a);
    }
  }
  if (a.Nk > 0) {
    a.tiles = (a.Nk + 127) / 128;
    a.splits = dkv_splits(a.B, a.Nq, a.Nk, a.Hkv, a.G, D, a.causal != 0);
    hipLaunchKernelGGL((mha_dkv_kernel<T, D, TURN>), dim3(static_cast<unsigned>(a.B * a.Hkv * a.tiles * a.splits)), dim3(256), 0, s, a);
    if (a.splits > 1) {
      if constexpr (TURN) hipLaunchKernelGGL((mha_turn_join_kernel<typename T::Io, D>), dim3(static_cast<unsigned>(join_groups<D>(a)), 2), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((mha_dkv_join_kernel<T, D>), dim3(static_cast<unsigned>((a.B * a.Hkv * a.Nk * (D / 4) + 255) / 256), 2), dim3(256), 0, s, a);
    }
  }
  return launch_status();
}

template <typename T>
int launch_fwd(MhaArgs& a, int32_t head_dim, hipStream_t s) { return head_dim == 64 ? launch_fwd<T, 64>(a, s) : launch_fwd<T, 128>(a, s); }
template <typename T, bool TURN>
int launch_bwd(MhaArgs& a, int32_t head_dim, hipStream_t s) { return head_dim == 64 ? launch_bwd<T, 64, TURN>(a, s) : launch_bwd<T, 128, TURN>(a, s); }

View view_of(const int64_t* s) { return View{s[0], s[1], s[2]}; }
// a staged tile's rows lie within 31 bits of bytes of its first: 64 tokens and the heads that share a key head
bool near_enough(const View& v, int64_t G) {
  return v.n >= 0 && v.h >= 0 && v.n < (1LL << 30) / 128 && v.h < (1LL << 30) / (2 * G);
}

}  // namespace

extern "C" {

int cnx_mha_supported(int32_t head_dim) { return head_dim == 64 || head_dim == 128; }

int64_t cnx_mha_ws_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t head_dim) {
  if (B <= 0 || Nq <= 0 || Nk <= 0 || H < 1 || Hkv < 1 || H % Hkv || !cnx_mha_supported(head_dim)) return 0;
  const int64_t tiles = row_tiles(Nq, H / Hkv);
  if (B > INT64_MAX / Hkv / tiles) return 0;
  const int s = splits_for(B * Hkv * tiles, Nk);
  return s > 1 ? static_cast<int64_t>(s) * B * H * Nq * (head_dim + 1) : 0;
}

int64_t cnx_mha_bwd_ws_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t head_dim, int32_t causal) {
  const int64_t dq = cnx_mha_ws_floats(B, Nq, Nk, H, Hkv, head_dim);
  if (B <= 0 || Nq <= 0 || Nk <= 0 || H < 1 || Hkv < 1 || H % Hkv || !cnx_mha_supported(head_dim)) return 0;
  const int s = dkv_splits(B, Nq, Nk, Hkv, H / Hkv, head_dim, causal != 0);
  const int64_t dkv = s > 1 ? static_cast<int64_t>(s) * 2 * B * Nk * Hkv * head_dim : 0;
  return dq > dkv ? dq : dkv;
}

int cnx_mha_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int32_t* q_lens, const int32_t* kv_lens, float* ws,
                const int64_t* strides, int dtype, int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t head_dim,
                int32_t causal, float scale, void* stream) {
  MhaArgs a = {};
  a.q = static_cast<const uint16_t*>(q); a.k = static_cast<const uint16_t*>(k); a.v = static_cast<const uint16_t*>(v);
  a.o = static_cast<uint16_t*>(out); a.lse = lse; a.part = ws; a.q_lens = q_lens; a.kv_lens = kv_lens;
  a.B = B; a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.causal = causal != 0; a.scale = scale;
  if (const int rc = check_args(a, dtype, head_dim)) return rc;
  if (B == 0 || Nq == 0) return APGD_OK;
  a.G = H / Hkv;
  if (!strides || !q || !out || (Nk > 0 && (!k || !v))) return APGD_ERR_NULL;
  if (cnx_mha_ws_floats(B, Nq, Nk, H, Hkv, head_dim) > 0 && !ws) return APGD_ERR_NULL;
  a.vq = view_of(strides); a.vk = view_of(strides + 3); a.vv = view_of(strides + 6); a.vo = view_of(strides + 9);
  if (!near_enough(a.vk, 1) || !near_enough(a.vv, 1)) return APGD_ERR_ARG;
  hipStream_t s = as_stream(stream);
  return dtype == APGD_BF16 ? launch_fwd<Bf16>(a, head_dim, s) : launch_fwd<Fp16>(a, head_dim, s);
}

int cnx_mha_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv,
                float* dvec, const int32_t* q_lens, const int32_t* kv_lens, float* ws, const int64_t* strides, int dtype, int64_t B,
                int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t head_dim, int32_t causal, float scale, void* stream) {
  MhaArgs a = {};
  a.q = static_cast<const uint16_t*>(q); a.k = static_cast<const uint16_t*>(k); a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<const uint16_t*>(out); a.dout = static_cast<const uint16_t*>(dout); a.lse = const_cast<float*>(lse);
  a.dq = static_cast<uint16_t*>(dq); a.dk = static_cast<uint16_t*>(dk); a.dv = static_cast<uint16_t*>(dv); a.dvec = dvec;
  a.part = ws; a.q_lens = q_lens; a.kv_lens = kv_lens;
  a.B = B; a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.causal = causal != 0; a.scale = scale;
  if (const int rc = check_args(a, dtype, head_dim)) return rc;
  if (B == 0 || (Nq == 0 && Nk == 0)) return APGD_OK;
  a.G = H / Hkv;
  if (!strides || (Nq > 0 && (!q || !out || !dout || !lse || !dq || !dvec)) || (Nk > 0 && (!k || !v || !dk || !dv))) return APGD_ERR_NULL;
  if (cnx_mha_bwd_ws_floats(B, Nq, Nk, H, Hkv, head_dim, causal) > 0 && !ws) return APGD_ERR_NULL;
  a.vq = view_of(strides); a.vk = view_of(strides + 3); a.vv = view_of(strides + 6); a.vo = view_of(strides + 9); a.vdo = view_of(strides + 12);
  a.vdq = view_of(strides + 15); a.vdk = view_of(strides + 18); a.vdv = view_of(strides + 21);
  if (!near_enough(a.vq, a.G) || !near_enough(a.vk, 1) || !near_enough(a.vv, 1) || !near_enough(a.vdo, a.G)) return APGD_ERR_ARG;
  hipStream_t s = as_stream(stream);
  return dtype == APGD_BF16 ? launch_bwd<Bf16, false>(a, head_dim, s) : launch_bwd<Fp16, false>(a, head_dim, s);
}

int cnx_attention_rope_fwd(const void* qkv, void* yq, void* yk, void* out, float* lse, float* ws, int dtype, const void* wq, const void* wk,
                           int w_dtype, const void* positions, int pos_dtype, int64_t pos_batch_stride, int32_t axes, const int32_t* sections,
                           const float* inv_freq, int64_t B, int32_t N, int32_t H, int32_t head_dim, float eps, int32_t norm,
                           int32_t interleaved, float scale, void* stream) {
  MhaArgs a = {};
  const bool turns = norm || positions, half = dtype == APGD_BF16 && norm;
  const int64_t D = head_dim, C = H * D;
  const uint16_t* x = static_cast<const uint16_t*>(qkv);
  a.B = B; a.Nq = a.Nk = N; a.H = a.Hkv = H; a.G = 1; a.scale = scale;
  if (const int rc = check_args(a, dtype, head_dim)) return rc;
  if (B == 0 || N == 0) return APGD_OK;
  if (!qkv || !out || (turns && (!yq || !yk))) return APGD_ERR_NULL;
  if (cnx_mha_ws_floats(B, N, N, H, H, head_dim) > 0 && !ws) return APGD_ERR_NULL;
  const View packed = {N * 3 * C, 3 * C, D}, dense = {N * C, C, D};
  if (!near_enough(packed, 1)) return APGD_ERR_ARG;
  hipStream_t s = as_stream(stream);
  if (turns) {
    const int64_t strides[12] = {packed.b, packed.n, D, packed.b, packed.n, D, dense.b, dense.n, D, dense.b, dense.n, D};
    if (const int rc = rope_forward(x, x + C, yq, yk, dtype, half, strides, wq, wk, w_dtype, positions, pos_dtype, pos_batch_stride, axes, sections,
                                    inv_freq, B, N, H, H, head_dim, eps, norm, interleaved, s))
      return rc;
  }
  a.q = turns ? static_cast<const uint16_t*>(yq) : x; a.k = turns ? static_cast<const uint16_t*>(yk) : x + C; a.v = x + 2 * C;
  a.vq = a.vk = turns ? dense : packed;
  a.vv = packed; a.vo = dense;
  a.o = static_cast<uint16_t*>(out); a.lse = lse; a.part = ws;
  if (half) return launch_fwd<Mixed>(a, head_dim, s);
  return dtype == APGD_BF16 ? launch_fwd<Bf16>(a, head_dim, s) : launch_fwd<Fp16>(a, head_dim, s);
}

// rows of partial weight gradients of a side: the workgroups of dq (of dk/dv), or of the join behind its splits
static int64_t turn_rows(int64_t B, int64_t N, int64_t H, int64_t D, bool joined) { return joined ? (B * H * N * (D / 4) + 255) / 256 : B * H * ((N + 127) / 128); }

int64_t cnx_attention_rope_bwd_ws_floats(int64_t B, int32_t N, int32_t H, int32_t head_dim, int32_t own_positions) {
  if (B <= 0 || N <= 0 || H < 1 || !cnx_mha_supported(head_dim)) return 0;
  const int64_t D = head_dim;                    // D of the rows; cosines and sines; sizes of v and dout; weight gradients; the splits' sums
  const int64_t most = std::max(turn_rows(B, N, H, D, false), turn_rows(B, N, H, D, true));
  return (B * H * N + 3) / 4 * 4 + (own_positions ? B : 1) * N * D + (2 * B * H * kPieces + 3) / 4 * 4 + 2 * most * D +
         cnx_mha_bwd_ws_floats(B, N, N, H, H, head_dim, 0);
}

int cnx_attention_rope_bwd(const void* qkv, const void* yq, const void* yk, const void* out, const void* dout, const float* lse, void* dqkv,
                           float* dwq, float* dwk, float* ws, const int64_t* dout_strides, int dtype, const float* wq, const float* wk,
                           const void* positions, int pos_dtype, int64_t pos_batch_stride, int32_t axes, const int32_t* sections,
                           const float* inv_freq, int64_t B, int32_t N, int32_t H, int32_t head_dim, float eps, int32_t norm,
                           int32_t interleaved, float scale, void* stream) {
  MhaArgs a = {};
  const int64_t D = head_dim, C = H * D;
  const bool want_w = dwq || dwk, turns = norm || positions, half = dtype == APGD_BF16 && norm;
  const uint16_t* x = static_cast<const uint16_t*>(qkv);
  a.B = B; a.Nq = a.Nk = N; a.H = a.Hkv = H; a.G = 1; a.scale = scale;
  a.eps = eps; a.norm = norm != 0; a.il = interleaved != 0;
  if (const int rc = check_args(a, dtype, head_dim)) return rc;
  if (!turns || (want_w && !norm)) return APGD_ERR_ARG;
  hipStream_t s = as_stream(stream);
  if (B == 0 || N == 0) return want_w ? rope_dw(nullptr, 0, nullptr, 0, head_dim, dwq, dwk, s) : APGD_OK;          // no row: zeros
  if (!qkv || !yq || !yk || !out || !dout || !lse || !dqkv || !ws || !dout_strides) return APGD_ERR_NULL;
  const View packed = {N * 3 * C, 3 * C, D}, dense = {N * C, C, D};
  a.q = static_cast<const uint16_t*>(yq); a.k = static_cast<const uint16_t*>(yk); a.v = x + 2 * C;
  a.out = static_cast<const uint16_t*>(out); a.dout = static_cast<const uint16_t*>(dout); a.lse = const_cast<float*>(lse);
  a.dq = static_cast<uint16_t*>(dqkv); a.dk = a.dq + C; a.dv = a.dk + C;
  a.vq = a.vk = a.vo = dense;
  a.vv = a.vdq = a.vdk = a.vdv = packed;
  a.vdo = view_of(dout_strides);
  if (!near_enough(packed, 1) || !near_enough(a.vdo, 1)) return APGD_ERR_ARG;
  const int64_t nq = turn_rows(B, N, H, D, splits_for(B * H * row_tiles(N, 1), N) > 1), nk = turn_rows(B, N, H, D, dkv_splits(B, N, N, H, 1, head_dim, false) > 1);
  a.dvec = ws;
  float* table = ws + (B * H * N + 3) / 4 * 4;
  float2* range = reinterpret_cast<float2*>(table + (pos_batch_stride ? B : 1) * N * D);
  float* pq = reinterpret_cast<float*>(range) + (2 * B * H * kPieces + 3) / 4 * 4;
  float* pk = pq + nq * D;
  a.part = pk + nk * D;
  a.tq = Turn{x, packed, wq, want_w ? pq : nullptr};
  a.tk = Turn{x + C, packed, wk, want_w ? pk : nullptr};
  if (positions) {
    a.cs = reinterpret_cast<const float2*>(table);
    a.cs_b = pos_batch_stride ? N * D / 2 : 0;
    if (const int rc = rope_table(positions, pos_dtype, pos_batch_stride, axes, sections, inv_freq, B, N, head_dim, reinterpret_cast<float2*>(table), s))
      return rc;
  }
  int rc;
  if (half) {
    a.range = range;
    a.pieces = static_cast<int32_t>(B * H >= 512 ? 1 : std::min<int64_t>(kPieces, (N + 127) / 128));
    const dim3 grid(static_cast<unsigned>(B * H * a.pieces));
    if (head_dim == 64) hipLaunchKernelGGL((mha_range_kernel<Bf16, 64>), grid, dim3(256), 0, s, a, range);
    else hipLaunchKernelGGL((mha_range_kernel<Bf16, 128>), grid, dim3(256), 0, s, a, range);
    rc = launch_bwd<Mixed, true>(a, head_dim, s);
  } else {
    rc = dtype == APGD_BF16 ? launch_bwd<Bf16, true>(a, head_dim, s) : launch_bwd<Fp16, true>(a, head_dim, s);
  }
  return rc || !want_w ? rc : rope_dw(pq, static_cast<int>(nq), pk, static_cast<int>(nk), head_dim, dwq, dwk, s);
}

}  // extern "C"
