// A paged KV cache in 8 or 4 bits: written as keys are rotated, read back, and read by the attention of single tokens and of prompts.
//
// Format.  A head's row of DH dims in groups of 32.  Each group has one power of two as its scale (a byte: exponent + 127; 255: the
// group held a NaN or an infinity and reads back as NaN) and elements of e2m1 (0 .5 1 1.5 2 3 4 6) or e4m3.  The exponent is the
// smallest with absmax <= 7 (464) 2^e, halfway between the largest element and where the next would be, so the largest value of a
// group is off by half a step of its binade like all others (a scale by the binade alone clips values of 6 to 8 to 6).  Its range, -100
// to 125 (119), keeps every element a normal bf16 number: what is read back is exact in bf16.  4.25 and 8.25 bits a value.
//
// Layout.  A page of one KV head is one run of bytes, 64 keys of elements, then their scales; each wide load of the attention is
// one operand of a matrix instruction as it stands:
//   keys     rows of DH elements (4 bits: even dim low): the A operand of v_mfma_scale_f32_16x16x128, which takes these formats and
//            their scales as they are.  Scales by group, the four score tiles of a page side by side (mx_key_scale)
//   values   units of 16 bytes with a lane's share of some keys: dims 2r and 2r + 1 of every group (mx_value_off); scales
//            [64 keys][groups].  A token's write fills whole bytes: no two tokens share one
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <algorithm>
#include "handover.h"

namespace xot {
namespace {

constexpr int PAGE = 64;
constexpr float NEG_BIG = -3.402823466e38f;  // a maximum of no scores: no finite score is below it
constexpr float FAR = 16777216.f;            // (Rows::weights)
constexpr float LOG2E = 1.4426950408889634f;

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int DH, bool FP8>
struct Mx {
  static constexpr int J = DH / 32;                   // groups of a row
  static constexpr int ROW = FP8 ? DH : DH / 2;       // bytes of a key's elements
  static constexpr int ELEMS = PAGE * ROW;            // elements of a page: its scales start here
  static constexpr int BYTES = ELEMS + PAGE * J;      // a page of one head
  static constexpr int NB = FP8 ? 2 * J : J;          // bytes of a key in a value unit
  static constexpr int KC = 16 / NB;                  // keys of a value unit
  static constexpr int EMAX = FP8 ? 8 : 2;            // exponent of the largest element
  static constexpr uint32_t TOP = FP8 ? 0x680000u : 0x600000u;  // mantissa of 464 / 256 and of 7 / 4
  static constexpr int HIGH = FP8 ? 119 : 125;
};
constexpr int LOW = -100;

// byte of key i's scale among a group's 64: score tile t, row c of the attention (below) is key 32 (t >> 1) + 4 (t & 1) + 8 (c >> 2) + (c & 3)
__device__ __forceinline__ int mx_key_scale(int i) { return 4 * (4 * ((i >> 3) & 3) + (i & 3)) + 2 * (i >> 5) + ((i >> 2) & 1); }
template <int DH, bool FP8>
__device__ __forceinline__ int mx_value_off(int key, int r) {
  using M = Mx<DH, FP8>;
  return ((key / M::KC) * 16 + r) * 16 + (key % M::KC) * M::NB;
}

// absmax bits of a group -> exponent of its scale
template <int DH, bool FP8>
__device__ __forceinline__ int mx_exponent(uint32_t a) {
  using M = Mx<DH, FP8>;
  const int e = (int)(a >> 23) - 127 - M::EMAX + ((a & 0x7fffffu) > M::TOP ? 1 : 0);
  return min(max(e, LOW), M::HIGH);
}
__device__ __forceinline__ bool mx_bad(uint32_t a) { return a >= 0x7f800000u; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// two values -> a byte of e2m1 (a low); the instruction divides by the scale, rounds to the nearest, ties to even, and saturates
__device__ __forceinline__ uint32_t to_fp4(float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, scale, 0) & 0xffu;
}
// two values (already divided) -> two bytes of e4m3; past 464 the instruction gives NaN, hence the clamp
__device__ __forceinline__ uint32_t to_fp8(float a, float b) {
  a = fminf(fmaxf(a, -448.f), 448.f);
  b = fminf(fmaxf(b, -448.f), 448.f);
  return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
// byte b of x, two e2m1 -> two bf16, times the power of two in the scale's exponent field (its other bits do not count; a field of 255
// gives NaN).  Exact.
__device__ __forceinline__ uint32_t from_fp4(uint32_t x, float scale, int b) {
  switch (b) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 3));
  }
}
// half h of x, two e4m3 -> two bf16
__device__ __forceinline__ uint32_t from_fp8(uint32_t x, float scale, int h) {
  return h ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true))
           : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false));
}
// byte j of x in a float's exponent field (the other bits are whatever stands beside it: from_fp4 and from_fp8 do not look)
__device__ __forceinline__ float scale_of(uint32_t x, int j) { return __uint_as_float(j == 3 ? x >> 1 : x << (23 - 8 * j)); }
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// largest value of N (8 or 16) neighbouring lanes, in all of them
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if (N == 16) v = max(v, row_turn<8>(v));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // the eight lanes mirrored
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));   // lane ^ 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));  // lane ^ 1
}

// ============================================================================ write
// Sixteen lanes a row of one head (q, k or v) of a token; a wave takes a head's rows of four neighbouring tokens, whose elements lie side
// by side in a page (keys 256 bytes, value units whole).  k is quantised from its rotation in fp32, v from its bf16; a group's largest
// value is found among the lanes that hold it (on the bits: a NaN counts as larger than everything).  The rotation's products and sums are
// rounded one by one, so that a value on the border between two elements falls the same way wherever it is computed.
// Bound by its launch at a few tokens (2.7 us up to 64), by memory at many: 4.8 to 5.3 TB/s at 8192 (a large copy: 4.9).
// N values under one scale -> N bytes of e4m3 or N / 2 of e2m1
template <bool FP8, int N>
__device__ __forceinline__ uint32_t mx_elements(const float (&x)[N], int e, bool bad) {
  uint32_t y = 0;
  const float s = pow2(FP8 ? -e : e);
#pragma unroll
  for (int i = 0; i < N; i += 2) y |= FP8 ? to_fp8(x[i] * s, x[i + 1] * s) << (8 * i) : to_fp4(x[i], x[i + 1], s) << (4 * i);
  return bad ? 0u : y;
}
template <int BYTES>
__device__ __forceinline__ void st_bytes(uint8_t* p, uint64_t v) {
  if constexpr (BYTES == 8) *reinterpret_cast<uint64_t*>(p) = v;
  else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = (uint32_t)v;
  else if constexpr (BYTES == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)v;
  else *p = (uint8_t)v;
}

template <int DH, bool FP8, int HB>
__global__ __launch_bounds__(256) void rope_kv_write_mx_kernel(const uint16_t* __restrict__ qkv, const int32_t* __restrict__ pos,
                                                               const float* __restrict__ cos_sin, const int64_t* __restrict__ slots,
                                                               uint16_t* __restrict__ q_out, uint8_t* __restrict__ kc,
                                                               uint8_t* __restrict__ vc, int T, int H, int Hkv, int max_pos, long nslots) {
#pragma clang fp contract(off)
  using M = Mx<DH, FP8>;
  constexpr int J = M::J, E = DH / 32, HALF = DH / 2, KB = FP8 ? E : E / 2;  // E: dims a lane takes of each half; KB: their bytes
  const int N = H + 2 * Hkv, groups = (N + HB - 1) / HB, w = blockIdx.x * 4 + (threadIdx.x >> 6), quad = w / groups;
  const int h0 = (w - quad * groups) * HB, t = 4 * quad + ((threadIdx.x >> 4) & 3), r = threadIdx.x & 15;
  if (t >= T) return;  // (sixteen lanes together)
  // a lane's share of a row is J dwords: E dims of each half to rotate, or two dims of each group of a value
  uint32_t raw[HB][J];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const int h = min(h0 + i, N - 1);
    const uint16_t* src = qkv + ((size_t)t * N + h) * DH;
    if (h < H + Hkv) {
      if constexpr (J == 4) {
        const uint64_t a = *reinterpret_cast<const uint64_t*>(src + E * r), b = *reinterpret_cast<const uint64_t*>(src + HALF + E * r);
        raw[i][0] = (uint32_t)a;
        raw[i][1] = (uint32_t)(a >> 32);
        raw[i][2] = (uint32_t)b;
        raw[i][3] = (uint32_t)(b >> 32);
      } else {
        raw[i][0] = *reinterpret_cast<const uint32_t*>(src + E * r);
        raw[i][1] = *reinterpret_cast<const uint32_t*>(src + HALF + E * r);
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) raw[i][j] = *reinterpret_cast<const uint32_t*>(src + 32 * j + 2 * r);
    }
  }
  const int64_t slot = slots[t];
  const bool kept = slot >= 0 && slot < nslots;
  const int off = (int)(slot & (PAGE - 1));
  float c[E], s[E];
  if (h0 < H + Hkv) {
    int p = pos[t];
    p = p < 0 ? 0 : (p >= max_pos ? max_pos - 1 : p);
    const float* cs = cos_sin + (size_t)p * DH + E * r;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      c[i] = cs[i];
      s[i] = cs[HALF + i];
    }
  }
#pragma unroll
  for (int n = 0; n < HB; ++n) {
    const int h = h0 + n;
    if (h >= N || (h >= H && !kept)) break;
    auto at = [&](int i) { return bf2f((uint16_t)(raw[n][i >> 1] >> (16 * (i & 1)))); };
    if (h < H + Hkv) {
      float lo[E], hi[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float x = at(i), y = at(E + i);
        lo[i] = x * c[i] - y * s[i];
        hi[i] = y * c[i] + x * s[i];
      }
      if (h < H) {
        uint8_t* dst = reinterpret_cast<uint8_t*>(q_out + ((size_t)t * H + h) * DH + E * r);
        uint64_t a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          a |= (uint64_t)f2bf(lo[i]) << (16 * i);
          b |= (uint64_t)f2bf(hi[i]) << (16 * i);
        }
        st_bytes<2 * E>(dst, a);
        st_bytes<2 * E>(dst + 2 * HALF, b);
        continue;
      }
      uint8_t* page = kc + ((size_t)(slot / PAGE) * Hkv + (h - H)) * M::BYTES;
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        a = max(a, __float_as_uint(lo[i]) & 0x7fffffffu);
        b = max(b, __float_as_uint(hi[i]) & 0x7fffffffu);
      }
      a = lanes_max<32 / E>(a);
      b = lanes_max<32 / E>(b);
      const int ea = mx_exponent<DH, FP8>(a), eb = mx_exponent<DH, FP8>(b);
      const bool na = mx_bad(a), nb = mx_bad(b);
      uint8_t* dst = page + off * M::ROW + KB * r;
      st_bytes<KB>(dst, mx_elements<FP8>(lo, ea, na));
      st_bytes<KB>(dst + M::ROW / 2, mx_elements<FP8>(hi, eb, nb));
      if (r % (32 / E) == 0) {
        const int j = E * r / 32;
        uint8_t* sc = page + M::ELEMS + mx_key_scale(off);
        sc[64 * j] = (uint8_t)(na ? 255 : ea + 127);
        sc[64 * (j + J / 2)] = (uint8_t)(nb ? 255 : eb + 127);
      }
      continue;
    }
    uint8_t* page = vc + ((size_t)(slot / PAGE) * Hkv + (h - H - Hkv)) * M::BYTES;
    uint64_t y = 0;
    uint32_t sc = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float x[2] = {at(2 * j), at(2 * j + 1)};
      const uint32_t a = lanes_max<16>(max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu));
      const int e = mx_exponent<DH, FP8>(a);
      y |= (uint64_t)mx_elements<FP8>(x, e, mx_bad(a)) << (FP8 ? 16 * j : 8 * j);
      sc |= (uint32_t)(mx_bad(a) ? 255 : e + 127) << (8 * j);
    }
    st_bytes<M::NB>(page + mx_value_off<DH, FP8>(off, r), y);
    if (r == 0) st_bytes<J>(page + M::ELEMS + off * J, sc);
  }
}

// ============================================================================ read
// One workgroup a page of one head: bf16 keys [64][DH] and values chunk-major (v_page_off), what the prompt attention reads.  Keys past
// the context are zeros, in pages that hold some and (skip unset) in those that lie wholly past it.  own: the table of what is written,
// entry i page i.  Bound by memory (mostly its writes).
template <int DH, bool FP8>
__global__ __launch_bounds__(256) void kv_read_mx_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                         const int32_t* __restrict__ tables, int width, const int32_t* __restrict__ ctx_lens,
                                                         uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, int Hkv,
                                                         int num_pages, bool skip, int32_t* __restrict__ own) {
  using M = Mx<DH, FP8>;
  const int kvh = (int)(blockIdx.x % Hkv), entry = (int)(blockIdx.x / Hkv), b = entry / width, w = entry - b * width;
  if (own != nullptr && kvh == 0 && threadIdx.x == 0) own[entry] = entry;
  const int live = min(max(ctx_lens[b] - w * PAGE, 0), PAGE);  // (a context past the table's width: whole pages)
  if (live == 0 && skip) return;
  const long page = min(max(tables[entry], 0), num_pages - 1);
  const uint8_t* kp = kc + ((size_t)page * Hkv + kvh) * M::BYTES;
  const uint8_t* vp = vc + ((size_t)page * Hkv + kvh) * M::BYTES;
  uint16_t* ko = k_out + ((size_t)entry * Hkv + kvh) * PAGE * DH;
  uint16_t* vo = v_out + ((size_t)entry * Hkv + kvh) * PAGE * DH;
  constexpr int CPR = DH / 8, KI = PAGE * CPR / 256;
  // eight dims of a key a thread and turn, all loads first
  uint32_t kx[KI][2], ks[KI];
#pragma unroll
  for (int n = 0; n < KI; ++n) {
    const int i = threadIdx.x + 256 * n, key = i / CPR, d = (i % CPR) * 8;
    if constexpr (FP8) {
      const uint64_t u = *reinterpret_cast<const uint64_t*>(kp + key * M::ROW + d);
      kx[n][0] = (uint32_t)u;
      kx[n][1] = (uint32_t)(u >> 32);
    } else {
      kx[n][0] = kx[n][1] = *reinterpret_cast<const uint32_t*>(kp + key * M::ROW + d / 2);
    }
    ks[n] = kp[M::ELEMS + 64 * (d >> 5) + mx_key_scale(key)];
  }
  // eight keys of the dims 2 r, 2 r + 1 of a group: two threads share a lane's units, and J / 2 groups each
  constexpr int VU = 8 / M::KC, JT = M::J / 2;
  const int r = threadIdx.x & 15, half = (threadIdx.x >> 4) & 1, k0 = 8 * (threadIdx.x >> 5);
  u32x4 v[VU];
  uint32_t vs[2 * M::J];
#pragma unroll
  for (int u = 0; u < VU; ++u) v[u] = *reinterpret_cast<const u32x4*>(vp + ((k0 / M::KC + u) * 16 + r) * 16);
#pragma unroll
  for (int u = 0; u < 2 * M::J; ++u) vs[u] = *reinterpret_cast<const uint32_t*>(vp + M::ELEMS + k0 * M::J + 4 * u);
#pragma unroll
  for (int n = 0; n < KI; ++n) {
    const int i = threadIdx.x + 256 * n, key = i / CPR, d = (i % CPR) * 8;
    const float s = scale_of(ks[n], 0);
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = FP8 ? from_fp8(kx[n][e >> 1], s, e & 1) : from_fp4(kx[n][0], s, e);
      y[e] = key < live ? y[e] : 0u;
    }
    *reinterpret_cast<u32x4*>(ko + key * DH + d) = y;
  }
#pragma unroll
  for (int jj = 0; jj < JT; ++jj) {
    u32x4 lo, hi;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      uint32_t y[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int key = 2 * n + m;
        // (both halves' groups are compile-time places: a thread converts one of the two)
        auto conv = [&](int j) {
          const int at = key * M::NB + (FP8 ? 2 * j : j), sa = key * M::J + j;
          const uint32_t x = v[at >> 4][(at >> 2) & 3];
          const float s = scale_of(vs[sa >> 2], sa & 3);
          return FP8 ? from_fp8(x, s, (at >> 1) & 1) : from_fp4(x, s, at & 3);
        };
        y[m] = half ? conv(JT + jj) : conv(jj);
        y[m] = k0 + key < live ? y[m] : 0u;
      }
      lo[n] = low_halves(y[0], y[1]);
      hi[n] = high_halves(y[0], y[1]);
    }
    uint16_t* o = vo + v_page_off(k0, 32 * (half ? JT + jj : jj) + 2 * r, DH);
    *reinterpret_cast<u32x4*>(o) = lo;
    *reinterpret_cast<u32x4*>(o + 8) = hi;
  }
}

// ============================================================================ attention of single tokens
// Scores S^T = K . Q^T: sixteen keys (A) by the query heads of a KV head (B columns) on v_mfma_scale_f32_16x16x128_f8f6f4, which reads the
// cache's elements and scales as they stand.  A query is the sum of two e4m3 numbers, one 1/16 of the other's scale: bf16 has 8
// significant bits, each of the two takes 4, so the split is exact down to 2^-21 of the query's largest value (below e4m3's normal
// range).  Heads of 128 take one instruction for each, heads of 64 both in the two halves of one.
// Operand maps (lane (g, c) = (l >> 4, l & 15)): e2m1 A: dims 32 g .. of row c, 16 bytes; e4m3: 16 g .. in the first 16 bytes, 64 + 16 g
// .. in the second; a scale byte counts for dims 32 g .. of its lane's row.  Score tile t's row c = 4 q + r is key 32 (t >> 1) + 8 q + 4 (t
// & 1) + r, so that a lane's scores of tiles 2 kk and 2 kk + 1 are the eight keys 32 kk + 8 g .. that it holds in the B operand of
// O^T = V^T . P^T: probabilities stay in their registers.
// Values: two e2m1 / e4m3 of a key become two bf16 (exact, scaled on the way), and two keys' pairs change halves: tile (j, e) of O^T
// has dims 32 j + 2 row + e.  P is rounded to bf16 (2^-8 of a weight at most): the values' own type, the widest that the unit multiplies at
// this rate, and what attention over a bf16 cache does; sums, maxima and the output before its rounding are fp32.
template <int DH, bool FP8>
struct PageRegs {
  using M = Mx<DH, FP8>;
  static constexpr int KV = FP8 && DH == 128 ? 2 : 1;  // 16-byte loads of a key row's share
  static constexpr int VU = 8 / M::KC;                 // value units of eight keys
  static constexpr int VS = M::J / 2;                  // 16-byte loads of eight keys' scales
  u32x4 k[4][KV], v[2][VU], vs[2][VS];
  uint32_t ks;
};

template <int DH, bool FP8>
__device__ __forceinline__ f32x4 score_mfma(const u32x4 (&k)[PageRegs<DH, FP8>::KV], const i32x8& q, f32x4 acc, uint32_t ks, int qs, int t) {
  constexpr int F = FP8 ? 0 : 4;
  i32x8 a;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = (int)k[0][i];
    a[4 + i] = !FP8 ? 0 : (int)k[PageRegs<DH, FP8>::KV - 1][i];
  }
  switch (t) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc, F, 0, 0, (int)ks, 0, qs);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc, F, 0, 1, (int)ks, 0, qs);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc, F, 0, 2, (int)ks, 0, qs);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc, F, 0, 3, (int)ks, 0, qs);
  }
}

struct AttnArgs {
  const uint16_t* q;
  const uint8_t *kc, *vc;
  const int32_t *tables, *ctx_lens, *cu_q;
  uint16_t* out;
  float *ws_o, *ws_ml;
  int* tickets;
  int T, B, width, H, Hkv, ppp, nparts, num_pages, units, per, order;  // units: of a KV head; per: unit_at
  float scale_log2;
};

// Four results O / L in bf16 (inv = 1 / L: the product is within 2^-23 of the quotient, far below bf16's step).
__device__ __forceinline__ void st_results(uint16_t* p, const f32x4& O, float inv) {
  s16x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = (short)f2bf(O[r] * inv);
  *reinterpret_cast<s16x4*>(p) = y;
}

// The sequence at place p of a decode step of at most 64.  order 1: the longest first, so that none starts late.  2 (units that all start at
// once, up to three a CU): the longer half, longest first, then the shorter, shortest first: the units that a CU gets, one of each round, are
// then of about the same length together.  Figures beside ops.kernels.mx_decode_order; finding the place costs a unit about 1 us.
__device__ __forceinline__ int sequence_at(const AttnArgs& A, int p) {
  const int lane = threadIdx.x & 63, B = A.T, half = (B + 1) >> 1;
  const int pages = lane < B ? (min(max(A.ctx_lens[lane], 0), A.width * PAGE) + PAGE - 1) / PAGE : 0;
  if (__ballot(lane < B && pages != __builtin_amdgcn_readfirstlane(pages)) == 0) return p;  // (all as long: as they are given)
  const uint32_t key = lane < B ? (uint32_t)pages * 64u + 63u - lane : 0;  // no two alike
  int rank = 0;
  for (int j0 = 0; j0 < B; j0 += 8)
#pragma unroll
    for (int j = 0; j < 8; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, j0 + j) > key ? 1 : 0;
  const int want = A.order == 1 || p < half ? p : B - 1 - (p - half);
  return __builtin_ctzll(__ballot(lane < B && rank == want));
}

// Unit u of a launch over new tokens: the sequence and the first of its R rows.  Sequence b's units start at floor(cu_q[b] G / R) + b, so that
// T G / R + B units hold them all, whatever the lengths, with at most two to spare a sequence: a step of one prompt of 2000 tokens and 511
// single ones has 6600 units of work where a grid of the longest's for each has a million.  64 sequences a look.  (cu_q that falls somewhere
// finds some sequence of the launch, or none.)  per: the longest's units for each sequence, where that is no more (prompts about alike: 4 of 64
// tokens behind 1000 15 us, 20 with a spare unit each, beside which others' CUs get two).
template <int R>
__device__ __forceinline__ bool unit_at(const AttnArgs& A, int u, int& b, int& row0, int& q0, int& q1) {
  const int lane = threadIdx.x & 63, G = A.H / A.Hkv;
  auto start = [&](int q, int i) { return (int)((uint32_t)(q * G) / R) + i; };
  if (A.per > 0) {
    b = u / A.per;
    row0 = (u - b * A.per) * R;
    q0 = min(max(A.cu_q[b], 0), A.T);
    q1 = min(max(A.cu_q[b + 1], 0), A.T);
    return true;
  }
  int k = 0, mine = 0, next = 0;
  b = 0;
  for (int n = A.B, step = 64; step > 1;) {
    step = (n + 63) >> 6;
    const int at = lane * step, i = b + min(at, n - 1);
    mine = min(max(A.cu_q[i], 0), A.T);
    next = min(max(A.cu_q[i + 1], 0), A.T);
    k = __builtin_popcountll(__ballot(at < n && start(mine, i) <= u)) - 1;
    if (k < 0) return false;
    b += k * step;
    n = min(step, n - k * step);
  }
  q0 = __builtin_amdgcn_readlane(mine, k);
  q1 = __builtin_amdgcn_readlane(next, k);
  row0 = (u - start(q0, b)) * R;
  return row0 >= 0;
}

// What a lane's eight keys hold past the context may be anything, NaN too: it becomes zeros (their probabilities are 0, but 0 NaN is
// NaN).  left: how many of the eight count
template <int DH, bool FP8, class V, class S>
__device__ __forceinline__ void cut_values(V& v, S& vs, int left) {  // u32x4 [VU], [VS]
  using M = Mx<DH, FP8>;
#pragma unroll
  for (int key = 0; key < 8; ++key) {
    const bool dead = key >= left;
    const uint32_t other = key & 1 ? 0xffffu : 0xffff0000u;
    if constexpr (M::NB >= 4) {
#pragma unroll
      for (int i = key * (M::NB / 4); i < (key + 1) * (M::NB / 4); ++i) v[i >> 2][i & 3] = dead ? 0u : v[i >> 2][i & 3];
    } else {
      v[key >> 3][(key >> 1) & 3] = dead ? v[key >> 3][(key >> 1) & 3] & other : v[key >> 3][(key >> 1) & 3];
    }
    if constexpr (M::J == 4) vs[key >> 2][key & 3] = dead ? 0x7f7f7f7fu : vs[key >> 2][key & 3];
    else vs[0][key >> 1] = dead ? (vs[0][key >> 1] & other) | (0x7f7f7f7fu & ~other) : vs[0][key >> 1];
  }
}

// group j of a lane's eight keys: the A operands of O^T's tiles (j, even dims) and (j, odd)
template <int DH, bool FP8, class V, class S>
__device__ __forceinline__ void value_pairs(const V& v, const S& vs, int j, u32x4& ae, u32x4& ao) {  // u32x4 [VU], [VS]
  using M = Mx<DH, FP8>;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    uint32_t y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = 2 * n + i, at = key * M::NB + (FP8 ? 2 * j : j), sa = key * M::J + j;  // bytes among the eight keys'
      const uint32_t w = v[at >> 4][(at >> 2) & 3];
      const float s = scale_of(vs[sa >> 4][(sa >> 2) & 3], sa & 3);
      y[i] = FP8 ? from_fp8(w, s, (at >> 1) & 1) : from_fp4(w, s, at & 3);
    }
    ae[n] = low_halves(y[0], y[1]);
    ao[n] = high_halves(y[0], y[1]);
  }
}

// A wave's 16 NB rows (queries) and what it has of them.  ONES: the weights are summed as products with ones, which costs registers and
// saves vector operations.
template <int DH, bool FP8, int NB, bool ONES>
struct Rows {
  using M = Mx<DH, FP8>;
  using R = PageRegs<DH, FP8>;
  static constexpr int J = M::J;
  // A row's weights are 2^(score - m).  m follows the largest score once that is past it by more than this.  Prompts: weights stay below 2^8, sums
  // far from overflow, and what the rows have is brought to a new m a few times, not at every second page (4096 tokens 158 -> 150 us; the
  // heaviest weight is then rounded to bf16 like the others, where it had been 1: errors 0.0017 -> 0.0020 of the output).  Single tokens gain
  // nothing by it and follow at once.
  static constexpr float LAZY = ONES ? 8.f : 0.f;
  i32x8 qhi[NB], qlo[NB];
  int shi[NB], slo[NB];
  float m[NB], l[NB];
  f32x4 o[NB][J][2], lacc[NB];

  // row c of block nb: the query at qp (dims 16 g ..) in two parts; !ok: zeros
  __device__ __forceinline__ void query(int nb, const uint16_t* qp, bool ok, int g) {
    m[nb] = NEG_BIG;
    l[nb] = 0.f;
    lacc[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < J; ++j) o[nb][j][0] = o[nb][j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    qhi[nb] = qlo[nb] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
    s16x8 x[DH / 32];
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) {
      x[i] = ld16(qp + (i >> 1) * 64 + (i & 1) * 8);
#pragma unroll
      for (int n = 0; n < 8; ++n) a = max(a, ((uint32_t)(uint16_t)x[i][n] << 16) & 0x7fffffffu);
    }
    auto most = [](uint32_t u, uint32_t v) { return max(u, v); };
    a = lane_xor<16>(lane_xor<32>(a, most), most);
    const int e = min(max((int)(a >> 23) - 127 - 7, -120), 120);
    const float inv = pow2(-e);
#pragma unroll
    for (int i = 0; i < DH / 32; ++i)
#pragma unroll
      for (int n = 0; n < 8; n += 4) {
        int hi = 0, lo = 0;
        const float f0 = bf2f(x[i][n]) * inv, f1 = bf2f(x[i][n + 1]) * inv, f2 = bf2f(x[i][n + 2]) * inv, f3 = bf2f(x[i][n + 3]) * inv;
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(f0, f1, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(f2, f3, hi, true);
        const f32x2_t h0 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), h1 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32((f0 - h0[0]) * 16.f, (f1 - h0[1]) * 16.f, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32((f2 - h1[0]) * 16.f, (f3 - h1[1]) * 16.f, lo, true);
        const int at = 2 * i + n / 4;  // dword of the operand
        if (!ok) hi = lo = 0;
        qhi[nb][at] = hi;
        if (DH == 128) qlo[nb][at] = lo;
        else qhi[nb][4 + at] = lo;
      }
    const bool bad = mx_bad(a) && ok;
    shi[nb] = bad ? 255 : e + 127;
    slo[nb] = bad ? 255 : e + 127 - 4;
    if (DH == 64 && g >= 2) shi[nb] = slo[nb];
  }

  // kt(t, k): this lane's share of score tile t
  template <class K>
  __device__ __forceinline__ void scores(K kt, uint32_t ks, f32x4 (&st)[NB][4]) const {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      u32x4 k[R::KV];
      kt(t, k);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        st[nb][t] = score_mfma<DH, FP8>(k, qhi[nb], f32x4{0.f, 0.f, 0.f, 0.f}, ks, shi[nb], t);
        if (DH == 128) st[nb][t] = score_mfma<DH, FP8>(k, qlo[nb], st[nb][t], ks, slo[nb], t);
      }
    }
  }
  // scores of keys that block nb's row does not see; left: how many of the keys from the lane's first on it does
  __device__ __forceinline__ static void mask(f32x4 (&st)[4], int left) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[t][r] = 32 * (t >> 1) + 4 * (t & 1) + r < left ? st[t][r] : -INFINITY;
  }
  // The page's weights in bf16, B operands of the products with its values; what the rows have so far is brought to the new maxima.
  // Weights are 2^fma(score, scale, -m): the product unrounded, m the largest one rounded.  Past 2^24 the two differ by more than 1, soon by
  // hundreds, and all weights of a row overflow or vanish: the scores of far rows are scaled, with m's rounding, before m is taken from them.
  // Single tokens branch (no slower); prompts, from whose registers a branch takes too many (one prompt of 4096 in mxfp8 of 64 dims 94 / 119 us),
  // leave far rows to a second pass over the unit with FARS (95 us; others within 1.5 %).
  template <bool FARS>
  __device__ __forceinline__ void weights(f32x4 (&st)[NB][4], float scale_log2, s16x8 (&pf)[NB][2]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, st[nb][t][r]);
      mx = xor_max<16>(mx);
      mx = xor_max<32>(mx) * scale_log2;  // (the scale is positive)
      if (__ballot(mx > m[nb] + LAZY)) {
        const float mn = fmaxf(m[nb], mx), alpha = __builtin_amdgcn_exp2f(m[nb] - mn);
        m[nb] = mn;
        if constexpr (ONES) lacc[nb] *= alpha;
        else l[nb] *= alpha;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          o[nb][j][0] *= alpha;
          o[nb][j][1] *= alpha;
        }
      }
      float scale = scale_log2;
      if constexpr (FARS) {
#pragma clang fp contract(off)
#pragma unroll
        for (int t = 0; t < 4; ++t) st[nb][t] *= scale_log2;
        scale = 1.f;
      } else if (!ONES && __ballot(fabsf(m[nb]) > FAR)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) st[nb][t] *= scale_log2;
        scale = 1.f;
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 pw;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(st[nb][2 * kk + (e >> 2)][e & 3], scale, -m[nb]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(st[nb][2 * kk + (e >> 2)][(e & 3) + 1], scale, -m[nb]));
          if constexpr (!ONES) l[nb] += p0 + p1;
          pw[e >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p0, p1}), bf16x2_t));
        }
        pf[nb][kk] = __builtin_bit_cast(s16x8, pw);
        constexpr short ONE = 0x3f80;
        if constexpr (ONES) lacc[nb] = mfma16(s16x8{ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE}, pf[nb][kk], lacc[nb]);
      }
    }
  }
  // The page's weights and their products with its values; vv(kk, v, vs): eight keys' units and scales.
  template <bool FARS, class V>
  __device__ __forceinline__ void weigh(V vv, f32x4 (&st)[NB][4], float scale_log2) {
    s16x8 pf[NB][2];
    weights<FARS>(st, scale_log2, pf);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 v[R::VU], vs[R::VS];
      vv(kk, v, vs);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        u32x4 ae, ao;
        value_pairs<DH, FP8>(v, vs, j, ae, ao);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          o[nb][j][0] = mfma16(__builtin_bit_cast(s16x8, ae), pf[nb][kk], o[nb][j][0]);
          o[nb][j][1] = mfma16(__builtin_bit_cast(s16x8, ao), pf[nb][kk], o[nb][j][1]);
        }
      }
    }
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (ONES) {
        l[nb] = lacc[nb][0];  // (every row of the product is the column's sum)
      } else {
        l[nb] = xor_sum<16>(l[nb]);
        l[nb] = xor_sum<32>(l[nb]);
      }
    }
  }
  // Whether some row of the wave is far, or was and overflowed before a larger score came (behind finish; sums of others stay below 2^9 a key)
  __device__ __forceinline__ bool far() const {
    bool bad = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) bad |= m[nb] > NEG_BIG && (fabsf(m[nb]) > FAR || !(l[nb] < 0x1p40f));
    return __ballot(bad) != 0;
  }
  // four neighbouring dims of block nb's row c: 32 j + 8 g + 4 half ..
  __device__ __forceinline__ f32x4 dims(int nb, int j, int half) const {
    const f32x4 &e = o[nb][j][0], &d = o[nb][j][1];
    return half ? f32x4{e[2], d[2], e[3], d[3]} : f32x4{e[0], d[0], e[1], d[1]};
  }
};

// One unit: 16 NB rows (tokens of a sequence x query heads of a KV head; single tokens: its G heads) against a part of the pages.
// NW waves share the part, wave w takes pages w, w + NW, ..., and meet in LDS.  REFILL: a page's registers are loaded anew as soon as
// they are consumed, keys behind the scores, values behind their products, so that a page's loads fly under the other half's math; without
// it a page is loaded and then computed, in fewer registers (mxfp4 126, four waves a SIMD; 155, three).  Many pairs have waves enough to
// hide the loads (512 sequences of 525 tokens 56 / 60 us with REFILL, 128 of 30 to 8000 103 / 110), few have not (64 of 30 to 2000 21.0 /
// 19.9, 8 on 32 KV heads 9.3 / 8.4); mxfp8 pages of 128 dims have no registers left for it.  Two sets of a page's registers, and three,
// leave two waves a SIMD: 59, 59, 107, 107 us of the first two.
// A context of several parts (at most nparts, of ppp pages and more) is merged by the workgroup that arrives last (a ticket a (rows, KV
// head), zero between launches), in the parts' order whoever it is.
// Bound by memory where the pairs of single tokens fill the chip: 512 sequences of 1500 tokens, 32 heads of 128 on 8, mxfp8 1.66 GB in 257
// us (6.5 TB/s), mxfp4 856 MB in 138 us (6.2 TB/s); of 525 tokens, 64 heads, mxfp4 54 us (5.7 TB/s of what counts).  A page of mxfp4 is
// about 330 vector operations a wave, 190 of them making bf16 values; K needs none.  Uncut contexts and no loads ahead: 8 sequences of
// 32000 tokens 239 us, now 48.
// Prompts (PROMPT) start with their last rows, which see the most keys; here where they are few (attn_prompt_mx_kernel): 4 sequences of 64 new
// tokens behind 1000, 32 heads of 128 on 8, mxfp4, 15 us.
// Bounds: four waves a SIMD where the registers suffice (single tokens of mxfp4, 128 dims: 54 us at 512 of 525 keys, 61 in three).
template <int DH, bool FP8, int NW, int NB, bool PROMPT, bool REFILL>
__global__ __launch_bounds__(64 * NW, NB > 1 && DH == 128 ? 2 : FP8 || REFILL || PROMPT ? 3 : 4) void attn_mx_kernel(const AttnArgs A) {
  static_assert(PROMPT || NB == 1, "a single token's heads are one column block");
  using M = Mx<DH, FP8>;
  using R = PageRegs<DH, FP8>;
  constexpr int J = M::J, LD = DH + 4;
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int kvh = blockIdx.x % A.Hkv, bp = blockIdx.x / A.Hkv, part = bp % A.nparts, bu = bp / A.nparts;
  int b = bu, row0 = 0, q0 = bu, q1 = bu + 1;
  if (PROMPT) {
    if (!unit_at<16 * NB>(A, A.units - 1 - bu, b, row0, q0, q1)) return;  // (the whole workgroup, here and below)
  } else if (A.order != 0) {
    q0 = b = sequence_at(A, bu);
  }
  int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int G = A.H / A.Hkv;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qlen = PROMPT ? max(q1 - q0, 0) : 1, nrows = qlen * G;
  if (PROMPT && row0 >= nrows) return;
  const int RN = PROMPT ? min(16 * NB, nrows - row0) : G, RS = PROMPT ? 16 * NB : G;  // rows, and from unit to unit
  const int ctx = min(max(A.ctx_lens[b], 0), A.width * PAGE), pos0 = ctx - qlen;       // pos0: keys before the new tokens
  const int seen = PROMPT ? max(0, pos0 + (row0 + RN - 1) / G + 1) : ctx;              // keys that the unit's last row sees
  const int pages = (seen + PAGE - 1) / PAGE;
  const int parts = max(1, min(A.nparts, (pages + A.ppp - 1) / A.ppp));
  if (part >= parts) return;
  const int share = pages / parts, rest = pages - share * parts;
  const int first = part * share + min(part, rest), last = first + share + (part < rest ? 1 : 0);

  Rows<DH, FP8, NB, PROMPT> rows;
  int sees[NB];  // the last key of the lane's row

  // the queries, and what follows from the lane
  auto lanes = [&] {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = row0 + 16 * nb + c, ti = PROMPT ? min(row, nrows - 1) / G : 0, hq = PROMPT ? min(row, nrows - 1) - ti * G : min(c, G - 1);
      sees[nb] = pos0 + ti;
      rows.query(nb, A.q + ((size_t)(q0 + ti) * A.H + kvh * G + hq) * DH + 16 * g, row < nrows, g);
    }
  };
  lanes();

  const int32_t* bt = A.tables + (size_t)b * A.width;
  auto page_of = [&](int p) -> long { return min(max(bt[min(p, last - 1)], 0), A.num_pages - 1); };  // (last > first)
  // (read once a launch: non-temporal, as fast as plain loads for small caches and up to 11 % faster for large ones)
  auto ld = [](const uint8_t* p) -> u32x4 {
    return PROMPT ? *reinterpret_cast<const u32x4*>(p) : __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  };
  // page p of the sequence, which lies at `page`.  Rows past the context read its last row again: no bytes that do not count
  // (512 contexts of 525 tokens end 13 tokens into a page)
  auto load_k = [&](int p, long page, R& x) {
    const uint8_t* kp = A.kc + ((size_t)page * A.Hkv + kvh) * M::BYTES;
    const int end = min(ctx - 1 - p * PAGE, PAGE - 1), krow = 8 * (c >> 2) + (c & 3);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < R::KV; ++i)
        x.k[t][i] = ld(kp + (uint32_t)(min(32 * (t >> 1) + 4 * (t & 1) + krow, end) * M::ROW + 16 * (DH == 64 && !FP8 ? g & 1 : g)) + 64 * i);
    x.ks = *reinterpret_cast<const uint32_t*>(kp + M::ELEMS + 64 * (g & (J - 1)) + 4 * c);
  };
  auto load_v = [&](int p, long page, R& x) {
    const uint8_t* vp = A.vc + ((size_t)page * A.Hkv + kvh) * M::BYTES;
    const int end = min(ctx - 1 - p * PAGE, PAGE - 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int u = 0; u < R::VU; ++u)
        x.v[kk][u] = ld(vp + (uint32_t)((min(32 * kk + 8 * g + u * M::KC, end) / M::KC) * 256 + 16 * c));
#pragma unroll
      for (int u = 0; u < R::VS; ++u) x.vs[kk][u] = ld(vp + M::ELEMS + (32 * kk + 8 * g) * J + 16 * u);
    }
  };
  R x;
  auto scores = [&](f32x4 (&st)[NB][4]) {
    rows.scores([&](int t, u32x4 (&k)[R::KV]) {
#pragma unroll
      for (int i = 0; i < R::KV; ++i) k[i] = x.k[t][i];
    }, x.ks, st);
  };
  auto weigh = [&](auto far, int p, f32x4 (&st)[NB][4]) {
    const int left = ctx - p * PAGE - 8 * g;  // keys of the context from the lane's first on
    // keys that some row does not see: past the context (the last page), or past a new token
    if ((PROMPT ? pos0 + row0 / G + 1 : ctx) - p * PAGE < PAGE) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) rows.mask(st[nb], (PROMPT ? sees[nb] + 1 : ctx) - p * PAGE - 8 * g);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) cut_values<DH, FP8>(x.v[kk], x.vs[kk], left - 32 * kk);
    }
    rows.template weigh<decltype(far)::value>([&](int kk, u32x4 (&v)[R::VU], u32x4 (&vs)[R::VS]) {
#pragma unroll
      for (int u = 0; u < R::VU; ++u) v[u] = x.v[kk][u];
#pragma unroll
      for (int u = 0; u < R::VS; ++u) vs[u] = x.vs[kk][u];
    }, st, A.scale_log2);
  };

  long nxt = last > first ? page_of(first + wave) : 0;  // (scalar reads of the table, ahead of the loads that need them)
  if (REFILL && first + wave < last) {
    load_k(first + wave, nxt, x);
    load_v(first + wave, nxt, x);
    nxt = page_of(first + wave + NW);
  }
  for (int p = first + wave; p < last; p += NW) {
    const std::false_type near;
    f32x4 st[NB][4];
    if constexpr (REFILL) {
      const bool more = p + NW < last;
      scores(st);
      if (more) load_k(p + NW, nxt, x);
      weigh(near, p, st);
      if (more) load_v(p + NW, nxt, x);
      nxt = page_of(p + 2 * NW);
    } else {
      load_k(p, nxt, x);
      load_v(p, nxt, x);
      nxt = page_of(p + NW);
      scores(st);
      weigh(near, p, st);
    }
  }
  rows.finish();
  if constexpr (PROMPT)
    if (__builtin_expect(rows.far(), 0)) {
      asm volatile("" : "+v"(lane));  // (what follows from the lane is found anew: none of it is kept through the first pass)
      g = lane >> 4;
      c = lane & 15;
      lanes();
      for (int p = first + wave; p < last; p += NW) {
        f32x4 st[NB][4];
        const long at = page_of(p);
        load_k(p, at, x);
        load_v(p, at, x);
        scores(st);
        weigh(std::true_type{}, p, st);
      }
      rows.finish();
    }

  const size_t row_ws = ((size_t)bu * A.nparts * A.Hkv + kvh) * RS, step = (size_t)A.Hkv * RS;  // partial results: part 0's first row, from part to part
  auto result = [&](int rw, int d, const f32x4& O, float inv) {
    const int row = row0 + rw, ti = PROMPT ? row / G : 0, hq = row - ti * G;
    uint16_t* p = A.out + ((size_t)(q0 + ti) * A.H + kvh * G + hq) * DH + d;
    if (pos0 + ti >= 0) st_results(p, O, inv);
    else *reinterpret_cast<s16x4*>(p) = s16x4{0, 0, 0, 0};  // a row without keys
  };
  auto leave = [&](int rw, int d, const f32x4& O, float mm, float L, float inv) {
    if (parts == 1) return result(rw, d, O, inv);
    const size_t row = row_ws + part * step + rw;
    agent_store4(A.ws_o + row * DH + d, O);
    if (d == 0) agent_store2(A.ws_ml + row * 2, mm, L);
  };
  if constexpr (NW == 1) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float inv = 1.f / rows.l[nb];
      if (16 * nb + c < RN)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            leave(16 * nb + c, 32 * j + 8 * g + 4 * half, rows.dims(nb, j, half), rows.m[nb], rows.l[nb], inv);
    }
  } else {  // the waves meet in LDS: [NW][RS][LD] sums, [NW][RS][2] maxima and sums of weights
    float* ml = sm + NW * RS * LD;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (16 * nb + c < RN) {
        const int at = wave * RS + 16 * nb + c;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half) *reinterpret_cast<f32x4*>(sm + at * LD + 32 * j + 8 * g + 4 * half) = rows.dims(nb, j, half);
        if (g == 0) {
          ml[at * 2] = rows.m[nb];
          ml[at * 2 + 1] = rows.l[nb];
        }
      }
    __syncthreads();
    for (int e = 4 * threadIdx.x; e < RN * DH; e += 4 * NW * 64) {
      const int rw = e / DH, d = e - rw * DH;
      float mm = NEG_BIG;
#pragma unroll
      for (int w = 0; w < NW; ++w) mm = fmaxf(mm, ml[(w * RS + rw) * 2]);
      float L = 0.f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {  // (a wave without pages: m = NEG_BIG, l = 0, o = 0)
        const float f = __builtin_amdgcn_exp2f(ml[(w * RS + rw) * 2] - mm);
        L += ml[(w * RS + rw) * 2 + 1] * f;
        O += *reinterpret_cast<const f32x4*>(sm + (w * RS + rw) * LD + d) * f;
      }
      leave(rw, d, O, mm, L, 1.f / L);
    }
  }
  if (parts == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the partial results have left
  __syncthreads();
  __shared__ int last_sm;
  int* t = A.tickets + bu * A.Hkv + kvh;
  if (threadIdx.x == 0) last_sm = __hip_atomic_fetch_add(t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
  __syncthreads();
  if (!last_sm) return;
  if (threadIdx.x == 0) __hip_atomic_store(t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int e = 4 * threadIdx.x; e < RN * DH; e += 4 * NW * 64) {
    const int rw = e / DH, d = e - rw * DH;
    float mm = NEG_BIG, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 8) {
      f32x2_t ml[8];
      f32x4 po[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i] = {NEG_BIG, 0.f};
        po[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (!PROMPT || s0 + i < parts) {  // (single tokens read the last again: a branch costs them registers; prompts' rows are many)
          const size_t row = row_ws + min(s0 + i, parts - 1) * step + rw;
          ml[i] = agent_load2(A.ws_ml + row * 2);
          po[i] = agent_load4(A.ws_o + row * DH + d);
        }
      }
      float mx = mm;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, ml[i][0]);
      const float f0 = __builtin_amdgcn_exp2f(mm - mx);
      L *= f0;
      O *= f0;
      mm = mx;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < parts) {
          const float f = __builtin_amdgcn_exp2f(ml[i][0] - mm);
          L += ml[i][1] * f;
          O += po[i] * f;
        }
    }
    result(rw, d, O, 1.f / L);
  }
}

// ============================================================================ attention of prompts
// 128 rows (token, head) of a (sequence, KV head) a workgroup: eight waves of 16, or four of 32 for heads of 64 (two workgroups a CU, three or
// four).  The pages they see pass through LDS: the keys as the cache holds them, their rows' 16-byte pieces exchanged so that the 16 rows of a
// score tile lie in 16 different pieces of 256 bytes (mx_swizzle; the loads' source addresses do it), the values made bf16 by the waves
// together, once for all their rows.  One barrier a page: behind it page p's values are there and page p + 1 has landed, page p + 1 + AHEAD is
// asked for, the values of p + 1 are made, page p is computed.
// Bound by the vector unit and the waits for each other: 32 rows of a page are 1100 cycles of matrix instructions and 1300 of vector ones
// (512 of them exponentials'), which overlap in part (46 % and 59 % busy; LDS 44 %).  One prompt, 32 heads on 8: of 128 dims, mxfp4, 4096
// tokens 150 us (900 TFLOP/s), 8192 507 to 535 (1030 and more), mxfp8 164 and 557 to 598; of 64 dims 92 and 288, 94 and 330; the bf16 kernel
// behind kv_read_mx 165 and 577, 165 and 580, 120 and 421, 120 and 424.  us of others, 4096 of 128 dims, mxfp4 / mxfp8: units of one wave that make their own values
// 149 / 192 (12 prompts of 512 62 / 68, here 56 / 59), four waves of 32 rows 158 / 164, half of the waves making values behind their products
// instead of before 156 / 171, six waves of 32 rows 244; mxfp4 of 64 dims eight waves of 16 rows 92, 12 prompts of 512 37 (36).
template <int DH, bool FP8>
struct PromptLds {
  using M = Mx<DH, FP8>;
  static constexpr int NB = DH == 128 ? 1 : 2, NW = 8 / NB;   // blocks of 16 rows of a wave, waves: four a SIMD and two
  static constexpr int AHEAD = FP8 && DH == 128 ? 1 : 2;     // pages in flight (two workgroups a CU have 80 KB each)
  static constexpr int KG = M::BYTES / 16;                   // pieces of a page's keys, and of its values
  static constexpr int NCH = (KG + 63) / 64;                 // loads of 64 pieces (1 KB of LDS) that hold them
  static constexpr int N = (2 * NCH + NW - 1) / NW;                // loads a wave and page
  static constexpr int RAW = NCH * 1024;
  static constexpr int VBUF = PAGE * DH * 2;                 // values in bf16: [half of the keys][group][even / odd][eight keys][16 dims][8]
  static constexpr int K0 = 0, V0 = (AHEAD + 2) * RAW, B0 = V0 + (AHEAD + 1) * RAW, FLAGS = B0 + 2 * VBUF, TOTAL = FLAGS + 64;
};
// which pieces of row r change places: x of its piece r (row / 16) + i becomes that number ^ x
template <int DH, bool FP8>
__device__ __forceinline__ int mx_swizzle(int r) {
  constexpr int RG = Mx<DH, FP8>::ROW / 16;
  const int q = (r >> 3) & 3;
  return RG == 8 ? 2 * q + ((r >> 1) & 1) : RG == 4 ? q : (q & 1) | (q & 2) << 2;
}

template <int DH, bool FP8>
__global__ __launch_bounds__(DH == 128 ? 512 : 256, 4) void attn_prompt_mx_kernel(const AttnArgs A) {
  using M = Mx<DH, FP8>;
  using R = PageRegs<DH, FP8>;
  using L = PromptLds<DH, FP8>;
  constexpr int J = M::J, NB = L::NB, RG = M::ROW / 16, AHEAD = L::AHEAD;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const PromptWork work = prompt_work(A.ctx_lens);
  const int b = __builtin_amdgcn_readfirstlane(work.seq), kvh = work.head, row0 = work.tile * 128;
  int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int G = A.H / A.Hkv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q0 = min(max(A.cu_q[b], 0), A.T), qlen = min(max(A.cu_q[b + 1], q0), A.T) - q0, nrows = qlen * G;
  if (row0 >= nrows) return;  // the whole workgroup
  const int ctx = min(max(A.ctx_lens[b], 0), A.width * PAGE), pos0 = ctx - qlen;  // pos0: keys before the new tokens
  const int pages = (max(0, pos0 + (min(row0 + 128, nrows) - 1) / G + 1) + PAGE - 1) / PAGE;
  const int wrow0 = row0 + 16 * NB * wave, wend = min(wrow0 + 16 * NB, nrows);
  const int wmin = pos0 + wrow0 / G, wmax = wend > wrow0 ? pos0 + (wend - 1) / G : -1;  // last keys of the wave's first and last rows

  // this lane's pieces of a page: load i of the wave brings chunk ch of the keys' or (from NCH on) the values' bytes.  Every wave has N loads in
  // flight, which the waits count, so the waves' loads are more than the chunks: of 128 dims 16 for 10 (mxfp4) and 24 for 18, of 64 8 for 6 and
  // 12 for 10; the surplus brings the last chunk's bytes once more
  int from[L::N], chunk[L::N];
  auto pieces = [&] {
#pragma unroll
    for (int i = 0; i < L::N; ++i) {
      chunk[i] = min(L::N * wave + i, 2 * L::NCH - 1);  // (past the last chunk: that again)
      const bool v = chunk[i] >= L::NCH;
      const int at = min(64 * (v ? chunk[i] - L::NCH : chunk[i]) + lane, L::KG - 1);  // (past the page: its last piece again)
      from[i] = 16 * (v || at >= M::ELEMS / 16 ? at : at ^ mx_swizzle<DH, FP8>(at / RG));
    }
  };
  // the table's entries as scalar loads, one page ahead of the loads that need them (a vector load there would be waited for behind the
  // pages in flight)
  typedef const __attribute__((address_space(4))) int32_t* table_t;
  const table_t bt = (table_t)(uintptr_t)(A.tables + (size_t)b * A.width);
  auto page_of = [&](int p) -> int { return min(max(bt[min(p, pages - 1)], 0), A.num_pages - 1); };  // (pages > 0)
  auto issue = [&](int p, long page) {
    const uint8_t* kp = A.kc + ((size_t)page * A.Hkv + kvh) * M::BYTES;
    const uint8_t* vp = A.vc + ((size_t)page * A.Hkv + kvh) * M::BYTES;
    uint8_t* kd = lds + L::K0 + p % (AHEAD + 2) * L::RAW;
    uint8_t* vd = lds + L::V0 + p % (AHEAD + 1) * L::RAW;
#pragma unroll
    for (int i = 0; i < L::N; ++i) {
      const bool v = chunk[i] >= L::NCH;
      uint32_t at = from[i];
      if constexpr (DH == 64) asm volatile("" : "+v"(at));  // (else it becomes a 64-bit constant of the loop, and a register too many is spilled)
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)((v ? vp : kp) + at),
                                       (__attribute__((address_space(3))) void*)((v ? vd - L::NCH * 1024 : kd) + chunk[i] * 1024), 16, 0, 0);
    }
  };
  // values of page p, landed, into bf16: the wave takes four octets of keys (lane group: octet) of one group of dims
  auto make_values = [&](int p) {
    const uint8_t* raw = lds + L::V0 + p % (AHEAD + 1) * L::RAW;
    uint8_t* to = lds + L::B0 + (p & 1) * L::VBUF;
    const int oct = 4 * (wave & 1) + g, left = ctx - p * PAGE - 8 * oct;
    u32x4 v[R::VU], vs[R::VS];
#pragma unroll
    for (int u = 0; u < R::VU; ++u) v[u] = *reinterpret_cast<const u32x4*>(raw + (8 * oct / M::KC + u) * 256 + 16 * c);
#pragma unroll
    for (int u = 0; u < R::VS; ++u) vs[u] = *reinterpret_cast<const u32x4*>(raw + M::ELEMS + 8 * oct * J + 16 * u);
    if (ctx - p * PAGE < PAGE) cut_values<DH, FP8>(v, vs, left);
    auto group = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      u32x4 ae, ao;
      value_pairs<DH, FP8>(v, vs, j, ae, ao);
      uint8_t* t = to + ((oct >> 2) * J + j) * 2048 + (oct & 3) * 256 + 16 * c;
      *reinterpret_cast<u32x4*>(t) = ae;
      *reinterpret_cast<u32x4*>(t + 1024) = ao;
    };
    if (wave < 2) group(std::integral_constant<int, 0>{});
    else if (wave < 4) group(std::integral_constant<int, 1>{});
    else if constexpr (J == 4) {
      if (wave < 6) group(std::integral_constant<int, 2>{});
      else group(std::integral_constant<int, 3>{});
    }
  };
  auto meet = [] {  // LDS of this wave done, all waves here
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  Rows<DH, FP8, NB, true> rows;
  int sees[NB];
  auto run = [&](auto far) {
    if constexpr (decltype(far)::value) {  // (what follows from the lane is found anew: none of it is kept through the first pass)
      asm volatile("" : "+v"(lane));
      g = lane >> 4;
      c = lane & 15;
    }
    pieces();
#pragma unroll
    for (int p = 0; p <= AHEAD; ++p)
      if (p < pages) issue(p, page_of(p));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = min(wrow0 + 16 * nb + c, nrows - 1), ti = row / G;
      sees[nb] = pos0 + ti;
      rows.query(nb, A.q + ((size_t)(q0 + ti) * A.H + kvh * G + row - ti * G) * DH + 16 * g, wrow0 + 16 * nb + c < nrows, g);
    }
    int nxt = pages > AHEAD + 1 ? page_of(AHEAD + 1) : 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the queries came behind the first pages)
    meet();
    if (pages > 0) make_values(0);
    for (int p = 0; p < pages; ++p) {
      if (AHEAD > 1 && p + AHEAD < pages)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 1) * L::N) : "memory");  // this wave's share of page p + 1 has landed
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      meet();
      if (p + 1 + AHEAD < pages) {
        issue(p + 1 + AHEAD, nxt);
        nxt = page_of(p + 2 + AHEAD);
      }
      if (p + 1 < pages) make_values(p + 1);
      if (p * PAGE > wmax) continue;  // every row of this wave is before the page
      const uint8_t* kr = lds + L::K0 + p % (AHEAD + 2) * L::RAW;
      const uint8_t* vb = lds + L::B0 + (p & 1) * L::VBUF;
      f32x4 st[NB][4];
      rows.scores([&](int t, u32x4 (&k)[R::KV]) {
        const int r = 32 * (t >> 1) + 4 * (t & 1) + 8 * (c >> 2) + (c & 3);
#pragma unroll
        for (int i = 0; i < R::KV; ++i)
          k[i] = *reinterpret_cast<const u32x4*>(kr + 16 * ((r * RG + (DH == 64 && !FP8 ? g & 1 : g) + 4 * i) ^ mx_swizzle<DH, FP8>(r)));
      }, *reinterpret_cast<const uint32_t*>(kr + M::ELEMS + 64 * (g & (J - 1)) + 4 * c), st);
      if (wmin + 1 - p * PAGE < PAGE) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) rows.mask(st[nb], sees[nb] + 1 - p * PAGE - 8 * g);
      }
      s16x8 pf[NB][2];
      rows.template weights<decltype(far)::value>(st, A.scale_log2, pf);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const s16x8 v = ld16(vb + ((kk * J + j) * 2 + e) * 1024 + g * 256 + 16 * c);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) rows.o[nb][j][e] = mfma16(v, pf[nb][kk], rows.o[nb][j][e]);
          }
    }
    rows.finish();
  };
  auto store = [&] {
    if (wmin < 0) {  // rows without keys: what they weighed with 0 may have been NaN
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) rows.o[nb][j][e] = sees[nb] >= 0 ? rows.o[nb][j][e] : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = wrow0 + 16 * nb + c, ti = row / G;
      if (row >= nrows) continue;
      const float inv = pos0 + ti >= 0 ? 1.f / rows.l[nb] : 0.f;  // a row without keys: zeros (its sums are)
      uint16_t* p = A.out + ((size_t)(q0 + ti) * A.H + kvh * G + row - ti * G) * DH + 8 * g;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) st_results(p + 32 * j + 4 * half, rows.dims(nb, j, half), inv);
    }
  };
  run(std::false_type{});
  const bool again = rows.far();
  uint32_t* flags = reinterpret_cast<uint32_t*>(lds + L::FLAGS);
  if (lane == 0) flags[wave] = again;
  if (!again) store();  // (once: a result may lie where its row's queries were)
  meet();  // (every page has landed and is read)
  uint32_t any = 0;
#pragma unroll
  for (int w = 0; w < L::NW; ++w) any |= flags[w];
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(any) != 0, 0)) {
    run(std::true_type{});
    if (again) store();
  }
}

// ============================================================================ bindings
#define XCHECK(cond, ...) TORCH_CHECK(cond, "xot kernel: ", __VA_ARGS__)
inline hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }
inline uint16_t* bf(const at::Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

void on_gpu(const char* op, const at::Tensor& t, at::ScalarType dt, const char* name, const at::Device& dev) {
  XCHECK(t.is_cuda() && t.device() == dev, op, ": ", name, " must be on the queries' GPU");
  XCHECK(t.scalar_type() == dt, op, ": ", name, " must be ", dt);
  XCHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}

int64_t page_bytes(int64_t Dh, bool fp8) { return PAGE * (fp8 ? Dh : Dh / 2) + PAGE * (Dh / 32); }

// both pools [pages, Hkv, bytes] of one format; true: e4m3
bool caches_ok(const char* op, const at::Tensor& k, const at::Tensor& v, int64_t Dh, const at::Device& dev) {
  XCHECK(Dh == 64 || Dh == 128, op, ": heads of 64 or 128 dims");
  on_gpu(op, k, at::kByte, "k_cache", dev);
  on_gpu(op, v, at::kByte, "v_cache", dev);
  XCHECK(k.dim() == 3 && v.sizes() == k.sizes(), op, ": caches must be two [pages, Hkv, page bytes] of the same size");
  XCHECK(k.size(0) >= 1 && k.size(0) < (int64_t(1) << 31) && k.size(1) >= 1, op, ": caches without pages or heads");
  const bool fp8 = k.size(2) == page_bytes(Dh, true);
  XCHECK(fp8 || k.size(2) == page_bytes(Dh, false), op, ": a page of ", k.size(2), " bytes is neither mxfp4 nor mxfp8 of heads of ", Dh);
  XCHECK((reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) % 16 == 0, op, ": caches must be aligned to 16 bytes");
  return fp8;
}

#define MX_GO(fp8, Dh, GO)                  \
  do {                                      \
    if ((Dh) == 128) {                      \
      if (fp8) GO(128, true);               \
      else GO(128, false);                  \
    } else {                                \
      if (fp8) GO(64, true);                \
      else GO(64, false);                   \
    }                                       \
  } while (0)

// heads of a wave: four share its angles (which are as many bytes as its rows) where there are rows enough to fill the chip with fewer
// waves.  us at 1 / 4, mxfp4, heads of 128: 8192 tokens of 64 + 16 heads 69.7 / 58.9 (5.3 TB/s), of 32 + 16 43.2 / 36.8, 2048 of 64 + 16
// 16.2 / 15.0, of 32 + 16 10.9 / 11.2, 512 4.3 / 5.3, 1 2.7 / 4.0
constexpr int WRITE_HEADS = 4, WRITE_HEADS_ROWS = 1 << 17;

at::Tensor rope_kv_write_mx(const at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& cos_sin, const at::Tensor& slots,
                            const c10::optional<at::Tensor>& out, at::Tensor& k_cache, at::Tensor& v_cache, int64_t H, int64_t Hkv) {
  const char* op = "rope_kv_write_mx";
  XCHECK(qkv.is_cuda() && qkv.dim() == 2, op, ": qkv must be [T, (H + 2 Hkv) Dh] on a GPU");
  const at::Device dev = qkv.device();
  const c10::DeviceGuard guard(dev);
  const int64_t T = qkv.size(0);
  XCHECK(H >= 1 && Hkv >= 1 && qkv.size(1) % (H + 2 * Hkv) == 0, op, ": qkv columns are not H + 2 Hkv heads");
  const int64_t Dh = qkv.size(1) / (H + 2 * Hkv);
  on_gpu(op, qkv, at::kBFloat16, "qkv", dev);
  on_gpu(op, pos, at::kInt, "pos", dev);
  on_gpu(op, cos_sin, at::kFloat, "cos_sin", dev);
  on_gpu(op, slots, at::kLong, "slots", dev);
  at::Tensor q_out = out.has_value() ? *out : at::empty({T, H, Dh}, qkv.options());
  on_gpu(op, q_out, at::kBFloat16, "q_out", dev);
  const bool fp8 = caches_ok(op, k_cache, v_cache, Dh, dev);
  XCHECK(k_cache.size(1) == Hkv, op, ": the caches have ", k_cache.size(1), " heads");
  XCHECK(pos.numel() == T && slots.numel() == T && q_out.numel() == T * H * Dh, op, ": pos, slots or q_out of another length");
  XCHECK(cos_sin.dim() == 2 && cos_sin.size(1) == Dh && cos_sin.size(0) >= 1, op, ": cos_sin must be [positions, Dh]");
  if (T == 0) return q_out;
  XCHECK((reinterpret_cast<uintptr_t>(qkv.data_ptr()) | reinterpret_cast<uintptr_t>(q_out.data_ptr()) | reinterpret_cast<uintptr_t>(cos_sin.data_ptr())) % 16 == 0,
         op, ": qkv, q_out and cos_sin must be aligned to 16 bytes");
  XCHECK(T < (1 << 26) && H + 2 * Hkv < (1 << 20) && (T + 3) / 4 * (H + 2 * Hkv) < (int64_t(1) << 26), op, ": too many tokens for one launch");
  const int64_t hb = T * (H + 2 * Hkv) >= WRITE_HEADS_ROWS ? WRITE_HEADS : 1;
  const unsigned blocks = (unsigned)(((T + 3) / 4 * ((H + 2 * Hkv + hb - 1) / hb) + 3) / 4);
#define GO_HB(DHV, F, HB)                                                                                                               \
  rope_kv_write_mx_kernel<DHV, F, HB><<<blocks, 256, 0, stream()>>>(bf(qkv), pos.data_ptr<int32_t>(), cos_sin.data_ptr<float>(),        \
                                                                    slots.data_ptr<int64_t>(), bf(q_out), k_cache.data_ptr<uint8_t>(),  \
                                                                    v_cache.data_ptr<uint8_t>(), (int)T, (int)H, (int)Hkv,              \
                                                                    (int)cos_sin.size(0), (long)k_cache.size(0) * PAGE)
#define GO(DHV, F)                           \
  do {                                       \
    if (hb > 1) GO_HB(DHV, F, WRITE_HEADS);  \
    else GO_HB(DHV, F, 1);                   \
  } while (0)
  MX_GO(fp8, Dh, GO);
#undef GO
#undef GO_HB
  return q_out;
}

std::tuple<at::Tensor, at::Tensor> kv_read_mx(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& tables, const at::Tensor& ctx_lens,
                int64_t Dh, const c10::optional<at::Tensor>& k_opt, const c10::optional<at::Tensor>& v_opt, bool skip, const c10::optional<at::Tensor>& own) {
  const char* op = "kv_read_mx";
  XCHECK(k_cache.is_cuda(), op, ": k_cache must be on a GPU");
  const at::Device dev = k_cache.device();
  const c10::DeviceGuard guard(dev);
  on_gpu(op, tables, at::kInt, "block_tables", dev);
  on_gpu(op, ctx_lens, at::kInt, "ctx_lens", dev);
  XCHECK(tables.dim() == 2 && ctx_lens.numel() == tables.size(0), op, ": a row of block_tables for each of ctx_lens");
  const int64_t n = tables.numel(), Hkv = k_cache.dim() == 3 ? k_cache.size(1) : 0;
  const bool fp8 = caches_ok(op, k_cache, v_cache, Dh, dev);
  const auto bf16 = k_cache.options().dtype(at::kBFloat16);
  at::Tensor k_out = k_opt.has_value() ? *k_opt : at::empty({n, Hkv, PAGE, Dh}, bf16);
  at::Tensor v_out = v_opt.has_value() ? *v_opt : at::empty({n, Hkv, Dh, PAGE}, bf16);
  on_gpu(op, k_out, at::kBFloat16, "k_out", dev);
  on_gpu(op, v_out, at::kBFloat16, "v_out", dev);
  XCHECK(k_out.dim() == 4 && v_out.dim() == 4 && k_out.size(3) == Dh, op, ": k_out and v_out must be 4-D");
  XCHECK(k_out.size(0) == n && k_out.size(1) == Hkv && k_out.size(2) == PAGE && v_out.size(0) == n && v_out.size(1) == Hkv &&
             v_out.size(2) == Dh && v_out.size(3) == PAGE,
         op, ": k_out must be [entries, Hkv, 64, Dh], v_out [entries, Hkv, Dh, 64]");
  XCHECK((reinterpret_cast<uintptr_t>(k_out.data_ptr()) | reinterpret_cast<uintptr_t>(v_out.data_ptr())) % 16 == 0, op,
         ": k_out and v_out must be aligned to 16 bytes");
  if (own.has_value()) {
    on_gpu(op, *own, at::kInt, "own", dev);
    XCHECK(own->numel() == n, op, ": own must be of the entries' length");
  }
  if (n == 0) return {k_out, v_out};
  XCHECK(n < (int64_t(1) << 24) && n * Hkv < (int64_t(1) << 24), op, ": too many pages for one launch");
#define GO(DHV, F)                                                                                                                         \
  kv_read_mx_kernel<DHV, F><<<(unsigned)(n * Hkv), 256, 0, stream()>>>(                                                                    \
      k_cache.data_ptr<uint8_t>(), v_cache.data_ptr<uint8_t>(), tables.data_ptr<int32_t>(), (int)tables.size(1), ctx_lens.data_ptr<int32_t>(), \
      bf(k_out), bf(v_out), (int)Hkv, (int)k_cache.size(0), skip, own.has_value() ? own->data_ptr<int32_t>() : nullptr)
  MX_GO(fp8, Dh, GO);
#undef GO
  return {k_out, v_out};
}

// what both forms of the attention check; cu_q: several tokens a sequence
AttnArgs attn_args(const char* op, bool& fp8, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& tables,
                   const at::Tensor& ctx_lens, const at::Tensor* cu_q, at::Tensor& out, const c10::optional<at::Tensor>& ws_o,
                   const c10::optional<at::Tensor>& ws_ml, const c10::optional<at::Tensor>& tickets, int64_t units, int64_t unit_rows,
                   int64_t pages_per_part, int64_t nparts, double scale, int per = 0, int order = 0) {
  const at::Device dev = q.device();
  on_gpu(op, q, at::kBFloat16, "q", dev);
  on_gpu(op, out, at::kBFloat16, "out", dev);
  on_gpu(op, tables, at::kInt, "block_tables", dev);
  on_gpu(op, ctx_lens, at::kInt, "ctx_lens", dev);
  const int64_t T = q.size(0), H = q.size(1), Dh = q.size(2), Hkv = k_cache.dim() == 3 ? k_cache.size(1) : 0;
  const int64_t B = ctx_lens.numel();
  fp8 = caches_ok(op, k_cache, v_cache, Dh, dev);
  XCHECK(H >= 1 && H % Hkv == 0 && H / Hkv <= 16, op, ": ", H, " query heads on ", Hkv, " (at most 16 each)");
  XCHECK(tables.dim() == 2 && tables.size(0) == B, op, ": a row of block_tables for each of ctx_lens");
  XCHECK(B == 0 || (tables.size(1) >= 1 && tables.size(1) < (1 << 24)), op, ": block_tables of no or too many columns");
  if (cu_q != nullptr) {
    on_gpu(op, *cu_q, at::kInt, "cu_q", dev);
    XCHECK(cu_q->numel() == B + 1, op, ": cu_q must have one entry more than ctx_lens");
  } else {
    XCHECK(T == B, op, ": a length for each query");
  }
  XCHECK(T < (int64_t(1) << 31) / std::max<int64_t>(H, 1), op, ": too many tokens");
  XCHECK(out.sizes() == q.sizes(), op, ": out must have q's shape");
  XCHECK((reinterpret_cast<uintptr_t>(q.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) % 16 == 0, op, ": q and out must be aligned to 16 bytes");
  XCHECK(pages_per_part >= 1 && pages_per_part <= (1 << 24) && nparts >= 1, op, ": bad partitioning");
  // (what the kernels multiply by, the scale times log2 e as a float, stays a positive normal number: masked scores are -inf)
  XCHECK(scale >= 0x1p-125 && scale <= 0x1p126, op, ": the scale must be positive, 2^-125 to 2^126");
  XCHECK(nparts < (1 << 24) && units < (int64_t(1) << 24) && units * nparts < (int64_t(1) << 24) && units * nparts * Hkv < (int64_t(1) << 24), op,
         ": too many parts for one launch");
  float *o = nullptr, *ml = nullptr;
  int* tk = nullptr;
  if (nparts > 1) {
    XCHECK(ws_o.has_value() && ws_ml.has_value() && tickets.has_value(), op, ": parts need a workspace");
    on_gpu(op, *ws_o, at::kFloat, "ws_o", dev);
    on_gpu(op, *ws_ml, at::kFloat, "ws_ml", dev);
    on_gpu(op, *tickets, at::kInt, "tickets", dev);
    const int64_t rows = units * nparts * Hkv * unit_rows;
    XCHECK(tickets->numel() >= units * Hkv && ws_o->numel() >= rows * Dh && ws_ml->numel() >= rows * 2 &&
               (reinterpret_cast<uintptr_t>(ws_o->data_ptr()) | reinterpret_cast<uintptr_t>(ws_ml->data_ptr())) % 16 == 0,
           op, ": workspace small");
    o = ws_o->data_ptr<float>();
    ml = ws_ml->data_ptr<float>();
    tk = tickets->data_ptr<int32_t>();
  }
  return {bf(q), k_cache.data_ptr<uint8_t>(), v_cache.data_ptr<uint8_t>(), tables.data_ptr<int32_t>(), ctx_lens.data_ptr<int32_t>(),
          cu_q == nullptr ? nullptr : cu_q->data_ptr<int32_t>(), bf(out), o, ml, tk, (int)T, (int)B, (int)tables.size(1), (int)H, (int)Hkv, (int)pages_per_part,
          (int)nparts, (int)k_cache.size(0), (int)units, per, order, (float)scale * LOG2E};
}

at::Tensor attn_decode_mx(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& tables,
                    const at::Tensor& ctx_lens, const c10::optional<at::Tensor>& out_opt, const c10::optional<at::Tensor>& ws_o, const c10::optional<at::Tensor>& ws_ml,
                    const c10::optional<at::Tensor>& tickets, int64_t pages_per_part, int64_t nparts, int64_t waves, bool refill, int64_t order, double scale) {
  const char* op = "attn_decode_mx";
  XCHECK(q.is_cuda() && q.dim() == 3, op, ": q must be [B, H, Dh] on a GPU");
  const c10::DeviceGuard guard(q.device());
  bool fp8 = false;
  at::Tensor out = out_opt.has_value() ? *out_opt : at::empty_like(q);
  const int64_t H = q.size(1), Dh = q.size(2), Hkv = k_cache.dim() == 3 ? k_cache.size(1) : 1;
  const AttnArgs a = attn_args(op, fp8, q, k_cache, v_cache, tables, ctx_lens, nullptr, out, ws_o, ws_ml, tickets, q.size(0), H / std::max<int64_t>(Hkv, 1),
                               pages_per_part, nparts, scale, 0, (int)order);
  XCHECK(order == 0 || (order >= 1 && order <= 2 && q.size(0) <= 64), op, ": an order of at most 64 sequences");
  XCHECK(waves == 1 || waves == 2 || waves == 4, op, ": 1, 2 or 4 waves");
  if (q.size(0) == 0) return out;
  const size_t lds = waves == 1 ? 0 : (size_t)waves * (H / Hkv) * (Dh + 6) * sizeof(float);  // at most 34 KB
  const unsigned units = (unsigned)(q.size(0) * nparts * Hkv);
#define GO(DHV, F)                                                                                              \
  do {                                                                                                          \
    if (waves == 1) attn_mx_kernel<DHV, F, 1, 1, false, false><<<units, 64, lds, stream()>>>(a);                \
    else if (waves == 2) attn_mx_kernel<DHV, F, 2, 1, false, false><<<units, 128, lds, stream()>>>(a);          \
    else if (refill && !(F && DHV == 128)) attn_mx_kernel<DHV, F, 4, 1, false, !(F && DHV == 128)><<<units, 256, lds, stream()>>>(a); \
    else attn_mx_kernel<DHV, F, 4, 1, false, false><<<units, 256, lds, stream()>>>(a);                          \
  } while (0)
  MX_GO(fp8, Dh, GO);
#undef GO
  return out;
}

constexpr int PROMPT_WAVES = 4, PROMPT_BLOCKS = 2;  // of 16 rows

// new tokens against the pools: units of 32 rows of (token, head), of four waves that share the pages, or (tiles) attn_prompt_mx_kernel's of 128
at::Tensor attn_prompt_mx(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& tables, const at::Tensor& cu_q,
                          const at::Tensor& ctx_lens, const c10::optional<at::Tensor>& out_opt, const c10::optional<at::Tensor>& ws_o, const c10::optional<at::Tensor>& ws_ml,
                  const c10::optional<at::Tensor>& tickets, int64_t max_qlen, int64_t pages_per_part, int64_t nparts, bool tiles, double scale) {
  const char* op = "attn_prompt_mx";
  XCHECK(q.is_cuda() && q.dim() == 3, op, ": q must be [T, H, Dh] on a GPU");
  const c10::DeviceGuard guard(q.device());
  bool fp8 = false;
  at::Tensor out = out_opt.has_value() ? *out_opt : at::empty_like(q);
  const int64_t H = q.size(1), Dh = q.size(2), Hkv = k_cache.dim() == 3 ? k_cache.size(1) : 1, B = ctx_lens.numel();
  XCHECK(max_qlen >= 0 && max_qlen < (1 << 24), op, ": max_qlen");
  constexpr int64_t ROWS = 16 * PROMPT_BLOCKS, TILE = 128;
  tiles = tiles && Hkv < 65536 && B < 65536;  // (the grid's limits)
  const int64_t G = H / std::max<int64_t>(Hkv, 1), rows = tiles ? TILE : ROWS, per = (max_qlen * G + rows - 1) / rows;  // units of the longest
  const bool even = tiles || B * per <= q.size(0) * G / ROWS + B;
  const int64_t units = even ? B * per : q.size(0) * G / ROWS + B;
  const AttnArgs a = attn_args(op, fp8, q, k_cache, v_cache, tables, ctx_lens, &cu_q, out, ws_o, ws_ml, tickets, units, ROWS, pages_per_part, nparts, scale,
                               even ? (int)std::min<int64_t>(per, 1 << 24) : 0);
  if (B == 0 || max_qlen == 0) return out;
  if (tiles) {
    XCHECK(nparts == 1, op, ": parts are of units");
    const dim3 grid((unsigned)per, (unsigned)Hkv, (unsigned)B);
#define GO(DHV, F)                                                                                                             \
  do {                                                                                                                         \
    using L = PromptLds<DHV, F>;                                                                                               \
    auto* f = attn_prompt_mx_kernel<DHV, F>;                                                                                   \
    static const hipError_t set = hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);   \
    XCHECK(set == hipSuccess, op, ": LDS");                                                                                    \
    f<<<grid, 64 * L::NW, L::TOTAL, stream()>>>(a);                                                                            \
  } while (0)
    MX_GO(fp8, Dh, GO);
#undef GO
    return out;
  }
  const size_t lds = (size_t)PROMPT_WAVES * ROWS * (Dh + 6) * sizeof(float);  // 67 KB at heads of 128
  const unsigned grid = (unsigned)(units * nparts * Hkv);
#define GO(DHV, F)                                                                                                                         \
  do {                                                                                                                                     \
    auto* f = attn_mx_kernel<DHV, F, PROMPT_WAVES, PROMPT_BLOCKS, true, !(F && DHV == 128)>;                                               \
    static const hipError_t set = hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);              \
    XCHECK(set == hipSuccess, op, ": LDS");                                                                                                \
    f<<<grid, 64 * PROMPT_WAVES, lds, stream()>>>(a);                                                                                      \
  } while (0)
  MX_GO(fp8, Dh, GO);
#undef GO
  return out;
}

}  // namespace

void bind_kv_mx(pybind11::module& m) {
  m.def("rope_kv_write_mx", &rope_kv_write_mx);
  m.def("kv_read_mx", &kv_read_mx);
  m.def("attn_decode_mx", &attn_decode_mx);
  m.def("attn_prompt_mx", &attn_prompt_mx);
}

}  // namespace xot
