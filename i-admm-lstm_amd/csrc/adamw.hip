// The AdamW step over many tensors at once, with moments in 32 or in 8 bits, and the norm of many gradients.
//
//   g' = g min(1, max_norm / (norm + 1e-6))            (where clipping is asked for)
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// in fp32, each product and sum rounded by itself (with 8-bit moments the parameters' last steps are fused).  Bound:
// HBM, 28 bytes an element for fp32 parameters with 32-bit moments, 16 with 8-bit ones, 10 for bf16 parameters and
// gradients with 8-bit moments; a wave has all loads of its 1024 elements in flight, and nothing moves twice.
//
// Measured (MI355X; a copy of 1 GiB runs at 5.3 TB/s on it), one tensor of 100 M elements: fp32 with 32 bits 522 us =
// 5.4 TB/s, fp32 with 8 bits 299 us = 5.3, bf16 with 8 bits 194 us = 5.2 (where 47 vector instructions an element take
// nearly as long as the memory); mixed types at the same rate (32 bits: fp32 parameters with bf16 gradients 477 us, bf16
// with fp32 442, bf16 with bf16 407 = 5.4 TB/s; 8 bits: fp32 with bf16 254, bf16 with fp32 226 = 5.3 to 5.5); the 16 tensors of an h = 800 cell (2.6 M) 13.2 us, of an h = 200 cell 3.8 us.
//
// 8-bit moments.  256 elements (a wave's 64 lanes with 4 each: its maximum needs no LDS) share two powers of
// two.  m is a sign, 4 exponent and 3 mantissa bits under 2^em, v 5 and 3 bits without a sign under 2^ev:
//   |m| = 2^em * {n 2^-9 (e = 0), (8 + n) 2^(e - 10)},  v = 2^ev * {n 2^-33 (e = 0), (8 + n) 2^(e - 34)}
// (v's range, 2^-33 to 1.75, is about the square of m's, so that sqrt(v) keeps up with m).  Both layouts are
// fp32's with the lower mantissa bits cut off, once the number is scaled so that the code's exponent field is
// fp32's: bits >> 20 is the code, subnormals included, and bits << 20 the number.  A block whose largest value
// has a mantissa of 1.75 or more takes the next exponent, so no finite value reaches the codes of NaN (m) and
// infinity (v); these keep what overflowed visible.
//
// The cut is random: 20 hashed bits (12 for m) are added below the code's last bit.  A step changes v by
// (1 - b2) of itself, 0.1 % at b2 = 0.999, against half a code's 6 %: rounding to nearest would leave v where it
// is for good, rounding at random keeps its mean.  The same holds for bf16 parameters (half a step is 2^-9
// to 2^-8 of the value, lr is 1e-4).  A v that is not zero does not become zero: m / sqrt(v) would jump.
// The 32 bits belong to (seed, step, the tensor's place, the element's place), so a run can be repeated.
#include <string.h>

#include <type_traits>

#include "common.h"

namespace iadmm {

constexpr int kPer = 48;          // tensors that travel in a launch's arguments (3.5 KB of 4)
constexpr int kPlace = 55;        // tensors that adam_place_kernel's arguments carry (4 KB)
constexpr int kBlock8 = 256;      // elements under one pair of exponents
constexpr int kNormPer = 240, kNormBlocks = 1024;

enum { kHalfP = 1, kHalfG = 2 };  // AdamTensor::flags

struct AdamTensor {
  void* p;
  const void* g;
  void *m, *v, *e;
  int64_t n;
  float step_size, ibc2, decay;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
  uint32_t key;                  // (its slot, on the way to adam_place_kernel)
  uint32_t first;                // its first workgroup
  int flags;
};
static_assert(sizeof(AdamTensor) == 72, "words below");

struct AdamCommon {
  const float* norm;  // or null
  float b1, ob1, b2, ob2, eps, max_norm;
  int count;
};
// The tensors in the arguments, or in a table in memory that adam_place_kernel wrote: for more than kPer of them (216
// tensors of 100 M bf16 elements with 8-bit moments: 224 us, with five launches, each with a start and an end of its own,
// 262) and where the device counts (16 tensors of 2.6 M fp32 elements: 18.8 us; from the arguments 16.3).
struct AdamLaunch {
  AdamTensor t[kPer];
  AdamCommon c;
};
struct AdamTable {
  const AdamTensor* t;
  AdamCommon c;
};

// 32 well-mixed bits of 32: two odd multipliers between shifts, chosen by search for the least bias of any
// output bit's flip under any input bit's (0.4 % at most over 200 000 inputs).
__host__ __device__ inline uint32_t mix32_rest(uint32_t x) {
  x *= 0xDEFBD895u;
  x ^= x >> 15;
  x *= 0x066B4493u;
  return x ^ (x >> 16);
}
__host__ __device__ inline uint32_t mix32(uint32_t x) { return mix32_rest(x ^ x >> 16); }
__host__ __device__ inline uint32_t step_key(uint64_t seed, uint64_t step, int slot) {
  uint32_t k = mix32(static_cast<uint32_t>(seed) + 0x9E3779B9u);
  k = mix32(k ^ static_cast<uint32_t>(seed >> 32));
  k = mix32(k + static_cast<uint32_t>(step));
  return mix32(k ^ static_cast<uint32_t>(slot));
}

// Four neighbouring elements, at any address that the type may have; what lies behind the end is 0.
template <typename T> struct Quad { T v[4]; };
// FULL: none lies behind (a branch at each load would keep them from being in flight together).
template <bool FULL = false, typename T> IADMM_DEV Quad<T> load_quad(const T* p, int64_t left) {
  Quad<T> r;
  if (FULL || left >= 4) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = j < left ? p[j] : static_cast<T>(0);
  }
  return r;
}
template <bool FULL = false, typename T> IADMM_DEV void store_quad(T* p, const Quad<T>& r, int64_t left) {
  if (FULL || left >= 4) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = r.v[j];
  }
}

// The same for four codes, in one word (as members of their own they would be taken apart and put together again).
template <bool FULL> IADMM_DEV uint32_t load_codes(const uint8_t* p, int64_t left) {
  uint32_t r = 0;
  if (FULL || left >= 4) {
    __builtin_memcpy(&r, p, 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) r |= static_cast<uint32_t>(p[j]) << 8 * j;
  }
  return r;
}
template <bool FULL> IADMM_DEV void store_codes(uint8_t* p, uint32_t r, int64_t left) {
  if (FULL || left >= 4) {
    __builtin_memcpy(p, &r, 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = static_cast<uint8_t>(r >> 8 * j);
  }
}

IADMM_DEV float bits_f(uint32_t b) { return __uint_as_float(b); }
IADMM_DEV bool is_finite(float x) { return fabsf(x) < __builtin_inff(); }

IADMM_DEV float decode_m(uint32_t c, int e) {
  const float a = __builtin_amdgcn_ldexpf(bits_f((c & 127u) << 20), e + 120);
  return bits_f(__float_as_uint((c & 127u) == 127u ? __builtin_nanf("") : a) | (c & 128u) << 24);
}
IADMM_DEV float decode_v(uint32_t c, int e) {
  return c == 255u ? __builtin_inff() : __builtin_amdgcn_ldexpf(bits_f(c << 20), e + 96);
}
IADMM_DEV uint32_t encode_m(float m, int e, uint32_t bits) {
  const uint32_t a = __float_as_uint(__builtin_amdgcn_ldexpf(fabsf(m), -e - 120));
  uint32_t c = (a + (bits >> 20 << 8)) >> 20;
  c = c < 126u ? c : 126u;
  return (is_finite(m) ? c : 127u) | (m < 0.0f ? 128u : 0u);
}
IADMM_DEV uint32_t encode_v(float v, int e, uint32_t bits) {
  const uint32_t a = __float_as_uint(__builtin_amdgcn_ldexpf(v, -e - 96));
  uint32_t c = (a + (bits & 0xFFFFFu)) >> 20;
  c = c < 254u ? c : 254u;
  c = c == 0u && v > 0.0f ? 1u : c;
  return is_finite(v) ? c : 255u;
}
IADMM_DEV int block_exponent(uint32_t top, int shift, int low, int high) {
  const int e = static_cast<int>((top + 0x200000u) >> 23) - 127 - shift;
  return e < low ? low : (e > high ? high : e);
}
// The largest of the wave's values, as scalars: six maxima whose second operand comes from another lane (within rows
// of 16, then across them) instead of twelve instructions through LDS; two at a time, each in the other's wait states.
template <int CTRL> IADMM_DEV uint32_t umax_from(uint32_t v) {
  const uint32_t w = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
  return w > v ? w : v;
}
IADMM_DEV void wave_umax(uint32_t& a, uint32_t& b) {
  a = umax_from<0x111>(a), b = umax_from<0x111>(b);  // row_shr 1, 2, 4, 8: lane 15 of each row has its row's
  a = umax_from<0x112>(a), b = umax_from<0x112>(b);
  a = umax_from<0x114>(a), b = umax_from<0x114>(b);
  a = umax_from<0x118>(a), b = umax_from<0x118>(b);
  a = umax_from<0x142>(a), b = umax_from<0x142>(b);  // row_bcast 15, 31: lane 63 has the wave's
  a = umax_from<0x143>(a), b = umax_from<0x143>(b);
  a = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(a), 63));
  b = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), 63));
}

// Four codes at once, as the dword that they lie in.  The scales are products here, so the exponents have to
// leave 2^(e + 120) and its like normal: kFastM and kFastV, gradients below 10^4 or so; the others, and what is
// not finite, take the functions above.
constexpr int kFastM = 6, kFastV = 30;
IADMM_DEV float pow2(int e) { return bits_f(static_cast<uint32_t>(e + 127) << 23); }  // -126 <= e <= 127
IADMM_DEV bool ordinary_codes(uint32_t m, uint32_t v) {  // no NaN (m & 127 = 127), no infinity (v = 255)
  const uint32_t a = (m & 0x7F7F7F7Fu) + 0x01010101u, b = ((v & 0x7F7F7F7Fu) + 0x01010101u) & v;
  return ((a | b) & 0x80808080u) == 0u;
}
// Byte J of a word, moved to bits 20..27 (with its sign above, for m): one instruction each.
template <int J> IADMM_DEV uint32_t byte_up(uint32_t q) {
  uint32_t r;
  const uint32_t by = 20;
  if constexpr (J == 0) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 1) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 2) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 3) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(by), "v"(q));
  return r;
}
template <int J> IADMM_DEV uint32_t signed_byte_up(uint32_t q) {
  uint32_t r;
  const uint32_t by = 20;
  if constexpr (J == 0) asm("v_lshlrev_b32_sdwa %0, %1, sext(%2) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 1) asm("v_lshlrev_b32_sdwa %0, %1, sext(%2) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 2) asm("v_lshlrev_b32_sdwa %0, %1, sext(%2) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(by), "v"(q));
  if constexpr (J == 3) asm("v_lshlrev_b32_sdwa %0, %1, sext(%2) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(by), "v"(q));
  return r;
}
template <int J> IADMM_DEV float decode_m_of(uint32_t q, float scale) {
  return bits_f(signed_byte_up<J>(q) & 0x87F00000u) * scale;
}
template <int J> IADMM_DEV float decode_v_of(uint32_t q, float scale) { return bits_f(byte_up<J>(q)) * scale; }
// The code in the top byte (the blocks' exponents keep it below NaN's and infinity's).
IADMM_DEV uint32_t encode_m_top(float m, float scale, uint32_t bits) {
  const uint32_t a = (__float_as_uint(fabsf(m) * scale) + (bits >> 20 << 8)) << 4;
  return __float_as_uint(copysignf(bits_f(a), m));
}
// The median lifts what is below the first code onto it, and leaves 0 (and what fp32 itself holds with less than 20
// bits, below 2^-129) where it is: the scaled value is never above v.
IADMM_DEV uint32_t encode_v_top(float v, float scale, uint32_t bits) {
  const uint32_t x = __float_as_uint(v * scale), y = __float_as_uint(v), one = 1u << 20;
  const uint32_t lo = x < one ? x : one, hi = x < one ? one : x, mid = hi < y ? hi : y;
  return ((lo > mid ? lo : mid) + (bits & 0xFFFFFu)) << 4;  // (the median of x, y and one)
}
IADMM_DEV uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x00000703u), hi = __builtin_amdgcn_perm(d, c, 0x07030000u);
  return __builtin_amdgcn_perm(hi, lo, 0x07060100u);
}

// The last of `count` tensors whose first workgroup is not behind this one: 64 at a time from a stride apart, closer.
// (An empty tensor has its successor's first workgroup, and is never the last with it.)
template <typename T> IADMM_DEV int find_tensor(const T& t, int count, uint32_t block) {
  const int lane = threadIdx.x % kWave;
  int at = 0, n = count;
  for (;;) {
    const int stride = (n + kWave - 1) / kWave, k = lane * stride;
    const int reached = __popcll(__ballot(k < n && t[at + (k < n ? k : 0)].first <= block));
    at += (reached - 1) * stride;
    if (stride == 1) return __builtin_amdgcn_readfirstlane(at);
    n = n - (reached - 1) * stride < stride ? n - (reached - 1) * stride : stride;
  }
}

// The new parameters of four elements; `bits` are 0 for fp32.  SAFE: NaN keeps its bits (random ones added to a payload
// of ones would carry into the sign; where the moments are finite, a NaN is a bf16 parameter's own, with lower bits 0).
template <typename P, bool SAFE> IADMM_DEV Quad<P> new_params(const float (&np)[4], const uint32_t (&bits)[4]) {
  Quad<P> q;
  if constexpr (sizeof(P) == 2) {
    uint32_t b[4], w[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] = __float_as_uint(np[j]) + (bits[j] >> 16);
      if (SAFE) b[j] = np[j] != np[j] ? 0x7FC00000u : b[j];
    }
    w[0] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302u);
    w[1] = __builtin_amdgcn_perm(b[3], b[2], 0x07060302u);
    __builtin_memcpy(&q, w, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) q.v[j] = np[j];
  }
  return q;
}

// QUADS x 256 elements per wave.
template <typename P, typename G, bool EIGHT, int QUADS, bool FULL>
IADMM_DEV void adam_wave(const AdamCommon& a, const AdamTensor& t, float clip, int64_t at) {
  const int lane = threadIdx.x % kWave;
  P* p = static_cast<P*>(t.p);
  const G* g = static_cast<const G*>(t.g);
  float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
  uint8_t *m8 = static_cast<uint8_t*>(t.m), *v8 = static_cast<uint8_t*>(t.v);
  int8_t* e = static_cast<int8_t*>(t.e) + at / kBlock8 * 2;
  Quad<P> qp[QUADS];
  Quad<G> qg[QUADS];
  Quad<float> qm[QUADS], qv[QUADS];
  uint32_t cm[QUADS], cv[QUADS];
  int8_t old[2 * QUADS], now[2 * QUADS];
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int64_t i = at + u * 256 + lane * 4, left = t.n - i;
    qp[u] = load_quad<FULL>(p + i, left);
    qg[u] = load_quad<FULL>(g + i, left);
    if constexpr (EIGHT) {
      cm[u] = load_codes<FULL>(m8 + i, left);
      cv[u] = load_codes<FULL>(v8 + i, left);
    } else {
      qm[u] = load_quad<FULL>(m + i, left);
      qv[u] = load_quad<FULL>(v + i, left);
    }
  }
  if constexpr (EIGHT) __builtin_memcpy(old, e, 2 * QUADS);  // (every quad here has elements)
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int64_t i = at + u * 256 + lane * 4, left = t.n - i;
    float fm[4], fv[4], np[4];
    uint32_t bits[4] = {0, 0, 0, 0};
    // the element's place and the key, with mix32's first step: for four neighbours from i, a multiple of 4, they
    // differ by an exclusive or with 0..3 alone
    const uint32_t first = static_cast<uint32_t>(i) ^ static_cast<uint32_t>(i >> 32) * 0x9E3779B9u ^ t.key;
    const uint32_t mixed = first ^ first >> 16;
    bool odd = false;
    if constexpr (EIGHT) {
      const int em = __builtin_amdgcn_readfirstlane(old[2 * u]), ev = __builtin_amdgcn_readfirstlane(old[2 * u + 1]);
      if (em <= kFastM && ev <= kFastV && __all(ordinary_codes(cm[u], cv[u]))) {
        const float sm = pow2(em + 120), sv = pow2(ev + 96);
        fm[0] = decode_m_of<0>(cm[u], sm), fm[1] = decode_m_of<1>(cm[u], sm);
        fm[2] = decode_m_of<2>(cm[u], sm), fm[3] = decode_m_of<3>(cm[u], sm);
        fv[0] = decode_v_of<0>(cv[u], sv), fv[1] = decode_v_of<1>(cv[u], sv);
        fv[2] = decode_v_of<2>(cv[u], sv), fv[3] = decode_v_of<3>(cv[u], sv);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) fm[j] = decode_m(cm[u] >> 8 * j & 255u, em), fv[j] = decode_v(cv[u] >> 8 * j & 255u, ev);
        odd = true;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) fm[j] = qm[u].v[j], fv[j] = qv[u].v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gr = static_cast<float>(qg[u].v[j]) * clip;
      fm[j] = a.b1 * fm[j] + a.ob1 * gr;
      fv[j] = a.b2 * fv[j] + a.ob2 * (gr * gr);
      const float kept = static_cast<float>(qp[u].v[j]) * t.decay;
      if constexpr (EIGHT) {
        // the hardware's root and reciprocal, 1 ulp each: with 8-bit moments the arithmetic takes as long as the
        // memory, and their correctly rounded forms are a third of it
        const float d = fmaf(__builtin_amdgcn_sqrtf(fv[j]), t.ibc2, a.eps);
        np[j] = fmaf(-t.step_size, fm[j] * __builtin_amdgcn_rcpf(d), kept);
      } else {
        np[j] = kept - t.step_size * (fm[j] / (sqrtf(fv[j]) * t.ibc2 + a.eps));
      }
      if constexpr (EIGHT || sizeof(P) == 2) bits[j] = mix32_rest(mixed ^ static_cast<uint32_t>(j));
    }
    if constexpr (!EIGHT) {
      store_quad<FULL>(p + i, new_params<P, true>(np, bits), left);
#pragma unroll
      for (int j = 0; j < 4; ++j) qm[u].v[j] = fm[j], qv[u].v[j] = fv[j];
      store_quad<FULL>(m + i, qm[u], left);
      store_quad<FULL>(v + i, qv[u], left);
    } else {
      // (elements behind the end are 0; v is never negative.  NaN is none of tm's: where a gradient made m infinite or NaN,
      // v is so too, and where the state had it, `odd` says so)
      uint32_t tm = __float_as_uint(fmaxf(fmaxf(fabsf(fm[0]), fabsf(fm[1])), fmaxf(fabsf(fm[2]), fabsf(fm[3]))));
      uint32_t tv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) tv = __float_as_uint(fv[j]) > tv ? __float_as_uint(fv[j]) : tv;
      wave_umax(tm, tv);
      int ne = block_exponent(tm, 8, -117, 120), nv = block_exponent(tv, 0, -93, 127);
      if (!odd && tv < 0x7F800000u && ne <= kFastM && nv <= kFastV) {
        store_quad<FULL>(p + i, new_params<P, false>(np, bits), left);
        const float sm = pow2(-ne - 120), sv = pow2(-nv - 96);
        uint32_t tops[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) tops[j] = encode_m_top(fm[j], sm, bits[j]);
        cm[u] = top_bytes(tops[0], tops[1], tops[2], tops[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) tops[j] = encode_v_top(fv[j], sv, bits[j]);
        cv[u] = top_bytes(tops[0], tops[1], tops[2], tops[3]);
      } else {  // the exponents are the finite values'
        store_quad<FULL>(p + i, new_params<P, true>(np, bits), left);
        tm = tv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t bm = is_finite(fm[j]) ? __float_as_uint(fabsf(fm[j])) : 0u;
          const uint32_t bv = is_finite(fv[j]) ? __float_as_uint(fv[j]) : 0u;
          tm = bm > tm ? bm : tm;
          tv = bv > tv ? bv : tv;
        }
        wave_umax(tm, tv);
        ne = block_exponent(tm, 8, -117, 120);
        nv = block_exponent(tv, 0, -93, 127);
        cm[u] = cv[u] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          cm[u] |= encode_m(fm[j], ne, bits[j]) << 8 * j;
          cv[u] |= encode_v(fv[j], nv, bits[j]) << 8 * j;
        }
      }
      now[2 * u] = static_cast<int8_t>(ne);
      now[2 * u + 1] = static_cast<int8_t>(nv);
      store_codes<FULL>(m8 + i, cm[u], left);
      store_codes<FULL>(v8 + i, cv[u], left);
    }
  }
  if constexpr (EIGHT)
    if (lane == 0) __builtin_memcpy(e, now, 2 * QUADS);
}

template <typename P, typename G, bool EIGHT, int QUADS>
IADMM_DEV void adam_chunk(const AdamCommon& a, const AdamTensor& t, float clip) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t at = (static_cast<int64_t>(blockIdx.x - t.first) * 4 + wave) * (QUADS * 256);
  if (at + QUADS * 256 <= t.n) {
    adam_wave<P, G, EIGHT, QUADS, true>(a, t, clip, at);
  } else {
    for (int u = 0; u < QUADS; ++u)
      if (at + u * 256 < t.n) adam_wave<P, G, EIGHT, 1, false>(a, t, clip, at + u * 256);
  }
}

template <bool EIGHT, int QUADS> IADMM_DEV void adam_any(const AdamCommon& a, const AdamTensor& t) {
  float clip = 1.0f;
  if (a.norm) {
    const float c = a.max_norm / (*a.norm + 1e-6f);
    clip = c > 1.0f ? 1.0f : c;  // (a norm that is NaN reaches every parameter)
  }
  switch (t.flags) {
    case 0: adam_chunk<float, float, EIGHT, QUADS>(a, t, clip); break;
    case kHalfG: adam_chunk<float, __bf16, EIGHT, QUADS>(a, t, clip); break;
    case kHalfP: adam_chunk<__bf16, float, EIGHT, QUADS>(a, t, clip); break;
    default: adam_chunk<__bf16, __bf16, EIGHT, QUADS>(a, t, clip); break;
  }
}
template <bool EIGHT, int QUADS> __global__ void __launch_bounds__(256) adam_kernel(const AdamLaunch a) {
  adam_any<EIGHT, QUADS>(a.c, a.t[find_tensor(a.t, a.c.count, blockIdx.x)]);
}
template <bool EIGHT, int QUADS> __global__ void __launch_bounds__(256) adam_table_kernel(const AdamTable a) {
  const AdamTensor* from = a.t + find_tensor(a.t, a.c.count, blockIdx.x);
  int w[sizeof(AdamTensor) / 4];  // the same for the workgroup: scalars
  __builtin_memcpy(w, from, sizeof(w));
#pragma unroll
  for (unsigned i = 0; i < sizeof(w) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
  AdamTensor t;
  __builtin_memcpy(&t, w, sizeof(w));
  adam_any<EIGHT, QUADS>(a.c, t);
}

// Writes tensors into the table; where the steps are counted on the device (a captured step has to count by itself),
// counts, and works out what depends on the count.
struct AdamPlace {
  AdamTensor t[kPlace];
  AdamTensor* to;
  int64_t* steps;
  const float* lr;
  double lr_host, b1, b2, decay;
  uint64_t seed;
  int count;
};
static_assert(sizeof(AdamPlace) <= 4096 && kPlace <= 64 && kPlace >= kPer, "a launch's arguments, one wave");
__global__ void adam_place_kernel(const AdamPlace a) {
  const int k = threadIdx.x;
  if (k >= a.count) return;
  AdamTensor d = a.t[k];
  if (a.steps) {
    const int slot = static_cast<int>(d.key);
    const int64_t step = a.steps[slot] + 1;
    a.steps[slot] = step;
    const double lr = a.lr ? static_cast<double>(*a.lr) : a.lr_host, t = static_cast<double>(step);
    d.step_size = static_cast<float>(lr / (1.0 - pow(a.b1, t)));
    d.ibc2 = static_cast<float>(1.0 / sqrt(1.0 - pow(a.b2, t)));
    d.decay = static_cast<float>(1.0 - lr * a.decay);
    d.key = step_key(a.seed, static_cast<uint64_t>(step), slot);
  }
  a.to[k] = d;
}

// The codes' values, 1024 per wave.  HBM: 2 bytes in and 4 (bf16) out an element; 100 M of them 98 us = 6.1 TB/s, partly
// from the last-level cache that the step left them in.
template <typename T, int QUADS, bool FULL> IADMM_DEV void decode_wave(int64_t n, const uint8_t* m8, const uint8_t* v8,
                                                                       const int8_t* e, T* m, T* v, int64_t at) {
  const int lane = threadIdx.x % kWave;
  Quad<uint8_t> qm[QUADS], qv[QUADS];
  int em[QUADS], ev[QUADS];
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int64_t i = at + u * 256 + lane * 4;
    qm[u] = load_quad<FULL>(m8 + i, n - i);
    qv[u] = load_quad<FULL>(v8 + i, n - i);
    em[u] = e[(at + u * 256) / kBlock8 * 2], ev[u] = e[(at + u * 256) / kBlock8 * 2 + 1];
  }
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int64_t i = at + u * 256 + lane * 4;
    Quad<T> om, ov;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      om.v[j] = static_cast<T>(decode_m(qm[u].v[j], em[u]));
      ov.v[j] = static_cast<T>(decode_v(qv[u].v[j], ev[u]));
    }
    store_quad<FULL>(m + i, om, n - i);
    store_quad<FULL>(v + i, ov, n - i);
  }
}
template <typename T> __global__ void __launch_bounds__(256) adam_decode_kernel(int64_t n, const uint8_t* m8, const uint8_t* v8,
                                                                                const int8_t* e, T* m, T* v) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * 1024;
  if (at + 1024 <= n) {
    decode_wave<T, 4, true>(n, m8, v8, e, m, v, at);
  } else {
    for (int u = 0; u < 4; ++u)
      if (at + u * 256 < n) decode_wave<T, 1, false>(n, m8, v8, e, m, v, at + u * 256);
  }
}

// ---------------------------------------------------------------------------------------------- the norm
// sqrt(sum g^2), HBM bound: the workgroups sum every 1024th chunk, so that neighbouring ones are read at the same time (a
// run of neighbours each: 400 M fp32 282 us, now 258), one more the workgroups' sums.
// 100 M bf16 elements in 200 tensors 33 us = 6.1 TB/s, 2.6 M fp32 ones 5 us on the GPU and 8.4 a call (two launches).
struct NormTensor {  // 16 bytes, so that 240 travel in a launch's arguments
  uint64_t g;      // the address, and the highest bit for bf16
  uint32_t first;  // its first chunk: all of them are whole up to the next tensor's, but for the last one's
  uint32_t tail;   // elements
};
constexpr uint64_t kHalf = uint64_t{1} << 63;
struct NormLaunch {
  NormTensor t[kNormPer];
  double* part;
  uint32_t chunks;
  int count;
};

// Squares in 64 bits: they neither overflow (fp32's do from 1.8e19 on) nor lose small tensors beside large ones;
// the conversion and the product cost a third of the time that the bytes take.
template <typename T, int QUADS, bool FULL> IADMM_DEV double square_sum_of(const T* g, int n) {
  Quad<T> q[QUADS];
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int i = u * 1024 + static_cast<int>(threadIdx.x) * 4;
    q[u] = load_quad<FULL>(g + i, n - i);
  }
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < QUADS; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double d = static_cast<double>(static_cast<float>(q[u].v[j]));
      s = fma(d, d, s);
    }
  return s;
}
template <typename T, int QUADS> IADMM_DEV double square_sum(const T* g, int n) {
  return n == QUADS * 1024 ? square_sum_of<T, QUADS, true>(g, n) : square_sum_of<T, QUADS, false>(g, n);
}
// Chunk c of a tensor whose successor's first is `next` (or that of all behind it): its number of elements.
template <int SIZE> IADMM_DEV int chunk_elements(const NormTensor& t, uint32_t next, uint32_t c) {
  return c + 1 == next ? static_cast<int>(t.tail) : SIZE;
}
template <typename T> IADMM_DEV const T* chunk_at(const NormTensor& t, int64_t at) {
  return reinterpret_cast<const T*>(t.g & ~kHalf) + at;
}

// The workgroup's sum, in all its threads: adds whose second operand comes from another lane (a step through LDS waits
// for some hundred cycles), within 16 lanes, the wave, and over its waves' values (4 or 16).
template <int CTRL> IADMM_DEV double add_from(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xF, 0xF, true);
  return v + __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
template <int BLOCK> IADMM_DEV double block_sum_f64(double s, double* red) {
  static_assert(BLOCK == 256 || BLOCK == 1024, "");
  s = add_from<0x140>(add_from<0x141>(add_from<0x4E>(add_from<0xB1>(s))));  // lanes 1, 2 apart, half rows, rows mirrored
  s = add_from<0x143>(add_from<0x142>(s));                                  // row_bcast 15, 31: lane 63 has the wave's
  if (threadIdx.x % kWave == kWave - 1) red[threadIdx.x / kWave] = s;
  __syncthreads();
  s = add_from<0x4E>(add_from<0xB1>(red[threadIdx.x % (BLOCK / kWave)]));
  return BLOCK == 256 ? s : add_from<0x140>(add_from<0x141>(s));
}

// The launch's tensors lie in LDS, as a chunk's is looked for each time: four ballots (from the arguments 40 us for 33).
template <int QUADS> __global__ void __launch_bounds__(256) norm_kernel(const NormLaunch a) {
  __shared__ double red[4];
  __shared__ NormTensor table[256 + 1];
  static_assert(kNormPer <= 256, "one entry per thread");
  const int lane = threadIdx.x % kWave;
  for (int i = threadIdx.x; i < 256 + 1; i += 256) table[i] = i < a.count ? a.t[i] : NormTensor{0, a.chunks, 0};
  __syncthreads();
  double s = 0.0;
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    int k = -1;
#pragma unroll
    for (int j = 0; j < 256; j += kWave) k += __popcll(__ballot(table[j + lane].first <= c));
    const NormTensor t = table[k];
    const int64_t at = static_cast<int64_t>(c - t.first) * (QUADS * 1024);
    const int n = __builtin_amdgcn_readfirstlane(chunk_elements<QUADS * 1024>(t, table[k + 1].first, c));
    s += t.g & kHalf ? square_sum<__bf16, QUADS>(chunk_at<__bf16>(t, at), n)
                     : square_sum<float, QUADS>(chunk_at<float>(t, at), n);
  }
  s = block_sum_f64<256>(s, red);
  if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(1024) norm_end_kernel(const double* part, int count, float* norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 4096) {  // four loads in flight
    double v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = part[i + j * 1024 < count ? i + j * 1024 : i];
#pragma unroll
    for (int j = 0; j < 4; ++j) s += i + j * 1024 < count ? v[j] : 0.0;
  }
  s = block_sum_f64<1024>(s, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
}

// Workgroups take 2048 elements at a time up to this many in all, 8192 above: 168 000 of them 7.1 us against 7.7 (with the
// last sum's launch; both since 1 us less), 2.6 M 8.2 against 8.0.  Between these the two are within each other's spread
// (GPU time in a graph: 100 000 4.3 against 4.9, 524 000 4.5 against 4.6, 1.2 M 4.8 against 4.9, 2.6 M 5.3 against 5.1).
constexpr int64_t kNormSmall = int64_t{1} << 19;
// Chunks of 1024 that one workgroup sums alone (16 waves, two rounds): 16 tensors of 2000 elements 5.8 us a call, 8.3 with
// two launches; with four rounds the GPU takes longer than for the two.
constexpr int64_t kNormFew = 32;
static void place_chunks(NormLaunch& a, const int64_t* n, int64_t size) {  // (none is empty)
  uint64_t chunks = 0;
  for (int k = 0; k < a.count; ++k) {
    const int64_t whole = (n[k] - 1) / size;
    a.t[k].first = static_cast<uint32_t>(chunks);
    a.t[k].tail = static_cast<uint32_t>(n[k] - whole * size);
    chunks += static_cast<uint64_t>(whole) + 1;
  }
  a.chunks = static_cast<uint32_t>(chunks);
}
template <int QUADS> static int launch_norm(NormLaunch& a, const int64_t* n, hipStream_t st) {  // gives its workgroups
  place_chunks(a, n, QUADS * 1024);
  const uint32_t chunks = a.chunks;
  const int blocks = chunks < kNormBlocks ? static_cast<int>(chunks) : kNormBlocks;
  hipLaunchKernelGGL(norm_kernel<QUADS>, dim3(blocks), dim3(256), 0, st, a);
  return blocks;
}

// Few elements: one workgroup and one launch, 1024 elements to a wave at a time.
struct NormFew {
  NormLaunch a;
  float* norm;
};
static_assert(sizeof(NormFew) <= 4096, "a launch's arguments");
__global__ void __launch_bounds__(1024) norm_few_kernel(const NormFew f) {
  __shared__ double red[16];
  const int lane = threadIdx.x % kWave;
  double s = 0.0;
  for (uint32_t c = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); c < f.a.chunks; c += 16) {
    const int k = find_tensor(f.a.t, f.a.count, c);
    const NormTensor& t = f.a.t[k];
    const int n = chunk_elements<1024>(t, k + 1 < f.a.count ? f.a.t[k + 1].first : f.a.chunks, c);
    const int64_t at = static_cast<int64_t>(c - t.first) * 1024;
    for (int u = 0; u < 4; ++u) {
      const int i = u * 256 + lane * 4;
      if (t.g & kHalf) {
        const Quad<__bf16> q = load_quad(chunk_at<__bf16>(t, at) + i, n - i);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma(static_cast<float>(q.v[j]), static_cast<double>(static_cast<float>(q.v[j])), s);
      } else {
        const Quad<float> q = load_quad(chunk_at<float>(t, at) + i, n - i);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma(static_cast<double>(q.v[j]), static_cast<double>(q.v[j]), s);
      }
    }
  }
  s = block_sum_f64<1024>(s, red);
  if (threadIdx.x == 0) *f.norm = static_cast<float>(sqrt(s));
}

// Workgroups of 1024 elements up to this many in all, of 4096 above: 168 000 of them 7.9 us against 8.9 (with the
// counting launch), 2.6 M 17.9 against 16.6.  Between (GPU time in a graph, fp32 with 32 bits; bf16 with 8 in brackets):
// 524 000 6.9 (6.6) against 7.8 (7.8), 1.2 M 9.1 (8.0) against 11.2 (11.1), 2.6 M 15.3 (10.3) against 14.7 (11.7).
constexpr int64_t kAdamSmall = int64_t{1} << 19;
template <bool EIGHT, int QUADS> static void launch_adam(const AdamLaunch& a, const AdamTensor* table, unsigned blocks,
                                                       hipStream_t st) {
  if (table)
    hipLaunchKernelGGL((adam_table_kernel<EIGHT, QUADS>), dim3(blocks), dim3(256), 0, st, AdamTable{table, a.c});
  else
    hipLaunchKernelGGL((adam_kernel<EIGHT, QUADS>), dim3(blocks), dim3(256), 0, st, a);
}

}  // namespace iadmm

using namespace iadmm;

extern "C" int64_t iadmm_grad_norm_ws_bytes(int64_t count) {
  if (count <= 0) return 0;
  return (count + kNormPer - 1) / kNormPer * kNormBlocks * static_cast<int64_t>(sizeof(double));
}

extern "C" int iadmm_grad_norm(int64_t count, const iadmm_grad_tensor* grads, float* norm, void* ws, int64_t ws_bytes,
                               void* stream) {
  if (count < 0 || !norm || (count > 0 && (!grads || !ws)) || ws_bytes < iadmm_grad_norm_ws_bytes(count)) return IADMM_E_ARG;
  if (!aligned16(ws)) return IADMM_E_ALIGN;
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (grads[i].n < 0 || (grads[i].n > 0 && !grads[i].g) || (grads[i].dtype != IADMM_F32 && grads[i].dtype != IADMM_BF16))
      return IADMM_E_ARG;
    if (grads[i].n > (int64_t{1} << 40) || (all += grads[i].n) > (int64_t{1} << 40)) return IADMM_E_SIZE;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(ws);
  int parts = 0;
  NormFew f;
  NormLaunch& a = f.a;
  int64_t n[kNormPer], total = 0, few = 0, filled = 0;
  for (int64_t i = 0; i < count; ++i) few += (grads[i].n + 1023) / 1024, filled += grads[i].n > 0;
  const bool alone = filled <= kNormPer && few <= kNormFew;
  a.count = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (grads[i].n > 0) {
      n[a.count] = grads[i].n;
      a.t[a.count++] = NormTensor{reinterpret_cast<uint64_t>(grads[i].g) | (grads[i].dtype == IADMM_BF16 ? kHalf : 0), 0u, 0u};
      total += grads[i].n;
    }
    if (!alone && a.count > 0 && (a.count == kNormPer || i == count - 1)) {
      a.part = part + parts;
      const int blocks = total <= kNormSmall ? launch_norm<2>(a, n, st) : launch_norm<8>(a, n, st);
      IADMM_CHECK_LAUNCH();
      parts += blocks;
      a.count = 0;
      total = 0;
    }
  }
  if (alone) {
    place_chunks(a, n, 1024);
    a.part = nullptr, f.norm = norm;
    hipLaunchKernelGGL(norm_few_kernel, dim3(1), dim3(1024), 0, st, f);
    IADMM_CHECK_LAUNCH();
    return IADMM_OK;
  }
  hipLaunchKernelGGL(norm_end_kernel, dim3(1), dim3(1024), 0, st, part, parts, norm);
  IADMM_CHECK_LAUNCH();
  return IADMM_OK;
}

extern "C" int64_t iadmm_adamw_ws_bytes(int64_t count) {
  return count <= 0 ? 0 : count * static_cast<int64_t>(sizeof(AdamTensor));
}

extern "C" int iadmm_adamw_step(int64_t count, const iadmm_adamw_tensor* tensors, int state_bits, double lr, const float* lr_dev,
                                double beta1, double beta2, double eps, double weight_decay, const float* norm,
                                double max_norm, uint64_t seed, int64_t* steps_dev, void* ws, int64_t ws_bytes,
                                void* stream) {
  const bool eight = state_bits == 8, table = steps_dev || count > kPer;
  if (count < 0 || (count > 0 && !tensors) || (!eight && state_bits != 32)) return IADMM_E_ARG;
  if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) ||
      !(weight_decay >= 0.0) || (norm && !(max_norm > 0.0)) || (lr_dev && !steps_dev))
    return IADMM_E_ARG;
  if (table && (!ws || ws_bytes < iadmm_adamw_ws_bytes(count))) return IADMM_E_ARG;
  if (table && !aligned16(ws)) return IADMM_E_ALIGN;
  if (count > 0x7FFFFFFF) return IADMM_E_SIZE;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    const iadmm_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.slot < 0 || (t.n > 0 && (!t.p || !t.g || !t.m || !t.v || (eight && !t.e))) ||
        (!steps_dev && t.step < 1) || (t.dtype != IADMM_F32 && t.dtype != IADMM_BF16) ||
        (t.gdtype != IADMM_F32 && t.gdtype != IADMM_BF16))
      return IADMM_E_ARG;
    if (t.n > (int64_t{1} << 36) || (total += t.n) > (int64_t{1} << 36)) return IADMM_E_SIZE;
  }
  const int64_t each = total <= kAdamSmall ? 1024 : 4096;
  uint64_t blocks = 0;
  for (int64_t i = 0; i < count; ++i) blocks += (static_cast<uint64_t>(tensors[i].n) + each - 1) / each;
  if (blocks > 0xFFFFFFu) return IADMM_E_SIZE;  // 2^32 threads
  hipStream_t st = static_cast<hipStream_t>(stream);
  AdamPlace a{};
  a.steps = steps_dev, a.lr = lr_dev, a.lr_host = lr, a.b1 = beta1, a.b2 = beta2, a.decay = weight_decay, a.seed = seed;
  a.to = static_cast<AdamTensor*>(ws);
  int64_t step = 0;
  float step_size = 0.0f, ibc2 = 0.0f;
  uint32_t first = 0;
  for (int64_t i = 0; i < count; ++i) {
    const iadmm_adamw_tensor& t = tensors[i];
    if (!steps_dev && t.step != step) {
      step = t.step;
      step_size = static_cast<float>(lr / (1.0 - pow(beta1, static_cast<double>(step))));
      ibc2 = static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, static_cast<double>(step))));
    }
    AdamTensor& d = a.t[a.count++];
    d.p = t.p, d.g = t.g, d.m = t.m, d.v = t.v, d.e = t.e, d.n = t.n, d.first = first;
    d.flags = (t.dtype == IADMM_BF16 ? kHalfP : 0) | (t.gdtype == IADMM_BF16 ? kHalfG : 0);
    d.step_size = step_size, d.ibc2 = ibc2, d.decay = static_cast<float>(1.0 - lr * weight_decay);
    d.key = steps_dev ? static_cast<uint32_t>(t.slot) : step_key(seed, static_cast<uint64_t>(t.step), t.slot);
    first += static_cast<uint32_t>((t.n + each - 1) / each);
    if (table && (a.count == kPlace || i == count - 1)) {
      hipLaunchKernelGGL(adam_place_kernel, dim3(1), dim3(64), 0, st, a);
      IADMM_CHECK_LAUNCH();
      a.to += a.count;
      a.count = 0;
    }
  }
  if (blocks == 0) return IADMM_OK;
  AdamLaunch l;
  if (!table) memcpy(l.t, a.t, sizeof(l.t));
  l.c = AdamCommon{norm, static_cast<float>(beta1), static_cast<float>(1.0 - beta1), static_cast<float>(beta2),
                   static_cast<float>(1.0 - beta2), static_cast<float>(eps), static_cast<float>(max_norm),
                   static_cast<int>(count)};
  const AdamTensor* in = table ? static_cast<const AdamTensor*>(ws) : nullptr;
  const unsigned n = static_cast<unsigned>(blocks);
  if (eight && each == 1024) launch_adam<true, 1>(l, in, n, st);
  else if (eight) launch_adam<true, 4>(l, in, n, st);
  else if (each == 1024) launch_adam<false, 1>(l, in, n, st);
  else launch_adam<false, 4>(l, in, n, st);
  IADMM_CHECK_LAUNCH();
  return IADMM_OK;
}

extern "C" int iadmm_adamw_decode8(int64_t n, const void* m8, const void* v8, const void* e, int dtype, void* m, void* v,
                                   void* stream) {
  if (n < 0 || (dtype != IADMM_F32 && dtype != IADMM_BF16)) return IADMM_E_ARG;
  if (n == 0) return IADMM_OK;
  if (!m8 || !v8 || !e || !m || !v) return IADMM_E_ARG;
  if ((n + 4095) / 4096 > 0xFFFFFF) return IADMM_E_SIZE;  // 2^32 threads
  const dim3 grid(static_cast<unsigned>((n + 4095) / 4096));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint8_t *cm = static_cast<const uint8_t*>(m8), *cv = static_cast<const uint8_t*>(v8);
  const int8_t* ex = static_cast<const int8_t*>(e);
  if (dtype == IADMM_BF16)
    hipLaunchKernelGGL((adam_decode_kernel<__bf16>), grid, dim3(256), 0, st, n, cm, cv, ex, static_cast<__bf16*>(m),
                       static_cast<__bf16*>(v));
  else
    hipLaunchKernelGGL((adam_decode_kernel<float>), grid, dim3(256), 0, st, n, cm, cv, ex, static_cast<float*>(m),
                       static_cast<float*>(v));
  IADMM_CHECK_LAUNCH();
  return IADMM_OK;
}
