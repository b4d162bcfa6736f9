// gdn_recurrence.cuh -- what the channelwise gated linear recurrence's
// kernels share: element types, the gates, affine maps and their composition,
// the 8-bit group format, and the words that chunks hand to one another.
//
// Recurrence, per channel c (fp32 state, gates as in the GDN kernels):
//   z_t = a_t + dt_bias,  lg_t = -exp(A_log) softplus(z_t),  g_t = exp(lg_t)
//   h_t = g_t h_{t-1} + sigmoid(b_t) x_t,   out_t = h_t
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gdn_common.cuh"
#include "gdn_wait.cuh"

namespace gdn {
namespace rec {

constexpr int kWarps = 8;  // of a decode or checkpoint CTA
constexpr int kThreads = kWarps * 32;
constexpr int kTileCh = 128;  // channels of a decode warp: 4 a lane

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kEmptyWord = ~0ull;  // a word that has not been handed over

// ---- four channels of one token, raw as loaded ------------------------------
template <typename E>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void pairs(uint64_t &p, uint64_t &q) const {
    p = f2_pack(bf16_lo(v.x), bf16_hi(v.x));
    q = f2_pack(bf16_lo(v.y), bf16_hi(v.y));
  }
};
template <>
struct Raw<__half> {
  uint2 v;
  __device__ __forceinline__ void pairs(uint64_t &p, uint64_t &q) const {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
    p = f2_pack(a.x, a.y);
    q = f2_pack(b.x, b.y);
  }
};
template <>
struct Raw<float> {
  float4 v;
  __device__ __forceinline__ void pairs(uint64_t &p, uint64_t &q) const {
    p = f2_pack(v.x, v.y);
    q = f2_pack(v.z, v.w);
  }
};

// Channels of a lane: with kVec 4 neighbours (one 8- or 16-byte access), else
// lane, lane + 32, lane + 64, lane + 96 of the tile, so that single-element
// accesses of a warp still fall next to one another.
// left: channels of the tile that exist (D - first channel; may exceed 128).
// kReadOnly: nothing writes to the data while the kernel runs.
template <typename E, bool kVec, bool kReadOnly = true>
__device__ __forceinline__ Raw<E> load4(const E *p, int lane, int left) {
  Raw<E> r;
  if constexpr (kVec) {
    r.v = {};
    if (4 * lane < left) {
      const auto *q = reinterpret_cast<const decltype(r.v) *>(p) + lane;
      r.v = kReadOnly ? __ldg(q) : *q;
    }
  } else {
    E e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = lane + 32 * j < left ? p[lane + 32 * j] : E(0.f);
    memcpy(&r.v, e, sizeof(r.v));
  }
  return r;
}

template <typename E, bool kVec>
__device__ __forceinline__ void store4(E *p, int lane, int left, uint64_t a, uint64_t b) {
  const float f[4] = {f2_lo(a), f2_hi(a), f2_lo(b), f2_hi(b)};
  if constexpr (sizeof(E) == 4) {
    if constexpr (kVec) {
      if (4 * lane < left) reinterpret_cast<float4 *>(p)[lane] = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < left) p[lane + 32 * j] = f[j];
    }
  } else {
    // the one rounding of a result: to nearest even
    uint2 u;
    if constexpr (std::is_same<E, __half>::value) {
      const __half2 lo = __floats2half2_rn(f[0], f[1]), hi = __floats2half2_rn(f[2], f[3]);
      u = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    } else {
      u = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
    }
    if constexpr (kVec) {
      if (4 * lane < left) reinterpret_cast<uint2 *>(p)[lane] = u;
    } else {
      E e[4];
      memcpy(e, &u, sizeof(u));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < left) p[lane + 32 * j] = e[j];
    }
  }
}

// fp32 rows in channel order (states, A_log, dt_bias).
template <bool kVec>
__device__ __forceinline__ float4 load_f32(const float *p, int lane, int left) {
  if constexpr (kVec) {
    return 4 * lane < left ? reinterpret_cast<const float4 *>(p)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = lane + 32 * j < left ? p[lane + 32 * j] : 0.f;
    return make_float4(f[0], f[1], f[2], f[3]);
  }
}
template <bool kVec>
__device__ __forceinline__ void store_f32(float *p, int lane, int left, float4 v) {
  if constexpr (kVec) {
    if (4 * lane < left) reinterpret_cast<float4 *>(p)[lane] = v;
  } else {
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 32 * j < left) p[lane + 32 * j] = f[j];
  }
}

// ---- arithmetic on channel pairs ---------------------------------------------
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_dup(float x) { return f2_pack(x, x); }

// 2^x (relative error about 2 ulp) and 1 / x (1 ulp), one instruction each.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The gates are evaluated in base 2: with w = (a + dt_bias) log2(e) and
// e = 2^-|w|, softplus(z) log2(e) = max(w, 0) + log2(1 + e), so that
// g = 2^(-exp(A_log) softplus(z) log2(e)).
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) { return f2_pack(ex2(f2_lo(x)), ex2(f2_hi(x))); }
__device__ __forceinline__ uint64_t ex2_neg_abs(uint64_t x) {
  return f2_pack(ex2(-fabsf(f2_lo(x))), ex2(-fabsf(f2_hi(x))));
}
// log2(1 + e) for e in [0, 1], added to max(w, 0): e Q(e), with the polynomial Q
// of degree 8 of least relative error for log1p(e) / e (weighted least squares
// iterated to the minimax, 3e-8; 1.8e-7 with its coefficients and steps in
// fp32), times log2(e).  A logarithm of 1 + e would lose the relative error
// where e is small, which is where a gate remembers longest.  NaN stays NaN
// (through e).
__device__ __forceinline__ uint64_t softplus2(uint64_t w, uint64_t e) {
  uint64_t q = f2_dup(0.00754917785525322f);
  q = f2_fma(q, e, f2_dup(-0.042567044496536255f));
  q = f2_fma(q, e, f2_dup(0.11285616457462311f));
  q = f2_fma(q, e, f2_dup(-0.19711895287036896f));
  q = f2_fma(q, e, f2_dup(0.27564141154289246f));
  q = f2_fma(q, e, f2_dup(-0.35840848088264465f));
  q = f2_fma(q, e, f2_dup(0.480692982673645f));
  q = f2_fma(q, e, f2_dup(-0.7213402390480042f));
  q = f2_fma(q, e, f2_dup(1.442694902420044f));
  return f2_fma(q, e, f2_pack(fmaxf(f2_lo(w), 0.f), fmaxf(f2_hi(w), 0.f)));
}

// 1 / (1 + exp(-b)): exp(-b) may be infinite, its reciprocal is then 0.
__device__ __forceinline__ uint64_t sigmoid_pair(uint64_t b) {
  const uint64_t d = f2_add(ex2_pair(f2_mul(b, f2_dup(-kLog2e))), f2_dup(1.f));
  return f2_pack(rcp(f2_lo(d)), rcp(f2_hi(d)));
}

// A channel's constants: dt = dt_bias log2(e), c = -exp(A_log).
__device__ __forceinline__ float param_dt(float dt_bias) { return dt_bias * kLog2e; }
__device__ __forceinline__ float param_c(float A_log) { return -expf(A_log); }
struct Params {
  uint64_t dt[2], c[2];
};
template <bool kVec>
__device__ __forceinline__ Params load_params(const float *A_log, const float *dt_bias, int lane, int left) {
  const float4 a = load_f32<kVec>(A_log, lane, left), d = load_f32<kVec>(dt_bias, lane, left);
  Params p;
  p.dt[0] = f2_pack(param_dt(d.x), param_dt(d.y));
  p.dt[1] = f2_pack(param_dt(d.z), param_dt(d.w));
  p.c[0] = f2_pack(param_c(a.x), param_c(a.y));
  p.c[1] = f2_pack(param_c(a.z), param_c(a.w));
  return p;
}

// A gate 2^(c s), with s = softplus(z) log2(e).  Near 1 the hardware's exponential
// is low by 0.32 2^-24 on average (measured over [-1/4, 0]), which a gate that
// remembers n tokens adds up n times; kLift / log2(e) = 0.31 2^-24 in the
// argument, with the product's own rounding, takes it out (what is left of the
// mean: at most 0.08 2^-24 down to 1 - g = 1/350, 0.2 2^-24 beyond) at no cost.
// It leaves 2^0 at 1.  Over 65536 tokens x 1024 channels in fp32 the outputs are
// then off by 3.1e-7 in norm instead of 1.5e-6.  A cubic for 1 - g from x = -1/8
// on, which has no such mean, gave 1.8e-7 and took 10 % more time.
constexpr float kLift = 2.67e-8f;
__device__ __forceinline__ uint64_t gate_of(uint64_t c, uint64_t s) {
  return ex2_pair(f2_fma(c, s, f2_dup(kLift)));
}

// g and u = sigmoid(b) x of one channel pair.
__device__ __forceinline__ void gate_pair(uint64_t x, uint64_t a, uint64_t b, uint64_t dt, uint64_t c,
                                          uint64_t &g, uint64_t &u) {
  const uint64_t w = f2_fma(a, f2_dup(kLog2e), dt);
  g = gate_of(c, softplus2(w, ex2_neg_abs(w)));
  u = f2_mul(sigmoid_pair(b), x);
}

// ---- affine maps h -> A h + H, per channel -----------------------------------
// A is never negative as a product of gates; a set sign bit marks a map that
// restarts (h -> H whatever h is, even where h is infinite or NaN).
__device__ __forceinline__ bool restarts(float A) { return __float_as_uint(A) >> 31; }
__device__ __forceinline__ float apply(float A, float H, float h) { return restarts(A) ? H : fmaf(A, h, H); }

// ---- words handed from chunk to chunk -----------------------------------------
// A word is a map (A low, H high) or a state (0 low, h high) in 64 bits that is
// stored and loaded whole, so a word that is not kEmptyWord is complete: no
// flag and no fence goes with it.  Arithmetic never makes that bit pattern (a
// NaN that an operation returns is 0x7fffffff); keep_apart covers the case that
// a NaN was only passed through.
__device__ __forceinline__ uint64_t keep_apart(uint64_t w) { return w == kEmptyWord ? w >> 1 : w; }

// ---- 8-bit groups ---------------------------------------------------------------
// 128 neighbouring values of a row share one power of two 2^(E - 127), E in one
// byte; a value is the int8 q = rint(v / 2^(E-127)), |q| <= 127.  E is the
// smallest exponent with max|v| <= 127 2^(E-127), at least 1 and at most
// `cap`, the largest for which 127 2^(E-127) is finite in the type (values
// beyond then become +-127).  A power of two makes v / 2^(E-127) exact, so
// rounding to int8 (half a unit, to even) is the only error, and int8 times a
// power of two is exact in bf16 and fp32.  A group with a NaN or an infinity
// gets E = 255 and reads back as NaN.
constexpr int kGroupValues = 128;
constexpr uint32_t kExpNonFinite = 255;
template <typename E>
__device__ __forceinline__ constexpr uint32_t exp_cap() {
  return std::is_same<E, __half>::value ? 9u + 127u : 121u + 127u;
}
// from the largest |v| of the group as fp32 bits (order of bits = order of values)
__device__ __forceinline__ uint32_t group_exponent(uint32_t amax_bits, uint32_t cap) {
  if (amax_bits >= 0x7f800000u) return kExpNonFinite;
  // amax = m 2^k, m in [1, 2): k - 6 if m <= 127/64, else k - 5
  const int e = static_cast<int>((amax_bits + 0x1ffffu) >> 23) - 6;
  return min(static_cast<uint32_t>(max(e, 1)), cap);
}
__device__ __forceinline__ float group_scale(uint32_t E) { return __uint_as_float(E << 23); }
__device__ __forceinline__ float group_inverse(uint32_t E) {  // 2^(127 - E); 0 for a non-finite group
  return E == kExpNonFinite ? 0.f : __uint_as_float((254u - E) << 23);
}
// q of two (four) values as bytes.  v inv is exact and below 2^7 in magnitude
// (2^7.01 in a capped group), so adding 1.5 2^23 rounds it to an integer, half
// to even, in the sum's low byte.
__device__ __forceinline__ uint32_t quantise2(uint64_t a, float inv) {  // E below the cap
  a = f2_fma(a, f2_dup(inv), f2_dup(12582912.f));
  return __byte_perm(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), 0x0040);
}
__device__ __forceinline__ uint32_t quantise2(uint64_t a, uint32_t E, uint32_t cap) {
  if (E == kExpNonFinite) return 0u;  // 0 times infinity reads back as NaN
  const uint64_t magic = f2_dup(12582912.f);
  if (E == cap) {
    const float lim = 127.f, inv = group_inverse(E);
    a = f2_add(f2_pack(fminf(fmaxf(f2_lo(a) * inv, -lim), lim), fminf(fmaxf(f2_hi(a) * inv, -lim), lim)), magic);
  } else {
    a = f2_fma(a, f2_dup(group_inverse(E)), magic);
  }
  return __byte_perm(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), 0x0040);
}
__device__ __forceinline__ uint32_t quantise4(uint64_t a, uint64_t b, uint32_t E, uint32_t cap) {
  return __byte_perm(quantise2(a, E, cap), quantise2(b, E, cap), 0x5410);
}
// The values that four bytes stand for.  A byte q + 128 put into the mantissa
// of 2^23 is the fp32 number 2^23 + 128 + q: a byte permute and an addition
// instead of a conversion, which would share the slow pipe with the gates'
// exponentials.
__device__ __forceinline__ uint64_t dequantise2(uint32_t q, uint32_t E) {
  const uint32_t s = q ^ 0x8080u, m = 0x4b000000u;
  const uint64_t v = f2_pack(__uint_as_float(__byte_perm(s, m, 0x7650)), __uint_as_float(__byte_perm(s, m, 0x7651)));
  return f2_mul(f2_add(v, f2_dup(-8388736.f)), f2_dup(group_scale(E)));
}
__device__ __forceinline__ void dequantise4(uint32_t q, uint32_t E, uint64_t &a, uint64_t &b) {
  const uint64_t scale = f2_dup(group_scale(E)), off = f2_dup(-8388736.f);
  const uint32_t s = q ^ 0x80808080u, m = 0x4b000000u;
  const uint64_t lo = f2_pack(__uint_as_float(__byte_perm(s, m, 0x7650)), __uint_as_float(__byte_perm(s, m, 0x7651)));
  const uint64_t hi = f2_pack(__uint_as_float(__byte_perm(s, m, 0x7652)), __uint_as_float(__byte_perm(s, m, 0x7653)));
  a = f2_mul(f2_add(lo, off), scale);
  b = f2_mul(f2_add(hi, off), scale);
}
// largest |v| of four values as bits; NaN and infinities come out >= 0x7f800000
__device__ __forceinline__ uint32_t abs_max_bits(uint64_t a, uint64_t b) {
  const uint32_t m = 0x7fffffffu;
  return max(max(static_cast<uint32_t>(a) & m, static_cast<uint32_t>(a >> 32) & m),
             max(static_cast<uint32_t>(b) & m, static_cast<uint32_t>(b >> 32) & m));
}

}  // namespace rec
}  // namespace gdn
