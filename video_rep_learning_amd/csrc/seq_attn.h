// What the attention kernels over packed sequences and over a paged cache share (seq_attn.hip, seq_attn_bwd.hip, paged_attn.hip).
//
// Every kernel here OWNS 32 rows per wave (queries, or keys in the dK / dV kernel) and STREAMS blocks of the other side's rows through
// LDS.  Products run on the 32x32 matrix instruction with the streamed row on the accumulator's row and the owned row on its column:
//   lane (r = lane & 31, h = lane >> 5) holds A[row r][k = 8h + j], B[k = 8h + j][col r], D[row 8 (e >> 2) + 4h + (e & 3)][col r]
// so a softmax row lives in one lane and its partner lane ^ 32, and registers 8s .. 8s + 7 of an accumulator tile, rounded to the operand
// format, ARE the B operand of the next product over the 16 streamed rows  16s + {4h .. 4h + 3, 8 + 4h .. 8 + 4h + 3}:  nothing crosses
// lanes or LDS between two products.  The matching A operand is the streamed matrix transposed, fetched in that row order.
// The order of k inside a product is free as long as A and B agree, so fp32 runs the same code on v_mfma_f32_32x32x2_f32: "one
// fragment" is then 8 floats per lane and eight instructions.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <type_traits>
#include "../../include/mvf_hip.h"
#include "common.h"

namespace seq_attn {

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(8))) float f32x8_t;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_INF = -__builtin_huge_valf();

__device__ __forceinline__ float other_half(float x) {   // value of lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------------------------------------- operand formats
template <bool F16>
struct Op16 {
  typedef uint16_t E;
  typedef bf16x8_t Frag;
  static constexpr int SZ = 2;
  static __device__ __forceinline__ f32x16_t mma(const Frag& a, const Frag& b, const f32x16_t& c) {
    if constexpr (F16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_native_t, a), __builtin_bit_cast(f16x8_native_t, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // registers 8 s .. 8 s + 7 as a B operand: one rounding of the probability (or of dS) to the operands' own format, the least that
  // the 16-bit matrix instruction takes
  static __device__ __forceinline__ Frag pack(const f32x16_t& x, int s) {
    union { Frag v; uint32_t u[4]; } f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.u[j] = pack16x2<F16>(x[8 * s + 2 * j], x[8 * s + 2 * j + 1]);
    return f.v;
  }
  static constexpr uint32_t EXP = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
  static __device__ __forceinline__ bool any_nonfinite(const Frag& a) {
    union { Frag v; uint32_t u[4]; } f;
    f.v = a;
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= (f.u[j] & EXP) + ONE;     // an all-ones exponent carries into the sign bit
    return (bad & 0x80008000u) != 0;
  }
  static __device__ __forceinline__ float get(const Frag& a, int j) {
    const uint16_t x = (uint16_t)a[j];
    return F16 ? f16_to_f32(x) : bf16_to_f32(x);
  }
  static __device__ __forceinline__ void set(Frag& a, int j, float x) { a[j] = (short)(F16 ? f32_to_f16(x) : f32_to_bf16(x)); }
  static __device__ __forceinline__ void store4(E* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack16x2<F16>(a, b), pack16x2<F16>(c, d));
  }
};
template <int DT>
struct Op;
template <>
struct Op<MVF_BF16> : Op16<false> {};
template <>
struct Op<MVF_F16> : Op16<true> {};
template <>
struct Op<MVF_F32> {
  typedef float E;
  typedef f32x8_t Frag;
  static constexpr int SZ = 4;
  static __device__ __forceinline__ f32x16_t mma(const Frag& a, const Frag& b, f32x16_t c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag pack(const f32x16_t& x, int s) {
    Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = x[8 * s + j];
    return f;
  }
  static __device__ __forceinline__ bool any_nonfinite(const Frag& a) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) bad |= !(fabsf(a[j]) < __builtin_huge_valf());
    return bad;
  }
  static __device__ __forceinline__ float get(const Frag& a, int j) { return a[j]; }
  static __device__ __forceinline__ void set(Frag& a, int j, float x) { a[j] = x; }
  static __device__ __forceinline__ void store4(E* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
};

__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// acc + A . B where B holds weights that are exactly 0 in masked places and A the data those weights multiply.  0 * NaN is NaN, so a
// NaN or infinity of a key that a row must not see would reach it through the product.  In tiles with masked places (SAFE) non-finite
// data is therefore taken out of A and put back where its weight is not 0: counts of +inf, -inf and NaN per accumulator element come
// out of one more product (at most 16 of each per step: 1, 64 and 4096 do not meet).  SIGNED: weights of both signs (the gradients'):
// any of them makes the element NaN.
template <class O, bool SAFE, bool SIGNED>
__device__ __forceinline__ f32x16_t mma_weighted(const typename O::Frag& data, const typename O::Frag& w, const f32x16_t& acc) {
  if constexpr (!SAFE) {
    return O::mma(data, w, acc);
  } else {
    if (__builtin_amdgcn_ballot_w64(O::any_nonfinite(data)) == 0) return O::mma(data, w, acc);
    typename O::Frag fin = data, mark, hit;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = O::get(data, j), p = O::get(w, j);
      const bool bad = !(fabsf(x) < __builtin_huge_valf());
      if (bad) O::set(fin, j, 0.f);
      O::set(mark, j, !bad ? 0.f : (SIGNED || x != x) ? 4096.f : x > 0.f ? 1.f : 64.f);
      O::set(hit, j, p == 0.f ? 0.f : 1.f);
    }
    f32x16_t out = O::mma(fin, w, acc);
    const f32x16_t m = O::mma(mark, hit, zero16());
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int n = (int)m[e];
      const bool pos = (n & 63) != 0, neg = ((n >> 6) & 63) != 0;
      if (n != 0) out[e] += (n >= 4096 || (pos && neg)) ? __builtin_nanf("") : pos ? __builtin_huge_valf() : -__builtin_huge_valf();
    }
    return out;
  }
}

// ---------------------------------------------------------------------------------------------- LDS images
// Rows of DP elements in 16-byte chunks, chunk c of row i stored at c ^ swz(i).  Two kinds of reads have to be free of bank conflicts:
//   row fragments: ds_read_b128, 16 lanes at a time, one chunk of 16 different rows;
//   transposed fragments: ds_read_b64_tr_b16, 32 lanes at a time, 4 consecutive rows x 64 bytes (4 aligned chunks).
// A row of C chunks starts at chunk position C * i (mod 16, the 256 bytes of the banks); swz fills the positions that leaves.
template <class O, int DP>
struct Img {
  static constexpr int RB = DP * O::SZ, C = RB / 16;
  static __device__ __forceinline__ int swz(int i) {
    if constexpr (C == 4 || C == 12) return (i >> 2) & 3;
    else if constexpr (C == 8 || C == 24) return (((i >> 1) & 1) << 2) | ((i >> 2) & 3);
    else return ((i & 3) << 2) | ((i >> 2) & 3);
  }
  static __device__ __forceinline__ int off(int i, int c) { return i * RB + ((c ^ swz(i)) << 4); }
  // A operand = 32 rows of the image from row0 on: lane (r, h) <- X[row0 + r][16 ks + 8h .. + 8]
  static __device__ __forceinline__ typename O::Frag rows(const char* img, int row0, int ks, int lane) {
    const int i = row0 + (lane & 31), h = lane >> 5;
    if constexpr (O::SZ == 2) {
      return *reinterpret_cast<const bf16x8_t*>(img + off(i, 2 * ks + h));
    } else {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(img + off(i, 4 * ks + 2 * h));
      const f32x4_t b = *reinterpret_cast<const f32x4_t*>(img + off(i, 4 * ks + 2 * h + 1));
      return (f32x8_t){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // A operand = the image transposed, columns 32 dt .. + 32 on the rows, the 16 image rows from row0 on in the accumulators' order on k
  static __device__ __forceinline__ typename O::Frag cols(const char* img, int row0, int dt, int lane) {
    const int h = lane >> 5;
    if constexpr (O::SZ == 2) {
      const int li = lane & 15, g = (lane >> 4) & 1;
      union { bf16x8_t v; bf16x4_t q[2]; } f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = row0 + 8 * j + 4 * h + (li >> 2), c = 4 * dt + 2 * g + ((li & 3) >> 1);
        f.q[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4_t*)(img + off(i, c) + 8 * (li & 1)));
      }
      return f.v;
    } else {
      f32x8_t f;
      const int d = 32 * dt + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = row0 + (j < 4 ? 4 * h + j : 8 + 4 * h + j - 4);
        f[j] = *reinterpret_cast<const float*>(img + off(i, d >> 2) + 4 * (d & 3));
      }
      return f;
    }
  }
};

// ---------------------------------------------------------------------------------------------- which rows meet
struct Span { int lo, hi; };
// largest b < n with cu[b] <= row < cu[b + 1], as [start, end) cut to [0, T); {0, 0} for a row of no sequence
__device__ __forceinline__ Span sequence_of(const int* __restrict__ cu, int n, int T, int row) {
  int lo = 0, hi = n;                      // the first index with cu > row lies in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid + 1;
    else hi = mid;
  }
  if (lo == 0) return {0, 0};
  const int s = max(cu[lo - 1], 0), e = min(cu[lo], T);
  return row < e ? Span{s, e} : Span{0, 0};
}
// keys that query `row` sees: its sequence's, up to the end of its own group of `frame` tokens (frame = 0: all)
__device__ __forceinline__ Span keys_of(Span s, int frame, int row) {
  if (s.hi == 0 || frame == 0) return s;
  const long lim = ((long)((row - s.lo) / frame) + 1) * frame;
  return {s.lo, (int)min((long)s.hi, s.lo + lim)};
}
// queries that see key `row`
__device__ __forceinline__ Span queries_of(Span s, int frame, int row) {
  if (s.hi == 0 || frame == 0) return s;
  return {s.lo + (row - s.lo) / frame * frame, s.hi};
}

// Spans of a wave's 32 owned rows (both halves of the wave hold the same rows): any = the union, all = what every valid row meets
// (rows of no sequence are left out: nothing of theirs is kept).
struct WaveSpan { Span any, all; };
__device__ __forceinline__ WaveSpan wave_span(Span s) {
  const bool valid = s.hi > s.lo;
  int a = valid ? s.lo : 0x7fffffff, b = valid ? s.hi : 0, c = valid ? s.lo : 0, d = valid ? s.hi : 0x7fffffff;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a = min(a, __shfl_xor(a, o, 64));
    b = max(b, __shfl_xor(b, o, 64));
    c = max(c, __shfl_xor(c, o, 64));
    d = min(d, __shfl_xor(d, o, 64));
  }
  a = __builtin_amdgcn_readfirstlane(a); b = __builtin_amdgcn_readfirstlane(b);
  c = __builtin_amdgcn_readfirstlane(c); d = __builtin_amdgcn_readfirstlane(d);
  return {{b == 0 ? 0 : a, b}, {c, d}};
}

// ---------------------------------------------------------------------------------------------- softmax state of a row
// m: the maximum its exponents are taken against (raw scores), nm = -m * c, l: this lane's share of the row sum.
struct RowMax {
  float m = NEG_INF, nm = 0.f, l = 0.f;
  // mx: the row's maximum over the new scores.  The accumulators are only rescaled when some row's maximum grew by more than `thr`
  // (2^8 in the probability: far from any format's limit); returns true with the factor in alpha then.
  __device__ __forceinline__ bool grow(float mx, float c, float thr, float& alpha) {
    if (__builtin_amdgcn_ballot_w64(mx > m + thr) == 0) return false;
    const float to = fmaxf(m, mx);
    alpha = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((m - to) * c);
    m = to;
    nm = to == NEG_INF ? 0.f : -to * c;
    l *= alpha;
    return true;
  }
};

}  // namespace seq_attn
