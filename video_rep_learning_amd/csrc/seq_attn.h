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
#include <algorithm>
#include <type_traits>
#include "../../include/mvf_hip.h"
#include "common.h"

namespace seq_attn {

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(8))) float f32x8_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
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
  // what pack() rounded away (exact in 32 bits), rounded in turn
  static __device__ __forceinline__ Frag pack_rest(const f32x16_t& x, const Frag& b, int s) {
    union { Frag v; uint32_t u[4]; } f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.u[j] = pack16x2<F16>(x[8 * s + 2 * j] - get(b, 2 * j), x[8 * s + 2 * j + 1] - get(b, 2 * j + 1));
    return f.v;
  }
  // a 16-byte chunk holds a NaN or an infinity: an all-ones exponent carries into the sign bit
  static __device__ __forceinline__ bool nonfinite(const u32x4_t& x) {
    constexpr uint32_t EXP = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
    return ((((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE)) & 0x80008000u) != 0;
  }
  // four elements as fp32
  static __device__ __forceinline__ f32x4_t load4(const char* p) {
    const u32x2_t u = *reinterpret_cast<const u32x2_t*>(p);
    float x[4];
    unpack16x2<F16>(u.x, x[0], x[1]);
    unpack16x2<F16>(u.y, x[2], x[3]);
    return (f32x4_t){x[0], x[1], x[2], x[3]};
  }
  static __device__ __forceinline__ float get(const Frag& a, int j) {
    const uint16_t x = (uint16_t)a[j];
    return F16 ? f16_to_f32(x) : bf16_to_f32(x);
  }
  static __device__ __forceinline__ void store4(E* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack16x2<F16>(a, b), pack16x2<F16>(c, d));
  }
  // registers 4 e .. 4 e + 7 of an accumulator tile as the 8 channels 8 (e + h) .. of the lane's row (h: its half), and what the rounding took away
  static __device__ __forceinline__ void pack8_rest(const f32x16_t& x, int e, u32x4_t& out, u32x4_t& rest) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t u[2], r[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a = x[4 * (e + i) + 2 * j], b = x[4 * (e + i) + 2 * j + 1];
        float ra, rb;
        u[i] = pack16x2<F16>(a, b);
        unpack16x2<F16>(u[i], ra, rb);
        r[i] = pack16x2<F16>(a - ra, b - rb);
      }
      const auto p = __builtin_amdgcn_permlane32_swap(u[0], u[1], false, false), q = __builtin_amdgcn_permlane32_swap(r[0], r[1], false, false);
      out[j] = p[0]; out[2 + j] = p[1];
      rest[j] = q[0]; rest[2 + j] = q[1];
    }
  }
  // ... and to r what the rounding took away
  static __device__ __forceinline__ void store4_rest(E* p, E* r, float a, float b, float c, float d) {
    const uint2 u = make_uint2(pack16x2<F16>(a, b), pack16x2<F16>(c, d));
    *reinterpret_cast<uint2*>(p) = u;
    float x[4];
    unpack16x2<F16>(u.x, x[0], x[1]);
    unpack16x2<F16>(u.y, x[2], x[3]);
    store4(r, a - x[0], b - x[1], c - x[2], d - x[3]);
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
  static __device__ __forceinline__ bool nonfinite(const u32x4_t& x) {
    constexpr uint32_t EXP = 0x7f800000u, ONE = 0x00800000u;
    return ((((x.x & EXP) + ONE) | ((x.y & EXP) + ONE) | ((x.z & EXP) + ONE) | ((x.w & EXP) + ONE)) & 0x80000000u) != 0;
  }
  static __device__ __forceinline__ f32x4_t load4(const char* p) { return *reinterpret_cast<const f32x4_t*>(p); }
  static __device__ __forceinline__ float get(const Frag& a, int j) { return a[j]; }
  static __device__ __forceinline__ void store4(E* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
  static __device__ __forceinline__ void store4_rest(E* p, E*, float a, float b, float c, float d) { store4(p, a, b, c, d); }
};

__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// ---------------------------------------------------------------------------------------------- LDS images
// Rows of DP elements in 16-byte chunks, chunk c of row i stored at c ^ swz(i).  Two kinds of reads have to be free of bank conflicts:
//   row fragments: ds_read_b128, 16 lanes at a time, one chunk of 16 different rows;
//   transposed fragments: ds_read_b64_tr_b16, 32 lanes at a time, 4 consecutive rows x 64 bytes (4 aligned chunks).
// A row of C chunks starts at chunk position C * i (mod 16, the 256 bytes of the banks); swz fills the positions that leaves.
// An address inside an image is a lane part XOR a constant plus a constant, so one register per kind of read serves all fragments; launder()
// keeps the compiler from holding every sum in a register of its own across the loop.
typedef __attribute__((address_space(3))) const char* lds_t;
__device__ __forceinline__ lds_t lds_at(uint32_t a) { return (lds_t)(uintptr_t)a; }
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }
template <class T>
__device__ __forceinline__ T lds_read(uint32_t a) { return *reinterpret_cast<__attribute__((address_space(3))) const T*>(lds_at(a)); }
__device__ __forceinline__ uint32_t launder(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
template <class O, int DP>
struct Img {
  static constexpr int RB = DP * O::SZ, C = RB / 16;
  static constexpr int M = C == 4 || C == 12 ? 3 : C == 8 || C == 24 ? 7 : 15;       // chunk bits that swz touches
  static __device__ __forceinline__ int swz(int i) {
    if constexpr (M == 3) return (i >> 2) & 3;
    else if constexpr (M == 7) return (((i >> 1) & 1) << 2) | ((i >> 2) & 3);
    else return ((i & 3) << 2) | ((i >> 2) & 3);
  }
  static __device__ __forceinline__ int off(int i, int c) { return i * RB + ((c ^ swz(i)) << 4); }
  // chunk c of a row at `lane` (image base, a multiple of 256, + lane part): the low bits meet swz, the others are added
  static __device__ __forceinline__ uint32_t at(uint32_t lane, int c, int x) {
    return (lane ^ (uint32_t)(((c & M) ^ x) << 4)) + (uint32_t)((c & ~M) << 4);
  }
  // A operand = 32 rows of the image from `img` on: lane (r, h) <- X[r][16 ks + 8h .. + 8]
  static __device__ __forceinline__ uint32_t row_part(int lane) { return off(lane & 31, (lane >> 5) * (O::SZ / 2)); }
  static __device__ __forceinline__ typename O::Frag rows(uint32_t lane, int ks) {
    if constexpr (O::SZ == 2) {
      return lds_read<bf16x8_t>(at(lane, 2 * ks, 0));
    } else {
      const f32x4_t a = lds_read<f32x4_t>(at(lane, 4 * ks, 0)), b = lds_read<f32x4_t>(at(lane, 4 * ks + 1, 0));
      return (f32x8_t){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // A operand = the image transposed, columns 32 dt .. + 32 on the rows, rows 16 s .. + 16 of the image in the accumulators' order on k
  static __device__ __forceinline__ uint32_t col_part(int lane) {
    const int h = lane >> 5, li = lane & 15;
    if constexpr (O::SZ == 2) return off(4 * h + (li >> 2), 2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) + 8 * (li & 1);
    else return off(4 * h, (lane & 31) >> 2) + 4 * (lane & 3);
  }
  static __device__ __forceinline__ typename O::Frag cols(uint32_t lane, int s, int dt) {
    if constexpr (O::SZ == 2) {
      union { bf16x8_t v; bf16x4_t q[2]; } f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f.q[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4_t*)lds_at(
            at(lane, 4 * dt, 2 * j) + (16 * s + 8 * j) * RB));
      return f.v;
    } else {
      f32x8_t f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {     // row 16 s + 8 (j >> 2) + 4 h + (j & 3)
        const int x = (M == 7 ? ((j >> 1) & 1) << 2 : (j & 3) << 2) ^ (2 * (j >> 2));
        f[j] = lds_read<float>(at(lane, 8 * dt, x) + (16 * s + 8 * (j >> 2) + (j & 3)) * RB);
      }
      return f;
    }
  }
};

// acc (rows d, columns owned) += X^T w over a 32-row tile X of an image, w its weights in accumulator order.  Weights are exactly 0 in masked
// places, but 0 * NaN is NaN: through the product a NaN or infinity of a row would reach the columns that must not see it.  So in
// tiles with masked places the kernels look for non-finite values, and a wave that met one goes over its rows again, element by
// element and visible pairs only (their slow()), after the loop.
// LOW: what the rounding of w to the operands' 16 bits left over goes through a second product, so that w counts with 16 bits and more.
template <class O, int DP, bool LOW = false>
__device__ __forceinline__ void accumulate(f32x16_t (&acc)[DP / 32], const f32x16_t& w, uint32_t lane) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const typename O::Frag b = O::pack(w, s);
    typename O::Frag low;
    if constexpr (LOW) low = O::pack_rest(w, b, s);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      const typename O::Frag x = Img<O, DP>::cols(lane, s, dt);
      acc[dt] = O::mma(x, b, acc[dt]);
      if constexpr (LOW) acc[dt] = O::mma(x, low, acc[dt]);
    }
  }
}
// the same behind a branch (low is wave-uniform), with the image's fragments read again: what the loops of long walks are kept lean with
template <class O, int DP>
__device__ __forceinline__ void accumulate_if(bool low, f32x16_t (&acc)[DP / 32], f32x16_t w, uint32_t lane) {
  accumulate<O, DP>(acc, w, lane);
  if constexpr (O::SZ == 2) {
    if (__builtin_expect(low, 0)) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const typename O::Frag r = O::pack_rest(w, O::pack(w, s), s);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = O::mma(Img<O, DP>::cols(lane, s, dt), r, acc[dt]);
      }
    }
  }
}
template <class O, int DP>
__device__ __forceinline__ bool tile_nonfinite(uint32_t img, int lane) {
  typedef Img<O, DP> I;
  bool bad = false;
#pragma unroll 2
  for (int i = 0; i < I::C / 2; ++i) bad |= O::nonfinite(lds_read<u32x4_t>(img + (i * 64 + lane) * 16));
  return __builtin_amdgcn_ballot_w64(bad) != 0;
}
// The second operand of LOW may be 0 or of the other sign, so an infinity of the streamed rows can come out as NaN: where sums that took it
// are not finite (in lanes that are kept), the wave goes over its rows again too.
template <int N>
__device__ __forceinline__ bool not_finite(const f32x16_t (&x)[N], bool kept) {
  float t = 0.f;
#pragma unroll
  for (int dt = 0; dt < N; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) t = fmaf(x[dt][e], 0.f, t);
  return __builtin_amdgcn_ballot_w64(kept && t != 0.f) != 0;      // (a NaN is not equal to 0)
}
// the slow forms' pieces: a dot product of a row in fragments with a row in memory (whole in both lanes of a pair), and acc += w * row
template <class O, int DP>
__device__ __forceinline__ float slow_dot(const typename O::Frag (&f)[DP / 16], const char* row, int D, int hh) {
  float s = 0.f;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int d = 16 * ks + 8 * hh;
    if (d < D) {
      const typename O::Frag x = *reinterpret_cast<const typename O::Frag*>(row + d * O::SZ);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(O::get(f[ks], j), O::get(x, j), s);
    }
  }
  return pair_sum(s);
}
template <class O, int DP>
__device__ __forceinline__ void slow_add(f32x16_t (&acc)[DP / 32], float w, const char* row, int D, int hh) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < D) {
        const f32x4_t x = O::load4(row + d * O::SZ);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[dt][4 * g + j] = fmaf(w, x[j], acc[dt][4 * g + j]);
      }
    }
}

// ---------------------------------------------------------------------------------------------- streaming
// One LDS-DMA piece: 64 lanes x 16 bytes from per-lane addresses to 1 KiB of LDS at the wave-uniform byte address `lds`; a lane that
// is switched off leaves its 16 bytes as they were.  Written in assembly because behind the builtin the compiler orders every later
// transposing LDS read after ALL outstanding DMAs; the counted waits and barriers below order them.  (s_nop: no hazards are padded
// around inline assembly.)
__device__ __forceinline__ void dma16(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void dma4(const float* src, uint32_t lds) {      // 64 lanes x 4 bytes
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_dma() {           // all but the wave's last N pieces have landed, its LDS reads have too
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// A workgroup of NW waves streams blocks of KB rows of two matrices (a and b) through a ring of three buffers: its first half fetches a's
// pieces, its second half b's, block n + 2 is asked for right behind the one barrier of block n (with two buffers: block n + 1).  A row
// behind the last one repeats it; chunks behind the row's D elements are not fetched (the caller cleared the buffers once).
template <class O, int DP, int NBUF = 3, int NW = 4>
struct Ring {
  typedef Img<O, DP> I;
  static constexpr int KB = I::RB <= 64 ? 128 : I::RB <= 128 || NW == 8 ? 64 : 32;
  static constexpr int IMG = KB * I::RB, BUF = 2 * IMG, NB = NBUF, HW = NW / 2, PP = IMG / (1024 * HW);     // PP: pieces per wave and block
  const char* p[PP];
  long ld;
  uint32_t on, lds;
  __device__ __forceinline__ void start(const char* a, long lda, const char* b, long ldb, int row, int D, int wave, int lane, uint32_t lds0) {
    ld = wave < HW ? lda : ldb;
    const char* base = (wave < HW ? a : b) + (long)row * ld;
    lds = lds0 + wave * PP * 1024;
    on = 0;
#pragma unroll
    for (int j = 0; j < PP; ++j) {
      const int idx = (wave % HW * PP + j) * 64 + lane, r = idx / I::C, ch = (idx % I::C) ^ I::swz(r);
      p[j] = base + r * ld + ch * 16;
      on |= (uint32_t)(ch * 16 < D * O::SZ) << j;
    }
  }
  // block of rows [row, row + KB) of the rows before `end`, into buffer `buf`
  template <bool PAD>
  __device__ __forceinline__ void issue(int row, int end, int buf, int wave, int lane) {
    const bool last = row + KB > end;
    lane = launder(lane);
#pragma unroll
    for (int j = 0; j < PP; ++j) {
      const char* q = p[j];
      if (last) {
        const int over = row + ((wave % HW * PP + j) * 64 + lane) / I::C - (end - 1);
        if (over > 0) q -= over * ld;
      }
      if (!PAD || ((on >> j) & 1)) dma16(q, lds + buf * BUF + j * 1024);
      p[j] += KB * ld;
    }
  }
};

// A wave streams 32-row tiles of two matrices through buffers of its own (one or two): no barrier, nothing shared.
template <class O, int DP, int NBUF = (DP * O::SZ <= 256 ? 2 : 1)>
struct Tiles {
  typedef Img<O, DP> I;
  static constexpr int IMG = 32 * I::RB, BUF = 2 * IMG, NB = NBUF, NP = I::C;    // NP: pieces per tile
  template <bool PAD, class RowAt>      // RowAt(i): byte offsets of the tile's row i in a and in b
  static __device__ __forceinline__ void issue(const char* a, const char* b, RowAt&& at, int D, int lane, uint32_t lds) {
#pragma unroll
    for (int j = 0; j < NP / 2; ++j) {
      const int idx = j * 64 + lane, r = idx / I::C, ch = (idx % I::C) ^ I::swz(r);
      long oa, ob;
      at(r, oa, ob);
      if (!PAD || ch * 16 < D * O::SZ) {
        dma16(a + oa + ch * 16, lds + j * 1024);
        dma16(b + ob + ch * 16, lds + IMG + j * 1024);
      }
    }
  }
};

// ... of consecutive rows: the pieces' addresses walk along, 32 * NW rows a step
template <class O, int DP, int NW, class S>
struct TileWalk {
  typedef Img<O, DP> I;
  static constexpr int H = S::NP / 2;
  const char *pa[H], *pb[H];
  long lda, ldb;
  __device__ __forceinline__ void start(const char* a, long lda_, const char* b, long ldb_, int row, int lane) {
    lda = lda_;
    ldb = ldb_;
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int idx = j * 64 + lane, r = idx / I::C, ch = (idx % I::C) ^ I::swz(r);
      pa[j] = a + (row + r) * lda + ch * 16;
      pb[j] = b + (row + r) * ldb + ch * 16;
    }
  }
  // the tile of rows [row, row + 32) of the rows before `end` (a row behind repeats the last), and on to the wave's next tile
  template <bool PAD>
  __device__ __forceinline__ void issue(int row, int end, int D, int lane, uint32_t lds) {
    const bool last = row + 32 > end;
    lane = launder(lane);
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const char *qa = pa[j], *qb = pb[j];
      if (last) {
        const int over = row + (j * 64 + lane) / I::C - (end - 1);
        if (over > 0) { qa -= over * lda; qb -= over * ldb; }
      }
      bool on = true;
      if constexpr (PAD) {
        const int idx = j * 64 + lane;
        on = ((idx % I::C) ^ I::swz(idx / I::C)) * 16 < D * O::SZ;
      }
      if (on) {
        dma16(qa, lds + j * 1024);
        dma16(qb, lds + S::IMG + j * 1024);
      }
      pa[j] += 32 * NW * lda;
      pb[j] += 32 * NW * ldb;
    }
  }
};

__device__ __forceinline__ void clear_lds(char* p, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
}

// blockIdx -> (head, tile).  Workgroups go round the 8 XCDs; a head's keys and values should stay in one XCD's cache, every XCD should get the
// same share of long and short tiles, and the tiles should start in their order.  Heads a multiple of 8: an eighth of them on each XCD; of
// 4: a quarter on each pair of XCDs, which take the tiles in turn; else: all heads' tiles in turn.  (Runs of one head's tiles after the other
// instead share more of a cache, but start long tiles late: 2 x 8192 causal D 128, 10 heads on 2, forward / backward 458 / 1639 us, in
// turn 376 / 1310; not causal, 32 x 785 D 64, 6 heads: 65 / 187, 68 / 197.)
// `level`: all workgroups are on the card at once, nobody comes later to even out what a compute unit got.  An XCD's units then go out to its 32
// compute units there and back, so that who got the longest of one round gets the shortest of the next (1 x 7000 causal D 80, 15 heads:
// 206 / 660, with it 178 / 534; 8 x 1440 fp32 D 32, 6 heads on 3: 98 / 314, 80 / 254; where later workgroups even out, it costs: 1 x 4096
// D 128 with two waves a tile 101, 118).
struct Unit { int head, tile; };
__device__ __forceinline__ Unit xcd_unit(int heads, int tiles, bool level = false) {
  const int x = blockIdx.x & 7;
  int s = blockIdx.x >> 3;
  if (level && (s & 32)) {
    const int row = s & ~31;
    s = row + min(32, (int)(gridDim.x >> 3) - row) - 1 - (s - row);
  }
  if ((heads & 7) == 0) {
    const int h = heads >> 3;
    return {x * h + s % h, s / h};
  }
  if ((heads & 3) == 0) {
    const int h = heads >> 2, t = 2 * (s / h) + (x >> 2);
    return {t < tiles ? (x & 3) * h + s % h : -1, t};
  }
  const int u = s * 8 + x;
  return {u < heads * tiles ? u % heads : -1, u / heads};
}
// how many workgroups of a kernel the card holds (found once), and a sixteenth: so many of a grid's last ones own no rows
static inline long card_holds(const void* f, int threads, size_t lds, long& n) {
  if (n == 0) {
    hipFuncAttributes at;
    if (hipFuncGetAttributes(&at, f) != hipSuccess) {
      (void)hipGetLastError();
      return 0;
    }
    const long waves = std::min(8, 512 / std::max(8, (at.numRegs + 7) / 8 * 8)) * 4;
    n = 272 * std::min<long>(163840 / std::max<size_t>(lds + at.sharedSizeBytes, 1), waves * 64 / threads);
  }
  return n;
}
static inline unsigned xcd_grid(long heads, long tiles) {
  return (unsigned)((heads & 7) == 0 ? heads * tiles : (heads & 3) == 0 ? heads * ((tiles + 1) / 2 * 2) : (heads * tiles + 7) / 8 * 8);
}

// Waves of a split forward's workgroup: eight, a tile each at a time, for walks of 512 and more where two such workgroups fit a unit's LDS
// (1 x 4096 bf16 D 64 12 heads: 59 us, with four 73; 2 x 1440 fp32 D 32 the same), else four with two tiles each.  The backward, which
// holds more registers, keeps four (1 x 4096: 173 us, with eight 205; 2 x 1440: 108, 114).
template <class O, int DP>
constexpr int SPLIT_WAVES = DP * O::SZ <= 128 ? 8 : 4;
template <class O, int DP, int NW>
using SplitTiles = Tiles<O, DP, ((NW == 8 && DP * O::SZ > 64) || DP * O::SZ > 256) ? 1 : 2>;
static inline bool long_walks(long T, long n_seqs) { return T >= 512 * n_seqs; }

// The wide form with eight waves (H = 2): two for each 32 rows, which take the tiles of 64-row blocks in turn and join their sums in LDS.  A walk
// is half as long and a block half as many barriers, for an unchanged amount of work: it pays where few, long and unequal walks fill the
// compute units once, at rows of 256 bytes.  Measured, us, forward / backward with one and two waves a row tile, causal: 1 x 2048 bf16 D 128
// 16 heads on 4: 60 / 195, 45 / 153; 1 x 4096: 117 / 380, 94 / 320; 2 x 2048: 63 / 211, 55 / 195; 4 x 2048 fp32 D 64 8 heads: 210 / 633,
// 158 / 529; 2 x 1600: 50 / 170, 44 / 150; but 3 x 1300, 560 workgroups: 48 / 168, 57 / 183; 1 x 6000, 800 workgroups: forward 193, 191;
// not causal, 4 x 2048 8 heads D 128: 82, 90; shorter rows, 2 x 4096 D 96 12 heads: 108, 115.
template <class O, int DP>
constexpr bool PAIRS = DP * O::SZ == 256;
template <int DP>
constexpr int HALF = (DP / 8 + 1) * 1024;        // bytes of 32 rows' sums in the accumulators' order, and a float2 for each lane
template <int DP>
__device__ __forceinline__ void put_half(char* half, const f32x16_t (&o)[DP / 32]) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4_t*>(half + (4 * dt + g) * 1024) = (f32x4_t){o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
}
template <int DP>
__device__ __forceinline__ void add_half(const char* half, f32x16_t (&o)[DP / 32]) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(half + (4 * dt + g) * 1024);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[dt][4 * g + j] += x[j];
    }
}

// ---------------------------------------------------------------------------------------------- which rows meet
struct Span { int lo, hi; };
// Which rows a workgroup owns.  Up to SEQ_TILES sequences every sequence is cut into tiles of its own (a tile across two sequences would walk
// both: twice the longest path), and so are the rows before the first and behind the last one; beyond that, the packed rows are, and
// every row looks its sequence up.
constexpr int SEQ_TILES = 510;
struct OwnTile { int row0, end; Span seq; };      // rows [row0, end); seq: their sequence ({0, 0}: none)
template <int ROWS>
static inline long tile_bound(long T, long n) {   // no fewer than the tiles there are
  return n > SEQ_TILES ? (T + ROWS - 1) / ROWS : (T + (ROWS - 1) * (n + 2 < T ? n + 2 : T)) / ROWS;
}
static inline bool use_pairs(long T, long n_seqs, long heads, int frame) {
  const long wide = tile_bound<128>(T, n_seqs) * heads;
  return frame > 0 && wide <= 640 && T >= (wide > 512 ? 1536 : 1280) * n_seqs;
}
// Which form: `wide` = the wide one's workgroups.  Below one for each of the 256 compute units the split form is faster (measured, us: 1 x 512
// bf16 D 128 16 heads, 80 workgroups: wide 20, split 13; 4 x 197 D 64, 96: 10.5, 9.5), above it the wide one (16 x 197 D 64, 384: 13, 23;
// 4 x 1024 D 128, 544: 43, 96) unless few workgroups walk far: up to two for each unit and 4096 tokens a sequence (1 x 4096 D 64, 408: 99,
// 59), in fp32, whose walks are 8 times as long, 1024 (4 x 1024 D 128, 280: 157, 131; 8 x 400 D 64, 384: 65, 83).  Pairs of waves move
// that border (wide and split, forward / backward, causal: 1 x 2048 bf16 D 128 8 heads, 152: 41 / 139, 37 / 94; 1 x 1300 16 heads, 208:
// 31 / 108, 43 / 112; 1 x 5000 8 heads, 336: 100 / 324, 167 / 419; 2 x 2048 fp32 D 64, 272: 151 / 487, 128 / 372; 3 x 2048, 408: 151 /
// 488, 182 / 526).
static inline bool use_split(long wide, int dtype, long T, long n_seqs, bool pairs) {
  if (pairs) return wide < (dtype == MVF_F32 ? 352 : 192);
  return wide < 256 || (wide < 512 && T >= (dtype == MVF_F32 ? 1024 : 4096) * n_seqs);
}
// The t-th tile, found by every wave for itself.  Up to 62 sequences the tiles come in the order of their walks, longest first (causal: the
// tile's place in its sequence, counted from the end that sees most; else the sequence's length), so that the last workgroups to
// finish are short ones: lane i holds segment i, and the walk w of the t-th tile is found by 64 candidates at a time, F(w) = tiles
// that walk at least w.  Beyond that sequence by sequence, with a prefix sum per 64 of them.
enum class Walk { ALL, LATE, EARLY };             // non-causal; causal: late rows walk far (queries), early rows do (keys)
__device__ __forceinline__ int nth_bit(uint64_t m, int k) {
  for (; k > 0; --k) m &= m - 1;
  return __builtin_ctzll(m);
}
template <int ROWS>
__device__ __forceinline__ OwnTile find_tile(const int* __restrict__ cu, int n, int T, int t, int bound, Walk walk) {
  const int lane = threadIdx.x & 63;
  if (n > SEQ_TILES) {
    if (walk == Walk::LATE) t = bound - 1 - t;
    return {t * ROWS, min(T, t * ROWS + ROWS), {0, 0}};
  }
  if (n <= 62) {
    const int i = lane;                             // segment 0: rows before cu[0]; i: sequence i - 1; n + 1: rows behind cu[n]
    const int lo = i == 0 ? 0 : min(max(cu[min(i - 1, n)], 0), T), hi = i > n ? T : min(max(cu[min(i, n)], 0), T);
    const int tiles = i < n + 2 && hi > lo ? (hi - lo + ROWS - 1) / ROWS : 0;
    const int c = i > 0 && i <= n ? tiles : 0;      // of sequences
    int most = 0, total = 0;
    for (int k0 = 0; k0 <= n; k0 += 8)              // (lanes behind n hold 0)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int x = __builtin_amdgcn_readlane(c, k0 + k);
        most = max(most, x);
        total += x;
      }
    if (t >= total) {                               // rows of no sequence
      const int g0 = __builtin_amdgcn_readlane(tiles, 0), j = t - total, seg = j < g0 ? 0 : n + 1, k = j < g0 ? j : j - g0;
      if (seg != 0 && k >= __builtin_amdgcn_readlane(tiles, n + 1)) return {0, 0, {0, 0}};
      const int l = __builtin_amdgcn_readlane(lo, seg), h = __builtin_amdgcn_readlane(hi, seg);
      return {l + k * ROWS, min(h, l + k * ROWS + ROWS), {0, 0}};
    }
    int w0 = 1, w1 = most + 1, above = 0;           // the smallest w with F(w) <= t; above = F(w)
    while (true) {
      const int step = (w1 - w0 + 62) / 63, w = min(w0 + lane * max(step, 1), w1);
      int f = 0;
      for (int k0 = 0; k0 <= n; k0 += 8) {
        if (walk == Walk::ALL) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int x = __builtin_amdgcn_readlane(c, k0 + k);
            f += x >= w ? x : 0;
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) f += max(__builtin_amdgcn_readlane(c, k0 + k) - w + 1, 0);
        }
      }
      const uint64_t ok = __builtin_amdgcn_ballot_w64(f <= t);       // never 0: lane 63 stands at w1
      const int j = __builtin_ctzll(ok);
      const int at = __builtin_amdgcn_readlane(w, j);
      if (j == 0 || step <= 1) {
        w1 = at;
        above = __builtin_amdgcn_readlane(f, j);
        break;
      }
      w0 = __builtin_amdgcn_readlane(w, j - 1) + 1;
      w1 = at;
    }
    const int w = w1 - 1, r = t - above;            // the tile's walk, its place among those
    const int seg = walk == Walk::ALL ? nth_bit(__builtin_amdgcn_ballot_w64(c == w), r / w) : nth_bit(__builtin_amdgcn_ballot_w64(c >= w), r);
    const int j = walk == Walk::ALL ? r % w : walk == Walk::LATE ? w - 1 : __builtin_amdgcn_readlane(c, seg) - w;
    const int l = __builtin_amdgcn_readlane(lo, seg), h = __builtin_amdgcn_readlane(hi, seg);
    return {l + j * ROWS, min(h, l + j * ROWS + ROWS), {l, h}};
  }
  if (walk == Walk::LATE) t = bound - 1 - t;
  int before = 0;
  for (int s0 = 0; s0 < n + 2; s0 += 64) {
    const int i = s0 + lane;
    const int lo = i == 0 ? 0 : min(max(cu[min(i - 1, n)], 0), T), hi = i > n ? T : min(max(cu[i], 0), T);
    const int tiles = i < n + 2 && hi > lo ? (hi - lo + ROWS - 1) / ROWS : 0;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o, 64);
      if (lane >= o) sum += up;
    }
    const uint64_t in = __builtin_amdgcn_ballot_w64(t >= before + sum - tiles && t < before + sum);
    if (in != 0) {
      const int j = __builtin_ctzll(in);
      const int l = __builtin_amdgcn_readlane(lo, j), h = __builtin_amdgcn_readlane(hi, j);
      const int first = before + __builtin_amdgcn_readlane(sum - tiles, j), r0 = l + (t - first) * ROWS;
      const int seg = s0 + j;
      return {r0, min(h, r0 + ROWS), seg == 0 || seg == n + 1 ? Span{0, 0} : Span{l, h}};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {0, 0, {0, 0}};
}
// largest b < n with cu[b] <= row < cu[b + 1], as [start, end) cut to [0, T); {0, 0} for a row of no sequence
__device__ __forceinline__ Span sequence_of(const int* __restrict__ cu, int n, int T, int row) {
  int lo = 0, hi = n;                      // the first index with cu > row lies in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid + 1;
    else hi = mid;
  }
  const int s = max(cu[max(lo - 1, 0)], 0), e = min(cu[lo], T);
  return lo > 0 && row < e ? Span{s, e} : Span{0, 0};
}
__device__ __forceinline__ Span sequence_of(const OwnTile& t, const int* __restrict__ cu, int n, int T, int row) {
  if (row >= t.end) return {0, 0};
  return n > SEQ_TILES ? sequence_of(cu, n, T, row) : t.seq;
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

// Walks of up to four tiles take their 16-bit weights and dS whole (in two operands).  Of a few terms, and of a sum as small beside them as
// dP - delta, the operands' roundings are what is left of an error; over long walks they average to one rounding beside the result's own,
// and second operands cost: 2 x 8192 bf16, 16 heads of 128 on 4, a training pass 2.50 -> 3.51 ms with all of them, the backward 1.88 -> 2.27
// with dS's alone; 4 prompts of up to 7001 fp16 D 80 190 -> 261 us.
__device__ __forceinline__ bool short_walk(const WaveSpan& ws) { return ws.any.hi - ws.any.lo <= 128; }

// ---------------------------------------------------------------------------------------------- softmax state of a row
// m: the maximum its exponents are taken against (raw scores), nm = -m * c, l: this lane's share of the row sum.
struct RowMax {
  float m = NEG_INF, nm = 0.f, l = 0.f;
  // (finite, also for a scale so small that no scores differ: -infinity + infinity would compare as no growth at all)
  static __device__ __forceinline__ float threshold(float c) { return fminf(8.f / c, 3e38f); }
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
  // The exponents s c + nm all carry the rounding of nm, which cancels against the row's sum; beyond this size it could push them out of
  // the formats' range (one step of nm is 2 there), so the wave takes its slow form, whose exponents are (s - m) c.
  __device__ __forceinline__ bool steep(bool kept) const { return __builtin_amdgcn_ballot_w64(kept && fabsf(nm) > 16777216.f) != 0; }
  // the slow forms' step: one more score; its weight, and what everything so far is multiplied with
  __device__ __forceinline__ float add(float s, float c, float& alpha) {
    const float to = fmaxf(m, s);
    alpha = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((m - to) * c);
    m = to;
    nm = to == NEG_INF ? 0.f : -to * c;
    return __builtin_amdgcn_exp2f((to == NEG_INF ? s : s - to) * c);
  }
};

// The backward's probabilities in fp16 carry this power of two (in the rows' exponent offsets, so it costs nothing): of sequences of ten
// thousands of tokens they lie where fp16 has few bits, and they are at most 1.
constexpr int PSHIFT = 15;

// union of the four waves' spans (a barrier inside)
__device__ __forceinline__ Span block_span(const WaveSpan& ws, int* s_span, int lane, int wave, int nw) {
  if (lane == 0) { s_span[2 * wave] = ws.any.hi > 0 ? ws.any.lo : 0x7fffffff; s_span[2 * wave + 1] = ws.any.hi; }
  __syncthreads();
  Span s = {0x7fffffff, 0};
  for (int w = 0; w < nw; ++w) { s.lo = min(s.lo, s_span[2 * w]); s.hi = max(s.hi, s_span[2 * w + 1]); }
  // nothing: {0, 0}, so that sums with .lo stay in range
  return {__builtin_amdgcn_readfirstlane(s.hi == 0 ? 0 : s.lo), __builtin_amdgcn_readfirstlane(s.hi)};
}

// NW waves hold partial softmaxes of the same 32 rows: sums o^T against their own maxima.  Joins them in LDS (fixed order) and hands
// use(row, first channel of four, unnormalised sums, maximum in the exponent's units, sum of weights) for every row and channel.  All
// threads; the caller's earlier LDS reads are behind a barrier.
template <int DP, int NW = 4>
constexpr int JOIN_BYTES = NW * 32 * (DP + 4) * 4;
template <int DP, int NW = 4, class Use>
__device__ __forceinline__ void join_waves(float* so, float (*s_m)[32], float (*s_l)[32], const f32x16_t (&o)[DP / 32], const RowMax& st,
                                           int rows, int D, int wave, int lane, Use&& use) {
  constexpr int ROWF = DP + 4;
  const int r = lane & 31, hh = lane >> 5;
  const float l = pair_sum(st.l);
  if (hh == 0) { s_m[wave][r] = st.m == NEG_INF ? NEG_INF : -st.nm; s_l[wave][r] = l; }
  if (r < rows) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t*>(so + (wave * 32 + r) * ROWF + 32 * dt + 8 * g + 4 * hh) =
            (f32x4_t){o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (DP / 4); i += 64 * NW) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= D) continue;
    float mx = NEG_INF;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w][row]);
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = s_m[w][row], lw = s_l[w][row];
      if (m == NEG_INF && lw == lw) continue;                 // saw nothing (a NaN sum with no maximum saw a NaN)
      const float f = m == NEG_INF ? lw : __builtin_amdgcn_exp2f(m - mx);
      sum = fmaf(f, lw, sum);
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(so + (w * 32 + row) * ROWF + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(f, x[j], acc[j]);
    }
    use(row, d, acc, mx, sum);
  }
}

}  // namespace seq_attn
