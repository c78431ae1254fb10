// Backward of seq_attn.hip.  With P the probabilities (recomputed from the forward's row statistics) and dP = dO V^T:
//   dV = P^T dO,   dS = P o (dP - delta),  delta = rowsum(dO o O),   dQ = scale dS K,   dK = scale dS^T Q,
// dK and dV summed over the query heads of a group.  Two kernels, each owning what it writes, so no atomics and the same bits every time:
//   dQ:     owns 32 queries per wave, streams K and V;       also writes delta, which the second kernel reads
//   dK/dV:  owns 32 keys per wave, streams Q and dO of every head of the group (the sum over the group stays in registers)
// Each in the three forms of the forward: wide (four waves of 32 rows share the streamed blocks), pairs (eight waves do) and split (one
// 32-row tile, every wave walks its own quarter of the streamed tiles, the four sums are added at the end in a fixed order).
// P and dS are rounded to the operands' format where they enter a product (whole in short walks: short_walk()); the sums, delta and the row
// statistics are 32 bits.  delta is taken from the output and what its rounding took away: from the rounded output alone it leaves
// gradients of short sequences off by up to 30 roundings, of long ones by 1.55.  Errors in bf16: 1.7e-3 of the gradient's size in short
// walks, one rounding, and in long ones, with dS's own (2^-9 relative, random in sign), sqrt(2) of that, 2.4e-3.
// Measured, 2 x 8192 causal bf16, 16 query heads of 128 on 4: dQ 0.87 ms (946 TFLOP/s of its three products), dK / dV 1.28 ms (862 of its
// four) and 25 us for the sum of the parts.  Bound by registers: dK / dV holds 2 x 32 x 128 sums and a wave's K rows, so two waves a SIMD
// are all that fit, and their waits are not all covered.
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using namespace seq_attn;

struct BwdArgs {
  const char *q, *k, *v;
  long ldq, hsq, ldk, hsk, ldv, hsv;   // token and head strides in BYTES
  const int* cu;
  int n_seqs;
  const char *out, *rest, *d_out;      // [T, Hq, D]; rest may be NULL
  const float* stat;                   // [2][Hq][T] of the forward
  float* delta;                        // [Hq][T]
  float* part;                         // parts > 1: [parts][2 (dk, dv)][T][Hk][D]
  int parts;                           // workgroups that share a group's heads
  char *dq, *dk, *dv;                  // [T, Hq, D], [T, Hk, D] x 2
  int T, Hq, Hk, D, frame, ntiles, level;
  float c, scale;                      // scale * log2(e); scale over 2^PSHIFT
  float pinv;                          // 1 over 2^PSHIFT
};

// a row as the B operand's fragments.  (A row of no sequence may hold anything: it stays in its own lanes and is not stored.)
template <class O, int DP>
__device__ __forceinline__ void load_row(typename O::Frag (&f)[DP / 16], const char* src, int D, int hh) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int d = 16 * ks + 8 * hh;
    typename O::Frag x = {};
    if (d < D) x = *reinterpret_cast<const typename O::Frag*>(src + d * O::SZ);
    f[ks] = x;
  }
}

template <class O, int DP>
__device__ __forceinline__ void store_rows(char* base, size_t row_elems, const f32x16_t (&x)[DP / 32], float f, bool some, int D, int hh) {
  typename O::E* dst = reinterpret_cast<typename O::E*>(base) + row_elems;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < D) {
        if (some) O::store4(dst + d, x[dt][4 * g] * f, x[dt][4 * g + 1] * f, x[dt][4 * g + 2] * f, x[dt][4 * g + 3] * f);
        else O::store4(dst + d, 0.f, 0.f, 0.f, 0.f);
      }
    }
}

// the fp32 format of the partial sums
typedef Op<MVF_F32> Part;

// fp16 holds 2^-14 to 2^16 with all of its bits, and dS = P (dP - delta) of a long sequence lies below.  A column (an owned row, the pair of
// lanes that holds it) therefore enters its product multiplied with a power of two of its own, which follows the largest dS so
// far: it is brought to 2^10 .. 2^11, and again only when one passes 2^15 (the sums follow; all of this is exact).  32 x 785, 12 heads of 64:
// 355 us for 328 without.
template <int DT>
struct DsScale {
  float f = 0x1p30f;       // smaller dS than 2^-15 leave it
  template <int N>
  __device__ __forceinline__ void fit(f32x16_t& x, f32x16_t (&acc)[N]) {
    if constexpr (DT == MVF_F16) {
      float mx = 0.f, top[5];
#pragma unroll
      for (int e = 0; e < 5; ++e) top[e] = fmaxf(fmaxf(fabsf(x[3 * e]), fabsf(x[3 * e + 1])), fabsf(x[3 * e + 2]));
      mx = fmaxf(fmaxf(fmaxf(top[0], top[1]), top[2]), fmaxf(fmaxf(top[3], top[4]), fabsf(x[15])));
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx * f > 32768.f) != 0, 0)) {
        mx = pair_max(mx);
        const float to = mx * f > 32768.f && mx < -NEG_INF ? ldexpf(1.f, 11 - __builtin_amdgcn_frexp_expf(mx)) : f;
        const float by = to / f;                  // (powers of two)
        f = to;
#pragma unroll
        for (int dt = 0; dt < N; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[dt][e] *= by;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= f;
    }
  }
  template <int N>
  __device__ __forceinline__ void undo(f32x16_t (&acc)[N]) const {
    if constexpr (DT == MVF_F16) {
      const float by = 1.f / f;
#pragma unroll
      for (int dt = 0; dt < N; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] *= by;
    }
  }
};

// The waves' sums of the same 32 rows, added in order, out as [row][D].  All threads; barriers inside.
template <class O, int DP>
__device__ __forceinline__ void store_joined(float* so, const f32x16_t (&x)[DP / 32], char* base, int row0, int rows, long stride, float f,
                                             int D, int wave, int lane) {
  constexpr int ROWF = DP + 4;
  const int r = lane & 31, hh = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4_t*>(so + (wave * 32 + r) * ROWF + 32 * dt + 8 * g + 4 * hh) =
          (f32x4_t){x[dt][4 * g], x[dt][4 * g + 1], x[dt][4 * g + 2], x[dt][4 * g + 3]};
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (DP / 4); i += 256) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= D) continue;
    f32x4_t acc = *reinterpret_cast<const f32x4_t*>(so + row * ROWF + d);
#pragma unroll
    for (int w = 1; w < 4; ++w) acc += *reinterpret_cast<const f32x4_t*>(so + (w * 32 + row) * ROWF + d);
    O::store4(reinterpret_cast<typename O::E*>(base) + (long)(row0 + row) * stride + d, acc[0] * f, acc[1] * f, acc[2] * f, acc[3] * f);
  }
}

// ------------------------------------------------------------------------------------------------ dQ
// Small heads take dS whole in long walks too: their keys' weighted mean is large beside the keys' spread, dS (whose sum is 0) takes it out of
// the gradient but not out of dS's roundings (dQ of heads of 16 to 40: 1.5 to 1.6 of one rounding, whole 1.1; of 64: 1.47, for 9 % of the
// backward's time).
constexpr int SMALL_HEAD = 48;
template <int DT, int DP>
struct Dq {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typename O::Frag qf[DP / 16], dof[DP / 16];
  f32x16_t dq[DP / 32];
  Span own;
  float c, off, inv, dl;
  int lane;
  uint32_t rpart, cpart;
  bool bad = false;        // a tile with masked places held a value that is not finite
  DsScale<DT> ds;
  bool low = false;        // dS's second operand: see accumulate()

  __device__ __forceinline__ void start(const BwdArgs& a, int head, int row, int lane_, bool write_delta) {
    lane = lane_;
    rpart = I::row_part(lane);
    cpart = I::col_part(lane);
    c = a.c;
    const int hh = lane >> 5, rr = min(row, a.T - 1);
    load_row<O, DP>(qf, a.q + (long)rr * a.ldq + head * a.hsq, a.D, hh);
    const size_t orow = ((size_t)rr * a.Hq + head) * a.D * O::SZ;
    load_row<O, DP>(dof, a.d_out + orow, a.D, hh);
    dl = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * hh;
      typename O::Frag x = {};
      if (d < a.D) x = *reinterpret_cast<const typename O::Frag*>(a.out + orow + d * O::SZ);
#pragma unroll
      for (int j = 0; j < 8; ++j) dl = fmaf(O::get(dof[ks], j), O::get(x, j), dl);
    }
    if (O::SZ == 2 && a.rest != nullptr) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = 16 * ks + 8 * hh;
        typename O::Frag x = {};
        if (d < a.D) x = *reinterpret_cast<const typename O::Frag*>(a.rest + orow + d * O::SZ);
#pragma unroll
        for (int j = 0; j < 8; ++j) dl = fmaf(O::get(dof[ks], j), O::get(x, j), dl);
      }
    }
    dl = pair_sum(dl);
    const size_t at = (size_t)head * a.T + rr;
    off = a.stat[at];
    inv = DT == MVF_F32 ? a.stat[(size_t)a.Hq * a.T + at] : 1.f;
    if (write_delta && hh == 0) a.delta[at] = dl;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(qf[ks]), "+v"(dof[ks]));      // landed before any DMA is in flight
    asm volatile("" : "+v"(off), "+v"(inv), "+v"(dl));
  }
  __device__ __forceinline__ void tile(uint32_t ik, uint32_t iv, int key0, bool mask) {
    const uint32_t rk = launder(rpart + ik), rv = launder(rpart + iv), ck = launder(cpart + ik);
    f32x16_t s = zero16(), dp = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(rk, ks), qf[ks], s);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) dp = O::mma(I::rows(rv, ks), dof[ks], dp);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[e], c, off));
      if constexpr (DT == MVF_F32) p *= inv;
      s[e] = p * (dp[e] - dl);
    }
    if (mask) {
      bad |= tile_nonfinite<O, DP>(ik, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = key0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        s[e] = key >= own.lo && key < own.hi ? s[e] : 0.f;
      }
    }
    ds.fit(s, dq);
    accumulate_if<O, DP>(low, dq, s, ck);
  }
  __device__ __forceinline__ void slow(const BwdArgs& a, const char* kb, const char* vb, int first, int step, int end) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = zero16();
#pragma unroll 1
    for (int k0 = first; k0 < end; k0 += step)
#pragma unroll 1
      for (int key = k0; key < min(k0 + 32, end); ++key) {
        const float s = slow_dot<O, DP>(qf, kb + (long)key * a.ldk, a.D, lane >> 5);
        const float dp = slow_dot<O, DP>(dof, vb + (long)key * a.ldv, a.D, lane >> 5);
        if (key < own.lo || key >= own.hi) continue;
        slow_add<O, DP>(dq, __builtin_amdgcn_exp2f(fmaf(s, c, off)) * inv * (dp - dl), kb + (long)key * a.ldk, a.D, lane >> 5);
      }
  }
  __device__ __forceinline__ void any_tile(const WaveSpan& ws, uint32_t ik, uint32_t iv, int key0) {
    if (key0 >= ws.any.hi || key0 + 32 <= ws.any.lo) return;
    tile(ik, iv, key0, key0 < ws.all.lo || key0 + 32 > ws.all.hi);
  }
};

template <int DT, int DP, bool PAD, int H>
__global__ __launch_bounds__(256 * H, DT == MVF_F32 && DP > 32 ? H : 2) void packed_attn_dq_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typedef Ring<O, DP, 3, 4 * H> R;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ int s_span[8 * H];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit u = xcd_unit(a.Hq, a.ntiles, a.level);
  if (u.head < 0) return;
  const int head = u.head;
  const OwnTile own = find_tile<128>(a.cu, a.n_seqs, a.T, u.tile, a.ntiles, a.frame == 0 ? Walk::ALL : Walk::LATE);
  if (own.row0 >= own.end) return;
  const int row = own.row0 + (wave & 3) * 32 + (lane & 31);
  Dq<DT, DP> f;
  f.start(a, head, row, lane, row < own.end && wave < 4);
  f.own = keys_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws) || a.D <= SMALL_HEAD;
  if constexpr (PAD) clear_lds(smem, R::NB * R::BUF);
  const Span span = block_span(ws, s_span, lane, wave, 4 * H);
  const int g = a.Hq / a.Hk;
  const char *kb = a.k + head / g * a.hsk, *vb = a.v + head / g * a.hsv;
  R ring;
  ring.start(kb, a.ldk, vb, a.ldv, span.lo, a.D, wave, lane, lds_addr(smem));
  if (span.lo < span.hi) ring.template issue<PAD>(span.lo, span.hi, 0, wave, lane);
  if (span.lo + R::KB < span.hi) ring.template issue<PAD>(span.lo + R::KB, span.hi, 1, wave, lane);
  int buf = 0;
  for (int b0 = span.lo; b0 < span.hi; b0 += R::KB) {
    if (b0 + R::KB < span.hi) wait_dma<R::PP>();
    else wait_dma<0>();
    __builtin_amdgcn_s_barrier();
    if (b0 + 2 * R::KB < span.hi) ring.template issue<PAD>(b0 + 2 * R::KB, span.hi, buf == 0 ? 2 : buf - 1, wave, lane);
    const uint32_t ik = lds_addr(smem) + buf * R::BUF;
#pragma unroll 1
    for (int t = wave >> 2; t < R::KB / 32; t += H) f.any_tile(ws, ik + t * 32 * I::RB, ik + R::IMG + t * 32 * I::RB, b0 + 32 * t);
    buf = buf == 2 ? 0 : buf + 1;
  }
  f.ds.undo(f.dq);
  if (O::SZ == 2 && f.low) f.bad |= not_finite(f.dq, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kb, vb, span.lo + 32 * (wave >> 2), 32 * H, ws.any.hi);
  if constexpr (H == 2) {
    __syncthreads();
    char* half = smem + (wave & 3) * HALF<DP> + lane * 16;
    if (wave >= 4) put_half<DP>(half, f.dq);
    __syncthreads();
    if (wave >= 4) return;
    add_half<DP>(half, f.dq);
  }
  if (row < own.end) store_rows<O, DP>(a.dq, ((size_t)row * a.Hq + head) * a.D, f.dq, a.scale, f.own.hi > 0, a.D, lane >> 5);
}

template <int DT, int DP, bool PAD>
__global__ __launch_bounds__(256, 1) void packed_attn_dq_split_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef SplitTiles<O, DP, 4> S;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit u = xcd_unit(a.Hq, a.ntiles);
  if (u.head < 0) return;
  const int head = u.head;
  const OwnTile own = find_tile<32>(a.cu, a.n_seqs, a.T, u.tile, a.ntiles, a.frame == 0 ? Walk::ALL : Walk::LATE);
  if (own.row0 >= own.end) return;
  const int row0 = own.row0, row = row0 + (lane & 31);
  Dq<DT, DP> f;
  f.start(a, head, row, lane, wave == 0 && row < own.end);
  f.own = keys_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws) || a.D <= SMALL_HEAD;
  if constexpr (PAD) clear_lds(smem, 4 * S::NB * S::BUF);
  const int g = a.Hq / a.Hk;
  const char *kb = a.k + head / g * a.hsk, *vb = a.v + head / g * a.hsv;
  const uint32_t lds = lds_addr(smem) + wave * S::NB * S::BUF;
  TileWalk<O, DP, 4, S> walk;
  walk.start(kb, a.ldk, vb, a.ldv, ws.any.lo + wave * 32, lane);
  auto issue = [&](int key0, int buf) __attribute__((always_inline)) {
    walk.template issue<PAD>(key0, ws.any.hi, a.D, lane, lds + buf * S::BUF);
  };
  int key0 = ws.any.lo + wave * 32, buf = 0;
  if (key0 < ws.any.hi) issue(key0, 0);
  for (; key0 < ws.any.hi; key0 += 128) {
    const bool more = key0 + 128 < ws.any.hi;
    if (S::NB == 2 && more) { issue(key0 + 128, buf ^ 1); wait_dma<S::NP>(); }
    else wait_dma<0>();
    f.any_tile(ws, lds + buf * S::BUF, lds + buf * S::BUF + S::IMG, key0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S::NB == 2) buf ^= 1;
    else if (more) issue(key0 + 128, 0);
  }
  f.ds.undo(f.dq);
  if (O::SZ == 2 && f.low) f.bad |= not_finite(f.dq, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kb, vb, ws.any.lo + wave * 32, 128, ws.any.hi);
  if (f.own.hi == 0) {           // rows of no sequence rode along in unmasked tiles
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) f.dq[dt] = zero16();
  }
  store_joined<O, DP>(reinterpret_cast<float*>(smem), f.dq, a.dq + (size_t)head * a.D * O::SZ, row0, own.end - row0, (long)a.Hq * a.D,
                      a.scale, a.D, wave, lane);
}

// ------------------------------------------------------------------------------------------------ dK, dV
// VL: the wave's own V rows as an image in LDS instead of registers: 16-bit D = 128 then fits two waves on a SIMD, whose products and
// exponentials overlap (2 x 8192 causal, 16 heads on 4: 1.29 ms; one wave with everything in registers: 2.2).  There is no room for second
// operands there: 2 x 2048 112 us, with them behind their branch 122.
template <int DT, int DP, bool VL>
struct Dkv {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typename O::Frag kf[DP / 16], vf[VL ? 1 : DP / 16];
  uint32_t vimg;
  f32x16_t dk[DP / 32], dv[DP / 32];
  Span own;
  float c;
  int lane;
  uint32_t rpart, cpart;
  bool bad = false;        // a tile with masked places held a value that is not finite
  DsScale<DT> ds;
  bool low = false;        // dS's second operand: see accumulate()

  __device__ __forceinline__ void start(const BwdArgs& a, int kh, int row, int lane_, char* own_v) {
    lane = lane_;
    rpart = I::row_part(lane);
    cpart = I::col_part(lane);
    c = a.c;
    const int rr = min(row, a.T - 1);
    load_row<O, DP>(kf, a.k + (long)rr * a.ldk + kh * a.hsk, a.D, lane >> 5);
    if constexpr (VL) {
      typename O::Frag x[DP / 16];
      load_row<O, DP>(x, a.v + (long)rr * a.ldv + kh * a.hsv, a.D, lane >> 5);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) *reinterpret_cast<typename O::Frag*>(own_v + I::off(lane & 31, 2 * ks + (lane >> 5))) = x[ks];
      vimg = lds_addr(own_v);
    } else {
      load_row<O, DP>(vf, a.v + (long)rr * a.ldv + kh * a.hsv, a.D, lane >> 5);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(vf[ks]));
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) { dk[dt] = zero16(); dv[dt] = zero16(); }
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(kf[ks]));
  }
  // soff: the tile's row statistics in LDS, planes of `plane` bytes: exponent offset, delta, (fp32: 1 / l)
  __device__ __forceinline__ void tile(uint32_t iq, uint32_t id, uint32_t soff, int plane, int q0, bool mask) {
    const uint32_t rq = launder(rpart + iq), rd = launder(rpart + id), cq = launder(cpart + iq), cd = launder(cpart + id);
    f32x16_t s = zero16(), dp = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(rq, ks), kf[ks], s);
    const uint32_t ro = VL ? launder(rpart + vimg) : 0;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) dp = O::mma(I::rows(rd, ks), VL ? I::rows(ro, ks) : vf[VL ? 0 : ks], dp);
    const uint32_t at = launder(soff + 16 * (lane >> 5));
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4_t off = lds_read<f32x4_t>(at + 32 * g), dl = lds_read<f32x4_t>(at + plane + 32 * g);
      f32x4_t inv = {1.f, 1.f, 1.f, 1.f};
      if constexpr (DT == MVF_F32) inv = lds_read<f32x4_t>(at + 2 * plane + 32 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * g + j;
        float p = __builtin_amdgcn_exp2f(fmaf(s[e], c, off[j]));
        if constexpr (DT == MVF_F32) p *= inv[j];
        s[e] = p;
        dp[e] = p * (dp[e] - dl[j]);
      }
    }
    if (mask) {
      bad |= tile_nonfinite<O, DP>(id, lane) | tile_nonfinite<O, DP>(iq, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int q = q0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        const bool sees = q >= own.lo && q < own.hi;
        s[e] = sees ? s[e] : 0.f;
        dp[e] = sees ? dp[e] : 0.f;
      }
    }
    accumulate_if<O, DP>(!VL && low, dv, s, cd);
    ds.fit(dp, dk);
    accumulate_if<O, DP>(!VL && low, dk, dp, cq);
  }
  // over tiles it = first, first + step, ... of (head h0 + .. of g, 32-query tile, of which a head has a multiple of `per`)
  __device__ __forceinline__ void slow(const BwdArgs& a, int kh, int row, int h0, int g, Span any, int first, int step, int per = 1) {
    typename O::Frag vf[DP / 16];
    load_row<O, DP>(vf, a.v + (long)min(row, a.T - 1) * a.ldv + kh * a.hsv, a.D, lane >> 5);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) { dk[dt] = zero16(); dv[dt] = zero16(); }
    const int nt = (((any.hi - any.lo + 31) >> 5) + per - 1) / per * per;
#pragma unroll 1
    for (int it = first; it < nt * g; it += step) {
      const int h = h0 + it / nt, q0 = any.lo + it % nt * 32;
#pragma unroll 1
      for (int q = q0; q < min(q0 + 32, any.hi); ++q) {
        const char *qr = a.q + (long)q * a.ldq + h * a.hsq, *dr = a.d_out + ((size_t)q * a.Hq + h) * a.D * O::SZ;
        const float s = slow_dot<O, DP>(kf, qr, a.D, lane >> 5), dp = slow_dot<O, DP>(vf, dr, a.D, lane >> 5);
        if (q < own.lo || q >= own.hi) continue;
        const size_t at = (size_t)h * a.T + q;
        const float p = __builtin_amdgcn_exp2f(fmaf(s, c, a.stat[at])) * (DT == MVF_F32 ? a.stat[(size_t)a.Hq * a.T + at] : 1.f);
        slow_add<O, DP>(dv, p, dr, a.D, lane >> 5);
        slow_add<O, DP>(dk, p * (dp - a.delta[at]), qr, a.D, lane >> 5);
      }
    }
  }
  __device__ __forceinline__ void any_tile(const WaveSpan& ws, uint32_t iq, uint32_t id, uint32_t soff, int plane, int q0) {
    if (q0 >= ws.any.hi || q0 + 32 <= ws.any.lo) return;
    tile(iq, id, soff, plane, q0, q0 < ws.all.lo || q0 + 32 > ws.all.hi);
  }
};

constexpr int planes(int dt) { return dt == MVF_F32 ? 3 : 2; }
// float f of the statistics of rows row .. row + n of head h: plane f / n (offset, delta, 1 / l), row f % n
__device__ __forceinline__ const float* stat_at(const BwdArgs& a, int h, int row, int f, int n) {
  const int plane = f / n;
  const float* base = plane == 1 ? a.delta : plane == 0 ? a.stat : a.stat + (size_t)a.Hq * a.T;
  return base + (size_t)h * a.T + min(row + f % n, a.T - 1);
}

template <int DT, int DP>
constexpr bool V_IN_LDS = DT != MVF_F32 && DP == 128;
template <int DT, int DP, int H>
using DkvRing = Ring<Op<DT>, DP, V_IN_LDS<DT, DP> ? 2 : 3, 4 * H>;

template <int DT, int DP, bool PAD, int H>
__global__ __launch_bounds__(256 * H, DT == MVF_F32 && DP > 32 ? H : 2) void packed_attn_dkv_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typedef DkvRing<DT, DP, H> R;
  constexpr bool VL = V_IN_LDS<DT, DP>;
  constexpr int NF = planes(DT) * R::KB, SB = (NF + 63) / 64 * 256;     // floats of a block's statistics, bytes of their buffer
  static_assert(NF <= 256, "one piece per wave");
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ int s_span[8 * H];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit u = xcd_unit(a.Hk * a.parts, a.ntiles, a.level);
  if (u.head < 0) return;
  const int kh = u.head / a.parts, part = u.head % a.parts;
  const OwnTile own = find_tile<128>(a.cu, a.n_seqs, a.T, u.tile, a.ntiles, a.frame == 0 ? Walk::ALL : Walk::EARLY);
  if (own.row0 >= own.end) return;
  const int row = own.row0 + (wave & 3) * 32 + (lane & 31);
  Dkv<DT, DP, VL> f;
  f.start(a, kh, row, lane, smem + R::NB * (R::BUF + SB) + (wave & 3) * 32 * I::RB);      // (two waves write the same V rows)
  f.own = queries_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws);
  if constexpr (PAD) clear_lds(smem, R::NB * R::BUF);
  const Span span = block_span(ws, s_span, lane, wave, 4 * H);
  const int g = a.Hq / a.Hk / a.parts, h0 = kh * (a.Hq / a.Hk) + part * g;
  const int nblk = span.hi > span.lo ? (span.hi - span.lo + R::KB - 1) / R::KB : 0, total = nblk * g;
  const uint32_t lds0 = lds_addr(smem), stat0 = lds0 + R::NB * R::BUF;
  const int sp = min(wave, SB / 256 - 1);                                 // (a wave without a piece of its own repeats the last one)
  R ring;
  int ih = h0, ib = 0;                                                    // head and block that are asked for next
  auto issue = [&](int buf) __attribute__((always_inline)) {
    if (ib == 0)
      ring.start(a.q + ih * a.hsq, a.ldq, a.d_out + (size_t)ih * a.D * O::SZ, (long)a.Hq * a.D * O::SZ, span.lo, a.D, wave, lane, lds0);
    const int b0 = span.lo + ib * R::KB;
    ring.template issue<PAD>(b0, span.hi, buf, wave, lane);
    dma4(stat_at(a, ih, b0, min(sp * 64 + lane, NF - 1), R::KB), stat0 + buf * SB + sp * 256);
    if (++ib == nblk) { ib = 0; ++ih; }
  };
  if (total > 0) issue(0);
  if (R::NB == 3 && total > 1) issue(1);
  int buf = 0, b0 = span.lo;
  for (int it = 0; it < total; ++it) {
    if (R::NB == 3 && it + 1 < total) wait_dma<R::PP + 1>();
    else wait_dma<0>();
    __builtin_amdgcn_s_barrier();
    if (it + R::NB - 1 < total) issue(buf == 0 ? R::NB - 1 : buf - 1);
    const uint32_t iq = lds0 + buf * R::BUF, so = stat0 + buf * SB;
#pragma unroll 1
    for (int t = wave >> 2; t < R::KB / 32; t += H)
      f.any_tile(ws, iq + t * 32 * I::RB, iq + R::IMG + t * 32 * I::RB, so + t * 128, R::KB * 4, b0 + 32 * t);
    buf = buf == R::NB - 1 ? 0 : buf + 1;
    b0 += R::KB;
    if (b0 >= span.hi) b0 = span.lo;
  }
  f.ds.undo(f.dk);
  if (O::SZ == 2 && !VL && f.low) f.bad |= not_finite(f.dk, f.own.hi > f.own.lo) | not_finite(f.dv, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kh, row, h0, g, {span.lo, ws.any.hi}, wave >> 2, H, H);
  if constexpr (H == 2) {
    char* half = smem + (wave & 3) * HALF<DP> + lane * 16;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
      if (wave >= 4) put_half<DP>(half, i == 0 ? f.dk : f.dv);
      __syncthreads();
      if (wave < 4) add_half<DP>(half, i == 0 ? f.dk : f.dv);
    }
    if (wave >= 4) return;
  }
  if (row >= own.end) return;
  const size_t at = ((size_t)row * a.Hk + kh) * a.D;
  if (a.parts > 1) {
    const size_t plane = (size_t)a.T * a.Hk * a.D;
    char* base = reinterpret_cast<char*>(a.part + 2 * part * plane);
    store_rows<Part, DP>(base, at, f.dk, a.scale, f.own.hi > 0, a.D, lane >> 5);
    store_rows<Part, DP>(base, plane + at, f.dv, a.pinv, f.own.hi > 0, a.D, lane >> 5);
  } else {
    store_rows<O, DP>(a.dk, at, f.dk, a.scale, f.own.hi > 0, a.D, lane >> 5);
    store_rows<O, DP>(a.dv, at, f.dv, a.pinv, f.own.hi > 0, a.D, lane >> 5);
  }
}

template <int DT, int DP, bool PAD>
__global__ __launch_bounds__(256, DT != MVF_F32 && DP <= 64 ? 2 : 1) void packed_attn_dkv_split_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef SplitTiles<O, DP, 4> S;
  constexpr int NF = planes(DT) * 32, NSP = (NF + 63) / 64, SB = NSP * 256;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit u = xcd_unit(a.Hk * a.parts, a.ntiles);
  if (u.head < 0) return;
  const int kh = u.head / a.parts, part = u.head % a.parts;
  const OwnTile own = find_tile<32>(a.cu, a.n_seqs, a.T, u.tile, a.ntiles, a.frame == 0 ? Walk::ALL : Walk::EARLY);
  if (own.row0 >= own.end) return;
  const int row0 = own.row0, row = row0 + (lane & 31);
  Dkv<DT, DP, false> f;
  f.start(a, kh, row, lane, nullptr);
  f.own = queries_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws);
  if constexpr (PAD) clear_lds(smem, 4 * S::NB * S::BUF);
  const int g = a.Hq / a.Hk / a.parts, h0 = kh * (a.Hq / a.Hk) + part * g, nt = (ws.any.hi - ws.any.lo + 31) >> 5, total = nt * g;
  const uint32_t lds = lds_addr(smem) + wave * S::NB * S::BUF, stat0 = lds_addr(smem) + 4 * S::NB * S::BUF + wave * S::NB * SB;
  TileWalk<O, DP, 4, S> walk;
  int ih = -1, it = wave;                      // the next tile: it of head ih's, wave by wave through (head, tile)
  auto issue = [&](int n, int buf) __attribute__((always_inline)) {
    const int h = h0 + n / nt, q0 = ws.any.lo + n % nt * 32;
    if (h != ih) {
      ih = h;
      walk.start(a.q + h * a.hsq, a.ldq, a.d_out + (size_t)h * a.D * O::SZ, (long)a.Hq * a.D * O::SZ, q0, lane);
    }
    walk.template issue<PAD>(q0, ws.any.hi, a.D, lane, lds + buf * S::BUF);
#pragma unroll
    for (int j = 0; j < NSP; ++j) dma4(stat_at(a, h, q0, min(j * 64 + lane, NF - 1), 32), stat0 + buf * SB + j * 256);
  };
  int buf = 0;
  if (it < total) issue(it, 0);
  for (; it < total; it += 4) {
    const bool more = it + 4 < total;
    if (S::NB == 2 && more) { issue(it + 4, buf ^ 1); wait_dma<S::NP + NSP>(); }
    else wait_dma<0>();
    f.any_tile(ws, lds + buf * S::BUF, lds + buf * S::BUF + S::IMG, stat0 + buf * SB, 128, ws.any.lo + it % nt * 32);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S::NB == 2) buf ^= 1;
    else if (more) issue(it + 4, 0);
  }
  f.ds.undo(f.dk);
  if (O::SZ == 2 && f.low) f.bad |= not_finite(f.dk, f.own.hi > f.own.lo) | not_finite(f.dv, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kh, row, h0, g, ws.any, wave, 4);
  if (f.own.hi == 0) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) { f.dk[dt] = zero16(); f.dv[dt] = zero16(); }
  }
  const int rows = own.end - row0;
  float* so = reinterpret_cast<float*>(smem);
  if (a.parts > 1) {
    const size_t plane = (size_t)a.T * a.Hk * a.D;
    float* base = a.part + 2 * part * plane + (size_t)kh * a.D;
    store_joined<Part, DP>(so, f.dk, reinterpret_cast<char*>(base), row0, rows, (long)a.Hk * a.D, a.scale, a.D, wave, lane);
    store_joined<Part, DP>(so, f.dv, reinterpret_cast<char*>(base + plane), row0, rows, (long)a.Hk * a.D, a.pinv, a.D, wave, lane);
  } else {
    store_joined<O, DP>(so, f.dk, a.dk + (size_t)kh * a.D * O::SZ, row0, rows, (long)a.Hk * a.D, a.scale, a.D, wave, lane);
    store_joined<O, DP>(so, f.dv, a.dv + (size_t)kh * a.D * O::SZ, row0, rows, (long)a.Hk * a.D, a.pinv, a.D, wave, lane);
  }
}

// dk and dv from the parts, added in order: n elements each (a multiple of 4)
template <int DT>
__global__ __launch_bounds__(256) void packed_attn_sum_kernel(const float* part, int parts, size_t n, char* dk, char* dv) {
  typedef Op<DT> O;
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= 2 * n) return;
  f32x4_t acc = *reinterpret_cast<const f32x4_t*>(part + i);
  for (int p = 1; p < parts; ++p) acc += *reinterpret_cast<const f32x4_t*>(part + 2 * n * p + i);
  O::store4(reinterpret_cast<typename O::E*>(i < n ? dk : dv) + (i < n ? i : i - n), acc[0], acc[1], acc[2], acc[3]);
}

// Into how many parts a group's heads are cut in the dK / dV kernel: the smallest divisor that gives it four workgroups for each of the 256
// compute units (causal walks are of all lengths), or all of them.  2 x 8192 bf16 D 128 16/4 heads: 1 part 3.19 ms, 4 parts 1.32 + 0.03;
// 1 x 2048: 436 us (dQ included), 175.  The parts' fp32 sums cost 16 bytes an element and part, so short walks only fill the units once
// (16 x 64 D 128 32/8: 4 parts 65 us, 1 part 44).
int head_parts(long T, long n_seqs, int Hq, int Hk, int dtype) {
  const int g = Hq / Hk;
  const bool split = use_split(tile_bound<128>(T, n_seqs) * Hq, dtype, T, n_seqs, false);     // near enough: any number of parts is right
  const long units = (split ? tile_bound<32>(T, n_seqs) : tile_bound<128>(T, n_seqs)) * Hk, want = T >= 512 * n_seqs ? 1024 : 256;
  for (int p = 1; p < g; ++p)
    if (g % p == 0 && units * p >= want) return p;
  return g;
}

template <int DT, int DP, bool PAD, int H>
int launch_dq(BwdArgs a, hipStream_t st) {
  typedef Ring<Op<DT>, DP, 3, 4 * H> R;
  constexpr size_t lds = R::NB * R::BUF;
  static_assert(H == 1 || lds >= 4 * HALF<DP>);
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dq_kernel<DT, DP, PAD, H>), lds, attr)) return rc;
  static long holds = 0;
  const unsigned grid = xcd_grid(a.Hq, a.ntiles);
  a.level = grid <= card_holds(reinterpret_cast<const void*>(packed_attn_dq_kernel<DT, DP, PAD, H>), 256 * H, lds, holds);
  hipLaunchKernelGGL((packed_attn_dq_kernel<DT, DP, PAD, H>), dim3(grid), dim3(256 * H), lds, st, a);
  return MVF_OK;
}
template <int DT, int DP, bool PAD, int H>
int launch_dkv(BwdArgs a, hipStream_t st) {
  typedef DkvRing<DT, DP, H> R;
  constexpr size_t lds = R::NB * (R::BUF + (planes(DT) * R::KB + 63) / 64 * 256) + (V_IN_LDS<DT, DP> ? 128 * Img<Op<DT>, DP>::RB : 0);
  static_assert(H == 1 || lds >= 4 * HALF<DP>);
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dkv_kernel<DT, DP, PAD, H>), lds, attr)) return rc;
  static long holds = 0;
  const unsigned grid = xcd_grid((long)a.Hk * a.parts, a.ntiles);
  a.level = grid <= card_holds(reinterpret_cast<const void*>(packed_attn_dkv_kernel<DT, DP, PAD, H>), 256 * H, lds, holds);
  hipLaunchKernelGGL((packed_attn_dkv_kernel<DT, DP, PAD, H>), dim3(grid), dim3(256 * H), lds, st, a);
  return MVF_OK;
}
template <int DT, int DP, bool PAD>
int launch(BwdArgs a, hipStream_t st) {
  typedef SplitTiles<Op<DT>, DP, 4> S;
  constexpr int H = PAIRS<Op<DT>, DP> ? 2 : 1;
  static uint64_t attr[2] = {0, 0};
  const bool pairs = PAIRS<Op<DT>, DP> && use_pairs(a.T, a.n_seqs, a.Hq, a.frame);
  const bool split = use_split(tile_bound<128>(a.T, a.n_seqs) * a.Hq, DT, a.T, a.n_seqs, pairs);
  a.ntiles = (int)(split ? tile_bound<32>(a.T, a.n_seqs) : tile_bound<128>(a.T, a.n_seqs));
  if (split) {
    const size_t lds = std::max(4 * S::NB * S::BUF, (JOIN_BYTES<DP>));
    if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dq_split_kernel<DT, DP, PAD>), lds, attr[0])) return rc;
    hipLaunchKernelGGL((packed_attn_dq_split_kernel<DT, DP, PAD>), dim3(xcd_grid(a.Hq, a.ntiles)), dim3(256), lds, st, a);
  } else {
    if (int rc = pairs ? launch_dq<DT, DP, PAD, H>(a, st) : launch_dq<DT, DP, PAD, 1>(a, st)) return rc;
  }
  MVF_LAUNCH_CHECK();
  if (split) {
    const size_t lds = std::max(4 * S::NB * (S::BUF + (planes(DT) * 32 + 63) / 64 * 256), (JOIN_BYTES<DP>));
    if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dkv_split_kernel<DT, DP, PAD>), lds, attr[1])) return rc;
    hipLaunchKernelGGL((packed_attn_dkv_split_kernel<DT, DP, PAD>), dim3(xcd_grid((long)a.Hk * a.parts, a.ntiles)), dim3(256), lds, st, a);
  } else {
    const bool two = use_pairs(a.T, a.n_seqs, (long)a.Hk * a.parts, a.frame);
    if (int rc = two ? launch_dkv<DT, DP, PAD, H>(a, st) : launch_dkv<DT, DP, PAD, 1>(a, st)) return rc;
  }
  MVF_LAUNCH_CHECK();
  if (a.parts > 1) {
    const size_t n = (size_t)a.T * a.Hk * a.D;
    hipLaunchKernelGGL((packed_attn_sum_kernel<DT>), dim3((unsigned)((2 * n / 4 + 255) / 256)), dim3(256), 0, st, a.part, a.parts, n, a.dk, a.dv);
    MVF_LAUNCH_CHECK();
  }
  return MVF_OK;
}
template <int DT, int DP>
int launch_p(const BwdArgs& a, hipStream_t st) { return a.D == DP ? launch<DT, DP, false>(a, st) : launch<DT, DP, true>(a, st); }
template <int DT>
int launch_d(const BwdArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch_p<DT, 32>(a, st) : a.D <= 64 ? launch_p<DT, 64>(a, st) : a.D <= 96 ? launch_p<DT, 96>(a, st) : launch_p<DT, 128>(a, st);
}

}  // namespace

extern "C" size_t mvf_packed_attn_bwd_workspace_bytes(int dtype, int T, int n_seqs, int Hq, int Hk, int D) {
  if (T <= 0 || n_seqs <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || D <= 0) return 0;
  const size_t delta = ((size_t)Hq * T + 3) / 4 * 4;
  const int parts = head_parts(T, n_seqs, Hq, Hk, dtype);
  return (delta + (parts > 1 ? 2 * parts * (size_t)T * Hk * D : 0)) * sizeof(float);
}

extern "C" int mvf_packed_attn_bwd(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                   long ldv, long hsv, const int* cu_seqlens, int n_seqs, const void* out, const void* d_out,
                                   const float* stat, void* workspace, size_t ws_bytes, void* dq, void* dk, void* dv, int T, int Hq, int Hk,
                                   int D, int frame, float scale, hipStream_t st) {
  return mvf_packed_attn_bwd_rest(dtype, q, ldq, hsq, k, ldk, hsk, v, ldv, hsv, cu_seqlens, n_seqs, out, nullptr, d_out, stat, workspace,
                                  ws_bytes, dq, dk, dv, T, Hq, Hk, D, frame, scale, st);
}

extern "C" int mvf_packed_attn_bwd_rest(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                        long ldv, long hsv, const int* cu_seqlens, int n_seqs, const void* out, const void* rest,
                                        const void* d_out, const float* stat, void* workspace, size_t ws_bytes, void* dq, void* dk,
                                        void* dv, int T, int Hq, int Hk, int D, int frame, float scale, hipStream_t st) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && k && v && cu_seqlens && out && d_out && stat && workspace && dq && dk && dv);
  MVF_CHECK_ARG(T > 0 && n_seqs > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && frame >= 0);
  MVF_CHECK_ARG(scale > 0.f && scale < 1e30f && T < (1 << 30) && tile_bound<32>(T, n_seqs) * Hq < (1l << 30));
  if (D <= 0 || D > 128 || D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  const long s[6] = {ldq * sz, hsq * sz, ldk * sz, hsk * sz, ldv * sz, hsv * sz};
  for (long x : s) MVF_CHECK_ARG(x > 0 && x % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk |
                  (uintptr_t)dv | (uintptr_t)workspace | (uintptr_t)rest) & 15) == 0);
  MVF_CHECK_ARG(ws_bytes >= mvf_packed_attn_bwd_workspace_bytes(dtype, T, n_seqs, Hq, Hk, D));
  float* delta = (float*)workspace;
  const int parts = head_parts(T, n_seqs, Hq, Hk, dtype);
  MVF_CHECK_ARG(tile_bound<32>(T, n_seqs) * Hk * parts < (1l << 30) && (size_t)T * Hk * D / 512 < (1ul << 31));
  BwdArgs a = {(const char*)q, (const char*)k, (const char*)v, s[0], s[1], s[2], s[3], s[4], s[5], cu_seqlens, n_seqs, (const char*)out,
               (const char*)rest, (const char*)d_out, stat, delta, delta + ((size_t)Hq * T + 3) / 4 * 4, parts, (char*)dq, (char*)dk, (char*)dv, T, Hq, Hk, D,
               frame, 0, 0, scale * LOG2E, scale * (dtype == MVF_F16 ? 1.f / (1 << PSHIFT) : 1.f), dtype == MVF_F16 ? 1.f / (1 << PSHIFT) : 1.f};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
