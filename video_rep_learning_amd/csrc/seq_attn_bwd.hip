// Backward of seq_attn.hip.  With P the probabilities (recomputed from the forward's row statistics) and dP = dO V^T:
//   dV = P^T dO,   dS = P o (dP - delta),  delta = rowsum(dO o O),   dQ = scale dS K,   dK = scale dS^T Q,
// dK and dV summed over the query heads of a group.  Two kernels, each owning what it writes, so no atomics and the same bits every time:
//   dQ:     owns 32 queries per wave, streams K and V;       also writes delta, which the second kernel reads
//   dK/dV:  owns 32 keys per wave, streams Q and dO of every head of the group (the sum over the group stays in registers)
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using namespace seq_attn;

struct BwdArgs {
  const char *q, *k, *v;
  long ldq, hsq, ldk, hsk, ldv, hsv;   // token and head strides in BYTES
  const int* cu;
  int n_seqs;
  const char *out, *d_out;             // [T, Hq, D]
  const float* stat;                   // [2][Hq][T] of the forward
  float* delta;                        // [Hq][T]
  char *dq, *dk, *dv;                  // [T, Hq, D], [T, Hk, D] x 2
  int T, Hq, Hk, D, frame, ntiles;
  float c, scale;
};

template <class O, int DP, int ROWS>
__device__ __forceinline__ void stage(char* img, const char* src, long ld, int row0, int end, int D, int tid, int nthreads) {
  typedef Img<O, DP> I;
  for (int i = tid; i < ROWS * I::C; i += nthreads) {
    const int r = i / I::C, ch = i % I::C;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row0 + r < end && ch * 16 < D * O::SZ) x = *reinterpret_cast<const uint4*>(src + (long)(row0 + r) * ld + ch * 16);
    *reinterpret_cast<uint4*>(img + I::off(r, ch)) = x;
  }
}

// a row as the B operand's fragments (zeros where it is not wanted)
template <class O, int DP>
__device__ __forceinline__ void load_row(typename O::Frag (&f)[DP / 16], const char* src, int D, int hh, bool want) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int d = 16 * ks + 8 * hh;
    typename O::Frag x = {};
    if (want && d < D) x = *reinterpret_cast<const typename O::Frag*>(src + d * O::SZ);
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

__device__ __forceinline__ Span block_span(const WaveSpan& ws, int* s_span, int lane, int wave, int nw) {
  if (lane == 0) { s_span[2 * wave] = ws.any.hi > 0 ? ws.any.lo : 0x7fffffff; s_span[2 * wave + 1] = ws.any.hi; }
  __syncthreads();
  Span s = {0x7fffffff, 0};
  for (int w = 0; w < nw; ++w) { s.lo = min(s.lo, s_span[2 * w]); s.hi = max(s.hi, s_span[2 * w + 1]); }
  return s;
}

// ------------------------------------------------------------------------------------------------ dQ
template <int DT, int DP>
__global__ __launch_bounds__(256, 1) void packed_attn_dq_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  constexpr int KROWS = 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_span[8];
  char* sk = smem;
  char* sv = smem + KROWS * I::RB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int r = lane & 31, hh = lane >> 5;
  const int head = blockIdx.x % a.Hq, tile = a.ntiles - 1 - (int)(blockIdx.x / a.Hq);
  const int row = (tile * nw + wave) * 32 + r, rr = min(row, a.T - 1);
  Span own = {0, 0};
  if (row < a.T) own = keys_of(sequence_of(a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(own);
  const Span span = block_span(ws, s_span, lane, wave, nw);
  const bool want = own.hi > 0;
  typename O::Frag qf[DP / 16], dof[DP / 16];
  load_row<O, DP>(qf, a.q + (long)rr * a.ldq + head * a.hsq, a.D, hh, want);
  const size_t orow = ((size_t)rr * a.Hq + head) * a.D * O::SZ;
  load_row<O, DP>(dof, a.d_out + orow, a.D, hh, want);
  float dl = 0.f;
  {
    typename O::Frag of[DP / 16];
    load_row<O, DP>(of, a.out + orow, a.D, hh, want);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) dl = fmaf(O::get(dof[ks], j), O::get(of[ks], j), dl);
    dl = pair_sum(dl);
  }
  const size_t at = (size_t)head * a.T + rr;
  const float off = want ? a.stat[at] : NEG_INF, inv = DT == MVF_F32 && want ? a.stat[(size_t)a.Hq * a.T + at] : 1.f;
  if (row < a.T && hh == 0) a.delta[at] = dl;
  f32x16_t dq[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = zero16();
  const char* kb = a.k + (head / (a.Hq / a.Hk)) * a.hsk;
  const char* vb = a.v + (head / (a.Hq / a.Hk)) * a.hsv;

  auto tile32 = [&](auto mask_tag, int t, int key0) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16_t s = zero16(), dp = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      s = O::mma(I::rows(sk, t * 32, ks, lane), qf[ks], s);
      dp = O::mma(I::rows(sv, t * 32, ks, lane), dof[ks], dp);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int key = key0 + 8 * (e >> 2) + 4 * hh + (e & 3);
      float p = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, off));
      if constexpr (DT == MVF_F32) p *= inv;
      const float ds = p * (dp[e] - dl);
      s[e] = !MASK || (key >= own.lo && key < own.hi) ? ds : 0.f;
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename O::Frag ds = O::pack(s, s2);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = mma_weighted<O, MASK, true>(I::cols(sk, t * 32 + 16 * s2, dt, lane), ds, dq[dt]);
    }
  };
  for (int b0 = span.lo; b0 < span.hi; b0 += KROWS) {
    __syncthreads();
    stage<O, DP, KROWS>(sk, kb, a.ldk, b0, span.hi, a.D, threadIdx.x, blockDim.x);
    stage<O, DP, KROWS>(sv, vb, a.ldv, b0, span.hi, a.D, threadIdx.x, blockDim.x);
    __syncthreads();
    for (int t = 0; t < KROWS / 32; ++t) {
      const int key0 = b0 + 32 * t;
      if (key0 >= ws.any.hi || key0 + 32 <= ws.any.lo) continue;
      if (key0 >= ws.all.lo && key0 + 32 <= ws.all.hi) tile32(std::false_type{}, t, key0);
      else tile32(std::true_type{}, t, key0);
    }
  }
  if (row < a.T) store_rows<O, DP>(a.dq, ((size_t)row * a.Hq + head) * a.D, dq, a.scale, want, a.D, hh);
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <int DT, int DP>
__global__ __launch_bounds__(256, 1) void packed_attn_dkv_kernel(BwdArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  constexpr int QROWS = 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_span[8];
  __shared__ __attribute__((aligned(16))) float s_off[QROWS], s_inv[QROWS], s_dl[QROWS];
  char* sq = smem;
  char* sd = smem + QROWS * I::RB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int r = lane & 31, hh = lane >> 5;
  const int kh = blockIdx.x % a.Hk, tile = blockIdx.x / a.Hk;
  const int row = (tile * nw + wave) * 32 + r, rr = min(row, a.T - 1);
  Span own = {0, 0};
  if (row < a.T) own = queries_of(sequence_of(a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(own);
  const Span span = block_span(ws, s_span, lane, wave, nw);
  const bool want = own.hi > 0;
  typename O::Frag kf[DP / 16], vf[DP / 16];
  load_row<O, DP>(kf, a.k + (long)rr * a.ldk + kh * a.hsk, a.D, hh, want);
  load_row<O, DP>(vf, a.v + (long)rr * a.ldv + kh * a.hsv, a.D, hh, want);
  f32x16_t dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) { dk[dt] = zero16(); dv[dt] = zero16(); }

  auto tile32 = [&](auto mask_tag, int t, int q0) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16_t s = zero16(), dp = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      s = O::mma(I::rows(sq, t * 32, ks, lane), kf[ks], s);
      dp = O::mma(I::rows(sd, t * 32, ks, lane), vf[ks], dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int i = t * 32 + 8 * g + 4 * hh;
      const f32x4_t off = *reinterpret_cast<const f32x4_t*>(s_off + i), dl = *reinterpret_cast<const f32x4_t*>(s_dl + i);
      f32x4_t inv = {1.f, 1.f, 1.f, 1.f};
      if constexpr (DT == MVF_F32) inv = *reinterpret_cast<const f32x4_t*>(s_inv + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * g + j, q = q0 + 8 * g + 4 * hh + j;
        float p = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, off[j]));
        if constexpr (DT == MVF_F32) p *= inv[j];
        const float ds = p * (dp[e] - dl[j]);
        const bool sees = !MASK || (q >= own.lo && q < own.hi);
        s[e] = sees ? p : 0.f;
        dp[e] = sees ? ds : 0.f;
      }
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename O::Frag p = O::pack(s, s2), ds = O::pack(dp, s2);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        dv[dt] = mma_weighted<O, MASK, false>(I::cols(sd, t * 32 + 16 * s2, dt, lane), p, dv[dt]);
        dk[dt] = mma_weighted<O, MASK, true>(I::cols(sq, t * 32 + 16 * s2, dt, lane), ds, dk[dt]);
      }
    }
  };
  const int g = a.Hq / a.Hk;
  for (int h = kh * g; h < (kh + 1) * g; ++h) {
    const char* qb = a.q + h * a.hsq;
    const char* db = a.d_out + (size_t)h * a.D * O::SZ;
    for (int b0 = span.lo; b0 < span.hi; b0 += QROWS) {
      __syncthreads();
      stage<O, DP, QROWS>(sq, qb, a.ldq, b0, span.hi, a.D, threadIdx.x, blockDim.x);
      stage<O, DP, QROWS>(sd, db, (long)a.Hq * a.D * O::SZ, b0, span.hi, a.D, threadIdx.x, blockDim.x);
      if (threadIdx.x < QROWS) {
        const int i = b0 + threadIdx.x;
        const size_t at = (size_t)h * a.T + min(i, a.T - 1);
        s_off[threadIdx.x] = i < span.hi ? a.stat[at] : NEG_INF;
        s_inv[threadIdx.x] = i < span.hi ? a.stat[(size_t)a.Hq * a.T + at] : 0.f;
        s_dl[threadIdx.x] = i < span.hi ? a.delta[at] : 0.f;
      }
      __syncthreads();
      for (int t = 0; t < QROWS / 32; ++t) {
        const int q0 = b0 + 32 * t;
        if (q0 >= ws.any.hi || q0 + 32 <= ws.any.lo) continue;
        if (q0 >= ws.all.lo && q0 + 32 <= ws.all.hi) tile32(std::false_type{}, t, q0);
        else tile32(std::true_type{}, t, q0);
      }
    }
  }
  if (row < a.T) {
    store_rows<O, DP>(a.dk, ((size_t)row * a.Hk + kh) * a.D, dk, a.scale, want, a.D, hh);
    store_rows<O, DP>(a.dv, ((size_t)row * a.Hk + kh) * a.D, dv, 1.f, want, a.D, hh);
  }
}

template <int DT, int DP>
int launch(BwdArgs a, hipStream_t st) {
  const size_t lds = 2 * 64 * Img<Op<DT>, DP>::RB;
  static uint64_t attr1 = 0, attr2 = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dq_kernel<DT, DP>), lds, attr1)) return rc;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_dkv_kernel<DT, DP>), lds, attr2)) return rc;
  const int nw = 4;
  a.ntiles = ceil_div(a.T, 32 * nw);
  hipLaunchKernelGGL((packed_attn_dq_kernel<DT, DP>), dim3((unsigned)a.ntiles * a.Hq), dim3(64 * nw), lds, st, a);
  MVF_LAUNCH_CHECK();
  hipLaunchKernelGGL((packed_attn_dkv_kernel<DT, DP>), dim3((unsigned)a.ntiles * a.Hk), dim3(64 * nw), lds, st, a);
  MVF_LAUNCH_CHECK();
  return MVF_OK;
}
template <int DT>
int launch_d(const BwdArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch<DT, 32>(a, st) : a.D <= 64 ? launch<DT, 64>(a, st) : a.D <= 96 ? launch<DT, 96>(a, st) : launch<DT, 128>(a, st);
}

}  // namespace

extern "C" int mvf_packed_attn_bwd(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                   long ldv, long hsv, const int* cu_seqlens, int n_seqs, const void* out, const void* d_out,
                                   const float* stat, float* delta, void* dq, void* dk, void* dv, int T, int Hq, int Hk, int D, int frame,
                                   float scale, hipStream_t st) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && k && v && cu_seqlens && out && d_out && stat && delta && dq && dk && dv);
  MVF_CHECK_ARG(T > 0 && n_seqs > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && frame >= 0);
  MVF_CHECK_ARG(scale > 0.f && scale < 1e30f && (long)T * Hq < (1l << 36) && (long)ceil_div(T, 32) * Hq < (1l << 31));
  if (D <= 0 || D > 128 || D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  const long s[6] = {ldq * sz, hsq * sz, ldk * sz, hsk * sz, ldv * sz, hsv * sz};
  for (long x : s) MVF_CHECK_ARG(x > 0 && x % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk |
                  (uintptr_t)dv) & 15) == 0);
  BwdArgs a = {(const char*)q, (const char*)k, (const char*)v, s[0], s[1], s[2], s[3], s[4], s[5], cu_seqlens, n_seqs, (const char*)out,
               (const char*)d_out, stat, delta, (char*)dq, (char*)dk, (char*)dv, T, Hq, Hk, D, frame, 0, scale * LOG2E, scale};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
