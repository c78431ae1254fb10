// Self-attention over packed sequences of different lengths, grouped heads, causal by token or by frame:
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / g]) v[j, h / g],   j in i's sequence, j < (i / frame + 1) frame inside it
// Tiles are cut out of the packed rows, not out of each sequence: a tile may hold the end of one sequence and the start of the next,
// every row has its own [lo, hi) of keys, and a tile walks the union.  So nothing but the number of rows sizes the grid (no host copy
// of the lengths), empty sequences cost nothing, short ones share a tile, and rows behind the last sequence come out as zeros.
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using namespace seq_attn;

struct FwdArgs {
  const char *q, *k, *v;
  long ldq, hsq, ldk, hsk, ldv, hsv;   // token and head strides in BYTES
  const int* cu;
  int n_seqs;
  char* out;                           // [T, Hq, D]
  float* stat;                         // NULL, or [2][Hq][T]: see below
  int T, Hq, Hk, D, frame, ntiles;
  float c;                             // scale * log2(e)
};

// rows [row0, row0 + ROWS) of a strided matrix into an image; rows from `end` on and columns from D on are zeros
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

template <int DT, int DP>
__global__ __launch_bounds__(256, 1) void packed_attn_fwd_kernel(FwdArgs a) {
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
  const int row = (tile * nw + wave) * 32 + r;
  Span own = {0, 0};
  if (row < a.T) own = keys_of(sequence_of(a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(own);
  if (lane == 0) { s_span[2 * wave] = ws.any.hi > 0 ? ws.any.lo : 0x7fffffff; s_span[2 * wave + 1] = ws.any.hi; }
  __syncthreads();
  int lo = 0x7fffffff, hi = 0;
  for (int w = 0; w < nw; ++w) { lo = min(lo, s_span[2 * w]); hi = max(hi, s_span[2 * w + 1]); }

  typename O::Frag qf[DP / 16];
  {
    const char* src = a.q + (long)min(row, a.T - 1) * a.ldq + head * a.hsq;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * hh;
      typename O::Frag f = {};
      if (d < a.D && own.hi > 0) f = *reinterpret_cast<const typename O::Frag*>(src + d * O::SZ);
      qf[ks] = f;
    }
  }
  f32x16_t o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
  RowMax st;
  const float thr = 8.f / a.c;
  const char* kb = a.k + (head / (a.Hq / a.Hk)) * a.hsk;
  const char* vb = a.v + (head / (a.Hq / a.Hk)) * a.hsv;

  auto tile32 = [&](auto mask_tag, int t, int key0) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16_t s = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(sk, t * 32, ks, lane), qf[ks], s);
    if constexpr (MASK) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = key0 + 8 * (e >> 2) + 4 * hh + (e & 3);
        s[e] = key >= own.lo && key < own.hi ? s[e] : NEG_INF;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = pair_max(mx);
    float alpha;
    if (st.grow(mx, a.c, thr, alpha)) {
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, st.nm));
      st.l += s[e];
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename O::Frag p = O::pack(s, s2);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) o[dt] = mma_weighted<O, MASK, false>(I::cols(sv, t * 32 + 16 * s2, dt, lane), p, o[dt]);
    }
  };

  for (int b0 = lo; b0 < hi; b0 += KROWS) {
    __syncthreads();
    stage<O, DP, KROWS>(sk, kb, a.ldk, b0, hi, a.D, threadIdx.x, blockDim.x);
    stage<O, DP, KROWS>(sv, vb, a.ldv, b0, hi, a.D, threadIdx.x, blockDim.x);
    __syncthreads();
    for (int t = 0; t < KROWS / 32; ++t) {
      const int key0 = b0 + 32 * t;
      if (key0 >= ws.any.hi || key0 + 32 <= ws.any.lo) continue;
      if (key0 >= ws.all.lo && key0 + 32 <= ws.all.hi) tile32(std::false_type{}, t, key0);
      else tile32(std::true_type{}, t, key0);
    }
  }
  if (row >= a.T) return;
  const float l = pair_sum(st.l);
  const bool some = own.hi > own.lo && l != 0.f;          // (l is NaN where a score was)
  const float inv = some ? 1.0f / l : 0.f;
  // What the backward needs to have the same probabilities again.  fp32: the exponent's offset and 1 / l, applied as here (one log2-sum
  // would round at the size of its integer part: 1e-6 of a probability); 16-bit: one offset that holds both.
  if (a.stat != nullptr && hh == 0) {
    const size_t at = (size_t)head * a.T + row;
    a.stat[at] = !some ? NEG_INF : DT == MVF_F32 ? st.nm : st.nm - __builtin_amdgcn_logf(l);
    a.stat[(size_t)a.Hq * a.T + at] = inv;
  }
  typename O::E* dst = reinterpret_cast<typename O::E*>(a.out) + ((size_t)row * a.Hq + head) * a.D;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < a.D) {
        if (some) O::store4(dst + d, o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv);
        else O::store4(dst + d, 0.f, 0.f, 0.f, 0.f);
      }
    }
}

template <int DT, int DP>
int launch(FwdArgs a, hipStream_t st) {
  const size_t lds = 2 * 64 * Img<Op<DT>, DP>::RB;
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_fwd_kernel<DT, DP>), lds, attr)) return rc;
  const int nw = 4;
  a.ntiles = ceil_div(a.T, 32 * nw);
  hipLaunchKernelGGL((packed_attn_fwd_kernel<DT, DP>), dim3((unsigned)a.ntiles * a.Hq), dim3(64 * nw), lds, st, a);
  MVF_LAUNCH_CHECK();
  return MVF_OK;
}
template <int DT>
int launch_d(const FwdArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch<DT, 32>(a, st) : a.D <= 64 ? launch<DT, 64>(a, st) : a.D <= 96 ? launch<DT, 96>(a, st) : launch<DT, 128>(a, st);
}

}  // namespace

extern "C" int mvf_packed_attn_fwd(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                   long ldv, long hsv, const int* cu_seqlens, int n_seqs, void* out, float* stat, int T, int Hq, int Hk,
                                   int D, int frame, float scale, hipStream_t st) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && k && v && cu_seqlens && out && T > 0 && n_seqs > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && frame >= 0);
  MVF_CHECK_ARG(scale > 0.f && scale < 1e30f && (long)T * Hq < (1l << 36) && (long)ceil_div(T, 32) * Hq < (1l << 31));
  if (D <= 0 || D > 128 || D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  const long s[6] = {ldq * sz, hsq * sz, ldk * sz, hsk * sz, ldv * sz, hsv * sz};
  for (long x : s) MVF_CHECK_ARG(x > 0 && x % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0);
  FwdArgs a = {(const char*)q, (const char*)k, (const char*)v, s[0], s[1], s[2], s[3], s[4], s[5], cu_seqlens, n_seqs, (char*)out, stat,
               T, Hq, Hk, D, frame, 0, scale * LOG2E};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
