// Rotary positions with up to three axes: channel pair p of every head turns by the angle  pos[t, axis(p)] * freq[p],
//   (x0, x1) -> (x0 cos - x1 sin, x1 cos + x0 sin),      backward: the same with the angle negated.
// HBM-bound: every element is read and written once; the angles are computed once per token into LDS and used by all heads.
// The angle is reduced in 64 bits -- turns = pos * freq / (2 pi), minus the nearest quarter -- because at position 10^6 a 32-bit product
// is off by 0.06 rad; what is left (|angle| <= pi / 4) goes through the Taylor polynomials of sin and cos in 32 bits, whose first
// dropped terms are 2e-9 and 1e-10 there.
// The appending form writes the turned keys and the values into pages of a cache instead: token t of stream seq[t] at index[t] goes to
// row index % page of page table[seq][index / page].
// Measured: 50176 tokens, 12 + 12 heads of 64, bf16: 67 us, 4.6 TB/s (a copy of 2 GiB: 4.9); 24 prompts into their pages, 16 + 2 x 2 heads of
// 128, 354 MB: 78 us, 4.5 TB/s; 48 tokens in fp32: 7 us, a launch.
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using seq_attn::Op;

struct RotArgs {
  const char* x[3];       // q, k, v
  long ld[3], hs[3];      // token and head strides in BYTES
  char* y[3];             // q: [T, Hq, D]; k, v: [T, Hk, D] or the caches' pages [n_pages, page, Hk, D]
  int h0, h1, h2;         // heads of q; of q and k; of q, k and v
  const void* pos;        // [T, axes]
  const double* freq;     // [P]
  const int *table, *seq, *index;
  int T, D, P, axes, e0, e1;     // pairs [0, e0) axis 0, [e0, e1) axis 1, [e1, P) axis 2
  int tb, width, n_seqs, n_pages, page;
  float sign;
};

__device__ __forceinline__ float2 cos_sin_of_turns(double turns) {
  const double r = turns - rint(turns);             // [-1/2, 1/2]
  const double q = rint(4.0 * r);                   // nearest quarter
  const float a = (float)((r - 0.25 * q) * 6.283185307179586476925286766559);
  const float z = a * a;
  const float s = a * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int n = (int)q & 3;                         // cos, sin of a + n pi / 2
  const float cc = (n & 1) ? s : c, ss = (n & 1) ? c : s;
  return make_float2((n == 1 || n == 2) ? -cc : cc, (n >= 2) ? -ss : ss);
}

template <int N>
struct Bytes { uint32_t u[N / 4]; };
template <int N>
__device__ __forceinline__ void copy_bytes(void* d, const void* s) {
  if constexpr (N >= 16) {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) reinterpret_cast<uint4*>(d)[i] = reinterpret_cast<const uint4*>(s)[i];
  } else if constexpr (N == 8) {
    *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(s);
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(s);
  } else {
    *reinterpret_cast<uint16_t*>(d) = *reinterpret_cast<const uint16_t*>(s);
  }
}

template <int DT>
__device__ __forceinline__ float ld1(const void* p) {
  if constexpr (DT == MVF_F32) return *reinterpret_cast<const float*>(p);
  else return DT == MVF_F16 ? f16_to_f32(*reinterpret_cast<const uint16_t*>(p)) : bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
}
template <int DT>
__device__ __forceinline__ void st1(void* p, float v) {
  if constexpr (DT == MVF_F32) *reinterpret_cast<float*>(p) = v;
  else *reinterpret_cast<uint16_t*>(p) = DT == MVF_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}

// V pairs per item; IL: pair p is channels 2p, 2p + 1, else p, P + p; POS: 0 int32, 1 int64, 2 float32; PAGED: the appending form
template <int DT, int V, bool IL, int POS, bool PAGED>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
  constexpr int SZ = DT == MVF_F32 ? 4 : 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2* cs = reinterpret_cast<float2*>(smem);                        // [tb][P]
  long* slot = reinterpret_cast<long*>(smem + (size_t)a.tb * a.P * 8);  // [tb] cache row of a token, -1: none
  const int t0 = blockIdx.x * a.tb, nt = min(a.tb, a.T - t0);
  for (int i = threadIdx.x; i < nt * a.P; i += 256) {
    const int t = i / a.P, p = i % a.P;
    const int axis = (p >= a.e0) + (p >= a.e1);
    const size_t at = (size_t)(t0 + t) * a.axes + axis;
    const double x = POS == 0 ? (double)reinterpret_cast<const int*>(a.pos)[at] :
                     POS == 1 ? (double)reinterpret_cast<const long long*>(a.pos)[at] : (double)reinterpret_cast<const float*>(a.pos)[at];
    float2 v = cos_sin_of_turns(x * a.freq[p] * 0.15915494309189533576888376337251);
    v.y *= a.sign;
    cs[i] = v;
  }
  if constexpr (PAGED)
    for (int t = threadIdx.x; t < nt; t += 256) {
      const int b = a.seq[t0 + t], i = a.index[t0 + t];
      long s = -1;
      if (b >= 0 && b < a.n_seqs && i >= 0 && i / a.page < a.width) {
        const int pg = a.table[(long)b * a.width + i / a.page];
        if (pg >= 0 && pg < a.n_pages) s = (long)pg * a.page + i % a.page;
      }
      slot[t] = s;
    }
  __syncthreads();
  const int np = a.P / V, items = np + (a.D - 2 * a.P) / V, per = a.h2 * items;
  for (int i = threadIdx.x; i < nt * per; i += 256) {
    const int t = i / per, rem = i % per, hd = rem / items, it = rem % items;
    const int w = (hd >= a.h0) + (hd >= a.h1), h = hd - (w == 0 ? 0 : w == 1 ? a.h0 : a.h1);
    const int nh = w == 0 ? a.h0 : a.h1 - a.h0;
    const char* src = a.x[w] + (long)(t0 + t) * a.ld[w] + h * a.hs[w];
    long row = t0 + t;
    if (PAGED && w > 0) {
      row = slot[t];
      if (row < 0) continue;
    }
    char* dst = a.y[w] + (row * nh + h) * (long)a.D * SZ;
    if (it >= np) {                                // channels behind the turned ones
      const int d = 2 * a.P + (it - np) * V;
      copy_bytes<V * SZ>(dst + d * SZ, src + d * SZ);
      continue;
    }
    const int d0 = IL ? 2 * it * V : it * V, d1 = IL ? d0 + V : a.P + it * V;
    __attribute__((aligned(16))) char in[2 * V * SZ], out[2 * V * SZ];
    copy_bytes<V * SZ>(in, src + d0 * SZ);
    copy_bytes<V * SZ>(in + V * SZ, src + d1 * SZ);
    if (PAGED && w == 2) {                         // values go in as they are
      copy_bytes<V * SZ>(dst + d0 * SZ, in);
      copy_bytes<V * SZ>(dst + d1 * SZ, in + V * SZ);
      continue;
    }
    const float2* c = cs + t * a.P + it * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i0 = IL ? 2 * j : j, i1 = IL ? 2 * j + 1 : V + j;
      const float x0 = ld1<DT>(in + i0 * SZ), x1 = ld1<DT>(in + i1 * SZ);
      st1<DT>(out + i0 * SZ, x0 * c[j].x - x1 * c[j].y);
      st1<DT>(out + i1 * SZ, x1 * c[j].x + x0 * c[j].y);
    }
    copy_bytes<V * SZ>(dst + d0 * SZ, out);
    copy_bytes<V * SZ>(dst + d1 * SZ, out + V * SZ);
  }
}

template <int DT, int V, bool IL, bool PAGED>
int launch(RotArgs a, int pos_type, hipStream_t st) {
  // tokens per workgroup: about four items per thread, and the angles within 32 KB
  const int per = a.h2 * (a.P / V + (a.D - 2 * a.P) / V);
  a.tb = std::max(1, std::min({1024 / std::max(per, 1), 32768 / (8 * a.P), a.T}));
  const dim3 grid((unsigned)ceil_div(a.T, a.tb));
  const size_t lds = (size_t)a.tb * (8 * a.P + 8);
  if (pos_type == 0) hipLaunchKernelGGL((rotary_kernel<DT, V, IL, 0, PAGED>), grid, dim3(256), lds, st, a);
  else if (pos_type == 1) hipLaunchKernelGGL((rotary_kernel<DT, V, IL, 1, PAGED>), grid, dim3(256), lds, st, a);
  else hipLaunchKernelGGL((rotary_kernel<DT, V, IL, 2, PAGED>), grid, dim3(256), lds, st, a);
  MVF_LAUNCH_CHECK();
  return MVF_OK;
}
template <int DT, bool PAGED>
int launch_v(const RotArgs& a, int il, int pos_type, hipStream_t st) {
  const int v = a.P % 8 == 0 ? 8 : a.P % 4 == 0 ? 4 : 1;       // pairs per item that the rows' alignment and the pair count allow
  if (v == 8) return il ? launch<DT, 8, true, PAGED>(a, pos_type, st) : launch<DT, 8, false, PAGED>(a, pos_type, st);
  if (v == 4) return il ? launch<DT, 4, true, PAGED>(a, pos_type, st) : launch<DT, 4, false, PAGED>(a, pos_type, st);
  return il ? launch<DT, 1, true, PAGED>(a, pos_type, st) : launch<DT, 1, false, PAGED>(a, pos_type, st);
}

int fill(RotArgs& a, int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* pos, int pos_type,
         const double* freqs, int s0, int s1, int s2, int T, int Hq, int Hk, int D) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && pos && freqs && pos_type >= 0 && pos_type <= 2 && T > 0 && Hq > 0 && Hk >= 0 && (k || Hk == 0));
  MVF_CHECK_ARG(s0 > 0 && s1 >= 0 && s2 >= 0 && (s1 > 0 || s2 == 0));
  MVF_CHECK_ARG(D > 0 && D <= 4096 && (long)s0 + s1 + s2 <= D / 2 && (long)Hq + 2l * Hk <= 65536);
  if (D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  MVF_CHECK_ARG(ldq > 0 && hsq > 0 && ldq * sz % 16 == 0 && hsq * sz % 16 == 0 && ((uintptr_t)q & 15) == 0);
  MVF_CHECK_ARG(Hk == 0 || (ldk > 0 && hsk > 0 && ldk * sz % 16 == 0 && hsk * sz % 16 == 0 && ((uintptr_t)k & 15) == 0));
  a = {};
  a.x[0] = (const char*)q; a.ld[0] = ldq * sz; a.hs[0] = hsq * sz;
  a.x[1] = (const char*)k; a.ld[1] = ldk * sz; a.hs[1] = hsk * sz;
  a.h0 = Hq; a.h1 = a.h2 = Hq + Hk;
  a.pos = pos; a.freq = freqs;
  a.T = T; a.D = D; a.P = s0 + s1 + s2; a.e0 = s0; a.e1 = s0 + s1;
  a.axes = 1 + (s1 > 0) + (s2 > 0);
  return MVF_OK;
}

}  // namespace

extern "C" int mvf_rotary(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* pos, int pos_type,
                          const double* freqs, int s0, int s1, int s2, int interleaved, int inverse, void* q_out, void* k_out, int T,
                          int Hq, int Hk, int D, hipStream_t st) {
  RotArgs a;
  if (int rc = fill(a, dtype, q, ldq, hsq, k, ldk, hsk, pos, pos_type, freqs, s0, s1, s2, T, Hq, Hk, D)) return rc;
  MVF_CHECK_ARG(q_out && (k_out || Hk == 0) && (((uintptr_t)q_out | (uintptr_t)k_out) & 15) == 0);
  a.y[0] = (char*)q_out; a.y[1] = (char*)k_out;
  a.sign = inverse ? -1.f : 1.f;
  return dtype == MVF_F32 ? launch_v<MVF_F32, false>(a, interleaved, pos_type, st) :
         dtype == MVF_BF16 ? launch_v<MVF_BF16, false>(a, interleaved, pos_type, st) : launch_v<MVF_F16, false>(a, interleaved, pos_type, st);
}

extern "C" int mvf_rotary_append(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v, long ldv,
                                 long hsv, const void* pos, int pos_type, const double* freqs, int s0, int s1, int s2, int interleaved,
                                 void* q_out, void* k_cache, void* v_cache, const int* block_table, int table_width, int n_seqs,
                                 const int* seq, const int* index, int n_pages, int page, int T, int Hq, int Hk, int D, hipStream_t st) {
  RotArgs a;
  if (int rc = fill(a, dtype, q, ldq, hsq, k, ldk, hsk, pos, pos_type, freqs, s0, s1, s2, T, Hq, Hk, D)) return rc;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  MVF_CHECK_ARG(v && q_out && k_cache && v_cache && block_table && seq && index && Hk > 0);
  MVF_CHECK_ARG(table_width > 0 && n_seqs > 0 && n_pages > 0 && page > 0);
  MVF_CHECK_ARG(ldv > 0 && hsv > 0 && ldv * sz % 16 == 0 && hsv * sz % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0);
  a.x[2] = (const char*)v; a.ld[2] = ldv * sz; a.hs[2] = hsv * sz;
  a.h2 = Hq + 2 * Hk;
  a.y[0] = (char*)q_out; a.y[1] = (char*)k_cache; a.y[2] = (char*)v_cache;
  a.table = block_table; a.width = table_width; a.n_seqs = n_seqs; a.seq = seq; a.index = index; a.n_pages = n_pages; a.page = page;
  a.sign = 1.f;
  return dtype == MVF_F32 ? launch_v<MVF_F32, true>(a, interleaved, pos_type, st) :
         dtype == MVF_BF16 ? launch_v<MVF_BF16, true>(a, interleaved, pos_type, st) : launch_v<MVF_F16, true>(a, interleaved, pos_type, st);
}
