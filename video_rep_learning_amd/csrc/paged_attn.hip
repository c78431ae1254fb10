// Attention of the newest tokens of each stream over its pages of a key-value cache:
//   out[b, i, h] = sum_j softmax_j(scale q[b, i, h] . K[b, j, h / g]) V[b, j, h / g]
// for the last n positions p = len[b] - n + i of stream b, j < min(len[b], (p / frame + 1) frame)   (frame = 0: j < len[b]).
// The n tokens x g heads that share a key head are the rows of ONE owned tile (up to 32), so every key and value is read once for all of
// them: HBM-bound on 2 len Hk D elements per stream.  A workgroup's four waves walk 32-key tiles of their own (staged by the wave
// itself: no barrier in the loop) and meet once at the end; the length is further split over workgroups, whose partial sums a second
// launch joins in a fixed order.  A page id outside the cache holds no keys.
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using namespace seq_attn;

constexpr int NW = 4;                  // waves per workgroup

struct PagedArgs {
  const char* q;                       // [B, n, Hq, D], strides in BYTES
  long qb, qn, qh;
  const char *k, *v;                   // [n_pages, page, Hk, D]
  const int *table, *len;              // [B, width], [B]
  char* out;                           // [B, n, Hq, D]
  float* part;                         // [B Hk R splits][D] sums, then [..][2] (maximum in the exponent's units, sum of weights)
  int B, n, Hq, Hk, D, g, R, rt, page, width, n_pages, frame, splits;
  float c;
};

template <int DT, int DP>
__global__ __launch_bounds__(64 * NW, 1) void paged_attn_kernel(PagedArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  constexpr int ROWF = DP + 4;                       // floats per row of the joining area
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float s_m[NW][32], s_l[NW][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int rt = unit % a.rt, kh = unit / a.rt % a.Hk, b = unit / a.rt / a.Hk;
  const int len = (int)max(0l, min((long)a.len[b], (long)a.width * a.page));
  const int ntile = (len + 31) >> 5, per = (ntile + a.splits - 1) / a.splits;
  const int t_end = min(ntile, (split + 1) * per);
  const int m0 = rt * 32, m = m0 + r, mi = m / a.g, rows = min(32, a.R - m0);
  int hi = 0;                                        // keys this row sees
  if (m < a.R) {
    const int p = len - a.n + mi;
    hi = a.frame == 0 ? len : p < 0 ? 0 : (int)min((long)len, ((long)(p / a.frame) + 1) * a.frame);
  }
  int hi_all = m < a.R ? hi : 0x7fffffff;            // keys that every row sees
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) hi_all = min(hi_all, __shfl_xor(hi_all, o, 64));
  typename O::Frag qf[DP / 16];
  {
    const char* src = a.q + b * a.qb + (long)min(mi, a.n - 1) * a.qn + (kh * a.g + m % a.g) * a.qh;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * hh;
      typename O::Frag f = {};
      if (d < a.D && m < a.R) f = *reinterpret_cast<const typename O::Frag*>(src + d * O::SZ);
      qf[ks] = f;
    }
  }
  char* sk = smem + wave * 64 * I::RB;
  char* sv = sk + 32 * I::RB;
  f32x16_t o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
  RowMax st;
  const float thr = 8.f / a.c;
  const long row_bytes = (long)a.Hk * a.D * O::SZ;
  const char* kb = a.k + (long)kh * a.D * O::SZ;
  const char* vb = a.v + (long)kh * a.D * O::SZ;
  const int* tab = a.table + (long)b * a.width;

  constexpr int NL = I::C / 2;                       // 16-byte pieces per lane of 32 rows
  uint4 kr[NL], vr[NL];
  uint32_t there = 0, there_next = 0;                // which of the tile's 32 keys exist
  auto load = [&](int t) __attribute__((always_inline)) {
    const int key = t * 32 + r;
    long off = -1;
    if (key < len) {
      const int pg = tab[key / a.page];
      if (pg >= 0 && pg < a.n_pages) off = ((long)pg * a.page + key % a.page) * row_bytes;
    }
    there_next = (uint32_t)__builtin_amdgcn_ballot_w64(off >= 0);
    const int lo32 = (int)off, hi32 = (int)(off >> 32);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = (i * 64 + lane) / I::C, ch = (i * 64 + lane) % I::C;
      const long at = (long)(((uint64_t)(uint32_t)__shfl(hi32, row, 64) << 32) | (uint32_t)__shfl(lo32, row, 64));
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0 && ch * 16 < a.D * O::SZ) {
        kr[i] = *reinterpret_cast<const uint4*>(kb + at + ch * 16);
        vr[i] = *reinterpret_cast<const uint4*>(vb + at + ch * 16);
      }
    }
  };
  auto tile = [&](auto mask_tag, int t) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    f32x16_t s = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(sk, 0, ks, lane), qf[ks], s);
    if constexpr (MASK) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 8 * (e >> 2) + 4 * hh + (e & 3);
        s[e] = t * 32 + i < hi && ((there >> i) & 1) ? s[e] : NEG_INF;
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
      for (int dt = 0; dt < DP / 32; ++dt) o[dt] = mma_weighted<O, MASK, false>(I::cols(sv, 16 * s2, dt, lane), p, o[dt]);
    }
  };
  int t = split * per + wave;
  if (t < t_end) load(t);
  for (; t < t_end; t += NW) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = (i * 64 + lane) / I::C, ch = (i * 64 + lane) % I::C;
      *reinterpret_cast<uint4*>(sk + I::off(row, ch)) = kr[i];
      *reinterpret_cast<uint4*>(sv + I::off(row, ch)) = vr[i];
    }
    there = there_next;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own stores, before its other lanes read them
    if (t + NW < t_end) load(t + NW);
    if (there == 0xffffffffu && t * 32 + 32 <= hi_all) tile(std::false_type{}, t);
    else tile(std::true_type{}, t);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // ---- the four waves' parts ----
  const float l = pair_sum(st.l);
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);           // [NW][32][ROWF]
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
    if (d >= a.D) continue;
    float mx = NEG_INF;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w][row]);
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = s_m[w][row] == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(s_m[w][row] - mx);
      if (s_m[w][row] == NEG_INF && !(s_l[w][row] != s_l[w][row])) continue;
      sum += f * s_l[w][row];
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(so + (w * 32 + row) * ROWF + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(f, x[j], acc[j]);
    }
    const int mm = m0 + row;
    if (a.splits == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      typename O::E* dst = reinterpret_cast<typename O::E*>(a.out) + (((long)b * a.n + mm / a.g) * a.Hq + kh * a.g + mm % a.g) * a.D + d;
      O::store4(dst, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      const size_t prow = (((size_t)b * a.Hk + kh) * a.R + mm) * a.splits + split;
      *reinterpret_cast<f32x4_t*>(a.part + prow * a.D + d) = acc;
      if (d == 0) {
        float* ml = a.part + (size_t)a.B * a.Hk * a.R * a.splits * a.D + prow * 2;
        ml[0] = mx;
        ml[1] = sum;
      }
    }
  }
}

// one workgroup per row: the splits' weights, then D channels x 8 groups of splits
template <int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  typedef Op<DT> O;
  __shared__ float s_w[256], s_red[8];
  __shared__ f32x4_t s_acc[256];
  const int prow = blockIdx.x;                                   // (b, kh, m)
  const float* ml = a.part + (size_t)a.B * a.Hk * a.R * a.splits * a.D + (size_t)prow * a.splits * 2;
  const float* po = a.part + (size_t)prow * a.splits * a.D;
  const int tid = threadIdx.x;
  float m = NEG_INF, l = 0.f;
  if (tid < a.splits) { m = ml[2 * tid]; l = ml[2 * tid + 1]; }
  const float mw = wave_max(m);
  if ((tid & 63) == 0) s_red[tid >> 6] = mw;
  __syncthreads();
  const float mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float w = m == NEG_INF ? (l != l ? l : 0.f) : __builtin_amdgcn_exp2f(m - mx);
  s_w[tid] = w;
  const float sum = wave_sum(w * l);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = sum;
  __syncthreads();
  const float total = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const float inv = total != 0.f ? 1.f / total : 0.f;
  const int d = (tid & 31) * 4;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  if (d < a.D)
    for (int s = tid >> 5; s < a.splits; s += 8)
      if (s_w[s] != 0.f) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(po + (size_t)s * a.D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(s_w[s], x[j], acc[j]);
      }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < 32 && d < a.D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) acc += s_acc[k * 32 + tid];
    const int mm = prow % a.R, kh = prow / a.R % a.Hk, b = prow / a.R / a.Hk;
    typename O::E* dst = reinterpret_cast<typename O::E*>(a.out) + (((long)b * a.n + mm / a.g) * a.Hq + kh * a.g + mm % a.g) * a.D + d;
    O::store4(dst, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
  }
}

// How many workgroups share a stream's keys.  The lengths are on the device; the host knows the longest possible one.
int split_count(long units, long max_keys) {
  const long fill = (512 + units - 1) / units;          // two workgroups per compute unit
  const long most = (max_keys + 255) / 256;             // two tiles per wave
  return (int)std::max(1l, std::min({std::max(fill, (max_keys + 1023) / 1024), most, 256l}));
}

template <int DT, int DP>
int launch(const PagedArgs& a, hipStream_t st) {
  typedef Img<Op<DT>, DP> I;
  const size_t lds = std::max((size_t)NW * 64 * I::RB, (size_t)NW * 32 * (DP + 4) * 4);
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(paged_attn_kernel<DT, DP>), lds, attr)) return rc;
  hipLaunchKernelGGL((paged_attn_kernel<DT, DP>), dim3((unsigned)a.B * a.Hk * a.rt * a.splits), dim3(64 * NW), lds, st, a);
  MVF_LAUNCH_CHECK();
  if (a.splits > 1) {
    hipLaunchKernelGGL((paged_join_kernel<DT>), dim3((unsigned)a.B * a.Hk * a.R), dim3(256), 0, st, a);
    MVF_LAUNCH_CHECK();
  }
  return MVF_OK;
}
template <int DT>
int launch_d(const PagedArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch<DT, 32>(a, st) : a.D <= 64 ? launch<DT, 64>(a, st) : a.D <= 96 ? launch<DT, 96>(a, st) : launch<DT, 128>(a, st);
}

}  // namespace

extern "C" size_t mvf_paged_attn_workspace_bytes(int B, int n_new, int Hq, int Hk, int D, int table_width, int page) {
  if (B <= 0 || n_new <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || D <= 0 || table_width <= 0 || page <= 0) return 0;
  const long R = (long)n_new * (Hq / Hk);
  const int splits = split_count((long)B * Hk * ((R + 31) / 32), (long)table_width * page);
  return splits == 1 ? 0 : (size_t)B * Hk * R * splits * (D + 2) * sizeof(float);
}

extern "C" int mvf_paged_attn(int dtype, const void* q, long q_batch, long q_token, long q_head, const void* k_cache, const void* v_cache,
                              const int* block_table, const int* lengths, void* out, void* workspace, size_t ws_bytes, int B, int n_new,
                              int Hq, int Hk, int D, int n_pages, int page, int table_width, int frame, float scale, hipStream_t st) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && k_cache && v_cache && block_table && lengths && out && B > 0 && n_new > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0);
  MVF_CHECK_ARG(n_pages > 0 && page > 0 && table_width > 0 && frame >= 0 && scale > 0.f && scale < 1e30f);
  if (D <= 0 || D > 128 || D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  MVF_CHECK_ARG(q_batch >= 0 && q_token >= 0 && q_head >= 0 && q_batch * sz % 16 == 0 && q_token * sz % 16 == 0 && q_head * sz % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0);
  const long R = (long)n_new * (Hq / Hk), rt = (R + 31) / 32, max_keys = (long)table_width * page;
  MVF_CHECK_ARG(R < (1l << 24) && max_keys < (1l << 31) - 64);
  const int splits = split_count((long)B * Hk * rt, max_keys);
  MVF_CHECK_ARG((long)B * Hk * rt * splits < (1l << 31) && (long)B * Hk * R < (1l << 31));
  const size_t need = splits == 1 ? 0 : (size_t)B * Hk * R * splits * (D + 2) * sizeof(float);
  MVF_CHECK_ARG(need == 0 || (workspace && ws_bytes >= need));
  PagedArgs a = {(const char*)q, q_batch * sz, q_token * sz, q_head * sz, (const char*)k_cache, (const char*)v_cache, block_table, lengths,
                 (char*)out, (float*)workspace, B, n_new, Hq, Hk, D, Hq / Hk, (int)R, (int)rt, page, table_width, n_pages, frame, splits,
                 scale * LOG2E};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
