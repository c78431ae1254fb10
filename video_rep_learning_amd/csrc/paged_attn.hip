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

// every stream cuts its own length evenly
__device__ __forceinline__ int tiles_per_split(int ntile, int splits) { return max((ntile + splits - 1) / splits, 1); }

template <int DT, int DP, bool PAD>
__global__ __launch_bounds__(64 * NW, 1) void paged_attn_kernel(PagedArgs a) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typedef Tiles<O, DP> S;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ float s_m[NW][32], s_l[NW][32];
  __shared__ int s_tab[NW][2][64];                    // page ids of a tile's 32 keys (twice)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int rt = unit % a.rt, kh = unit / a.rt % a.Hk, b = unit / a.rt / a.Hk;
  const int len = (int)max(0l, min((long)a.len[b], (long)a.width * a.page));
  const int ntile = (len + 31) >> 5, per = tiles_per_split(ntile, a.splits);
  if (split > 0 && split * per >= ntile) return;
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
  hi_all = __builtin_amdgcn_readfirstlane(hi_all);
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
  if constexpr (PAD) clear_lds(smem, NW * S::NB * S::BUF);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(qf[ks]));      // landed before any DMA is in flight
  f32x16_t o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
  RowMax st;
  const float thr = 8.f / a.c;
  const long row_bytes = (long)a.Hk * a.D * O::SZ;
  const char* kb = a.k + (long)kh * a.D * O::SZ;
  const char* vb = a.v + (long)kh * a.D * O::SZ;
  const int* tab = a.table + (long)b * a.width;
  const uint32_t lds = lds_addr(smem) + wave * S::NB * S::BUF, tlds = lds_addr(&s_tab[wave][0][0]);
  const uint32_t rpart = I::row_part(lane), cpart = I::col_part(lane);

  auto ask_pages = [&](int t, int buf) __attribute__((always_inline)) {
    dma4(reinterpret_cast<const float*>(tab + min((t * 32 + r) / a.page, a.width - 1)), tlds + buf * 256);
  };
  // where the tile's 32 keys lie, from the page ids; returns which of them exist (an absent one repeats one that does)
  auto place = [&](int t, int pg, long& off) __attribute__((always_inline)) {
    const int key = t * 32 + r;
    const bool is = key < len && pg >= 0 && pg < a.n_pages;
    const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(is);
    off = is ? ((long)pg * a.page + key % a.page) * row_bytes : 0;
    const int from = is ? r : there != 0 ? __builtin_ctz(there) : r;
    off = (long)(((uint64_t)(uint32_t)__shfl((int)(off >> 32), from, 64) << 32) | (uint32_t)__shfl((int)off, from, 64));
    return there;
  };
  auto ask_rows = [&](long off, int buf) __attribute__((always_inline)) {
    const int lo32 = (int)off, hi32 = (int)(off >> 32);
    S::template issue<PAD>(kb, vb, [&](int i, long& oa, long& ob) {
      oa = ob = (long)(((uint64_t)(uint32_t)__shfl(hi32, i, 64) << 32) | (uint32_t)__shfl(lo32, i, 64));
    }, a.D, lane, lds + buf * S::BUF);
  };
  bool bad = false;
  auto tile = [&](int t, uint32_t there, uint32_t ik, bool mask) __attribute__((always_inline)) {
    const uint32_t rl = launder(rpart + ik), cl = launder(cpart + ik + S::IMG);
    f32x16_t s = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(rl, ks), qf[ks], s);
    if (mask) {
      bad |= tile_nonfinite<O, DP>(ik + S::IMG, lane);
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
    accumulate<O, DP>(o, s, cl);
  };

  // Per tile: its page ids are asked for two tiles ahead, its rows one tile ahead (where the buffers allow two tiles).
  const int t0 = split * per + wave;
  int buf = 0;
  uint32_t there = 0, next = 0;
  long off;
  if (t0 < t_end) {
    ask_pages(t0, 0);
    ask_pages(t0 + NW, 1);
    wait_dma<1>();
    there = place(t0, s_tab[wave][0][lane], off);
    ask_rows(off, 0);
  }
  for (int t = t0, i = 0; t < t_end; t += NW, ++i) {
    const bool more = t + NW < t_end;
    const uint32_t ik = lds + buf * S::BUF;
    if (S::NB == 2 && more) {
      wait_dma<S::NP>();                             // the next tile's page ids are older than this tile's rows
      next = place(t + NW, s_tab[wave][(i + 1) & 1][lane], off);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      ask_pages(t + 2 * NW, i & 1);
      ask_rows(off, buf ^ 1);
      wait_dma<S::NP + 1>();
    } else {
      wait_dma<0>();
    }
    if (there != 0) tile(t, there, ik, there != 0xffffffffu || t * 32 + 32 > hi_all);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S::NB == 2) {
      buf ^= 1;
    } else if (more) {
      next = place(t + NW, s_tab[wave][(i + 1) & 1][lane], off);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      ask_pages(t + 2 * NW, i & 1);
      ask_rows(off, 0);
    }
    there = next;
  }
  if (bad) {                                          // a value that is not finite beside masked places: visible pairs only
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
    st = RowMax();
#pragma unroll 1
    for (int t = t0; t < t_end; t += NW)
#pragma unroll 1
      for (int key = t * 32; key < min(t * 32 + 32, len); ++key) {
        const int pg = tab[key / a.page];
        if (pg < 0 || pg >= a.n_pages) continue;
        const long at = ((long)pg * a.page + key % a.page) * row_bytes;
        const float s = slow_dot<O, DP>(qf, kb + at, a.D, hh);
        if (key >= hi) continue;
        const float to = fmaxf(st.m, s);
        const float alpha = st.m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((st.m - to) * a.c);
        st.m = to;
        st.nm = to == NEG_INF ? 0.f : -to * a.c;
        const float p = __builtin_amdgcn_exp2f(fmaf(s, a.c, st.nm));
        st.l = fmaf(st.l, alpha, hh == 0 ? p : 0.f);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        slow_add<O, DP>(o, p, vb + at, a.D, hh);
      }
  }
  __syncthreads();
  join_waves<DP, NW>(reinterpret_cast<float*>(smem), s_m, s_l, o, st, rows, a.D, wave, lane,
                 [&](int row, int d, const f32x4_t& acc, float mx, float l) {
    const int mm = m0 + row;
    if (a.splits == 1) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      O::store4(reinterpret_cast<typename O::E*>(a.out) + (((long)b * a.n + mm / a.g) * a.Hq + kh * a.g + mm % a.g) * a.D + d, acc[0] * inv,
                acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      const size_t prow = (((size_t)b * a.Hk + kh) * a.R + mm) * a.splits + split;
      *reinterpret_cast<f32x4_t*>(a.part + prow * a.D + d) = acc;
      if (d == 0) {
        float* ml = a.part + (size_t)a.B * a.Hk * a.R * a.splits * a.D + prow * 2;
        ml[0] = mx;
        ml[1] = l;
      }
    }
  });
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
  const int len = (int)max(0l, min((long)a.len[prow / a.R / a.Hk], (long)a.width * a.page)), ntile = (len + 31) >> 5;
  const int per = tiles_per_split(ntile, a.splits), n = max(1, (ntile + per - 1) / per);      // the splits that were written
  float m = NEG_INF, l = 0.f;
  if (tid < n) { m = ml[2 * tid]; l = ml[2 * tid + 1]; }
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
    for (int s = tid >> 5; s < n; s += 8)
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
  const long fill = (2048 / NW + units - 1) / units;          // two workgroups per compute unit
  const long most = (max_keys + 64 * NW - 1) / (64 * NW);             // two tiles per wave
  return (int)std::max(1l, std::min({std::max(fill, (max_keys + 1024 - 1) / 1024), most, 256l}));
}

template <int DT, int DP, bool PAD>
int launch(const PagedArgs& a, hipStream_t st) {
  typedef Tiles<Op<DT>, DP> S;
  const size_t lds = std::max(NW * S::NB * S::BUF, (JOIN_BYTES<DP, NW>));
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(paged_attn_kernel<DT, DP, PAD>), lds, attr)) return rc;
  hipLaunchKernelGGL((paged_attn_kernel<DT, DP, PAD>), dim3((unsigned)a.B * a.Hk * a.rt * a.splits), dim3(64 * NW), lds, st, a);
  MVF_LAUNCH_CHECK();
  if (a.splits > 1) {
    hipLaunchKernelGGL((paged_join_kernel<DT>), dim3((unsigned)a.B * a.Hk * a.R), dim3(256), 0, st, a);
    MVF_LAUNCH_CHECK();
  }
  return MVF_OK;
}
template <int DT, int DP>
int launch_p(const PagedArgs& a, hipStream_t st) { return a.D == DP ? launch<DT, DP, false>(a, st) : launch<DT, DP, true>(a, st); }
template <int DT>
int launch_d(const PagedArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch_p<DT, 32>(a, st) : a.D <= 64 ? launch_p<DT, 64>(a, st) : a.D <= 96 ? launch_p<DT, 96>(a, st) : launch_p<DT, 128>(a, st);
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
