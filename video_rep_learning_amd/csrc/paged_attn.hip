// Attention of the newest tokens of each stream over its pages of a key-value cache:
//   out[b, i, h] = sum_j softmax_j(scale q[b, i, h] . K[b, j, h / g]) V[b, j, h / g]
// for the last n positions p = len[b] - n + i of stream b, j < min(len[b], (p / frame + 1) frame)   (frame = 0: j < len[b]).
// The n tokens x g heads that share a key head are the rows of ONE owned tile (up to 32), so every key and value is read once for all of
// them: HBM-bound on 2 len Hk D elements per stream.  A workgroup's four waves walk 32-key tiles of their own (staged by the wave
// itself, two tiles ahead: no barrier in the loop, 128 KB in flight per compute unit at 16-bit D 128) and meet once per unit; long
// streams are further cut over workgroups, whose partial sums a second launch joins in a fixed order.  A page id outside the cache holds no
// keys.  Measured: 12 streams of 32768, bf16, 8 key heads of 128: 300 us, 5.4 TB/s (a copy of 2 GiB: 4.9); 64 of 4096, 4 heads: 105 us,
// 5.1 TB/s; 64 of 1 to 4096 (50 MB): 27 us, of which the first tile's chain of loads (length, page ids, rows) and the join are 12.
#include "mvf_hip_internal.h"
#include "seq_attn.h"

namespace {
using namespace seq_attn;

constexpr int NW = 4;                  // waves per workgroup
constexpr int MAX_GROUPS = 512;        // workgroups that share a call's work
// The weights of 16-bit tensors enter the second product as two operands, the rounded weight and the rounded rest: the matrix pipe waits for
// keys most of the time anyway (12 streams of 32768 bf16: 302 us a call, with one operand 301; 64 of 1 to 4096 fp16: 25.4, 25.0), and the
// result is one rounding of the 32-bit sum (bf16 1.7e-3 of its size, with one operand 2.3e-3; fp16 1.8e-4, 2.0e-4).
template <class O>
constexpr bool LOW = O::SZ == 2;

struct PagedArgs {
  const char* q;                       // [B, n, Hq, D], strides in BYTES
  long qb, qn, qh;
  const char *k, *v;                   // [n_pages, page, Hk, D]
  const int *table, *len;              // [B, width], [B]
  char* out;                           // [B, n, Hq, D]
  float* part;                         // [groups][2][RS][D] sums, then [..][2] (maximum in the exponent's units, sum of weights)
  int* shared;                         // [B Hk rt][2]: first and last workgroup of a unit
  int B, n, Hq, Hk, D, g, R, rt, RS, page, width, n_pages, frame, groups, extra;
  float c;
};

__device__ __forceinline__ int clamped_length(const PagedArgs& a, int b) {
  return (int)max(0l, min((long)a.len[b], (long)a.width * a.page));
}
__device__ __forceinline__ int rounds_of(int len) { return (len + 32 * NW - 1) / (32 * NW); }

// The work of a call as one line.  A unit is 32 rows of one key head of one stream; it walks rounds of NW tiles (one per wave), and where
// there are many units, `extra` = 1 more round's length stands for its beginning and end; unit by unit they lie behind each other, stream
// by stream.  Every workgroup takes an equal stretch of that line, whatever the lengths are, and finds where it lies from the
// lengths on the device.  A unit that two or more workgroups share leaves a partial sum in each one's slots: 0 for a unit that began in an
// earlier workgroup, 1 for one that begins here and goes on in the next; the first of them notes which they are.
struct Piece { int b, unit, len, start; };       // unit (of stream b, of that length), where it starts on the line
struct Line {                                    // by one whole wave
  int lane, len, sum;                            // of streams 0 .. 63: a lane's length, the sum on the line up to it
  int total;
  static __device__ __forceinline__ int scan(int x, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    return x;
  }
  static __device__ __forceinline__ int of(const PagedArgs& a, int len) { return rounds_of(len) + (len > 0 ? a.extra : 0); }
  static __device__ __forceinline__ int length(const PagedArgs& a, int b) { return b < a.B ? clamped_length(a, b) : 0; }
  __device__ __forceinline__ void start(const PagedArgs& a, int lane_) {
    lane = lane_;
    len = length(a, lane);
    sum = scan(of(a, len), lane);
    total = __builtin_amdgcn_readlane(sum, 63);
#pragma unroll 1
    for (int b = 64; b < a.B; b += 64) total += __builtin_amdgcn_readlane(scan(of(a, length(a, b + lane)), lane), 63);
  }
  // the unit that place `pos` of the line lies in (pos < total * units of a stream; length 0: there is none, so the lengths were changed
  // while this ran, which must not keep it here)
  __device__ __forceinline__ Piece find(const PagedArgs& a, int pos) const {
    const int per = a.Hk * a.rt, p = pos / per;
    int x = len, s = sum, base = 0, b0 = 0;
    uint64_t m = __builtin_amdgcn_ballot_w64(s > p);
#pragma unroll 1
    while (m == 0) {
      if (b0 >= a.B) return {0, 0, 0, 0};
      base += __builtin_amdgcn_readlane(s, 63);
      b0 += 64;
      x = length(a, b0 + lane);
      s = scan(of(a, x), lane);
      m = __builtin_amdgcn_ballot_w64(base + s > p);
    }
    const int j = __builtin_ctzll(m), l = __builtin_amdgcn_readlane(x, j), w = of(a, l);
    const int s0 = (base + __builtin_amdgcn_readlane(s, j) - w) * per, unit = max((pos - s0) / w, 0);
    return {b0 + j, unit, l, s0 + unit * w};
  }
};

__device__ __forceinline__ int stretch(int all, int groups) { return max((all + groups - 1) / groups, 2); }

// rounds [r0, r1) of a unit, by a whole workgroup
template <int DT, int DP, bool PAD, bool LINE>
__device__ __forceinline__ void walk_unit(const PagedArgs& a, const Piece& u, int r0, int r1, char* smem, float (&s_m)[NW][32],
                                          float (&s_l)[NW][32], int (&s_tab)[2][64], int lane, int wave) {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typedef Tiles<O, DP> S;
  const int r = lane & 31, hh = lane >> 5;
  const int rt = u.unit % a.rt, kh = u.unit / a.rt, b = u.b;
  const int len = u.len;
  const int t_end = min((len + 31) >> 5, r1 * NW);
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
  const int* tab = a.table + (long)b * a.width;
  const int t0 = r0 * NW + wave;
  const uint32_t lds = lds_addr(smem) + wave * S::NB * S::BUF, tlds = lds_addr(&s_tab[0][0]);
  auto ask_pages = [&](int t, int buf) __attribute__((always_inline)) {
    dma4(reinterpret_cast<const float*>(tab + min((t * 32 + r) / a.page, a.width - 1)), tlds + buf * 256);
  };
  if (t0 < t_end) {                      // the first page ids come beside the queries
    ask_pages(t0, 0);
    ask_pages(t0 + NW, 1);
  }
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
  const float thr = RowMax::threshold(a.c);
  const long row_bytes = (long)a.Hk * a.D * O::SZ;
  const char* kb = a.k + (long)kh * a.D * O::SZ;
  const char* vb = a.v + (long)kh * a.D * O::SZ;
  const uint32_t rpart = I::row_part(lane), cpart = I::col_part(lane);

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
      bad |= st.steep(m < a.R);
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
    accumulate<O, DP, LOW<O>>(o, s, cl);
  };

  // Per tile: its page ids are asked for two tiles ahead, its rows one tile ahead (where the buffers allow two tiles).
  int buf = 0;
  uint32_t there = 0, next = 0;
  long off;
  if (t0 < t_end) {
    wait_dma<0>();
    there = place(t0, s_tab[0][lane], off);
    ask_rows(off, 0);
  }
  for (int t = t0, i = 0; t < t_end; t += NW, ++i) {
    const bool more = t + NW < t_end;
    const uint32_t ik = lds + buf * S::BUF;
    if (S::NB == 2 && more) {
      wait_dma<S::NP>();                             // the next tile's page ids are older than this tile's rows
      next = place(t + NW, s_tab[(i + 1) & 1][lane], off);
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
      next = place(t + NW, s_tab[(i + 1) & 1][lane], off);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      ask_pages(t + 2 * NW, i & 1);
      ask_rows(off, 0);
    }
    there = next;
  }
  if constexpr (LOW<O>) bad |= not_finite(o, m < a.R);
  if (bad) {                                          // a value that is not finite beside masked places, or steep scores: visible pairs only
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
        float alpha;
        const float p = st.add(s, a.c, alpha);
        st.l = fmaf(st.l, alpha, hh == 0 ? p : 0.f);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        slow_add<O, DP>(o, p, vb + at, a.D, hh);
      }
  }
  const bool whole = !LINE || (r0 == 0 && r1 == rounds_of(len));
  __syncthreads();
  join_waves<DP, NW>(reinterpret_cast<float*>(smem), s_m, s_l, o, st, rows, a.D, wave, lane,
                 [&](int row, int d, const f32x4_t& acc, float mx, float l) {
    const int mm = m0 + row;
    if (whole) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      O::store4(reinterpret_cast<typename O::E*>(a.out) + (((long)b * a.n + mm / a.g) * a.Hq + kh * a.g + mm % a.g) * a.D + d, acc[0] * inv,
                acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      const size_t prow = ((size_t)blockIdx.x * 2 + (r0 == 0)) * a.RS + row;
      *reinterpret_cast<f32x4_t*>(a.part + prow * a.D + d) = acc;
      if (d == 0) {
        float* ml = a.part + (size_t)a.groups * 2 * a.RS * a.D + prow * 2;
        ml[0] = mx;
        ml[1] = l;
      }
    }
  });
  if constexpr (LINE) __syncthreads();                 // the next unit's tiles overwrite what was joined
}

// LINE: the workgroups share the line; else a workgroup per unit
template <int DT, int DP, bool PAD, bool LINE>
__global__ __launch_bounds__(64 * NW, 1) void paged_attn_kernel(PagedArgs a) {
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ float s_m[NW][32], s_l[NW][32];
  __shared__ int s_tab[NW][2][64];                    // page ids of a tile's 32 keys (twice)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = a.Hk * a.rt;
  if constexpr (!LINE) {
    const int b = (int)blockIdx.x / units, len = clamped_length(a, b);
    walk_unit<DT, DP, PAD, false>(a, {b, (int)blockIdx.x % units, len, 0}, 0, rounds_of(len), smem, s_m, s_l, s_tab[wave], lane, wave);
  } else {
    Line line;
    line.start(a, lane);
    const int all = line.total * units, per = stretch(all, a.groups), end = min(((int)blockIdx.x + 1) * per, all);
#pragma unroll 1
    for (int pos = blockIdx.x * per; pos < end;) {
      const Piece u = line.find(a, pos);
      if (u.len == 0) break;
      const int n = rounds_of(u.len), first = u.start + a.extra;       // place of the first round
      const int r0 = max(pos - first, 0), r1 = min(end - first, n);
      if (r1 > r0) {
        if (r0 == 0 && threadIdx.x == 0) {
          a.shared[(u.b * units + u.unit) * 2] = blockIdx.x;
          a.shared[(u.b * units + u.unit) * 2 + 1] = (first + n - 1) / per;
        }
        walk_unit<DT, DP, PAD, true>(a, u, r0, r1, smem, s_m, s_l, s_tab[wave], lane, wave);
      }
      pos = first + n;
    }
  }
}

// one workgroup per row that more than one workgroup of the first launch had: their weights, then D channels x 8 groups of the partial sums
template <int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  typedef Op<DT> O;
  __shared__ float s_w[MAX_GROUPS], s_l[MAX_GROUPS], s_red[8];
  __shared__ f32x4_t s_acc[256];
  const int prow = blockIdx.x, tid = threadIdx.x;                // (b, kh, m)
  const int m = prow % a.R, head = prow / a.R, b = head / a.Hk, kh = head % a.Hk;
  const int len = clamped_length(a, b), unit = head * a.rt + m / 32;
  // (not written for an empty stream; the bounds hold whatever the workspace holds)
  const int w0 = min(max(a.shared[unit * 2], 0), a.groups - 1), n = len > 0 ? min(max(a.shared[unit * 2 + 1], w0), a.groups - 1) - w0 + 1 : 0;
  if (n == 1) return;                                            // written by its one workgroup
  auto slot = [&](int i) { return ((size_t)(w0 + i) * 2 + (i == 0)) * a.RS + m % 32; };
  const float* ml = a.part + (size_t)a.groups * 2 * a.RS * a.D;
  float mx = NEG_INF;
  for (int i = tid; i < n; i += 256) {
    const float2 x = *reinterpret_cast<const float2*>(ml + slot(i) * 2);
    s_w[i] = x.x;
    s_l[i] = x.y;
    mx = fmaxf(mx, x.x);
  }
  mx = wave_max(mx);
  if ((tid & 63) == 0) s_red[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  float l = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float pm = s_w[i], pl = s_l[i];
    const float w = pm == NEG_INF ? (pl != pl ? pl : 0.f) : __builtin_amdgcn_exp2f(pm - mx);
    s_w[i] = w;
    l += w * pl;
  }
  l = wave_sum(l);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
  __syncthreads();
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int d = (tid & 31) * 4;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  if (d < a.D)
    for (int i = tid >> 5; i < n; i += 8)
      if (s_w[i] != 0.f) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part + slot(i) * a.D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(s_w[i], x[j], acc[j]);
      }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < 32 && d < a.D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) acc += s_acc[k * 32 + tid];
    typename O::E* dst = reinterpret_cast<typename O::E*>(a.out) + (((long)b * a.n + m / a.g) * a.Hq + kh * a.g + m % a.g) * a.D + d;
    O::store4(dst, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
  }
}

// How many workgroups share the line (0: a workgroup per unit, one launch: short streams, or many of up to 1024 keys).  The lengths are on
// the device; the host knows the longest possible one.  One workgroup per compute unit, as many as LDS holds of most forms (64 streams of 1 to
// 4096 bf16 D 128: 26 us, with 512 31; 16 of 8192 fp32 D 128: 68, 77); two where LDS holds two (D 32) and for very long lines, where
// they even out the units' unequal bandwidth (12 of 32768: 297, with 256 309).  Cutting every stream into the same number of parts, chosen from
// the longest possible length, instead: 64 streams of 1 to 4096 35 us, 32 fp32 ones 42 (the line: 29), 64 of 4096 113 (105), one stream
// of 32768 with one key head 16 (20), 12 of 32768 294 (297).
int group_count(int D, long units, long max_keys) {
  if (max_keys <= 64 * NW || (units >= 512 && max_keys <= 1024)) return 0;
  const long line = units * ((max_keys + 32 * NW - 1) / (32 * NW) + 1);
  return (int)std::min(line, D <= 32 || line >= 16384 ? 512l : 256l);
}
// sums, (maximum, weights) and the workgroups of each unit
size_t partial_bytes(int groups, int D, long R, long units) {
  return groups == 0 ? 0 : ((size_t)groups * 2 * std::min(R, 32l) * (D + 2) + units * 2) * 4;
}

template <int DT, int DP, bool PAD, bool LINE>
int launch_form(const PagedArgs& a, hipStream_t st) {
  typedef Tiles<Op<DT>, DP> S;
  const size_t lds = std::max(NW * S::NB * S::BUF, (JOIN_BYTES<DP, NW>));
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(paged_attn_kernel<DT, DP, PAD, LINE>), lds, attr)) return rc;
  hipLaunchKernelGGL((paged_attn_kernel<DT, DP, PAD, LINE>), dim3(LINE ? a.groups : (unsigned)a.B * a.Hk * a.rt), dim3(64 * NW), lds, st, a);
  MVF_LAUNCH_CHECK();
  return MVF_OK;
}
template <int DT, int DP, bool PAD>
int launch(const PagedArgs& a, hipStream_t st) {
  if (a.groups == 0) return launch_form<DT, DP, PAD, false>(a, st);
  if (int rc = launch_form<DT, DP, PAD, true>(a, st)) return rc;
  hipLaunchKernelGGL((paged_join_kernel<DT>), dim3((unsigned)a.B * a.Hk * a.R), dim3(256), 0, st, a);
  MVF_LAUNCH_CHECK();
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
  const long units = (long)B * Hk * ((R + 31) / 32);
  return partial_bytes(group_count(D, units, (long)table_width * page), D, R, units);
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
  MVF_CHECK_ARG(R < (1l << 24) && max_keys < (1l << 31) - 4096);
  MVF_CHECK_ARG((long)B * Hk < (1l << 31) && (long)B * Hk * R < (1l << 31));
  MVF_CHECK_ARG((double)B * Hk * rt * ((max_keys + 32 * NW - 1) / (32 * NW) + 1) < 2e9);
  const int groups = group_count(D, (long)B * Hk * rt, max_keys);
  const size_t need = partial_bytes(groups, D, R, (long)B * Hk * rt);
  MVF_CHECK_ARG(need == 0 || (workspace && ws_bytes >= need));
  PagedArgs a = {(const char*)q, q_batch * sz, q_token * sz, q_head * sz, (const char*)k_cache, (const char*)v_cache, block_table, lengths,
                 (char*)out, (float*)workspace, (int*)((float*)workspace + (size_t)groups * 2 * std::min(R, 32l) * (D + 2)), B, n_new, Hq,
                 Hk, D, Hq / Hk, (int)R, (int)rt, (int)std::min(R, 32l), page, table_width, n_pages, frame, groups,
                 (long)B * Hk * rt >= 256, scale * LOG2E};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
