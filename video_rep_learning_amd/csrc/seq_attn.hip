// Self-attention over packed sequences of different lengths, grouped heads, causal by token or by frame:
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / g]) v[j, h / g],   j in i's sequence, j < (i / frame + 1) frame inside it
// The running maximum and sum of a row's softmax stay in the row's lane, scores and weights in registers between the two products.
// Every sequence is cut into row tiles of its own, found on the device: nothing but the numbers of rows and sequences sizes the grid (no
// host copy of the lengths), empty sequences cost nothing, and rows outside every sequence come out as zeros.
//
// Three forms of the same tile arithmetic, chosen by use_split and use_pairs:
//   wide:   a workgroup owns 128 rows of one head (32 per wave) and its waves share each block of keys;
//   pairs:  the same with two waves for each 32 rows, which take a block's tiles in turn and join their sums at the end;
//   split:  a workgroup owns 32 rows, each wave walks every fourth (or eighth) 32-key tile by itself, the partial softmaxes are joined at
//           the end: four times as many workgroups and a quarter of the dependent steps, for four times the key traffic.
// The weights are rounded to the operands' format for the second product (relative 2^-9 in bf16, random in sign, so the sum is off by that
// much of its size, as the rounding of the result is; not in short walks: short_walk()); their sum is taken before, in 32 bits.
// Measured: 2 x 8192 causal bf16, 16 query heads of 128 on 4: 0.60 ms, 911 TFLOP/s of visible pairs (a large bf16 matrix product: 1130 to
// 1150); 32 x 785, 12 of 64: 114 us, 530; 8 x 1440 fp32 causal by 6, 8 of 32: 119 us, 72 (a large fp32 product: 148).  Bound by the waves'
// own chains: at D 96 the matrix pipe is busy 24 % of the cycles, the vector unit 31 %, and 32 % of the waves' time goes into waits.
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
  float* stat;                         // NULL, or [2][Hq][T]: see finish()
  int T, Hq, Hk, D, frame, ntiles, level;
  float c;                             // scale * log2(e)
  char* rest;                          // NULL, or (16-bit types) [T, Hq, D]: what out's rounding took away
};

// four channels of a row of the result
template <class O>
__device__ __forceinline__ void store_out(const FwdArgs& a, size_t at, float x, float y, float z, float w) {
  typedef typename O::E E;
  E* out = reinterpret_cast<E*>(a.out) + at;
  if (O::SZ == 2 && a.rest != nullptr) O::store4_rest(out, reinterpret_cast<E*>(a.rest) + at, x, y, z, w);
  else O::store4(out, x, y, z, w);
}

// 32 channels of a wave's rows, the first `left` of them: 16-bit formats trade quarters between the lanes of a pair, 16 bytes a store
template <class O>
__device__ __forceinline__ void store_tile(const FwdArgs& a, size_t at, int left, const f32x16_t& x, int lane) {
  const int hh = lane >> 5;
  if constexpr (O::SZ == 2) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      u32x4_t out, rest;
      O::pack8_rest(x, e, out, rest);
      const int d = 8 * (e + hh);
      if (d < left) {
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<typename O::E*>(a.out) + at + d) = out;
        if (a.rest != nullptr) *reinterpret_cast<u32x4_t*>(reinterpret_cast<typename O::E*>(a.rest) + at + d) = rest;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 8 * e + 4 * hh;
      if (d < left) O::store4(reinterpret_cast<typename O::E*>(a.out) + at + d, x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    }
  }
}

template <int DT, int DP>
struct Fwd {
  typedef Op<DT> O;
  typedef Img<O, DP> I;
  typename O::Frag qf[DP / 16];
  f32x16_t o[DP / 32];
  RowMax st;
  Span own;
  float c, thr;
  int lane;
  uint32_t rpart, cpart;
  bool bad = false;        // a tile with masked places held a value that is not finite, or the scores are steep
  bool low = false;        // the weights' second operand: see accumulate()

  __device__ __forceinline__ void start(const FwdArgs& a, int head, int row, int lane_) {
    lane = lane_;
    rpart = I::row_part(lane);
    cpart = I::col_part(lane);
    c = a.c;
    thr = RowMax::threshold(a.c);
    const int hh = lane >> 5;
    const char* src = a.q + (long)min(row, a.T - 1) * a.ldq + head * a.hsq;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * hh;
      typename O::Frag f = {};
      if (d < a.D) f = *reinterpret_cast<const typename O::Frag*>(src + d * O::SZ);
      qf[ks] = f;
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
  }
  // one 32-key tile; mask (wave-uniform): some row does not see all of it
  __device__ __forceinline__ void tile(uint32_t ik, uint32_t iv, int key0, bool mask) {
    const uint32_t rl = launder(rpart + ik), cl = launder(cpart + iv);
    f32x16_t s = zero16();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = O::mma(I::rows(rl, ks), qf[ks], s);
    if (mask) {
      bad |= tile_nonfinite<O, DP>(iv, lane);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = key0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        s[e] = key >= own.lo && key < own.hi ? s[e] : NEG_INF;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = pair_max(mx);
    float alpha;
    if (st.grow(mx, c, thr, alpha)) {
      bad |= st.steep(own.hi > own.lo);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, st.nm));
      st.l += s[e];
    }
    accumulate_if<O, DP>(low, o, s, cl);
  }
  // the same rows over 32-key tiles first, first + step, ..., one visible pair at a time
  __device__ __forceinline__ void slow(const FwdArgs& a, const char* kb, const char* vb, int first, int step, int end) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
    st = RowMax();
#pragma unroll 1
    for (int k0 = first; k0 < end; k0 += step)
#pragma unroll 1
      for (int key = k0; key < min(k0 + 32, end); ++key) {
        const float s = slow_dot<O, DP>(qf, kb + (long)key * a.ldk, a.D, lane >> 5);
        if (key < own.lo || key >= own.hi) continue;
        float alpha;
        const float p = st.add(s, c, alpha);
        st.l = fmaf(st.l, alpha, lane < 32 ? p : 0.f);                  // the pair's sum is taken at the end
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        slow_add<O, DP>(o, p, vb + (long)key * a.ldv, a.D, lane >> 5);
      }
  }
  __device__ __forceinline__ void any_tile(const WaveSpan& ws, uint32_t ik, uint32_t iv, int key0) {
    if (key0 >= ws.any.hi || key0 + 32 <= ws.any.lo) return;
    tile(ik, iv, key0, key0 < ws.all.lo || key0 + 32 > ws.all.hi);
  }
};

// What the backward needs to have the same probabilities again.  fp32: the exponent's offset and 1 / l, applied as in the forward (one
// log2-sum would round at the size of its integer part: 1e-6 of a probability); 16-bit: one offset that holds both (fp16: and PSHIFT).
template <int DT>
__device__ __forceinline__ void store_stat(const FwdArgs& a, int head, int row, float nm, float l, bool some) {
  const size_t at = (size_t)head * a.T + row;
  a.stat[at] = !some ? NEG_INF : DT == MVF_F32 ? nm : nm - __builtin_amdgcn_logf(l) + (DT == MVF_F16 ? PSHIFT : 0);
  a.stat[(size_t)a.Hq * a.T + at] = some ? 1.0f / l : 0.f;
}

// H = 2: eight waves, two for each 32 rows, which take every block's tiles in turn and join their halves at the end
template <int DT, int DP, bool PAD, int H>
__global__ __launch_bounds__(256 * H, DT == MVF_F32 && DP > 64 ? H : DT != MVF_F32 && DP == 128 && H == 1 ? 3 : 2) void packed_attn_fwd_kernel(FwdArgs a) {
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
  Fwd<DT, DP> f;
  f.start(a, head, row, lane);                 // (a row of no sequence may hold anything: it stays in its own lanes and is not stored)
  f.own = keys_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws);
  if constexpr (PAD) clear_lds(smem, R::NB * R::BUF);
  const Span span = block_span(ws, s_span, lane, wave, 4 * H);
  const int g = a.Hq / a.Hk;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(f.qf[ks]));      // landed before any DMA is in flight
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
  if (O::SZ == 2 && f.low) f.bad |= not_finite(f.o, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kb, vb, span.lo + 32 * (wave >> 2), 32 * H, ws.any.hi);
  if constexpr (H == 2) {
    __syncthreads();
    char* half = smem + (wave & 3) * HALF<DP> + lane * 16;
    if (wave >= 4) {
      put_half<DP>(half, f.o);
      *reinterpret_cast<float2*>(half + DP / 8 * 1024) = make_float2(f.st.m, f.st.l);
    }
    __syncthreads();
    if (wave >= 4) return;
    const float2 ml = *reinterpret_cast<const float2*>(half + DP / 8 * 1024);
    const float to = fmaxf(f.st.m, ml.x);
    const float f0 = f.st.m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((f.st.m - to) * a.c);
    const float f1 = ml.x == NEG_INF ? 0.f : __builtin_amdgcn_exp2f((ml.x - to) * a.c);
    f.st.nm = to == NEG_INF ? 0.f : -to * a.c;
    f.st.l = f.st.l * f0 + ml.y * f1;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(half + (dt * 4 + g) * 1024);
#pragma unroll
        for (int j = 0; j < 4; ++j) f.o[dt][4 * g + j] = f.o[dt][4 * g + j] * f0 + x[j] * f1;
      }
  }
  if (row >= own.end) return;
  const float l = pair_sum(f.st.l);
  const bool some = f.own.hi > f.own.lo && l != 0.f;          // (l is NaN where a score was)
  const float inv = some ? 1.0f / l : 0.f;
  if (a.stat != nullptr && lane < 32) store_stat<DT>(a, head, row, f.st.nm, l, some);
  const size_t at = ((size_t)row * a.Hq + head) * a.D;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
    for (int e = 0; e < 16; ++e) f.o[dt][e] = some ? f.o[dt][e] * inv : 0.f;
    store_tile<O>(a, at + 32 * dt, a.D - 32 * dt, f.o[dt], lane);
  }
}

template <int DT, int DP, bool PAD, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void packed_attn_fwd_split_kernel(FwdArgs a) {
  typedef Op<DT> O;
  typedef SplitTiles<O, DP, NW> S;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ float s_m[NW][32], s_l[NW][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit u = xcd_unit(a.Hq, a.ntiles);
  if (u.head < 0) return;
  const int head = u.head;
  const OwnTile own = find_tile<32>(a.cu, a.n_seqs, a.T, u.tile, a.ntiles, a.frame == 0 ? Walk::ALL : Walk::LATE);
  if (own.row0 >= own.end) return;
  const int row0 = own.row0, row = row0 + (lane & 31);
  Fwd<DT, DP> f;
  f.start(a, head, row, lane);                 // (a row of no sequence may hold anything: it stays in its own lanes and is not stored)
  f.own = keys_of(sequence_of(own, a.cu, a.n_seqs, a.T, row), a.frame, row);
  const WaveSpan ws = wave_span(f.own);
  f.low = short_walk(ws);
  if constexpr (PAD) clear_lds(smem, NW * S::NB * S::BUF);
  const int g = a.Hq / a.Hk;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) asm volatile("" : "+v"(f.qf[ks]));
  const char *kb = a.k + head / g * a.hsk, *vb = a.v + head / g * a.hsv;
  const uint32_t lds = lds_addr(smem) + wave * S::NB * S::BUF;
  TileWalk<O, DP, NW, S> walk;
  walk.start(kb, a.ldk, vb, a.ldv, ws.any.lo + wave * 32, lane);
  auto issue = [&](int key0, int buf) __attribute__((always_inline)) {
    walk.template issue<PAD>(key0, ws.any.hi, a.D, lane, lds + buf * S::BUF);
  };
  int key0 = ws.any.lo + wave * 32, buf = 0;
  if (key0 < ws.any.hi) issue(key0, 0);
  for (; key0 < ws.any.hi; key0 += 32 * NW) {
    const bool more = key0 + 32 * NW < ws.any.hi;
    if (S::NB == 2 && more) { issue(key0 + 32 * NW, buf ^ 1); wait_dma<S::NP>(); }
    else wait_dma<0>();
    f.any_tile(ws, lds + buf * S::BUF, lds + buf * S::BUF + S::IMG, key0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S::NB == 2) buf ^= 1;
    else if (more) issue(key0 + 32 * NW, 0);
  }
  if (O::SZ == 2 && f.low) f.bad |= not_finite(f.o, f.own.hi > f.own.lo);
  if (f.bad) f.slow(a, kb, vb, ws.any.lo + wave * 32, 32 * NW, ws.any.hi);
  if (f.own.hi == 0) {           // rows of no sequence rode along in unmasked tiles
    f.st = RowMax();
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) f.o[dt] = zero16();
  }
  __syncthreads();
  const bool stat = a.stat != nullptr;
  join_waves<DP, NW>(reinterpret_cast<float*>(smem), s_m, s_l, f.o, f.st, own.end - row0, a.D, wave, lane,
                 [&](int i, int d, const f32x4_t& acc, float mx, float l) {
    const bool some = l != 0.f;
    const float inv = some ? 1.0f / l : 0.f;
    if (stat && d == 0) store_stat<DT>(a, head, row0 + i, -mx, l, some);
    store_out<O>(a, ((size_t)(row0 + i) * a.Hq + head) * a.D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
  });
}

template <int DT, int DP, bool PAD, int NW>
int launch_split(FwdArgs a, hipStream_t st) {
  typedef SplitTiles<Op<DT>, DP, NW> S;
  const size_t lds = std::max(NW * S::NB * S::BUF, (JOIN_BYTES<DP, NW>));
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_fwd_split_kernel<DT, DP, PAD, NW>), lds, attr)) return rc;
  a.ntiles = (int)tile_bound<32>(a.T, a.n_seqs);
  hipLaunchKernelGGL((packed_attn_fwd_split_kernel<DT, DP, PAD, NW>), dim3(xcd_grid(a.Hq, a.ntiles)), dim3(64 * NW), lds, st, a);
  return MVF_OK;
}
template <int DT, int DP, bool PAD, int H>
int launch_wide(FwdArgs a, hipStream_t st) {
  typedef Ring<Op<DT>, DP, 3, 4 * H> R;
  constexpr size_t lds = std::max<size_t>(R::NB * R::BUF, H == 2 ? 4 * HALF<DP> : 0);
  static uint64_t attr = 0;
  if (int rc = mvf_ensure_lds(reinterpret_cast<const void*>(packed_attn_fwd_kernel<DT, DP, PAD, H>), lds, attr)) return rc;
  a.ntiles = (int)tile_bound<128>(a.T, a.n_seqs);
  static long holds = 0;
  const unsigned grid = xcd_grid(a.Hq, a.ntiles);
  a.level = grid <= card_holds(reinterpret_cast<const void*>(packed_attn_fwd_kernel<DT, DP, PAD, H>), 256 * H, lds, holds);
  hipLaunchKernelGGL((packed_attn_fwd_kernel<DT, DP, PAD, H>), dim3(grid), dim3(256 * H), lds, st, a);
  return MVF_OK;
}
template <int DT, int DP, bool PAD>
int launch(FwdArgs a, hipStream_t st) {
  const bool pairs = PAIRS<Op<DT>, DP> && use_pairs(a.T, a.n_seqs, a.Hq, a.frame);
  if (use_split(tile_bound<128>(a.T, a.n_seqs) * a.Hq, DT, a.T, a.n_seqs, pairs)) {
    constexpr int NW8 = SPLIT_WAVES<Op<DT>, DP>;
    if (int rc = long_walks(a.T, a.n_seqs) ? launch_split<DT, DP, PAD, NW8>(a, st) : launch_split<DT, DP, PAD, 4>(a, st)) return rc;
  } else {
    constexpr int H = PAIRS<Op<DT>, DP> ? 2 : 1;
    if (int rc = pairs ? launch_wide<DT, DP, PAD, H>(a, st) : launch_wide<DT, DP, PAD, 1>(a, st)) return rc;
  }
  MVF_LAUNCH_CHECK();
  return MVF_OK;
}
template <int DT, int DP>
int launch_p(const FwdArgs& a, hipStream_t st) { return a.D == DP ? launch<DT, DP, false>(a, st) : launch<DT, DP, true>(a, st); }
template <int DT>
int launch_d(const FwdArgs& a, hipStream_t st) {
  return a.D <= 32 ? launch_p<DT, 32>(a, st) : a.D <= 64 ? launch_p<DT, 64>(a, st) : a.D <= 96 ? launch_p<DT, 96>(a, st) : launch_p<DT, 128>(a, st);
}

}  // namespace

extern "C" int mvf_packed_attn_fwd(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                   long ldv, long hsv, const int* cu_seqlens, int n_seqs, void* out, float* stat, int T, int Hq, int Hk,
                                   int D, int frame, float scale, hipStream_t st) {
  return mvf_packed_attn_fwd_rest(dtype, q, ldq, hsq, k, ldk, hsk, v, ldv, hsv, cu_seqlens, n_seqs, out, nullptr, stat, T, Hq, Hk, D, frame,
                                  scale, st);
}

extern "C" int mvf_packed_attn_fwd_rest(int dtype, const void* q, long ldq, long hsq, const void* k, long ldk, long hsk, const void* v,
                                        long ldv, long hsv, const int* cu_seqlens, int n_seqs, void* out, void* rest, float* stat, int T,
                                        int Hq, int Hk, int D, int frame, float scale, hipStream_t st) {
  MVF_CHECK_ARG(dtype == MVF_F32 || dtype == MVF_BF16 || dtype == MVF_F16);
  MVF_CHECK_ARG(q && k && v && cu_seqlens && out && T > 0 && n_seqs > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && frame >= 0);
  MVF_CHECK_ARG(scale > 0.f && scale < 1e30f && T < (1 << 30) && tile_bound<32>(T, n_seqs) * Hq < (1l << 30));
  if (D <= 0 || D > 128 || D % 8 != 0) return MVF_ERR_UNSUPPORTED;
  const long sz = dtype == MVF_F32 ? 4 : 2;
  const long s[6] = {ldq * sz, hsq * sz, ldk * sz, hsk * sz, ldv * sz, hsv * sz};
  for (long x : s) MVF_CHECK_ARG(x > 0 && x % 16 == 0);
  MVF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest) & 15) == 0);
  FwdArgs a = {(const char*)q, (const char*)k, (const char*)v, s[0], s[1], s[2], s[3], s[4], s[5], cu_seqlens, n_seqs, (char*)out, stat,
               T, Hq, Hk, D, frame, 0, 0, scale * LOG2E, (char*)rest};
  return dtype == MVF_F32 ? launch_d<MVF_F32>(a, st) : dtype == MVF_BF16 ? launch_d<MVF_BF16>(a, st) : launch_d<MVF_F16>(a, st);
}
