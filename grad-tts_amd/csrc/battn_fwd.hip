// Attention with a learned relative position bias by buckets, gfx950, forward:
//   o_i = sum_j softmax_j(q_i . k_j scale + table[bucket(j - pos_i)][h]) v_j ,  pos_i = q_start + i
// T = fp32 / bf16 / fp16 operands on the matrix cores; scores, softmax statistics and sums in fp32, P rounded to T for
// the second product (its sum l is of the unrounded terms).
#include "battn_core.h"

namespace gt {
namespace {

// One pass over the keys with the running maximum m and sum l of each row. m moves only when a row's maximum has grown
// by 8 (in log2 units): terms stay below 2^8, and most tiles rescale nothing.
template <class T, int DP, int WR, int WS>
__global__ __launch_bounds__(64 * WR * WS, WS > 1 || sizeof(T) == 4 ? 1 : DP <= 64 ? 3 : 2) void ba_fwd_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  typedef Shape<T, DP, WS> SH;
  constexpr int KT = SH::KT, NB = SH::NB, KS = DP / 16, DB = DP / 32, NT = 64 * WR * WS;
  constexpr bool SPREAD = WS > 1;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wv % WR, ws = wv / WR;
  const int r = lane & 31, hh = lane >> 5;
  // ---- which rows
  int b, hk, g0, i0, split = 0;   // first head of the group and first query
  long blk = blockIdx.x;          // row block (spread: of all splits)
  if constexpr (SPREAD) {
    const int nbk = p.B * p.Hkv, ngb = (p.G + p.gp - 1) / p.gp;
    const long units = (long)nbk * ngb * p.ntile;
    split = (int)(blk / units);
    blk %= units;
    const int bk = (int)(blk % nbk), rest = (int)(blk / nbk);
    b = bk / p.Hkv; hk = bk % p.Hkv;
    g0 = rest % ngb * p.gp;
    i0 = tile_of(rest / ngb, p.ntile, 0) * p.qpb;
  } else {
    const int nbk = p.B * p.Hkv, bk = (int)(blk % nbk), rest = (int)(blk / nbk);
    b = bk / p.Hkv; hk = bk % p.Hkv;
    g0 = rest % p.G;
    i0 = tile_of(rest / p.G, p.ntile, p.zigzag) * 32 * WR;
  }
  const int gp = SPREAD ? p.gp : 1, rows = SPREAD ? p.qpb : 32 * WR;   // heads and queries of the workgroup
  const int qlen = clamp_len(p.qlen, b, p.Tq), klen = clamp_len(p.len, b, p.Tk), pos0 = start_of(p, b);
  const int wi0 = i0 + 32 * wr, wrows = SPREAD ? p.qpb : 32;           // this wave's queries
  const int gg = SPREAD ? r % gp : 0, qi = wi0 + (SPREAD ? min(r / gp, wrows - 1) : r);
  const int h = hk * p.G + min(g0 + gg, p.G - 1);
  const bool mine = SPREAD ? (r < gp * wrows && g0 + gg < p.G && qi < p.Tq) : qi < p.Tq, in = mine && qi < qlen;
  // ---- which keys
  int kend = klen;
  if (p.causal) kend = min(kend, pos0 + min(i0 + rows, qlen));
  if (i0 >= qlen) kend = 0;
  int kbeg = 0;
  if constexpr (SPREAD) {
    kbeg = split * p.split_keys;
    kend = min(kend, kbeg + p.split_keys);
  }
  const int elen = ext_len(p);
  float* ext0 = (float*)(smem + SH::BYTES);
  const float* ext = ext0 + (SPREAD ? gg * elen : 0) + p.dsat + EXT;   // ext[offset]
  const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h;
  const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h;
  auto tile = [&](int t, int which) { return smem + ((SH::NBUF == 2 ? t & 1 : 0) * 2 + which) * SH::TILE; };
  auto load = [&](int t) {
    stage<T, DP, KT, NT>(tile(t, 0), kb, p.ks.t, kbeg + t * KT, klen, p.D, p.vec, tid);
    stage<T, DP, KT, NT>(tile(t, 1), vb, p.vs.t, kbeg + t * KT, klen, p.D, p.vec, tid);
  };
  const int ntile = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;
  if (ntile && SH::NBUF == 2) load(0);
  frag qf[KS];
  {
    const T* qb = (const T*)p.q + b * p.qs.b + h * p.qs.h + (long)qi * p.qs.t;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = in ? load_row8(qb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
  }
  if (ntile) {
    if (p.vec && p.D < DP)
      for (int i = 0; i < 2 * SH::NBUF; ++i) clear_pad<T, DP>(smem + i * SH::TILE, KT, p.D, tid, NT);
    for (int g = 0; g < gp; ++g) build_ext<T>(p, hk * p.G + min(g0 + g, p.G - 1), ext0 + g * elen, tid, NT);
  }
  const float blo = table_at<T>(p, p.side - 1, h) * kLog2e, bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, h) * kLog2e;
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) zero16(o[d]);
  float m = -kInf, l = 0.f;
  const int pos = pos0 + qi, pmin = pos0 + wi0, pmax = pmin + wrows - 1;
  const int nkey = p.causal ? min(klen, pos + 1) : klen;                       // keys this lane's row sees
  const int wend = wi0 >= qlen ? 0 : p.causal ? min(kend, pmax + 1) : kend;    // keys this wave looks at
  for (int t = 0; t < ntile; ++t) {
    if constexpr (SH::NBUF == 2) {
      lds_ready();
      if (t + 1 < ntile) load(t + 1);
    } else {
      __syncthreads();
      load(t);
      lds_ready();
    }
    const int k0 = kbeg + t * KT + 32 * ws;
    if (k0 >= wend) continue;
    const char *sk = tile(t, 0), *sv = tile(t, 1);
    f32x16 s[NB];
    float off[NB], mt = -kInf;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int kk = k0 + 32 * WS * n, dmax = kk + 31 - pmin, dmin = kk - pmax;   // offsets of the block
      off[n] = 0.f;
      if (dmax <= -p.dsat) { off[n] = blo; zero16(s[n]); }
      else if (!p.causal && dmin >= p.dsat) { off[n] = bhi; zero16(s[n]); }
      else if (dmin > p.dsat) zero16(s[n]);   // causal, wholly unseen
      else {
        const float* e = ext + (kk + 4 * hh - pos);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[n][j] = e[acc_row(j, 0)];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) El<T>::mma(TL::row(sk, 32 * (ws + WS * n) + r, 2 * ks + hh), qf[ks], s[n]);
      if (kk + 31 >= klen || (p.causal && dmax > 0)) {
        const int lim = nkey - kk - 4 * hh;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[n][j] = acc_row(j, 0) < lim ? s[n][j] : -kInf;
      }
      float mx = fmaxf(fmaxf(s[n][0], s[n][1]), s[n][2]);
#pragma unroll
      for (int j = 3; j < 15; j += 2) mx = fmaxf(fmaxf(s[n][j], s[n][j + 1]), mx);
      mt = fmaxf(mt, __builtin_fmaf(fmaxf(mx, s[n][15]), p.c, off[n]));
    }
    mt = both_max(mt);
    if (__any(mt > m + 8.f || (m == -kInf && mt > -kInf))) {
      const float mn = fmaxf(m, mt), al = __builtin_amdgcn_exp2f(m - (mn == -kInf ? 0.f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] *= al;
    }
    const float mu = m == -kInf ? 0.f : m;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float pr[16], sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        pr[j] = expo<T>(s[n][j], p.c, off[n], mu);
        pr[j + 1] = expo<T>(s[n][j + 1], p.c, off[n], mu);
        sum0 += pr[j];
        sum1 += pr[j + 1];
      }
      l += sum0 + sum1;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const frag pf = El<T>::pack(pr + 8 * tt);
#pragma unroll
        for (int d = 0; d < DB; ++d) El<T>::mma(TL::col(sv, 32 * (ws + WS * n) + 16 * tt, d, lane), pf, o[d]);
      }
    }
  }
  l = both_sum(l);
  const long stat = ((long)b * p.Hq + h) * p.Tq + qi;
  if constexpr (!SPREAD) {
    if (!mine) return;
    T* ob = (T*)p.out + b * p.os.b + h * p.os.h + (long)qi * p.os.t;
    const bool live = in && l != 0.f;
    if (live) store_rows<T, DP>(ob, o, 1.f / l, p.D, p.vec, hh);
    else zero_rows<T, DP>(ob, p.D, p.vec, hh);
    if (p.lse && hh == 0) p.lse[stat] = live ? m + __builtin_amdgcn_logf(l) : kInf;
  } else {
    float* sml = ext0;   // [WS][2][32] (the bias table is done with)
    __syncthreads();
    if (hh == 0) { sml[ws * 64 + r] = m; sml[ws * 64 + 32 + r] = l; }
    __syncthreads();
    float M = -kInf, L = 0.f;
#pragma unroll
    for (int w = 0; w < WS; ++w) M = fmaxf(M, sml[w * 64 + r]);
    const float Mu = M == -kInf ? 0.f : M;
#pragma unroll
    for (int w = 0; w < WS; ++w) L += sml[w * 64 + 32 + r] * __builtin_amdgcn_exp2f(sml[w * 64 + r] - Mu);
    const float f = __builtin_amdgcn_exp2f(m - Mu);
    if (p.nsplit > 1) {
      const long at = blk * p.nsplit + split;
      if (tid < 32) {
        p.part_ml[at * 64 + r] = M;
        p.part_ml[at * 64 + 32 + r] = L;
      }
      if (ntile) join<DP, WS>(smem, o, f, ws, lane, tid, [&](int row, int d, const float* x) {
        float* q = p.part + (at * 32 + row) * p.D + d;
        if (p.D % 4 == 0) { if (d < p.D) *(f32x4*)q = (f32x4){x[0], x[1], x[2], x[3]}; }
        else
          for (int e = 0; e < 4; ++e) if (d + e < p.D) q[e] = x[e];
      });
      return;
    }
    const bool live = in && L != 0.f;
    if (mine && p.lse && tid < 32) p.lse[stat] = live ? M + __builtin_amdgcn_logf(L) : kInf;
    // the row's factor goes with the sum; dead rows come out as zeros whatever their lanes hold
    join<DP, WS>(smem, o, live ? f / L : 0.f, ws, lane, tid, [&](int row, int d, float* x) {
      const int g = g0 + row % gp, i = i0 + row / gp;
      if (row >= gp * wrows || g >= p.G || i >= p.Tq) return;
      if (!(i < qlen)) x[0] = x[1] = x[2] = x[3] = 0.f;
      store4_row((T*)p.out + b * p.os.b + (hk * p.G + g) * p.os.h + (long)i * p.os.t, d, x, p.D, p.vec);
    });
  }
}

// Joins the splits of a row: a wave a row, two channels a lane
template <class T> __global__ __launch_bounds__(256) void ba_join_kernel(BaParams p) {
  const int lane = threadIdx.x & 63;
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6), blk = id >> 5;
  const int row = (int)(id & 31);
  const int nbk = p.B * p.Hkv, ngb = (p.G + p.gp - 1) / p.gp;
  if (blk >= (long)nbk * ngb * p.ntile) return;
  const int bk = (int)(blk % nbk), rest = (int)(blk / nbk), b = bk / p.Hkv, hk = bk % p.Hkv;
  const int g = rest % ngb * p.gp + row % p.gp, i = tile_of(rest / ngb, p.ntile, 0) * p.qpb + row / p.gp;
  if (row >= p.gp * p.qpb || g >= p.G || i >= p.Tq) return;
  const float* ml = p.part_ml + blk * p.nsplit * 64 + row;
  float M = -kInf;
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, ml[(long)s * 64]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float Mu = M == -kInf ? 0.f : M;
  float L = 0.f, a0 = 0.f, a1 = 0.f;
  const float* part = p.part + (blk * p.nsplit * 32 + row) * p.D;
  for (int s = 0; s < p.nsplit; ++s) {
    const float ls = ml[(long)s * 64 + 32];
    if (ls == 0.f) continue;   // saw no key (its sums were not written)
    const float f = __builtin_amdgcn_exp2f(ml[(long)s * 64] - Mu);
    const float* q = part + (long)s * 32 * p.D;
    L = __builtin_fmaf(ls, f, L);
    if (lane < p.D) a0 = __builtin_fmaf(q[lane], f, a0);
    if (lane + 64 < p.D) a1 = __builtin_fmaf(q[lane + 64], f, a1);
  }
  const bool live = i < clamp_len(p.qlen, b, p.Tq) && L != 0.f;
  const int h = hk * p.G + g;
  T* ob = (T*)p.out + b * p.os.b + h * p.os.h + (long)i * p.os.t;
  if (lane < p.D) ob[lane] = (T)(live ? a0 / L : 0.f);
  if (lane + 64 < p.D) ob[lane + 64] = (T)(live ? a1 / L : 0.f);
  if (p.lse && lane == 0) p.lse[((long)b * p.Hq + h) * p.Tq + i] = live ? M + __builtin_amdgcn_logf(L) : kInf;
}

// ---------------------------------------------------------------- launches
// Shared form where it fills the chip (a workgroup of 128 rows for each CU), else the spread form: rows of all heads
// that share a key / value head packed into blocks of 32, four waves over the keys, and, where few blocks meet long
// caches, key ranges with workgroups of their own (about four a CU, of four tiles at least) joined afterwards.
constexpr int WSP = 4;
struct FwdPlan { bool spread; long units; };
FwdPlan plan_fwd(BaParams& p) {
  const long shared = (long)p.B * p.Hq * ((p.Tq + 127) / 128);
  FwdPlan f{shared < 256, 0};
  p.nsplit = 1;
  if (!f.spread) {
    p.ntile = (p.Tq + 127) / 128;
    p.zigzag = shared <= 1024;
    return f;
  }
  p.gp = p.G < 32 ? p.G : 32;
  while (p.gp > 1 && p.gp * host_ext_bytes(p) > 24 * 1024) p.gp = (p.gp + 1) / 2;
  p.qpb = 32 / p.gp;
  p.ntile = (p.Tq + p.qpb - 1) / p.qpb;
  f.units = (long)p.B * p.Hkv * ((p.G + p.gp - 1) / p.gp) * p.ntile;
  constexpr int KT = 32 * WSP;
  p.split_keys = (p.Tk + KT - 1) / KT * KT;
  if (f.units && f.units < 512 && p.Tk > 4 * KT) {
    long n = (1024 + f.units - 1) / f.units;
    if (n > 512) n = 512;
    long keys = ((p.Tk + n - 1) / n + KT - 1) / KT * KT;
    if (keys < 4 * KT) keys = 4 * KT;
    p.split_keys = (int)keys;
    p.nsplit = (int)((p.Tk + keys - 1) / keys);
  }
  return f;
}

template <class T, int DP> hipError_t fwd(const BaParams& p, const FwdPlan& f, hipStream_t s) {
  if (!f.spread)
    return launch(ba_fwd_kernel<T, DP, 4, 1>, (long)p.B * p.Hq * p.ntile, 256, Shape<T, DP, 1>::BYTES + host_ext_bytes(p), p, s);
  constexpr int joined = WSP * DP * 33 * 4, base = Shape<T, DP, WSP>::BYTES;
  static_assert(joined <= base && base + 24 * 1024 <= kLds, "LDS");
  int ext = p.gp * host_ext_bytes(p);
  if (ext < WSP * 64 * 4) ext = WSP * 64 * 4;
  hipError_t e = launch(ba_fwd_kernel<T, DP, 1, WSP>, f.units * p.nsplit, 64 * WSP, base + ext, p, s);
  if (e != hipSuccess || p.nsplit == 1) return e;
  const long blocks = (f.units * 32 + 3) / 4;
  if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((ba_join_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <class T> hipError_t fwd_t(const BaParams& p, const FwdPlan& f, hipStream_t s) {
  return p.D <= 64 ? fwd<T, 64>(p, f, s) : p.D <= 96 ? fwd<T, 96>(p, f, s) : fwd<T, 128>(p, f, s);
}

}  // namespace

size_t ba_forward_ws(const BaParams& p0, int) {
  BaParams p = p0;
  const FwdPlan f = plan_fwd(p);
  if (p.nsplit == 1) return 0;
  return up256((size_t)f.units * p.nsplit * 32 * p.D * 4) + (size_t)f.units * p.nsplit * 64 * 4 + 256;
}
hipError_t launch_ba_forward(BaParams p, int dtype, void* ws, hipStream_t s) {
  const FwdPlan f = plan_fwd(p);
  if (p.nsplit > 1) {
    char* w = align256(ws);
    p.part = (float*)w;
    p.part_ml = (float*)(w + up256((size_t)f.units * p.nsplit * 32 * p.D * 4));
  }
  return dtype == 0 ? fwd_t<float>(p, f, s) : dtype == 1 ? fwd_t<bf16>(p, f, s) : fwd_t<f16>(p, f, s);
}

}  // namespace gt
