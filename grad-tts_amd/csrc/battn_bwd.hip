// Attention with a learned relative position bias by buckets, gfx950, backward:
//   P = 2^(scores - lse),  dP = dO V^T,  delta = rowsum(P o dP) (= rowsum(o o dO)),  dS = P o (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,  dtable[c][h] = sum of dS over the pairs of bucket c
// Two kernels, each the sole writer of its rows, so that every sum has one order: dQ (with delta and the table's
// partial sums) streams keys past 32-row query blocks, dK dV streams queries past key blocks. Scores and dP are formed
// in both: 7 products instead of 5, against atomics or a T x T matrix in memory.
//
// Bound by the waves' own latency: at 128 channels the stationary rows, their sums and a block's fragments fill the
// registers of one wave a SIMD (dK dV) or two (dQ), so products wait for LDS reads and exponentials more than they
// overlap with them. 2 x 16 bf16 heads (4 key / value heads) of 2048 causal rows, 128 channels: dQ 93 us (0.55 PFLOP/s),
// dK dV 105 (0.65), sums of head groups 14 (4.8 TB/s), table 5; 3 x 6 fp16 heads of 777 rows, 80 channels: 40, 35, -, 4.
// Registers spill in some forms: 7 in the 16-bit dQ of 128 channels, 9 to 11 in the 16-bit dK dV of 64 channels and 128
// rows, 67 to 86 in the fp32 dK dV of 128 channels (2 x 16 heads, 4 key / value heads, 1024 causal rows: 296 us).
#include <type_traits>

#include "battn_core.h"

namespace gt {
namespace {

// Sums over the diagonals of a 32 x 32 block (rows: registers and lane half, columns: lane & 31): lane i of the result
// has those with row - column = 31 - i. Rows in ascending order, the running sums moving up a lane before each row:
// one add with a lane shift (v_add_f32, wave_shr:1) a row.
GT_DEV float diagonals(const float (&x)[16]) {
  float a = 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float lo[4], hi[4];   // rows 8 g + e and 8 g + 4 + e in lanes 0 .. 31, zeros above
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[4 * g + e]), 0u, false, false);
      lo[e] = __uint_as_float(w[0]);
      hi[e] = __uint_as_float(w[1]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float up = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(a), 0x138, 0xf, 0xf, true));
      a = up + (e < 4 ? lo[e & 3] : hi[e & 3]);
    }
  }
  return a;
}

// fp16 rounds P <= 1 below 2^-14 to steps of 2^-25: a row of thousands of keys loses digits of it. There dK dV forms
// 2^15 P, in the exponent, and takes the factor out of dV's sums and, by way of delta (kept times 2^-15) and one FMA in
// place of a subtraction, of dS. The other types have fp32's range.
template <class T> constexpr float kUp = std::is_same<T, f16>::value ? 15.f : 0.f;
template <class T> constexpr float kDown = std::is_same<T, f16>::value ? 0x1p-15f : 1.f;

// ================================================================ dQ, delta, table partials
// The product o . do with the rounded o, formed from rounded P, is off by about u |o| |do| (u = half a step of the
// type), which weighs when few keys share a row: dS = P (dP - delta) is then a small difference. Rows whose keys all lie
// in the first tile therefore sum P dP itself in fp32 (both are at hand; bf16, 14 keys: dq's error 2.5e-3 where the
// product's gave 5.4e-3). The others take the product, from the matrix cores in the channel order of dP: so does a row
// with one visible key (o = v), whose delta then equals dP bit for bit and whose dS is exactly zero.
template <class T, int DP, int WR, int WS>
__global__ __launch_bounds__(64 * WR * WS, WS > 2 || sizeof(T) == 4 ? 1 : 2) void ba_dq_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  typedef Shape<T, DP, WR, WS> SH;
  constexpr int KT = SH::KT, NB = SH::NB, KS = DP / 16, DB = DP / 32, NT = 64 * WR * WS, NW = WR * WS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int elen = ext_len(p);
  float* ext0 = (float*)(smem + SH::BYTES);
  const float* ext = ext0 + p.dsat + EXT;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wv % WR, ws = wv / WR;
  const int r = lane & 31, hh = lane >> 5, D = p.D;
  float* tacc = ext0 + (1 + wv) * elen + p.dsat + EXT;   // this wave's sums of dS by offset
  float* sat = ext0 + (1 + NW) * elen;                   // [NW][2]; [NW][32] before
  const int nbk = p.B * p.Hkv, bk = blockIdx.x % (unsigned)nbk, rest = blockIdx.x / (unsigned)nbk, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int h = hk * p.G + rest % p.G, rank = rest / p.G;
  const int qlen = clamp_len(p.qlen, b, p.Tq), pos0 = start_of(p, b), klen = keys_of(p, b, qlen, pos0);
  const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h;
  const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h;
  auto tile = [&](int t, int which) { return smem + ((SH::NBUF == 2 ? t & 1 : 0) * 2 + which) * SH::TILE; };
  Stage<T, DP, KT, NT> ks, vs;
  ks.init(kb, p.ks.t, klen, p.D, p.vec, tid);
  vs.init(vb, p.vs.t, klen, p.D, p.vec, tid);
  auto load = [&](int t) {
    ks.load(tile(t, 0), t * KT);
    vs.load(tile(t, 1), t * KT);
  };
  float slo = 0.f, shi = 0.f;   // dS beyond the last border
  const int tl = p.ntile - 1 - rank;   // the longest under a causal mask first
  const int q0 = tl * 32 * WR, wq0 = q0 + 32 * wr, qi = wq0 + r;
  int kend = klen;
  if (p.causal) kend = min(kend, pos0 + min(q0 + 32 * WR, qlen));
  if (q0 >= qlen) kend = 0;
  if (p.vec && D < DP)
    for (int i = 0; i < 2 * SH::NBUF; ++i) clear_pad<T, DP>(smem + i * SH::TILE, KT, D, tid, NT);
  const int ntile = kend > 0 ? (kend + KT - 1) / KT : 0;
  if (ntile && SH::NBUF == 2) load(0);
  const long srow = ((long)b * p.Hq + h) * p.Tq + qi;
  const bool in = qi < qlen;
  frag qf[KS], gf[KS];
  float delta = 0.f;
  if (qlen > 0) {   // rows past the last valid one repeat it: their P is zero (lse), their results are not kept
    const long row = min(qi, qlen - 1);
    frag of[KS];
    load_rows<T, KS>(qf, (const T*)p.q + b * p.qs.b + h * p.qs.h + row * p.qs.t, hh, D, p.vec);
    load_rows<T, KS>(gf, (const T*)p.dout + b * p.dos.b + h * p.dos.h + row * p.dos.t, hh, D, p.vec);
    load_rows<T, KS>(of, (const T*)p.o + b * p.os.b + h * p.os.h + row * p.os.t, hh, D, p.vec);
    f32x16 dg = mma0<T>(of[0], gf[0]);
#pragma unroll
    for (int s = 1; s < KS; ++s) El<T>::mma(of[s], gf[s], dg);
    // the diagonal: row r of column r, held by lane half (r >> 2) & 1 in register (r & 3) + 4 (r >> 3)
#pragma unroll
    for (int j = 0; j < 16; ++j) delta = acc_row(j, hh) == r ? dg[j] : delta;
    float a, c;
    halves(delta, a, c);
    delta = ((r >> 2) & 1) ? c : a;
  }
  const float lse = in ? p.lse[srow] : kInf;
  for (int i = tid; i < NW * elen; i += NT) ext0[elen + i] = 0.f;
  build_ext<T>(p, h, 1, h, ext0, tid, NT);
  const float blo = table_at<T>(p, p.side - 1, h) * kLog2e, bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, h) * kLog2e;
  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) zero16(dq[d]);
  const int pos = pos0 + qi, pmin = pos0 + wq0, pmax = pmin + 31;
  const int nkey = p.causal ? min(klen, pos + 1) : klen;                       // keys this lane's row sees
  const int wend = wq0 >= qlen ? 0 : p.causal ? min(kend, pmax + 1) : kend;    // keys this wave looks at
  // P and dP of the 32 keys from kk on (block j2 of the tile); unseen keys: 0
  auto probs = [&](const char* sk, const char* sv, int kk, int j2, float (&pr)[16], f32x16& dp) {
    const int dmax = kk + 31 - pmin, dmin = kk - pmax;
    f32x16 s;
    float off = 0.f;
    // fragments of each operand read together, then multiplied: four, at 128 channels two (their registers spilled
    // there: 111 us against 96 for 2 x 16 heads, 2048 causal rows)
    constexpr int CH = KS % 4 ? 3 : KS > 4 ? 2 : 4;
    frag a[CH], c[CH];
    auto read = [&](int k0) {
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        a[x] = TL::row(sk, 32 * j2 + r, 2 * (k0 + x) + hh);
        c[x] = TL::row(sv, 32 * j2 + r, 2 * (k0 + x) + hh);
      }
    };
    read(0);
    if (one_bias(dmin, dmax, p.dsat, p.causal)) {
      off = dmin < 0 ? blo : bhi;
      s = mma0<T>(a[0], qf[0]);
    } else {
      const float* e = ext + (kk + 4 * hh - pos);
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = e[acc_row(j, 0)];
      El<T>::mma(a[0], qf[0], s);
    }
    dp = mma0<T>(c[0], gf[0]);
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += CH) {
      if (k0) read(k0);
#pragma unroll
      for (int x = k0 ? 0 : 1; x < CH; ++x) {
        El<T>::mma(a[x], qf[k0 + x], s);
        El<T>::mma(c[x], gf[k0 + x], dp);
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) pr[j] = expo<T>(s[j], p.c, off, lse);
    if (kk + 31 >= klen || (p.causal && dmax > 0)) {
      int lim = nkey - kk - 4 * hh;
      in_branch(lim);
#pragma unroll
      for (int j = 0; j < 16; ++j) pr[j] = acc_row(j, 0) < lim ? pr[j] : 0.f;
    }
  };
  auto step = [&](int t, auto buf) {   // buf: t & 1, a constant at both calls
    if constexpr (SH::NBUF == 2) {
      lds_ready();
      if (t + 1 < ntile) load(t + 1);
    } else {
      __syncthreads();
      load(t);
      lds_ready();
    }
    const char *sk = tile(buf, 0), *sv = tile(buf, 1);
    if (t == 0 && (WS > 1 ? kend : wend) <= KT) {
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int kk = 32 * (ws + WS * n);
        if (kk >= wend) break;
        float pr[16];
        f32x16 dp;
        probs(sk, sv, kk, ws + WS * n, pr, dp);
#pragma unroll
        for (int j = 0; j < 16; ++j) sum = acc_row(j, hh) + kk < nkey ? __builtin_fmaf(pr[j], dp[j], sum) : sum;
      }
      sum = both_sum(sum);
      if constexpr (WS > 1) {   // all of the workgroup is here: its keys all lie in this tile
        if (hh == 0) sat[32 * wv + r] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WS; ++w) sum += sat[32 * (wr + WR * w) + r];
      }
      if (nkey > 1) delta = sum;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int j2 = ws + WS * n, kk = t * KT + 32 * j2;
      if (kk >= wend) break;
      const int dmax = kk + 31 - pmin, dmin = kk - pmax;
      float ds[16];
      f32x16 dp;
      probs(sk, sv, kk, j2, ds, dp);
      frag kc[DB];   // the first group's ahead of the arithmetic
#pragma unroll
      for (int d = 0; d < DB; ++d) kc[d] = TL::col(sk, 32 * j2, d, lane);
#pragma unroll
      for (int j = 0; j < 16; ++j) ds[j] *= dp[j] - delta;
      if (one_bias(dmin, dmax, p.dsat, p.causal)) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) a += ds[j];
        if (dmin < 0) slo += a;
        else shi += a;
      } else {
        const float a = diagonals(ds);   // lane i: offset kk - pmin + 31 - i
        if (lane < 63)                   // one add an offset and block, this wave's own array: one order
          __hip_atomic_fetch_add(tacc + (kk - pmin + 31 - lane), a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const frag df = El<T>::pack(ds + 8 * tt);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          El<T>::mma(kc[d], df, dq[d]);
          if (tt == 0) kc[d] = TL::col(sk, 32 * j2 + 16, d, lane);
        }
      }
    }
  };
  for (int t = 0; t < ntile; t += 2) {
    step(t, std::integral_constant<int, 0>());
    if (t + 1 < ntile) step(t + 1, std::integral_constant<int, 1>());
  }
  if (qi < p.Tq && hh == 0 && ws == 0) p.delta[srow] = in ? delta * kDown<T> : 0.f;
  if constexpr (WS == 1) {
    if (qi < p.Tq) {
      T* qo = (T*)p.dq + b * p.dqs.b + h * p.dqs.h + (long)qi * p.dqs.t;
      if (in) store_rows<T, DP>(qo, dq, p.scale, D, p.vec, hh);
      else zero_rows<T, DP>(qo, D, p.vec, hh);
    }
  } else {
    join<DP, WS>(smem, dq, p.scale, wr, ws, lane, [&](int row, int d, float* x) {
      const int i = wq0 + row;
      if (i >= p.Tq) return;
      if (!(i < qlen)) x[0] = x[1] = x[2] = x[3] = 0.f;
      store4_row((T*)p.dq + b * p.dqs.b + h * p.dqs.h + (long)i * p.dqs.t, d, x, D, p.vec);
    });
  }
  // table partials of the workgroup: a wave a bucket, its lanes over the bucket's offsets, then across the lanes in one order
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) {
    slo += __shfl_xor(slo, x);
    shi += __shfl_xor(shi, x);
  }
  __syncthreads();
  if (lane == 0) { sat[2 * wv] = slo; sat[2 * wv + 1] = shi; }
  __syncthreads();
  const long npart = (long)p.B * p.ntile;
  for (int c = wv; c < p.nb; c += NW) {
    const int side = c >= p.side, cc = side ? c - p.side : c;
    int d0, d1;   // distances of the bucket
    if (cc < p.exact) {
      d0 = cc;
      d1 = cc + 1;
    } else {
      d0 = cc == p.exact ? p.exact : p.border[cc - p.exact - 1];
      d1 = cc == p.side - 1 ? p.dsat + EXT + 1 : p.border[cc - p.exact];
    }
    if (side && d0 == 0) d0 = 1;   // offset 0 belongs to the first half
    float a = 0.f;
    for (int d = d0 + lane; d < d1; d += 64)
#pragma unroll
      for (int w = 0; w < NW; ++w) a += ext0[(1 + w) * elen + p.dsat + EXT + (side ? d : -d)];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) a += __shfl_xor(a, x);
    if (cc == p.side - 1)
      for (int w = 0; w < NW; ++w) a += sat[2 * w + side];
    if (lane == 0) p.tpart[((long)c * p.Hq + h) * npart + (long)b * p.ntile + rank] = a;
  }
}

template <class T> __global__ __launch_bounds__(64) void ba_dtable_kernel(const float* part, long npart, T* dtable) {
  const float* x = part + (long)blockIdx.x * npart;
  float a = 0.f;
  for (long i = threadIdx.x; i < npart; i += 64) a += x[i];
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) a += __shfl_xor(a, s);
  if (threadIdx.x == 0) dtable[blockIdx.x] = (T)a;
}

// ================================================================ dK, dV
// 32 WR keys of one key / value head over the query tiles of the heads that share it, or, where that leaves CUs idle, of
// a part of them (gsplit), summed afterwards in fp32.
template <class T, int DP, int WR, int WS>
__global__ __launch_bounds__(64 * WR * WS, WS > 2 || sizeof(T) == 4 || DP > 64 ? 1 : 2) void ba_dkv_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  typedef Shape<T, DP, WR, WS> SH;
  constexpr int QT = SH::KT, NB = SH::NB, KS = DP / 16, DB = DP / 32, NT = 64 * WR * WS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* stat = (float*)(smem + SH::BYTES);   // [NBUF][2][QT]: lse, delta of the tile's rows
  float* ext0 = stat + SH::NBUF * 2 * QT;
  const float* ext = ext0 + p.dsat + EXT;
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wv % WR, ws = wv / WR;
  const int nbk = p.B * p.Hkv, bk = blockIdx.x % (unsigned)nbk, rest = blockIdx.x / (unsigned)nbk, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int gpart = rest % p.gsplit, rank = rest / p.gsplit;
  const int qlen = clamp_len(p.qlen, b, p.Tq), pos0 = start_of(p, b), klen = keys_of(p, b, qlen, pos0);
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {   // a tile from the start and, paired, its mirror image
    if (pass && (!p.pair || 2 * rank >= p.ntile - 1)) break;
    const int lane = anew_v(tid & 63), r = lane & 31, hh = lane >> 5, D = anew_s(p.D);
    const int tl = pass ? p.ntile - 1 - rank : rank;
    const int k0 = tl * 32 * WR, wk0 = k0 + 32 * wr, ki = wk0 + r;
    if (pass) __syncthreads();   // the first pass's LDS is done with
    const int qbeg = (p.causal ? max(0, k0 - pos0) : 0) / QT * QT;   // first tile with a query that sees key k0
    const int qend = k0 < klen ? qlen : 0;
    const bool in = ki < klen;
    const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h + (long)min(ki, klen - 1) * p.ks.t;   // (rows past the last valid
    const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h + (long)min(ki, klen - 1) * p.vs.t;   // one repeat it, masked)
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) { zero16(dk[d]); zero16(dv[d]); }
    if (qbeg < qend) {
      frag kf[KS], vf[KS];
      load_rows<T, KS>(kf, kb, hh, D, p.vec);
      load_rows<T, KS>(vf, vb, hh, D, p.vec);
      if (p.vec && D < DP)
        for (int i = 0; i < 2 * SH::NBUF; ++i) clear_pad<T, DP>(smem + i * SH::TILE, QT, D, tid, NT);
      const int ntile = (qend - qbeg + QT - 1) / QT, hper = p.G / p.gsplit;
      for (int g = 0; g < hper; ++g) {
        const int h = hk * p.G + gpart * hper + g;
        const T* qb = (const T*)p.q + b * p.qs.b + h * p.qs.h;
        const T* gb = (const T*)p.dout + b * p.dos.b + h * p.dos.h;
        const float* lse = p.lse + ((long)b * p.Hq + h) * p.Tq;
        const float* del = p.delta + ((long)b * p.Hq + h) * p.Tq;
        auto tile = [&](int t, int which) { return smem + ((SH::NBUF == 2 ? t & 1 : 0) * 2 + which) * SH::TILE; };
        auto stats = [&](int t) { return stat + (SH::NBUF == 2 ? t & 1 : 0) * 2 * QT; };
        Stage<T, DP, QT, NT> qs, gs;
        qs.init(qb, p.qs.t, qlen, D, p.vec, tid);
        gs.init(gb, p.dos.t, qlen, D, p.vec, tid);
        auto load = [&](int t) {
          const int q0 = qbeg + t * QT;
          qs.load(tile(t, 0), q0);
          gs.load(tile(t, 1), q0);
          // one wave copies the row statistics of 64 rows at a time (rows past the last repeat it and are masked)
          const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
          for (int i = wave; i < 2 * ((QT + 63) / 64); i += NT / 64) {
            const int which = i & 1, row = (i >> 1) * 64 + lane;
            if (row < QT)
              __builtin_amdgcn_global_load_lds((const void*)((which ? del : lse) + min(q0 + row, qlen - 1)),
                                               (__attribute__((address_space(3))) void*)(stats(t) + which * QT + (i >> 1) * 64), 4, 0, 0);
          }
        };
        __syncthreads();   // the last head's tiles and bias are done with
        if (SH::NBUF == 2) load(0);
        build_ext<T>(p, h, 1, h, ext0, tid, NT);
        const float blo = table_at<T>(p, p.side - 1, h) * kLog2e + kUp<T>;
        const float bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, h) * kLog2e + kUp<T>;
        auto step = [&](int t, auto buf) {   // buf: t & 1, a constant at both calls
          if constexpr (SH::NBUF == 2) {
            lds_ready();
            if (t + 1 < ntile) load(t + 1);
          } else {
            __syncthreads();
            load(t);
            lds_ready();
          }
          const char *sq = tile(buf, 0), *sg = tile(buf, 1);
          const float* st = stats(buf);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const int j2 = ws + WS * n, qq = qbeg + t * QT + 32 * j2, pmin = pos0 + qq, pmax = pmin + 31;
            if (qq >= qend) break;
            if (p.causal && pmax < wk0) continue;
            const int dmax = wk0 + 31 - pmin, dmin = wk0 - pmax;
            f32x16 s, dp;
            float off = kUp<T>;
            constexpr int CH = KS % 4 ? 3 : 4;
            frag a[CH], c[CH];
            auto read = [&](int x0) {
#pragma unroll
              for (int x = 0; x < CH; ++x) {
                a[x] = TL::row(sq, 32 * j2 + r, 2 * (x0 + x) + hh);
                c[x] = TL::row(sg, 32 * j2 + r, 2 * (x0 + x) + hh);
              }
            };
            read(0);
            if (one_bias(dmin, dmax, p.dsat, p.causal)) {
              off = dmin < 0 ? blo : bhi;
              s = mma0<T>(a[0], kf[0]);
            } else {
              const float* e = ext + (ki - pmin - 4 * hh);
#pragma unroll
              for (int j = 0; j < 16; ++j) s[j] = e[-acc_row(j, 0)];
              El<T>::mma(a[0], kf[0], s);
            }
            dp = mma0<T>(c[0], vf[0]);
#pragma unroll
            for (int x0 = 0; x0 < KS; x0 += CH) {
              if (x0) read(x0);
#pragma unroll
              for (int x = x0 ? 0 : 1; x < CH; ++x) {
                El<T>::mma(a[x], kf[x0 + x], s);
                El<T>::mma(c[x], vf[x0 + x], dp);
              }
            }
            float pr[16], ds[16];
#pragma unroll
            for (int jg = 0; jg < 4; ++jg) {
              const f32x4 ls = *(const f32x4*)(st + 32 * j2 + 8 * jg + 4 * hh), de = *(const f32x4*)(st + QT + 32 * j2 + 8 * jg + 4 * hh);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = 4 * jg + e;
                pr[j] = expo<T>(s[j], p.c, off, ls[e]);
                ds[j] = pr[j] * (kDown<T> == 1.f ? dp[j] - de[e] : __builtin_fmaf(dp[j], kDown<T>, -de[e]));
              }
            }
            if (wk0 + 31 >= klen || qq + 31 >= qlen || (p.causal && dmax > 0)) {
              // rows that see this lane's key
              int first = p.causal ? ki - pmin - 4 * hh : -64, last = in ? qlen - qq - 4 * hh : -64;
              in_branch(first);
              in_branch(last);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const bool see = acc_row(j, 0) >= first && acc_row(j, 0) < last;
                pr[j] = see ? pr[j] : 0.f;
                ds[j] = see ? ds[j] : 0.f;
              }
            }
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
              frag x[DB];
#pragma unroll
              for (int d = 0; d < DB; ++d) x[d] = TL::col(sg, 32 * j2 + 16 * tt, d, lane);
              const frag pf = El<T>::pack(pr + 8 * tt), df = El<T>::pack(ds + 8 * tt);
#pragma unroll
              for (int d = 0; d < DB; ++d) {
                El<T>::mma(x[d], pf, dv[d]);
                x[d] = TL::col(sq, 32 * j2 + 16 * tt, d, lane);
              }
#pragma unroll
              for (int d = 0; d < DB; ++d) El<T>::mma(x[d], df, dk[d]);
            }
          }
        };
        for (int t = 0; t < ntile; t += 2) {
          step(t, std::integral_constant<int, 0>());
          if (t + 1 < ntile) step(t + 1, std::integral_constant<int, 1>());
        }
      }
    }
    // rows behind the sequence are zeros whatever the streamed rows hold
    const int v4 = D % 4 == 0;
    const long half = (long)p.gsplit * p.B * p.Tk * p.Hkv * p.D;
    auto part = [&](int row) { return p.gpart + ((((long)gpart * p.B + b) * p.Tk + row) * p.Hkv + hk) * p.D; };
    T* ko = (T*)p.dk + b * p.dks.b + hk * p.dks.h;
    T* vo = (T*)p.dv + b * p.dvs.b + hk * p.dvs.h;
    if constexpr (WS == 1) {
      if (ki >= p.Tk) {
        // no such row
      } else if (p.gsplit > 1) {
        if (in) {
          store_rows<float, DP>(part(ki), dk, p.scale, D, v4, hh);
          store_rows<float, DP>(part(ki) + half, dv, kDown<T>, D, v4, hh);
        } else {
          zero_rows<float, DP>(part(ki), D, v4, hh);
          zero_rows<float, DP>(part(ki) + half, D, v4, hh);
        }
      } else if (in) {
        store_rows<T, DP>(ko + (long)ki * p.dks.t, dk, p.scale, D, p.vec, hh);
        store_rows<T, DP>(vo + (long)ki * p.dvs.t, dv, kDown<T>, D, p.vec, hh);
      } else {
        zero_rows<T, DP>(ko + (long)ki * p.dks.t, D, p.vec, hh);
        zero_rows<T, DP>(vo + (long)ki * p.dvs.t, D, p.vec, hh);
      }
    } else {
      join<DP, WS>(smem, dk, p.scale, wr, ws, lane, [&](int row, int d, float* x) {
        if (wk0 + row >= p.Tk) return;
        if (wk0 + row >= klen) x[0] = x[1] = x[2] = x[3] = 0.f;
        if (p.gsplit > 1) store4_row(part(wk0 + row), d, x, D, v4);
        else store4_row(ko + (long)(wk0 + row) * p.dks.t, d, x, D, p.vec);
      });
      join<DP, WS>(smem, dv, kDown<T>, wr, ws, lane, [&](int row, int d, float* x) {
        if (wk0 + row >= p.Tk) return;
        if (wk0 + row >= klen) x[0] = x[1] = x[2] = x[3] = 0.f;
        if (p.gsplit > 1) store4_row(part(wk0 + row) + half, d, x, D, v4);
        else store4_row(vo + (long)(wk0 + row) * p.dvs.t, d, x, D, p.vec);
      });
    }
  }
}

// dk, dv from the head groups' sums, in order: four channels a thread, or one where D % 4
template <class T, int N> __global__ __launch_bounds__(256) void ba_gsum_kernel(BaParams p) {
  const long n = (long)p.B * p.Tk * p.Hkv * p.D, i = ((long)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= 2 * n) return;
  const bool second = i >= n;
  const long e = second ? i - n : i, row = e / p.D;
  const float* x = p.gpart + (second ? p.gsplit * n : 0) + e;
  float a[N];
#pragma unroll
  for (int c = 0; c < N; ++c) a[c] = 0.f;
  for (int g = 0; g < p.gsplit; ++g) {
    if constexpr (N == 4) {
      const f32x4 v = *(const f32x4*)(x + g * n);
#pragma unroll
      for (int c = 0; c < 4; ++c) a[c] += v[c];
    } else {
      a[0] += x[g * n];
    }
  }
  const BaStride st = second ? p.dvs : p.dks;
  const long pos = row / p.Hkv;
  T* out = (T*)(second ? p.dv : p.dk) + pos / p.Tk * st.b + pos % p.Tk * st.t + row % p.Hkv * st.h + e % p.D;
  if (N == 4 && p.vec) El<T>::store4(out, a);
  else
#pragma unroll
    for (int c = 0; c < N; ++c) out[c] = (T)a[c];
}

// ---------------------------------------------------------------- launches
constexpr int kSat = 4 * 32 * 4;   // bytes of `sat`, four waves
struct BwdPlan { int rows_q, rows_k, gsplit, ntq, ntk, ranks_k, pair_k; };
// Rows a workgroup, by how many workgroups that makes; us of the backward with 32 / 64 / 128 rows at (heads x batch, T,
// head size):
//   128 rows from two workgroups a CU on (fp32, not causal: one): bf16 (128, 512, 64) 148 / 84 / 67, causal 124 / 67 / 61,
//   below (64, 512, 64) 80 / 49 / 51; fp32 (64, 512, 128) 790 / 458 / 364; but not the 16-bit dQ of 128 channels, whose
//   registers spill there (2 x 16 causal heads, 2048 rows: dQ 97 us with 64, 116 with 128);
//   64 rows from 192 workgroups on: bf16 (64, 190, 64) 39 / 30, fp32 86 / 58; below (32, 190, 64) 28 / 30, 47 / 57. fp32
//   of more than 64 channels, one workgroup a CU either way: always (32, 190, 128) 118 / 101, (8, 64, 96) 52 / 46.
int rows_of(const BaParams& p, int dtype, long heads, int T) {
  const bool wide = dtype == 0;
  if (fills128(dtype, T) && heads * ((T + 127) / 128) >= (wide && !p.causal ? 256 : 512)) return 128;
  return heads * ((T + 63) / 64) >= 192 || (wide && p.D > 64) ? 64 : 32;
}
BwdPlan plan_bwd(const BaParams& p, int dtype) {
  BwdPlan b;
  const int dp = p.D <= 64 ? 64 : p.D <= 96 ? 96 : 128, spread = 1024 * dp;   // the spread Shape's bytes, any type
  b.rows_q = rows_of(p, dtype, (long)p.B * p.Hq, p.Tq);
  if (b.rows_q == 128 && dtype != 0 && dp == 128) b.rows_q = 64;
  // (the spread form's LDS does not hold the table sums of far borders)
  if (b.rows_q == 32 && spread + 5 * host_ext_bytes(p) + kSat > kLds) b.rows_q = 64;
  b.ntq = (p.Tq + b.rows_q - 1) / b.rows_q;
  const long kv = (long)p.B * p.Hkv;
  b.rows_k = rows_of(p, dtype, kv * p.G, p.Tk);
  b.ntk = (p.Tk + b.rows_k - 1) / b.rows_k;
  // causal dK dV: a tile and its mirror image a workgroup, so that all are equally long, unless every tile has a CU of its
  // own: bf16 (32, 2048, 128) 212 us paired, 271 not; (64, 190, 128) 51 and 41
  b.pair_k = p.causal && kv * p.G * b.ntk > 256;
  b.ranks_k = b.pair_k ? (b.ntk + 1) / 2 : b.ntk;
  // the heads of a group in several workgroups until every CU has one
  b.gsplit = 1;
  while (b.gsplit < p.G && kv * b.ranks_k * b.gsplit < 256)
    do ++b.gsplit; while (p.G % b.gsplit);
  return b;
}

template <class T, int DP, int WR> hipError_t bwd_q(BaParams p, const BwdPlan& b, hipStream_t s) {
  typedef Shape<T, DP, WR, 4 / WR> SH;
  static_assert(WR > 1 || SH::BYTES == 1024 * DP, "plan_bwd");
  const long grid = (long)p.B * p.Hq * b.ntq;
  p.ntile = b.ntq;
  return launch(ba_dq_kernel<T, DP, WR, 4 / WR>, grid, 256, SH::BYTES + 5 * host_ext_bytes(p) + kSat, p, s);
}
template <class T, int DP, int WR> hipError_t bwd_k(BaParams p, const BwdPlan& b, hipStream_t s) {
  typedef Shape<T, DP, WR, 4 / WR> SH;
  const long grid = (long)p.B * p.Hkv * b.gsplit * b.ranks_k;
  p.ntile = b.ntk;
  p.pair = b.pair_k;
  return launch(ba_dkv_kernel<T, DP, WR, 4 / WR>, grid, 256, SH::BYTES + SH::NBUF * 2 * SH::KT * 4 + host_ext_bytes(p), p, s);
}
template <class T, int DP> hipError_t bwd(const BaParams& p, const BwdPlan& b, hipStream_t s) {
  constexpr bool few = sizeof(T) == 2 || DP <= 64, many = sizeof(T) == 4 || DP < 128;   // as plan_bwd gives them
  hipError_t e = hipErrorInvalidValue;
  if (b.rows_q == 64) e = bwd_q<T, DP, 2>(p, b, s);
  if constexpr (many)
    if (b.rows_q == 128) e = bwd_q<T, DP, 4>(p, b, s);
  if constexpr (few)
    if (b.rows_q == 32) e = bwd_q<T, DP, 1>(p, b, s);
  if (e != hipSuccess) return e;
  e = hipErrorInvalidValue;
  if (b.rows_k == 128) e = bwd_k<T, DP, 4>(p, b, s);
  if (b.rows_k == 64) e = bwd_k<T, DP, 2>(p, b, s);
  if constexpr (few)
    if (b.rows_k == 32) e = bwd_k<T, DP, 1>(p, b, s);
  if (e != hipSuccess) return e;
  if (p.gsplit > 1) {
    const bool four = p.D % 4 == 0;
    const long n = 2L * p.B * p.Tk * p.Hkv * p.D / (four ? 4 : 1), blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    if (blocks && four) hipLaunchKernelGGL((ba_gsum_kernel<T, 4>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    else if (blocks) hipLaunchKernelGGL((ba_gsum_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  hipLaunchKernelGGL((ba_dtable_kernel<T>), dim3((unsigned)(p.nb * p.Hq)), dim3(64), 0, s, p.tpart, (long)p.B * b.ntq,
                     (T*)p.dtable);
  return hipGetLastError();
}
template <class T> hipError_t bwd_t(const BaParams& p, const BwdPlan& b, hipStream_t s) {
  return p.D <= 64 ? bwd<T, 64>(p, b, s) : p.D <= 96 ? bwd<T, 96>(p, b, s) : bwd<T, 128>(p, b, s);
}

size_t delta_bytes(const BaParams& p) { return up256((size_t)p.B * p.Hq * p.Tq * 4); }
size_t table_bytes(const BaParams& p, const BwdPlan& b) { return up256((size_t)p.nb * p.Hq * p.B * b.ntq * 4); }

}  // namespace

size_t ba_backward_ws(const BaParams& p, int dtype) {
  const BwdPlan b = plan_bwd(p, dtype);
  return delta_bytes(p) + table_bytes(p, b) + (b.gsplit > 1 ? (size_t)2 * b.gsplit * p.B * p.Tk * p.Hkv * p.D * 4 : 0) + 256;
}
hipError_t launch_ba_backward(BaParams p, int dtype, void* ws, hipStream_t s) {
  const BwdPlan b = plan_bwd(p, dtype);
  char* w = align256(ws);
  p.delta = (float*)w;
  p.tpart = (float*)(w + delta_bytes(p));
  p.gpart = (float*)(w + delta_bytes(p) + table_bytes(p, b));
  p.gsplit = b.gsplit;
  return dtype == 0 ? bwd_t<float>(p, b, s) : dtype == 1 ? bwd_t<bf16>(p, b, s) : bwd_t<f16>(p, b, s);
}

}  // namespace gt
