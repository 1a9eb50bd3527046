// Attention with a learned relative position bias by buckets, gfx950, forward:
//   o_i = sum_j softmax_j(q_i . k_j scale + table[bucket(j - pos_i)][h]) v_j ,  pos_i = q_start + i
// T = fp32 / bf16 / fp16 operands on the matrix cores; scores, softmax statistics and sums in fp32, P rounded to T for
// the second product (its sum l is of the unrounded terms).
//
// Many rows: bound by the matrix cores with the exponentials between their products, one wave's softmax beside another's
// products: 2 x 16 bf16 heads of 4096 causal rows, 64 channels (69 GFLOP) in 90 to 100 us, 0.7 PFLOP/s where a large
// library product reaches 1.17 (fp16 122); 16 heads of 2048 rows, 128 channels in 60 (there 2 to 44 registers spill). Rows
// off the 16-byte grid are read element by element: 2 x 16 causal bf16 heads of 2048 rows take 76 us with 104 channels,
// 376 with 100. Few rows: bound by memory, 32 sequences of up to 8192 keys, 4 x 128 channels (342 MB) in 75 us and 5 for
// the join, 4.5 TB/s where a copy reaches 4.9; in fp32, without copies in flight, up to 4096 keys (342 MB) in 130. Small
// calls: by latency, some 4 us from the launch to the first product (lengths, rows and table are dependent loads) and, in fp32,
// 2.6 us of products for each 32 x 32 block of 96 channels: one row over 190 keys 14 us.
#include <type_traits>

#include "battn_core.h"

namespace gt {
namespace {

// Reference m and sum l of a row's exponentials 2^(score - m), and its sums over v: `block` folds NB 32-key blocks in.
// SAFE: m is the running maximum, moved once a row's maximum has grown by 8 (in log2 units), and the sums follow it.
// Otherwise (kFixed) m is the maximum of the row's first keys and stays: neither maxima nor rescaling for any later block.
// Terms then grow up to 2^100 (69 nats), which `overflowed` sees in the sums; the workgroup's rows are then all done again
// the safe way: such a call takes about twice as long.
// Nothing is lost below: fp32 and bf16 hold terms down to 2^-126 of the first maximum.
// fp16 has no such range. It always takes the running maximum, and m lies kBelow = 7 below it: P of the largest term lies
// in [2^7, 2^15], so the 2^-25 by which rounding P can be off is 2^-32 of the largest term at most, below any sum's
// own rounding even where one key outweighs thousands (2 x 16 causal heads of 4096 rows, 64 channels: 122 us; a fixed
// reference took 112 and lost keys 13 nats below an early one).
template <class T, int DP> struct Softmax {
  typedef typename El<T>::frag frag;
  static constexpr bool kFixed = !std::is_same<T, f16>::value;
  static constexpr float kBelow = kFixed ? 0.f : 7.f;
  static constexpr int DB = DP / 32;
  f32x16 o[DB];
  float m, l;
  GT_DEV void clear() {
#pragma unroll
    for (int d = 0; d < DB; ++d) zero16(o[d]);
    m = -kInf;
    l = 0.f;
  }
  // (l well below the end of the range: the sums of the lane halves and of the streams, and 1 / l, are normal numbers)
  GT_DEV bool overflowed() const {
    bool bad = !(l < 0x1p100f);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) bad |= !(fabsf(o[d][j]) < kInf);
    return bad;
  }
  template <int NB> GT_DEV static float largest(const f32x16 (&s)[NB], const float (&off)[NB], float c) {
    float mt = -kInf;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float mx = fmaxf(fmaxf(s[n][0], s[n][1]), s[n][2]);
#pragma unroll
      for (int j = 3; j < 15; j += 2) mx = fmaxf(fmaxf(s[n][j], s[n][j + 1]), mx);
      mt = fmaxf(mt, __builtin_fmaf(fmaxf(mx, s[n][15]), c, off[n]));
    }
    return both_max(mt);
  }
  // s: scores / c (without off), -inf where unseen; col(n, tt, d): fragment of v for key group tt of block n
  template <bool SAFE, int NB, class Col> GT_DEV void block(const f32x16 (&s)[NB], const float (&off)[NB], float c, Col col) {
    static_assert(SAFE || kFixed, "range");
    if constexpr (SAFE) {
      const float mt = largest<NB>(s, off, c) - kBelow, mn = mt > m + 8.f || m == -kInf ? fmaxf(m, mt) : m;
      const float al = __builtin_amdgcn_exp2f(m - (mn == -kInf ? 0.f : mn));
      m = mn;
      l *= al;
      // (always: behind a branch the compiler copies the sums to other registers and back, which costs more)
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] *= al;
    } else if (__any(m == -kInf)) {
      float mt = largest<NB>(s, off, c);
      in_branch(mt);
      m = m == -kInf ? mt : m;
    }
    const float mu = m == -kInf ? 0.f : m;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      frag vf[2][DB];   // read ahead of the exponentials: an LDS read waited for before every product costs more than those
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int d = 0; d < DB; ++d) vf[tt][d] = col(n, tt, d);
      float pr[16], sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        pr[j] = expo<T>(s[n][j], c, off[n], mu);
        pr[j + 1] = expo<T>(s[n][j + 1], c, off[n], mu);
        sum0 += pr[j];
        sum1 += pr[j + 1];
      }
      l += sum0 + sum1;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const frag pf = El<T>::pack(pr + 8 * tt);
#pragma unroll
        for (int d = 0; d < DB; ++d) El<T>::mma(vf[tt][d], pf, o[d]);
      }
    }
  }
};

// A row's position in the sequence and what of the keys its wave looks at
struct Seen {
  int pos, pmin, pmax, nkey, wend;   // this lane's position, the wave's first and last; keys the lane sees, the wave visits
  float blo, bhi;                    // bias beyond the last border, log2 units
  const float* ext;                  // bias / scale by offset (this lane's head)
};
// scores / c of the 32 keys from kk on; a: their row fragments
template <class T, int KS>
GT_DEV void score_block(const BaParams& p, const Seen& w, int klen, int kk, int hh, const typename El<T>::frag (&a)[KS],
                        const typename El<T>::frag (&qf)[KS], f32x16& s, float& off) {
  const int dmax = kk + 31 - w.pmin, dmin = kk - w.pmax;   // offsets of the block
  if (one_bias(dmin, dmax, p.dsat, p.causal)) {
    off = dmin < 0 ? w.blo : w.bhi;
    s = mma0<T>(a[0], qf[0]);
  } else {
    const float* e = w.ext + (kk + 4 * hh - w.pos);
    off = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = e[acc_row(j, 0)];
    El<T>::mma(a[0], qf[0], s);
  }
#pragma unroll
  for (int ks = 1; ks < KS; ++ks) El<T>::mma(a[ks], qf[ks], s);
  if (kk + 31 >= klen || (p.causal && dmax > 0)) {
    int lim = w.nkey - kk - 4 * hh;
    in_branch(lim);
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = acc_row(j, 0) < lim ? s[j] : -kInf;
  }
}
template <class T> GT_DEV void far_bias(const BaParams& p, int h, Seen& w) {
  w.blo = table_at<T>(p, p.side - 1, h) * kLog2e;
  w.bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, h) * kLog2e;
}

// ================================================================ shared tiles
// K and V tiles copied straight to LDS, the next one's during this one's products; under a causal mask a workgroup takes a
// query tile and its mirror image, so that all are equally long.
template <class T, int DP, int WR, int WS>
__global__ __launch_bounds__(64 * WR * WS, sizeof(T) == 4 ? 1 : 2) void ba_fwd_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  typedef Shape<T, DP, WR, WS> SH;
  constexpr int KT = SH::KT, NB = SH::NB, KS = DP / 16, NT = 64 * WR * WS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wv % WR, ws = wv / WR;
  const int nbk = p.B * p.Hkv, bk = blockIdx.x % (unsigned)nbk, rest = blockIdx.x / (unsigned)nbk, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int h = hk * p.G + rest % p.G, rank = rest / p.G;
  float* ext0 = (float*)(smem + SH::BYTES);
  build_ext<T>(p, h, 1, h, ext0, tid, NT);
  const int qlen = clamp_len(p.qlen, b, p.Tq), pos0 = start_of(p, b), klen = keys_of(p, b, qlen, pos0);
  const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h;
  const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h;
  auto tile = [&](int t, int which) { return smem + ((SH::NBUF == 2 ? t & 1 : 0) * 2 + which) * SH::TILE; };   // LDS
  Stage<T, DP, KT, NT> ks, vs;
  ks.init(kb, p.ks.t, klen, p.D, p.vec, tid);
  vs.init(vb, p.vs.t, klen, p.D, p.vec, tid);
  auto load = [&](int t) {
    ks.load(tile(t, 0), t * KT);
    vs.load(tile(t, 1), t * KT);
  };
  Seen w;
  far_bias<T>(p, h, w);
  w.ext = ext0 + p.dsat + EXT;
  Softmax<T, DP> sm;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int lane = anew_v(tid & 63), r = lane & 31, hh = lane >> 5, D = anew_s(p.D);
    const int tl = pass ? rank : p.ntile - 1 - rank;
    if (pass && (!p.pair || 2 * rank >= p.ntile - 1)) break;
    const int i0 = tl * 32 * WR, wi0 = i0 + 32 * wr, qi = wi0 + r;
    const bool in = qi < qlen;
    int kend = klen;
    if (p.causal) kend = min(kend, pos0 + min(i0 + 32 * WR, qlen));
    if (i0 >= qlen) kend = 0;
    const int ntile = kend > 0 ? (kend + KT - 1) / KT : 0;
    if (pass) __syncthreads();   // the first pass's tiles are done with
    if (p.vec && D < DP && (WS > 1 || !pass))   // (a join has written over them)
      for (int i = 0; i < 2 * SH::NBUF; ++i) clear_pad<T, DP>(smem + i * SH::TILE, KT, D, tid, NT);
    frag qf[KS];   // (rows past the last valid one repeat it)
    if (ntile) load_rows<T, KS>(qf, (const T*)p.q + b * p.qs.b + h * p.qs.h + (long)min(qi, qlen - 1) * p.qs.t, hh, D, p.vec);
    w.pos = pos0 + qi;
    w.pmin = pos0 + wi0;
    w.pmax = w.pmin + 31;
    w.nkey = p.causal ? min(klen, w.pos + 1) : klen;
    w.wend = wi0 >= qlen ? 0 : p.causal ? min(kend, w.pmax + 1) : kend;
    // one tile; `buf`, a constant at both calls, is t & 1, so that LDS addresses do not depend on the loop
    auto step = [&](int t, auto buf, auto safe) {
      if constexpr (SH::NBUF == 2) {
        lds_ready();
        if (t + 1 < ntile) load(t + 1);
      } else {
        __syncthreads();
        load(t);
        lds_ready();
      }
      const int k0 = t * KT + 32 * ws;
      if (k0 >= w.wend) return;
      const char *sk = tile(buf, 0), *sv = tile(buf, 1);
      f32x16 s[NB];
      float off[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        frag a[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) a[ks] = TL::row(sk, 32 * (ws + WS * n) + r, 2 * ks + hh);
        score_block<T, KS>(p, w, klen, k0 + 32 * WS * n, hh, a, qf, s[n], off[n]);
      }
      sm.template block<decltype(safe)::value, NB>(s, off, p.c, [&](int n, int tt, int d) { return TL::col(sv, 32 * (ws + WS * n) + 16 * tt, d, lane); });
    };
    auto run = [&](auto safe) {
      if (ntile && SH::NBUF == 2) load(0);
      sm.clear();
      for (int t = 0; t < ntile; t += 2) {
        step(t, std::integral_constant<int, 0>(), safe);
        if (t + 1 < ntile) step(t + 1, std::integral_constant<int, 1>(), safe);
      }
    };
    if constexpr (Softmax<T, DP>::kFixed) {
      run(std::false_type());
      if (__syncthreads_or(sm.overflowed())) run(std::true_type());
    } else {
      run(std::true_type());
    }
    const float l = both_sum(sm.l);
    const long stat = ((long)b * p.Hq + h) * p.Tq + qi;
    T* ob = (T*)p.out + b * p.os.b + h * p.os.h;
    if constexpr (WS == 1) {
      if (qi >= p.Tq) continue;
      const bool live = in && l != 0.f;
      if (live) store_rows<T, DP>(ob + (long)qi * p.os.t, sm.o, 1.f / l, D, p.vec, hh);
      else zero_rows<T, DP>(ob + (long)qi * p.os.t, D, p.vec, hh);
      if (p.lse && hh == 0) p.lse[stat] = live ? sm.m + __builtin_amdgcn_logf(l) : kInf;
    } else {
      float* sml = ext0 + ext_len(p) + wr * WS * 64;   // [WR][WS][2][32]
      if (hh == 0) { sml[ws * 64 + r] = sm.m; sml[ws * 64 + 32 + r] = l; }
      __syncthreads();
      float M = -kInf, L = 0.f;
#pragma unroll
      for (int x = 0; x < WS; ++x) M = fmaxf(M, sml[x * 64 + r]);
      const float Mu = M == -kInf ? 0.f : M;
#pragma unroll
      for (int x = 0; x < WS; ++x) L += sml[x * 64 + 32 + r] * __builtin_amdgcn_exp2f(sml[x * 64 + r] - Mu);
      const bool live = in && L != 0.f;
      if (qi < p.Tq && p.lse && hh == 0 && ws == 0) p.lse[stat] = live ? M + __builtin_amdgcn_logf(L) : kInf;
      join<DP, WS>(smem, sm.o, live ? __builtin_amdgcn_exp2f(sm.m - Mu) / L : 0.f, wr, ws, lane, [&](int row, int d, float* x) {
        if (wi0 + row >= p.Tq) return;
        if (!(wi0 + row < qlen)) x[0] = x[1] = x[2] = x[3] = 0.f;
        store4_row(ob + (long)(wi0 + row) * p.os.t, d, x, D, p.vec);
      });
    }
  }
}

// ================================================================ spread rows
// 32 rows -- the queries and heads that share a key / value head, packed -- and four waves, each with every fourth 32-key
// block. No barrier in the loop. 16-bit: each wave has a slot of its own for K and one for V, refilled as soon as they are
// read: K's copies fly during the softmax and the second product, V's during the next first one, and the LDS left over
// holds a second workgroup. fp32: operands straight from memory (the transposed fragment's lanes are consecutive
// channels), all of a block's loads ahead of its products.
constexpr int WSP = 4;
template <class T, int DP> struct Spread {
  static constexpr bool RING = sizeof(T) == 2;
  static constexpr int SLOT = 32 * Tile<T, DP>::ROW, WAVE = 2 * SLOT, JOIN = WSP * DP * 33 * 4;
  static constexpr int BYTES = RING ? most(WSP * WAVE, JOIN) : JOIN;
  static constexpr int NI = SLOT / 1024;   // copies of one slot
};
template <int N> GT_DEV void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
GT_DEV void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <class T, int DP>
__global__ __launch_bounds__(64 * WSP, sizeof(T) == 2 || DP <= 96 ? 2 : 1) void ba_fwd_spread_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  typedef Spread<T, DP> SP;
  constexpr int KS = DP / 16, NT = 64 * WSP;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, ws = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  const int nbk = p.B * p.Hkv, ngb = (p.G + p.gp - 1) / p.gp;
  const unsigned units = (unsigned)nbk * ngb * p.ntile, blk = blockIdx.x % units;   // (the grid is below 2^31)
  const int split = blockIdx.x / units;
  const int bk = blk % (unsigned)nbk, rest = blk / (unsigned)nbk, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int g0 = rest % ngb * p.gp, i0 = (p.ntile - 1 - rest / ngb) * p.qpb, gp = p.gp;
  const int qlen = clamp_len(p.qlen, b, p.Tq), pos0 = start_of(p, b), klen = keys_of(p, b, qlen, pos0);
  float* ext0 = (float*)(smem + SP::BYTES);
  build_ext<T>(p, hk * p.G + g0, gp, hk * p.G + p.G - 1, ext0, tid, NT);
  const int gg = (unsigned)r % (unsigned)gp, qi = i0 + min((int)((unsigned)r / (unsigned)gp), p.qpb - 1), h = hk * p.G + min(g0 + gg, p.G - 1);
  const bool mine = r < gp * p.qpb && g0 + gg < p.G && qi < p.Tq, in = mine && qi < qlen;
  int kend = klen;
  if (p.causal) kend = min(kend, pos0 + min(i0 + p.qpb, qlen));
  if (i0 >= qlen) kend = 0;
  const int kbeg = split * p.split_keys;
  kend = min(kend, kbeg + p.split_keys);
  const int elen = ext_len(p);
  const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h;
  const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h;
  // this wave's blocks: keys kbeg + 32 (ws + 4 t)
  const int nblk = kend > kbeg + 32 * ws ? (kend - kbeg - 32 * ws + 32 * WSP - 1) / (32 * WSP) : 0;
  auto key0 = [&](int t) { return kbeg + 32 * (ws + WSP * t); };
  char* mem = smem + ws * SP::WAVE;   // K, V
  Stage<T, DP, 32, 64> ks, vs;
  ks.init(kb, p.ks.t, klen, p.D, p.vec, lane);
  vs.init(vb, p.vs.t, klen, p.D, p.vec, lane);
  if (SP::RING) {
    if (p.vec && p.D < DP)
      for (int i = 0; i < 2; ++i) clear_pad<T, DP>(mem + i * SP::SLOT, 32, p.D, lane, 64);
    if (nblk) {
      ks.load(mem, key0(0));
      vs.load(mem + SP::SLOT, key0(0));
    }
  }
  frag qf[KS];
  if (kend > kbeg) load_rows<T, KS>(qf, (const T*)p.q + b * p.qs.b + h * p.qs.h + (long)min(qi, qlen - 1) * p.qs.t, hh, p.D, p.vec);
  Seen w;
  far_bias<T>(p, h, w);
  w.ext = ext0 + gg * elen + p.dsat + EXT;
  w.pos = pos0 + qi;
  w.pmin = pos0 + i0;
  w.pmax = w.pmin + p.qpb - 1;
  w.nkey = p.causal ? min(klen, w.pos + 1) : klen;
  Softmax<T, DP> sm;
  sm.clear();
  lds_ready();   // the bias table (and the first blocks)
  for (int t = 0; t < nblk; ++t) {
    const int kk = key0(t);
    f32x16 s[1];
    float off[1];
    frag a[KS];
    if constexpr (SP::RING) {
      const bool more = t + 1 < nblk;
      wait_copies<SP::NI>();   // K of this block; its V may still be on its way (rows off the grid are there already)
#pragma unroll
      for (int x = 0; x < KS; ++x) a[x] = TL::row(mem, r, 2 * x + hh);
      score_block<T, KS>(p, w, klen, kk, hh, a, qf, s[0], off[0]);
      if (more) {
        reads_done();
        ks.load(mem, key0(t + 1));
        wait_copies<SP::NI>();   // V of this block, K of the next behind it
      } else {
        wait_copies<0>();
      }
      sm.template block<true, 1>(s, off, p.c, [&](int, int tt, int d) { return TL::col(mem + SP::SLOT, 16 * tt, d, lane); });
      if (more) {
        reads_done();
        vs.load(mem + SP::SLOT, key0(t + 1));
      }
    } else {
      frag v[2][DP / 32];
      load_rows<T, KS>(a, kb + (long)min(kk + r, klen - 1) * p.ks.t, hh, p.D, p.vec);
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const T* vr = vb + (long)min(kk + 16 * tt + acc_row(e, hh), klen - 1) * p.vs.t;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)   // (channels past the head size are not stored)
            El<T>::set(v[tt][d], e, vr[min(32 * d + r, p.D - 1)]);
        }
      score_block<T, KS>(p, w, klen, kk, hh, a, qf, s[0], off[0]);
      sm.template block<true, 1>(s, off, p.c, [&](int, int tt, int d) { return v[tt][d]; });
    }
  }
  const float l = both_sum(sm.l), m = sm.m;
  __syncthreads();     // the bias table is done with
  float* sml = ext0;   // [WSP][2][32]
  if (hh == 0) { sml[ws * 64 + r] = m; sml[ws * 64 + 32 + r] = l; }
  __syncthreads();
  float M = -kInf, L = 0.f;
#pragma unroll
  for (int x = 0; x < WSP; ++x) M = fmaxf(M, sml[x * 64 + r]);
  const float Mu = M == -kInf ? 0.f : M;
#pragma unroll
  for (int x = 0; x < WSP; ++x) L += sml[x * 64 + 32 + r] * __builtin_amdgcn_exp2f(sml[x * 64 + r] - Mu);
  const float f = __builtin_amdgcn_exp2f(m - Mu);
  if (p.nsplit > 1) {
    const long at = (long)blk * p.nsplit + split;
    if (tid < 32) {
      p.part_ml[at * 64 + r] = M;
      p.part_ml[at * 64 + 32 + r] = L;
    }
    if (kend > kbeg) join<DP, WSP>(smem, sm.o, f, 0, ws, lane, [&](int row, int d, const float* x) {
      float* q = p.part + (at * 32 + row) * p.D + d;
      if (p.D % 4 == 0) { if (d < p.D) *(f32x4*)q = (f32x4){x[0], x[1], x[2], x[3]}; }
      else
        for (int e = 0; e < 4; ++e) if (d + e < p.D) q[e] = x[e];
    });
    return;
  }
  const bool live = in && L != 0.f;
  if (mine && p.lse && tid < 32) p.lse[((long)b * p.Hq + h) * p.Tq + qi] = live ? M + __builtin_amdgcn_logf(L) : kInf;
  // the row's factor goes with the sum; dead rows come out as zeros whatever their lanes hold
  join<DP, WSP>(smem, sm.o, live ? f / L : 0.f, 0, ws, lane, [&](int row, int d, float* x) {
    const int g = g0 + row % gp, i = i0 + row / gp;
    if (row >= gp * p.qpb || g >= p.G || i >= p.Tq) return;
    if (!(i < qlen)) x[0] = x[1] = x[2] = x[3] = 0.f;
    store4_row((T*)p.out + b * p.os.b + (hk * p.G + g) * p.os.h + (long)i * p.os.t, d, x, p.D, p.vec);
  });
}

// Joins the splits of a row: a wave a row, two channels a lane. Latency (5 us), not bytes.
template <class T> __global__ __launch_bounds__(256) void ba_join_kernel(BaParams p) {
  const int lane = threadIdx.x & 63;
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6), blk = id >> 5;
  const int row = (int)(id & 31);
  const int nbk = p.B * p.Hkv, ngb = (p.G + p.gp - 1) / p.gp;
  if (blk >= (long)nbk * ngb * p.ntile) return;
  const int bk = (int)(blk % nbk), rest = (int)(blk / nbk), b = bk / p.Hkv, hk = bk % p.Hkv;
  const int g = rest % ngb * p.gp + row % p.gp, i = (p.ntile - 1 - rest / ngb) * p.qpb + row / p.gp;
  if (row >= p.gp * p.qpb || g >= p.G || i >= p.Tq) return;
  const float* ml = p.part_ml + blk * p.nsplit * 64 + row;
  float M = -kInf;
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, ml[(long)s * 64]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float Mu = M == -kInf ? 0.f : M;
  float L = 0.f, a0 = 0.f, a1 = 0.f;
  const float* part = p.part + (blk * p.nsplit * 32 + row) * p.D;
  const int d0 = min(lane, p.D - 1), d1 = min(lane + 64, p.D - 1);
  for (int s0 = 0; s0 < p.nsplit; s0 += 8) {   // eight splits' loads together
    float ms[8], ls[8], x0[8], x1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long s = min(s0 + e, p.nsplit - 1);
      ms[e] = ml[s * 64];
      ls[e] = ml[s * 64 + 32];
      x0[e] = part[s * 32 * p.D + d0];
      x1[e] = part[s * 32 * p.D + d1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // a split that saw no key has not written its sums
      if (s0 + e >= p.nsplit || ls[e] == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(ms[e] - Mu);
      L = __builtin_fmaf(ls[e], f, L);
      a0 = __builtin_fmaf(x0[e], f, a0);
      a1 = __builtin_fmaf(x1[e], f, a1);
    }
  }
  const bool live = i < clamp_len(p.qlen, b, p.Tq) && L != 0.f;
  const int h = hk * p.G + g;
  T* ob = (T*)p.out + b * p.os.b + h * p.os.h + (long)i * p.os.t;
  if (lane < p.D) ob[lane] = (T)(live ? a0 / L : 0.f);
  if (lane + 64 < p.D) ob[lane + 64] = (T)(live ? a1 / L : 0.f);
  if (p.lse && lane == 0) p.lse[((long)b * p.Hq + h) * p.Tq + i] = live ? M + __builtin_amdgcn_logf(L) : kInf;
}

// ---------------------------------------------------------------- launches
// Rows a workgroup, by how many workgroups that makes; us for spread / 64 / 128 rows at (heads x batch, T, head size):
//   128 rows from two workgroups a CU on (fp32, whose products outlast the copies: one): bf16 (128, 512, 64) 30 / 25 / 19,
//   below (64, 512, 128) 30 / 22 / 23, causal (64, 512, 64) 16 / 16 / 19; fp32 (64, 512, 128) 134 / 121 / 100;
//   64 rows from 192 workgroups on: bf16 (64, 512, 64) 18 / 15, fp32 (64, 190, 64) 20 / 17; below: fp32 (32, 190, 64)
//   12 / 16, bf16 causal (64, 190, 128) 12 / 18;
//   else spread rows, blocks of 32. Where these are fewer than the CUs and the cache is longer than 1024 keys, key ranges of
//   256 keys at least have workgroups of their own, one a CU in all, and are joined afterwards: one query of 16 bf16 heads
//   over 8192 keys 69 us alone, 16 split; 2 fp32 heads over 700 keys 12 alone, 13 split; over 2000 21 and 13. One range a
//   CU, not four: 32 sequences of 8192 keys 108 us against 117, one of 65536 55 against 69.
enum Form { SHARED4, SHARED2, SPREAD };
struct FwdPlan { Form form; long units; };
FwdPlan plan_fwd(BaParams& p, int dtype) {
  p.nsplit = 1;
  const long heads = (long)p.B * p.Hq;
  auto groups = [&](int rows) {
    p.ntile = (p.Tq + rows - 1) / rows;
    p.pair = p.causal && p.ntile > 1;
    return heads * (p.pair ? (p.ntile + 1) / 2 : p.ntile);
  };
  if (p.Tq > 32) {
    if (fills128(dtype, p.Tq) && groups(128) >= (dtype == 0 ? 256 : 512)) return {SHARED4, groups(128)};
    if (groups(64) >= 192) return {SHARED2, groups(64)};
  }
  FwdPlan f{SPREAD, 0};
  p.pair = 0;
  p.gp = p.G < 32 ? p.G : 32;
  while (p.gp > 1 && p.gp * host_ext_bytes(p) > 24 * 1024) p.gp = (p.gp + 1) / 2;
  p.qpb = 32 / p.gp;
  p.ntile = (p.Tq + p.qpb - 1) / p.qpb;
  f.units = (long)p.B * p.Hkv * ((p.G + p.gp - 1) / p.gp) * p.ntile;
  constexpr int KT = 32 * WSP;
  p.split_keys = (p.Tk + KT - 1) / KT * KT;
  if (f.units && f.units < 256 && p.Tk > 8 * KT) {
    const long n = (256 + f.units - 1) / f.units;
    long keys = ((p.Tk + n - 1) / n + KT - 1) / KT * KT;
    if (keys < 2 * KT) keys = 2 * KT;
    p.split_keys = (int)keys;
    p.nsplit = (int)((p.Tk + keys - 1) / keys);
  }
  return f;
}

template <class T, int DP, int WR, int WS> hipError_t shared(const BaParams& p, const FwdPlan& f, hipStream_t s) {
  const int smem = Shape<T, DP, WR, WS>::BYTES + host_ext_bytes(p) + (WS > 1 ? WR * WS * 64 * 4 : 0);
  return launch(ba_fwd_kernel<T, DP, WR, WS>, f.units, 64 * WR * WS, smem, p, s);
}
template <class T, int DP> hipError_t fwd(const BaParams& p, const FwdPlan& f, hipStream_t s) {
  if (f.form == SHARED4) return shared<T, DP, 4, 1>(p, f, s);
  if (f.form == SHARED2) return shared<T, DP, 2, 2>(p, f, s);
  constexpr int base = Spread<T, DP>::BYTES;
  static_assert(base + 24 * 1024 <= kLds, "LDS");
  int ext = p.gp * host_ext_bytes(p);
  if (ext < WSP * 64 * 4) ext = WSP * 64 * 4;
  hipError_t e = launch(ba_fwd_spread_kernel<T, DP>, f.units * p.nsplit, 64 * WSP, base + ext, p, s);
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

size_t ba_forward_ws(const BaParams& p0, int dtype) {
  BaParams p = p0;
  const FwdPlan f = plan_fwd(p, dtype);
  if (p.nsplit == 1) return 0;
  return up256((size_t)f.units * p.nsplit * 32 * p.D * 4) + (size_t)f.units * p.nsplit * 64 * 4 + 256;
}
hipError_t launch_ba_forward(BaParams p, int dtype, void* ws, hipStream_t s) {
  const FwdPlan f = plan_fwd(p, dtype);
  if (p.nsplit > 1) {
    char* w = align256(ws);
    p.part = (float*)w;
    p.part_ml = (float*)(w + up256((size_t)f.units * p.nsplit * 32 * p.D * 4));
  }
  return dtype == 0 ? fwd_t<float>(p, f, s) : dtype == 1 ? fwd_t<bf16>(p, f, s) : fwd_t<f16>(p, f, s);
}

}  // namespace gt
