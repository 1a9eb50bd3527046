// Attention with a learned relative position bias by buckets, gfx950:
//   o_i = sum_j softmax_j(q_i . k_j scale + table[bucket(j - pos_i)][h]) v_j ,  pos_i = q_start + i
// and its gradients. T = fp32 / bf16 / fp16 operands on the matrix cores, every sum, softmax statistic and gradient
// accumulator in fp32.
//
// All kernels hold one 32-row block a wave "stationary" (its rows are the lanes lane & 31 of every MFMA's B operand, in
// registers) and stream 32-row blocks of the other side through LDS (A operand):
//   forward, dQ   stationary queries, streamed keys:    S^T = K Q^T,  O^T += V^T P^T,  dQ^T += K^T dS^T
//   dK dV         stationary keys, streamed queries:    S = Q K^T,    dV^T += dO^T P,  dK^T += Q^T dS
// so that the P / dS block, which the first product leaves in the accumulator layout (column = lane & 31, rows
// acc_row(j, h)), is the second product's B operand as it stands: register j = 8 t + e holds key acc_row(8 t + e, h) of
// the 16-key step t, and the transposed A operand reads the same order (two 4-key groups a lane half).
//
// The bias enters as the C operand of the first product (bias / scale, from an LDS table over the offsets), or, where
// a 32 x 32 block lies wholly beyond the last border, as one constant: the exponent is a single FMA per score.
#include "battn.h"

#include "common.h"

namespace gt {
namespace {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kInf = __builtin_inff();

template <class T> struct El;
template <> struct El<float> {
  struct frag { f32x4 lo, hi; };
  static constexpr bool wide = true;
  GT_DEV static frag zero() { return frag{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}; }
  GT_DEV static float get(const frag& f, int e) { return e < 4 ? f.lo[e] : f.hi[e - 4]; }
  GT_DEV static void set(frag& f, int e, float v) { if (e < 4) f.lo[e] = v; else f.hi[e - 4] = v; }
  GT_DEV static frag load16(const float* p) { return frag{*(const f32x4*)p, *(const f32x4*)(p + 4)}; }
  GT_DEV static frag pack(const float* x) { return frag{{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}}; }
  GT_DEV static void store4(float* p, const float* x) { *(f32x4*)p = (f32x4){x[0], x[1], x[2], x[3]}; }
  GT_DEV static void mma(const frag& a, const frag& b, f32x16& c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[s], b.lo[s], c, 0, 0, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[s], b.hi[s], c, 0, 0, 0);
  }
};
template <> struct El<bf16> {
  typedef bf16x8 frag;
  static constexpr bool wide = false;
  GT_DEV static frag zero() { return __builtin_bit_cast(frag, make_uint4(0, 0, 0, 0)); }
  GT_DEV static float get(const frag& f, int e) { return (float)f[e]; }
  GT_DEV static void set(frag& f, int e, bf16 v) { f[e] = v; }
  GT_DEV static frag load16(const bf16* p) { return *(const frag*)p; }
  GT_DEV static frag pack(const float* x) { return __builtin_bit_cast(frag, f_to_item(x, bf16())); }
  GT_DEV static void store4(bf16* p, const float* x) { *(uint2*)p = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])); }
  GT_DEV static void mma(const frag& a, const frag& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct El<f16> {
  typedef f16x8 frag;
  static constexpr bool wide = false;
  GT_DEV static frag zero() { return __builtin_bit_cast(frag, make_uint4(0, 0, 0, 0)); }
  GT_DEV static float get(const frag& f, int e) { return (float)f[e]; }
  GT_DEV static void set(frag& f, int e, f16 v) { f[e] = v; }
  GT_DEV static frag load16(const f16* p) { return *(const frag*)p; }
  GT_DEV static frag pack(const float* x) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector((f32x8){x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}, f16x8);
  }
  GT_DEV static void store4(f16* p, const float* x) {
    *(f16x4*)p = __builtin_convertvector((f32x4){x[0], x[1], x[2], x[3]}, f16x4);
  }
  GT_DEV static void mma(const frag& a, const frag& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

GT_DEV void zero16(f32x16& x) {
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = 0.f;
}
// the other lane half's value
GT_DEV float other_half(float x) { return __shfl_xor(x, 32); }

// eight channels d .. d + 7 of one row (zero past D); `vec` as in BaParams
template <class T> GT_DEV typename El<T>::frag load_row8(const T* p, int d, int D, int vec) {
  if (vec) return d < D ? El<T>::load16(p + d) : El<T>::zero();
  typename El<T>::frag f = El<T>::zero();
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < D) El<T>::set(f, e, p[d + e]);
  return f;
}

// LDS image of a block of rows, DP channels each, as 16-byte chunks whose index is XORed with a function of the row:
// reads of one chunk of 16 consecutive rows (row fragments) and of 64 bytes of 4 consecutive rows (transposed
// fragments) both fall on 64 different banks.
template <class T, int DP> struct Tile {
  typedef typename El<T>::frag frag;
  static constexpr int ES = sizeof(T), NC = DP <= 64 ? 4 * ES : 8 * ES, ROW = NC * 16;   // chunks, bytes of a row
  GT_DEV static int swz(int row) {
    if constexpr (El<T>::wide) return ((row >> 2) & 1) * 8 + ((row >> 3) & 1) * 4 + (row & 3);
    else if constexpr (DP <= 64) return ((row >> 1) & 1) * 4 + ((row >> 2) & 3);
    else return (row & 3) * 4 + ((row >> 2) & 3);
  }
  GT_DEV static char* at(char* s, int row, int chunk) { return s + row * ROW + ((chunk ^ swz(row)) << 4); }
  // chunk8: group of eight channels
  GT_DEV static void put(char* s, int row, int chunk8, const frag& f) {
    if constexpr (El<T>::wide) {
      *(f32x4*)at(s, row, 2 * chunk8) = f.lo;
      *(f32x4*)at(s, row, 2 * chunk8 + 1) = f.hi;
    } else {
      *(frag*)at(s, row, chunk8) = f;
    }
  }
  GT_DEV static frag row(const char* s, int row, int chunk8) {
    if constexpr (El<T>::wide)
      return frag{*(const f32x4*)at((char*)s, row, 2 * chunk8), *(const f32x4*)at((char*)s, row, 2 * chunk8 + 1)};
    else
      return *(const frag*)at((char*)s, row, chunk8);
  }
  // channel 32 db + (lane & 31) of the rows r16 + acc_row(e, lane >> 5), e = 0 .. 7
  GT_DEV static frag col(const char* s, int r16, int db, int lane) {
    const int h = lane >> 5;
    if constexpr (El<T>::wide) {
      const int d = 32 * db + (lane & 31);
      frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.lo[e] = *(const float*)(at((char*)s, r16 + 4 * h + e, d >> 2) + (d & 3) * 4);
        f.hi[e] = *(const float*)(at((char*)s, r16 + 8 + 4 * h + e, d >> 2) + (d & 3) * 4);
      }
      return f;
    } else {
      // transposing read: within 16 lanes, lane i names row i >> 2, channels 4 (i & 3) .. + 3, and gets channel i of
      // the four rows
      const int i = lane & 15, rr = r16 + 4 * h + (i >> 2), d = 32 * db + (lane & 16) + 4 * (i & 3);
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at((char*)s, rr, d >> 3) + (d & 4) * 2));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at((char*)s, rr + 8, d >> 3) + (d & 4) * 2));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// ---------------------------------------------------------------- buckets
GT_DEV int bucket_of(const BaParams& p, int delta) {   // delta = key position - query position
  const int dist = p.causal ? (delta < 0 ? -delta : 0) : (delta < 0 ? -delta : delta);
  int b = dist < p.exact ? dist : p.exact;
  for (int k = 0; k < p.nborder; ++k) b += dist >= p.border[k];
  return b + ((!p.causal && delta > 0) ? p.side : 0);
}
// LDS table over the offsets -dsat - EXT .. dsat + EXT: a 32 x 32 block with an offset inside (-dsat, dsat) has all of
// its 63 offsets in it
constexpr int EXT = 64;
GT_DEV int ext_len(const BaParams& p) { return 2 * (p.dsat + EXT) + 1; }
template <class T> GT_DEV float table_at(const BaParams& p, int bucket, int h) {
  return (float)((const T*)p.table)[(long)bucket * p.Hq + h] * p.inv_scale;
}
template <class T> GT_DEV void build_ext(const BaParams& p, int h, float* ext, int tid, int nthreads) {
  for (int i = tid; i < ext_len(p); i += nthreads) ext[i] = table_at<T>(p, bucket_of(p, i - p.dsat - EXT), h);
}

GT_DEV int clamp_len(const int64_t* len, int b, int most) {
  if (!len) return most;
  const int64_t n = len[b];
  return n < 0 ? 0 : n > most ? most : (int)n;
}
GT_DEV int start_of(const BaParams& p, int b) {   // far beyond any offset that differs from the last bucket's
  const int64_t s = p.qstart ? p.qstart[b] : 0;
  return s < -(1 << 29) ? -(1 << 29) : s > (1 << 29) ? (1 << 29) : (int)s;
}

// work item -> (batch, query head, tile): the heads that share a key / value head run next to each other on the same
// XCD (workgroups go round the 8 XCDs in turn), the last query tiles, the longest under a causal mask, first
struct Item { int b, h, hk, tile; };
GT_DEV Item item_of(const BaParams& p, int id, int ntile) {
  const int nbk = p.B * p.Hkv, bk = id % nbk, rest = id / nbk, g = rest % p.G;
  Item it;
  it.b = bk / p.Hkv;
  it.hk = bk % p.Hkv;
  it.h = it.hk * p.G + g;
  it.tile = ntile - 1 - rest / p.G;
  return it;
}

// ---------------------------------------------------------------- streamed rows: global -> registers -> LDS
template <class T, int DP, int ROWS, int NT> struct Stream {
  static constexpr int C8 = DP / 8, N = (ROWS * C8 + NT - 1) / NT;
  typename El<T>::frag f[N];
  GT_DEV void fetch(const T* base, long st, int row0, int nrow, int D, int vec, int tid) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = tid + n * NT, row = i / C8, c = i % C8;
      f[n] = (i < ROWS * C8 && row0 + row < nrow) ? load_row8(base + (long)(row0 + row) * st, 8 * c, D, vec) : El<T>::zero();
    }
  }
  GT_DEV void put(char* s, int tid) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = tid + n * NT;
      if (i < ROWS * C8) Tile<T, DP>::put(s, i / C8, i % C8, f[n]);
    }
  }
};

// rows of a 32 x 32 x 32 db accumulator set (column = row of the output, registers = channels) to memory
template <class T, int DP> GT_DEV void store_rows(T* row, const f32x16 (&acc)[DP / 32], float mul, int D, int vec, int hh) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int jg = 0; jg < 4; ++jg) {
      const int d = 32 * db + 8 * jg + 4 * hh;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[db][4 * jg + e] * mul;
      if (vec) {
        if (d < D) El<T>::store4(row + d, x);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) row[d + e] = (T)x[e];
      }
    }
}
template <class T, int DP> GT_DEV void zero_rows(T* row, int D, int vec, int hh) {
  f32x16 z[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) zero16(z[db]);
  store_rows<T, DP>(row, z, 0.f, D, vec, hh);
}

// p = 2^(score - m) in the type's form. fp32 subtracts the rounded score, so that a row's largest term, and the only
// term of a row with one visible key, is exactly 1 (its output is then that value, its score gradient exactly 0); the
// 16-bit types round P and o, and take one FMA instead.
template <class T> GT_DEV float expo(float acc, float c, float off, float m) {
  if constexpr (El<T>::wide) return __builtin_amdgcn_exp2f(__builtin_fmaf(acc, c, off) - m);
  else return __builtin_amdgcn_exp2f(__builtin_fmaf(acc, c, off - m));
}

// ================================================================ forward
// Workgroup: NW waves x 32 queries of one head; key / value tiles of KT rows in LDS, the next tile's rows in registers.
template <class T> constexpr int kTile = El<T>::wide ? 32 : 64;

template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void ba_fwd_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  constexpr int KT = kTile<T>, KS = DP / 16, DB = DP / 32, NT = 64 * NW;
  extern __shared__ char smem[];
  char *sk = smem, *sv = smem + KT * TL::ROW;
  float* ext = (float*)(smem + 2 * KT * TL::ROW) + p.dsat + EXT;   // ext[offset]
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = lane & 31, hh = lane >> 5;
  const int ntile = (p.Tq + 32 * NW - 1) / (32 * NW);
  const Item it = item_of(p, blockIdx.x, ntile);
  const int qlen = clamp_len(p.qlen, it.b, p.Tq), klen = clamp_len(p.len, it.b, p.Tk), pos0 = start_of(p, it.b);
  const int q0 = it.tile * 32 * NW, qi = q0 + 32 * wv + r;
  int kend = klen;
  if (p.causal) kend = min(kend, pos0 + min(q0 + 32 * NW, qlen));
  if (q0 >= qlen) kend = 0;
  const T* kb = (const T*)p.k + it.b * p.ks.b + it.hk * p.ks.h;
  const T* vb = (const T*)p.v + it.b * p.vs.b + it.hk * p.vs.h;
  const T* qb = (const T*)p.q + it.b * p.qs.b + it.h * p.qs.h + (long)qi * p.qs.t;
  frag qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = qi < qlen ? load_row8(qb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
  if (kend > 0) build_ext<T>(p, it.h, ext - p.dsat - EXT, tid, NT);
  const float blo = table_at<T>(p, p.side - 1, it.h) * p.c, bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, it.h) * p.c;
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) zero16(o[d]);
  float m = -kInf, l = 0.f;
  const int wq0 = q0 + 32 * wv, pmin = pos0 + wq0, pmax = pmin + 31, pos = pos0 + qi;
  const int wend = wq0 >= qlen ? 0 : p.causal ? min(kend, pmax + 1) : kend;   // keys this wave looks at
  Stream<T, DP, KT, NT> ki, vi;
  if (kend > 0) {
    ki.fetch(kb, p.ks.t, 0, klen, p.D, p.vec, tid);
    vi.fetch(vb, p.vs.t, 0, klen, p.D, p.vec, tid);
  }
  for (int k0 = 0; k0 < kend; k0 += KT) {
    __syncthreads();
    ki.put(sk, tid);
    vi.put(sv, tid);
    if (k0 + KT < kend) {
      ki.fetch(kb, p.ks.t, k0 + KT, klen, p.D, p.vec, tid);
      vi.fetch(vb, p.vs.t, k0 + KT, klen, p.D, p.vec, tid);
    }
    __syncthreads();
#pragma unroll
    for (int j2 = 0; j2 < KT / 32; ++j2) {
      const int kk = k0 + 32 * j2;
      if (kk >= wend) break;
      const int dmax = kk + 31 - pmin, dmin = kk - pmax;   // offsets of the block
      f32x16 s;
      float off = 0.f;
      if (dmax <= -p.dsat) { off = blo; zero16(s); }
      else if (!p.causal && dmin >= p.dsat) { off = bhi; zero16(s); }
      else {
        const float* e = ext + (kk + 4 * hh - pos);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = e[acc_row(j, 0)];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) El<T>::mma(TL::row(sk, 32 * j2 + r, 2 * ks + hh), qf[ks], s);
      if (kk + 31 >= klen || (p.causal && dmax > 0)) {
        const int lim = (p.causal ? min(klen, pos + 1) : klen) - kk - 4 * hh;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = acc_row(j, 0) < lim ? s[j] : -kInf;
      }
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
      mx = fmaxf(mx, other_half(mx));
      const float mn = fmaxf(m, __builtin_fmaf(mx, p.c, off));
      const float mu = mn == -kInf ? 0.f : mn;
      const float al = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      float pr[16], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        pr[j] = expo<T>(s[j], p.c, off, mu);
        sum += pr[j];
      }
      l = l * al + sum;
      if (__any(al != 1.f)) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[d][j] *= al;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag pf = El<T>::pack(pr + 8 * t);
#pragma unroll
        for (int d = 0; d < DB; ++d) El<T>::mma(TL::col(sv, 32 * j2 + 16 * t, d, lane), pf, o[d]);
      }
    }
  }
  if (qi >= p.Tq) return;
  l += other_half(l);
  T* ob = (T*)p.out + it.b * p.os.b + it.h * p.os.h + (long)qi * p.os.t;
  const bool live = qi < qlen && l != 0.f;
  if (live) store_rows<T, DP>(ob, o, 1.f / l, p.D, p.vec, hh);
  else zero_rows<T, DP>(ob, p.D, p.vec, hh);
  if (p.lse && hh == 0) p.lse[((long)it.b * p.Hq + it.h) * p.Tq + qi] = live ? m + __builtin_amdgcn_logf(l) : kInf;
}

// ================================================================ backward: dQ, delta, table partials
// delta_i = sum_j P_ij dP_ij = o_i . do_i. The product with the rounded o, formed from rounded P, is off by about
// u |o| |do| (u = half a step of the type), which weighs when few keys share a row: dS = P (dP - delta) is then a small
// difference. Waves whose keys all lie in the first tile therefore sum P dP itself in fp32 (both are at hand; bf16, 14
// keys: dq's error 2.5e-3 where the product's gave 5.4e-3). The others take the product, from the matrix cores in the
// channel order of dP: so does a row with one visible key (o = v), whose delta then equals dP bit for bit and whose dS is
// exactly zero.
template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void ba_dq_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  constexpr int KT = kTile<T>, KS = DP / 16, DB = DP / 32, NT = 64 * NW;
  extern __shared__ char smem[];
  char *sk = smem, *sv = smem + KT * TL::ROW;
  const int elen = ext_len(p);
  float* ext0 = (float*)(smem + 2 * KT * TL::ROW);
  float* ext = ext0 + p.dsat + EXT;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = lane & 31, hh = lane >> 5;
  float* tacc = ext0 + (1 + wv) * elen + p.dsat + EXT;   // this wave's sums of dS by offset
  const int ntile = (p.Tq + 32 * NW - 1) / (32 * NW);
  const Item it = item_of(p, blockIdx.x, ntile);
  const int qlen = clamp_len(p.qlen, it.b, p.Tq), klen = clamp_len(p.len, it.b, p.Tk), pos0 = start_of(p, it.b);
  const int q0 = it.tile * 32 * NW, qi = q0 + 32 * wv + r;
  int kend = klen;
  if (p.causal) kend = min(kend, pos0 + min(q0 + 32 * NW, qlen));
  if (q0 >= qlen) kend = 0;
  const T* kb = (const T*)p.k + it.b * p.ks.b + it.hk * p.ks.h;
  const T* vb = (const T*)p.v + it.b * p.vs.b + it.hk * p.vs.h;
  const T* qb = (const T*)p.q + it.b * p.qs.b + it.h * p.qs.h + (long)qi * p.qs.t;
  const T* ob = (const T*)p.o + it.b * p.os.b + it.h * p.os.h + (long)qi * p.os.t;
  const T* gb = (const T*)p.dout + it.b * p.dos.b + it.h * p.dos.h + (long)qi * p.dos.t;
  const long srow = ((long)it.b * p.Hq + it.h) * p.Tq + qi;
  const bool in = qi < qlen;
  frag qf[KS], gf[KS];
  f32x16 dg;
  zero16(dg);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = in ? load_row8(qb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
    gf[s] = in ? load_row8(gb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
    const frag of = in ? load_row8(ob, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
    El<T>::mma(of, gf[s], dg);
  }
  const float lse = in ? p.lse[srow] : kInf;
  // the diagonal: row r of column r, held by lane half (r >> 2) & 1 in register (r & 3) + 4 (r >> 3)
  float delta = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) delta = acc_row(j, hh) == r ? dg[j] : delta;
  const float od = other_half(delta);
  delta = ((r >> 2) & 1) == hh ? delta : od;
  for (int i = tid; i < NW * elen; i += NT) ext0[elen + i] = 0.f;
  if (kend > 0) build_ext<T>(p, it.h, ext0, tid, NT);
  const float blo = table_at<T>(p, p.side - 1, it.h) * p.c, bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, it.h) * p.c;
  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) zero16(dq[d]);
  float slo = 0.f, shi = 0.f;   // dS beyond the last border
  const int wq0 = q0 + 32 * wv, pmin = pos0 + wq0, pmax = pmin + 31, pos = pos0 + qi;
  const int wend = wq0 >= qlen ? 0 : p.causal ? min(kend, pmax + 1) : kend;
  const int nkey = p.causal ? min(klen, pos + 1) : klen;   // keys this lane's row sees
  // scores (without `off`) and dP of the 32 keys from kk on
  auto scores = [&](int kk, int j2, f32x16& s, f32x16& dp, float& off) {
    const int dmax = kk + 31 - pmin, dmin = kk - pmax;
    zero16(dp);
    off = 0.f;
    if (dmax <= -p.dsat) { off = blo; zero16(s); }
    else if (!p.causal && dmin >= p.dsat) { off = bhi; zero16(s); }
    else {
      const float* e = ext + (kk + 4 * hh - pos);
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = e[acc_row(j, 0)];
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      El<T>::mma(TL::row(sk, 32 * j2 + r, 2 * ks + hh), qf[ks], s);
      El<T>::mma(TL::row(sv, 32 * j2 + r, 2 * ks + hh), gf[ks], dp);
    }
  };
  Stream<T, DP, KT, NT> ki, vi;
  if (kend > 0) {
    ki.fetch(kb, p.ks.t, 0, klen, p.D, p.vec, tid);
    vi.fetch(vb, p.vs.t, 0, klen, p.D, p.vec, tid);
  }
  for (int k0 = 0; k0 < kend; k0 += KT) {
    __syncthreads();
    ki.put(sk, tid);
    vi.put(sv, tid);
    if (k0 + KT < kend) {
      ki.fetch(kb, p.ks.t, k0 + KT, klen, p.D, p.vec, tid);
      vi.fetch(vb, p.vs.t, k0 + KT, klen, p.D, p.vec, tid);
    }
    __syncthreads();
    if (k0 == 0 && wend <= KT) {
      float sum = 0.f;
#pragma unroll
      for (int j2 = 0; j2 < KT / 32; ++j2) {
        if (32 * j2 >= wend) break;
        f32x16 s, dp;
        float off;
        scores(32 * j2, j2, s, dp, off);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sum += 32 * j2 + acc_row(j, hh) < nkey ? expo<T>(s[j], p.c, off, lse) * dp[j] : 0.f;
      }
      sum += other_half(sum);
      if (nkey > 1) delta = sum;
    }
#pragma unroll
    for (int j2 = 0; j2 < KT / 32; ++j2) {
      const int kk = k0 + 32 * j2;
      if (kk >= wend) break;
      const int dmax = kk + 31 - pmin, dmin = kk - pmax;
      const bool lo = dmax <= -p.dsat, hi = !p.causal && dmin >= p.dsat;
      f32x16 s, dp;
      float off;
      scores(kk, j2, s, dp, off);
      const int lim = nkey - kk - 4 * hh;
      const bool edge = kk + 31 >= klen || (p.causal && dmax > 0);
      float ds[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        ds[j] = expo<T>(s[j], p.c, off, lse) * (dp[j] - delta);
        if (edge) ds[j] = acc_row(j, 0) < lim ? ds[j] : 0.f;
      }
      if (lse == kInf) {   // no visible key (or no such row): nothing flows, whatever the operands hold
#pragma unroll
        for (int j = 0; j < 16; ++j) ds[j] = 0.f;
      }
      if (lo || hi) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) a += ds[j];
        slo += lo ? a : 0.f;
        shi += lo ? 0.f : a;
      } else {
        // one lane half at a time: the 32 lanes of a register then hold 32 different offsets, so every sum has one order
        float* e = tacc + (kk + 4 * hh - pos);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (hh == 0) __hip_atomic_fetch_add(e + acc_row(j, 0), ds[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (hh == 1) __hip_atomic_fetch_add(e + acc_row(j, 0), ds[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag df = El<T>::pack(ds + 8 * t);
#pragma unroll
        for (int d = 0; d < DB; ++d) El<T>::mma(TL::col(sk, 32 * j2 + 16 * t, d, lane), df, dq[d]);
      }
    }
  }
  if (qi < p.Tq) {
    if (hh == 0) p.delta[srow] = in ? delta : 0.f;
    T* qo = (T*)p.dq + it.b * p.dqs.b + it.h * p.dqs.h + (long)qi * p.dqs.t;
    if (in) store_rows<T, DP>(qo, dq, p.scale, p.D, p.vec, hh);
    else zero_rows<T, DP>(qo, p.D, p.vec, hh);
  }
  // table partials of this tile: a wave a bucket, its lanes over the bucket's offsets, then across the lanes in one order
  float* sat = (float*)smem;   // [NW][2] (the tiles are done with)
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) {
    slo += __shfl_xor(slo, x);
    shi += __shfl_xor(shi, x);
  }
  __syncthreads();
  if (lane == 0) { sat[2 * wv] = slo; sat[2 * wv + 1] = shi; }
  __syncthreads();
  const long npart = (long)p.B * ntile;
  for (int b = wv; b < p.nb; b += NW) {
    const int side = b >= p.side, bb = side ? b - p.side : b;
    int d0, d1;   // distances of the bucket
    if (bb < p.exact) {
      d0 = bb;
      d1 = bb + 1;
    } else {
      d0 = bb == p.exact ? p.exact : p.border[bb - p.exact - 1];
      d1 = bb == p.side - 1 ? p.dsat + EXT + 1 : p.border[bb - p.exact];
    }
    if (side && d0 == 0) d0 = 1;   // offset 0 belongs to the first half
    float a = 0.f;
    for (int d = d0 + lane; d < d1; d += 64)
#pragma unroll
      for (int w = 0; w < NW; ++w) a += ext0[(1 + w) * elen + p.dsat + EXT + (side ? d : -d)];
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) a += __shfl_xor(a, x);
    if (bb == p.side - 1)
      for (int w = 0; w < NW; ++w) a += sat[2 * w + side];
    if (lane == 0) p.tpart[((long)b * p.Hq + it.h) * npart + (long)it.b * ntile + it.tile] = a;
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

// ================================================================ backward: dK, dV
// Workgroup: NW waves x 32 keys of one key / value head, over the query tiles of all heads that share it.
template <class T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void ba_dkv_kernel(BaParams p) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  constexpr int QT = kTile<T>, KS = DP / 16, DB = DP / 32, NT = 64 * NW;
  extern __shared__ char smem[];
  char *sq = smem, *sg = smem + QT * TL::ROW;
  float* srow = (float*)(smem + 2 * QT * TL::ROW);   // [QT] lse, [QT] delta
  float* ext0 = srow + 2 * QT;
  float* ext = ext0 + p.dsat + EXT;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = lane & 31, hh = lane >> 5;
  const int nbk = p.B * p.Hkv, bk = blockIdx.x % nbk, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int k0 = (blockIdx.x / nbk) * 32 * NW, ki = k0 + 32 * wv + r;
  const int qlen = clamp_len(p.qlen, b, p.Tq), klen = clamp_len(p.len, b, p.Tk), pos0 = start_of(p, b);
  // first query that sees key k0 (causal: position >= k0)
  int qbeg = p.causal ? max(0, k0 - pos0) : 0;
  qbeg = qbeg / QT * QT;
  const int qend = k0 < klen ? qlen : 0;
  const T* kb = (const T*)p.k + b * p.ks.b + hk * p.ks.h + (long)ki * p.ks.t;
  const T* vb = (const T*)p.v + b * p.vs.b + hk * p.vs.h + (long)ki * p.vs.t;
  const bool in = ki < klen;
  frag kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = in ? load_row8(kb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
    vf[s] = in ? load_row8(vb, 16 * s + 8 * hh, p.D, p.vec) : El<T>::zero();
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) { zero16(dk[d]); zero16(dv[d]); }
  const int wk0 = k0 + 32 * wv;
  for (int g = 0; g < p.G; ++g) {
    const int h = hk * p.G + g;
    const T* qb = (const T*)p.q + b * p.qs.b + h * p.qs.h;
    const T* gb = (const T*)p.dout + b * p.dos.b + h * p.dos.h;
    const float* lse = p.lse + ((long)b * p.Hq + h) * p.Tq;
    const float* del = p.delta + ((long)b * p.Hq + h) * p.Tq;
    __syncthreads();
    if (qbeg < qend) build_ext<T>(p, h, ext0, tid, NT);
    const float blo = table_at<T>(p, p.side - 1, h) * p.c, bhi = p.causal ? 0.f : table_at<T>(p, 2 * p.side - 1, h) * p.c;
    Stream<T, DP, QT, NT> qi, gi;
    float rl = kInf, rd = 0.f;
    auto fetch = [&](int q0) {
      qi.fetch(qb, p.qs.t, q0, qlen, p.D, p.vec, tid);
      gi.fetch(gb, p.dos.t, q0, qlen, p.D, p.vec, tid);
      if (tid < QT) {
        const bool ok = q0 + tid < qlen;
        rl = ok ? lse[q0 + tid] : kInf;
        rd = ok ? del[q0 + tid] : 0.f;
      }
    };
    if (qbeg < qend) fetch(qbeg);
    for (int q0 = qbeg; q0 < qend; q0 += QT) {
      __syncthreads();
      qi.put(sq, tid);
      gi.put(sg, tid);
      if (tid < QT) { srow[tid] = rl; srow[QT + tid] = rd; }
      if (q0 + QT < qend) fetch(q0 + QT);
      __syncthreads();
#pragma unroll
      for (int j2 = 0; j2 < QT / 32; ++j2) {
        const int qq = q0 + 32 * j2, pmin = pos0 + qq, pmax = pmin + 31;
        if (qq >= qend) break;
        if (p.causal && pmax < wk0) continue;
        const int dmax = wk0 + 31 - pmin, dmin = wk0 - pmax;
        f32x16 s, dp;
        zero16(dp);
        float off = 0.f;
        if (dmax <= -p.dsat) { off = blo; zero16(s); }
        else if (!p.causal && dmin >= p.dsat) { off = bhi; zero16(s); }
        else {
          const float* e = ext + (ki - pmin - 4 * hh);
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] = e[-acc_row(j, 0)];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          El<T>::mma(TL::row(sq, 32 * j2 + r, 2 * ks + hh), kf[ks], s);
          El<T>::mma(TL::row(sg, 32 * j2 + r, 2 * ks + hh), vf[ks], dp);
        }
        float pr[16], ds[16];
        // query row visible to this lane's key: its position >= ki (causal), the key inside the sequence
        const int first = in ? (p.causal ? ki - pmin - 4 * hh : -64) : 64;
        const bool edge = wk0 + 31 >= klen || (p.causal && dmax > 0);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float ls = srow[32 * j2 + acc_row(j, hh)], de = srow[QT + 32 * j2 + acc_row(j, hh)];
          pr[j] = expo<T>(s[j], p.c, off, ls);
          if (edge) pr[j] = acc_row(j, 0) >= first ? pr[j] : 0.f;
          pr[j] = ls == kInf ? 0.f : pr[j];
          ds[j] = pr[j] * (dp[j] - de);
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 16; ++j) ds[j] = acc_row(j, 0) >= first ? ds[j] : 0.f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const frag pf = El<T>::pack(pr + 8 * t), df = El<T>::pack(ds + 8 * t);
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            El<T>::mma(TL::col(sg, 32 * j2 + 16 * t, d, lane), pf, dv[d]);
            El<T>::mma(TL::col(sq, 32 * j2 + 16 * t, d, lane), df, dk[d]);
          }
        }
      }
    }
  }
  if (ki >= p.Tk) return;
  T* ko = (T*)p.dk + b * p.dks.b + hk * p.dks.h + (long)ki * p.dks.t;
  T* vo = (T*)p.dv + b * p.dvs.b + hk * p.dvs.h + (long)ki * p.dvs.t;
  if (in) {
    store_rows<T, DP>(ko, dk, p.scale, p.D, p.vec, hh);
    store_rows<T, DP>(vo, dv, 1.f, p.D, p.vec, hh);
  } else {
    zero_rows<T, DP>(ko, p.D, p.vec, hh);
    zero_rows<T, DP>(vo, p.D, p.vec, hh);
  }
}

// ---------------------------------------------------------------- launches
template <class T, int DP> constexpr int tile_bytes() { return 2 * kTile<T> * Tile<T, DP>::ROW; }
int host_ext_bytes(const BaParams& p) { return (2 * (p.dsat + EXT) + 1) * 4; }


// launches over 64 KB of LDS need the kernel's limit raised
template <class K> hipError_t launch(K kernel, long grid, int threads, int smem, const BaParams& p, hipStream_t s) {
  if (grid > 0x7fffffffL) return hipErrorInvalidValue;
  if (grid == 0) return hipSuccess;
  if (smem > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), smem, s, p);
  return hipGetLastError();
}

template <class T, int DP> hipError_t fwd(const BaParams& p, hipStream_t s) {
  constexpr int NW = 4;
  const long ntile = (p.Tq + 32 * NW - 1) / (32 * NW);
  return launch(ba_fwd_kernel<T, DP, NW>, (long)p.B * p.Hq * ntile, 64 * NW, tile_bytes<T, DP>() + host_ext_bytes(p), p, s);
}
template <class T, int DP> hipError_t bwd(const BaParams& p, hipStream_t s) {
  constexpr int NW = 4;
  const long ntile = (p.Tq + 32 * NW - 1) / (32 * NW), nkt = (p.Tk + 32 * NW - 1) / (32 * NW);
  hipError_t e = launch(ba_dq_kernel<T, DP, NW>, (long)p.B * p.Hq * ntile, 64 * NW,
                        tile_bytes<T, DP>() + (1 + NW) * host_ext_bytes(p), p, s);
  if (e == hipSuccess)
    e = launch(ba_dkv_kernel<T, DP, NW>, (long)p.B * p.Hkv * nkt, 64 * NW,
               tile_bytes<T, DP>() + 2 * kTile<T> * 4 + host_ext_bytes(p), p, s);
  if (e != hipSuccess) return e;
  if (p.nb * p.Hq == 0) return hipSuccess;
  hipLaunchKernelGGL((ba_dtable_kernel<T>), dim3((unsigned)(p.nb * p.Hq)), dim3(64), 0, s, p.tpart, (long)p.B * ntile,
                     (T*)p.dtable);
  return hipGetLastError();
}
template <class T> hipError_t fwd_t(const BaParams& p, hipStream_t s) {
  return p.D <= 64 ? fwd<T, 64>(p, s) : p.D <= 96 ? fwd<T, 96>(p, s) : fwd<T, 128>(p, s);
}
template <class T> hipError_t bwd_t(const BaParams& p, hipStream_t s) {
  return p.D <= 64 ? bwd<T, 64>(p, s) : p.D <= 96 ? bwd<T, 96>(p, s) : bwd<T, 128>(p, s);
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
char* align256(void* ws) { return (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255); }

}  // namespace

size_t ba_forward_ws(const BaParams&, int) { return 0; }
size_t ba_backward_ws(const BaParams& p, int) {
  const long ntile = (p.Tq + 127) / 128;
  return up256((size_t)p.B * p.Hq * p.Tq * 4) + up256((size_t)p.nb * p.Hq * p.B * ntile * 4) + 256;
}
hipError_t launch_ba_forward(BaParams p, int dtype, void* ws, hipStream_t s) {
  (void)ws;
  return dtype == 0 ? fwd_t<float>(p, s) : dtype == 1 ? fwd_t<bf16>(p, s) : fwd_t<f16>(p, s);
}
hipError_t launch_ba_backward(BaParams p, int dtype, void* ws, hipStream_t s) {
  char* w = align256(ws);
  p.delta = (float*)w;
  p.tpart = (float*)(w + up256((size_t)p.B * p.Hq * p.Tq * 4));
  return dtype == 0 ? bwd_t<float>(p, s) : dtype == 1 ? bwd_t<bf16>(p, s) : bwd_t<f16>(p, s);
}

}  // namespace gt
