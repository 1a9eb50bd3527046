// Device side shared by the kernels of battn_fwd.hip and battn_bwd.hip: element types, LDS tiles and their staging,
// buckets and the bias table, softmax pieces.
//
// All kernels hold 32-row blocks "stationary" (a wave's rows are the lanes lane & 31 of every MFMA's B operand, in
// registers) and stream 32-row blocks of the other side through LDS (A operand):
//   forward, dQ   stationary queries, streamed keys:    S^T = K Q^T,  O^T += V^T P^T,  dQ^T += K^T dS^T
//   dK dV         stationary keys, streamed queries:    S = Q K^T,    dV^T += dO^T P,  dK^T += Q^T dS
// so that the P / dS block, which the first product leaves in the accumulator layout (column = lane & 31, rows
// acc_row(j, h)), is the second product's B operand as it stands: register j = 8 t + e holds key acc_row(8 t + e, h) of
// the 16-key step t, and the transposed A operand reads the same order (two 4-key groups a lane half).
//
// The bias enters as the C operand of the first product (bias / scale, from an LDS table over the offsets), or, where
// a 32 x 32 block lies wholly beyond the last border, as one constant: the exponent is a single FMA per score.
//
// A workgroup is WR row blocks x WS streams of waves: the WS waves of a row block take every WS-th 32-row block of the
// streamed side and join their sums through LDS at the end. WR = 4, WS = 1 shares each tile among 128 rows (long
// sequences, where the matrix cores bound), WR = 2, WS = 2 among 64 (twice the waves for as many rows), and WR = 1,
// WS = 4 spreads few rows over four waves (latency, memory).
#pragma once
#include "battn.h"
#include "battn_index.h"

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

// a b with nothing to add to: the zero stays an inline operand instead of 16 cleared registers
template <class T> GT_DEV f32x16 mma0(const typename El<T>::frag& a, const typename El<T>::frag& b) {
  f32x16 c = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  El<T>::mma(a, b, c);
  return c;
}
// keeps what follows inside its wave-uniform branch: the compiler would otherwise run such blocks always, with selects
template <class X> GT_DEV void in_branch(X& x) { asm volatile("" : "+v"(x)); }
// the value as if computed here: addresses and conditions formed from it are not kept in registers from before a loop
GT_DEV int anew_v(int x) { asm volatile("" : "+v"(x)); return x; }
GT_DEV int anew_s(int x) { asm volatile("" : "+s"(x)); return x; }
GT_DEV void zero16(f32x16& x) {
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = 0.f;
}
GT_DEV void halves(float x, float& lo, float& hi) {   // every lane: the low and the high half's value of its column
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}
GT_DEV float both_sum(float x) { float a, b; halves(x, a, b); return a + b; }
GT_DEV float both_max(float x) { float a, b; halves(x, a, b); return fmaxf(a, b); }

// eight channels d .. d + 7 of one row, zero past D (rows off the 16-byte grid)
template <class T> GT_DEV typename El<T>::frag load_row8(const T* p, int d, int D) {
  typename El<T>::frag f = El<T>::zero();
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < D) El<T>::set(f, e, p[d + e]);
  return f;
}
// a row's fragments, channels 16 s + 8 h .. + 7; `vec` as in BaParams: all loads, then the cleared channels past D
template <class T, int KS> GT_DEV void load_rows(typename El<T>::frag (&f)[KS], const T* row, int hh, int D, int vec) {
  if (vec) {
#pragma unroll
    for (int s = 0; s < KS; ++s) f[s] = El<T>::load16(row + min(16 * s + 8 * hh, D - 8));
    if (D < 16 * KS) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (16 * s + 8 * hh >= D) f[s] = El<T>::zero();
    }
  } else {
#pragma unroll
    for (int s = 0; s < KS; ++s) f[s] = load_row8(row, 16 * s + 8 * hh, D);
  }
}

// LDS image of a block of rows, DP channels each, as 16-byte chunks whose index is XORed, within groups of a power of
// two, with a function of the row: reads of one chunk of 16 consecutive rows (row fragments) and of 64 bytes of 4
// consecutive rows (transposed fragments) then fall on 64 different banks (fp32 transposed: 32 of two rows).
template <class T, int DP> struct Tile {
  typedef typename El<T>::frag frag;
  static constexpr int ES = sizeof(T), NC = DP * ES / 16, ROW = NC * 16;   // chunks, bytes of a row
  GT_DEV static constexpr int swz(int row) {
    if constexpr (NC == 32 || (NC == 16 && ES == 4)) return ((row >> 2) & 1) * 8 + ((row >> 3) & 1) * 4 + (row & 3);
    else if constexpr (NC == 16) return (row & 3) * 4 + ((row >> 2) & 3);
    else if constexpr (NC == 24) return (row >> 1) & 7;             // rows step by 32 banks
    else if constexpr (NC == 12) return (row >> 2) & 3;             // rows step by 48 banks
    else return ((row >> 1) & 1) * 4 + ((row >> 2) & 3);            // NC == 8: rows step by 32 banks
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
  for (int k = 0; k < p.nborder; k += 8)   // eight borders a scalar load; the unused ones lie beyond any distance
#pragma unroll
    for (int e = 0; e < 8; ++e) b += dist >= p.border[k + e];
  return b + ((!p.causal && delta > 0) ? p.side : 0);
}
GT_DEV int ext_len(const BaParams& p) { return ext_entries(p.dsat, p.causal); }
// Entries below -2^17 shut their bucket off as -inf does (rows that see only such keys are empty), entries above 2^17
// count as 2^17: exponents stay where one FMA is exact enough
template <class T> GT_DEV float table_at(const BaParams& p, int bucket, int h) {
  const float x = (float)((const T*)p.table)[(long)bucket * p.Hq + h];
  return x < -131072.f ? -kInf : x > 131072.f ? 131072.f : x;
}
// LDS tables of bias / scale by offset (battn_index.h) of the heads h0 .. h0 + nh - 1 (the last head again past h_last),
// ext_len entries each
template <class T> GT_DEV void build_ext(const BaParams& p, int h0, int nh, int h_last, float* ext, int tid, int nthreads) {
  const int n = ext_len(p);
  for (int i = tid; i < n; i += nthreads) {
    const int c = bucket_of(p, i - p.dsat - EXT);
    for (int g = 0; g < nh; ++g) ext[g * n + i] = table_at<T>(p, c, min(h0 + g, h_last)) * p.inv_scale;
  }
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
// keys of a batch entry that any of its queries sees: none past the last query's position under a causal mask, so what
// lies behind it in a cache (which zero probabilities would turn into NaN if it were not finite) is not read
GT_DEV int keys_of(const BaParams& p, int b, int qlen, int pos0) {
  const int n = clamp_len(p.len, b, p.Tk);
  return p.causal ? min(n, max(pos0 + qlen, 0)) : n;
}

// Work item -> batch, heads and tile: batch entry and key / value head go round first, so that the workgroups that read
// the same keys run on the same XCD (workgroups go round the 8 XCDs in turn). Under a causal mask a workgroup takes a tile
// from the end and its mirror image from the start (`pair`): all have the same work, and none runs on alone.

// ---------------------------------------------------------------- streamed rows: global -> LDS
// Aligned rows go by direct copies to LDS (16 bytes a lane; the lane's slot decides which chunk it fetches, so the image
// comes out swizzled); rows past the last valid one repeat it, and whoever reads them masks the products. Others go
// through registers, zero-padded. Visible after lds_ready().
template <class T, int DP, int ROWS, int NT> struct Stage {
  typedef Tile<T, DP> TL;
  static constexpr int SLOTS = ROWS * TL::NC, N = (SLOTS + NT - 1) / NT;
  const T* base;
  long st;
  int nrow, D, vec, tid, wave;   // wave: LDS bytes of the wave's first lane
  bool whole;                    // every chunk of a row is copied
  unsigned off[N];               // of this thread's chunks from the tile's first row
  GT_DEV static int row_of(int i) { return i / TL::NC; }
  GT_DEV static int chunk_of(int i) { return (i % TL::NC) ^ TL::swz(row_of(i)); }
  GT_DEV void init(const T* base_, long st_, int nrow_, int D_, int vec_, int tid_) {
    base = base_; st = st_; nrow = nrow_; D = D_; vec = vec_; tid = tid_;
    wave = __builtin_amdgcn_readfirstlane((tid & ~63) * 16);
    whole = vec && D == DP;
#pragma unroll
    for (int n = 0; n < N; ++n) off[n] = (unsigned)(row_of(n * NT + tid) * (int)(st * TL::ES)) + chunk_of(n * NT + tid) * 16;
  }
  GT_DEV void copy(char* lds, const char* from, unsigned o, int n) const {
    __builtin_amdgcn_global_load_lds((const void*)(from + o),
                                     (__attribute__((address_space(3))) void*)(lds + n * NT * 16 + wave), 16, 0, 0);
  }
  GT_DEV void load(char* lds, int row0) const {
    const char* from = (const char*)(base + (long)row0 * st);
    if (__builtin_expect(whole && row0 + ROWS <= nrow, 1)) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (SLOTS % NT == 0 || n * NT + tid < SLOTS) copy(lds, from, off[n], n);
      asm volatile("; whole tile");   // (keeps the compiler from folding the two forms' copies into one behind branches)
    } else if (vec) {
      const int last = nrow - 1 - row0;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int i = n * NT + tid, over = max(row_of(i) - last, 0);
        if ((SLOTS % NT == 0 || i < SLOTS) && chunk_of(i) * (16 / TL::ES) < D) copy(lds, from, off[n] - over * (int)(st * TL::ES), n);
      }
      asm volatile("; part of a tile");
    } else {
      constexpr int C8 = DP / 8;
      for (int i = tid; i < ROWS * C8; i += NT) {
        const int row = i / C8, c = i % C8;
        TL::put(lds, row, c, row0 + row < nrow ? load_row8(base + (long)(row0 + row) * st, 8 * c, D) : El<T>::zero());
      }
    }
  }
};
GT_DEV void lds_ready() {   // this wave's copies have landed, then everyone's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
// chunks past the head size are never copied: cleared once, apart from the others (the first lds_ready orders it)
template <class T, int DP> GT_DEV void clear_pad(char* lds, int rows, int D, int tid, int nthreads) {
  typedef Tile<T, DP> TL;
  for (int i = tid; i < rows * TL::NC; i += nthreads)
    if ((((i % TL::NC) ^ TL::swz(i / TL::NC)) * (16 / TL::ES)) >= D) *(uint4*)(lds + i * 16) = make_uint4(0, 0, 0, 0);
}

// rows of an accumulator set (column = row of the output, registers = channels) to memory
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

// fp32, whose time is its products: 128 rows where their last tile is not half empty and one of few ((416 heads, 189 rows,
// 80 channels): forward 118 us with 128 rows, 113 with 64, backward 422 and 397; 16-bit gains by 128 all the same)
inline bool fills128(int dtype, int T) { return dtype != 0 || T > 256 || (T - 1) % 128 >= 64; }

// Tiles shared by a workgroup: 64 streamed rows (fp32: 32 WS), two buffers, the next tile's copies in flight during this
// one's products (fp32 with WS > 1: one, its products are long).
constexpr int most(int a, int b) { return a > b ? a : b; }
template <class T, int DP, int WR, int WS> struct Shape {
  static constexpr int ES = sizeof(T);
  static constexpr int KT = WS > 2 ? 32 * WS : ES == 2 ? 64 : 32 * WS;
  static constexpr int NBUF = ES == 4 && WS > 1 ? 1 : 2;
  static constexpr int NB = KT / 32 / WS;                       // 32-row blocks of a tile for each wave
  static constexpr int TILE = KT * Tile<T, DP>::ROW;            // bytes of one operand's tile
  static constexpr int JOIN = WS > 1 ? WR * WS * DP * 33 * 4 : 0;
  static constexpr int BYTES = most(2 * NBUF * TILE, JOIN);
};

// Sum over the WS waves of a row block, through LDS ([row block][wave][channel][33], the tiles are done with): afterwards
// each thread of the row block's waves holds four channels of a row at a time, handed to `out(row, d, x[4])`. `mul`:
// this wave's factor for its row (lane & 31); 0: none of the wave's sums count, finite or not (a row that saw no key).
template <int DP, int WS, class F>
GT_DEV void join(char* smem, const f32x16 (&acc)[DP / 32], float mul, int wr, int ws, int lane, F out) {
  float* s = (float*)smem + wr * (WS * DP * 33);
  const int r = lane & 31, hh = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) s[(ws * DP + 32 * db + acc_row(j, hh)) * 33 + r] = mul == 0.f ? 0.f : acc[db][j] * mul;
  __syncthreads();
  for (int i = ws * 64 + lane; i < 32 * DP / 4; i += 64 * WS) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WS; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += s[(w * DP + d + e) * 33 + row];
    out(row, d, x);
  }
}
template <class T> GT_DEV void store4_row(T* row, int d, const float* x, int D, int vec) {
  if (vec) {
    if (d < D) El<T>::store4(row + d, x);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < D) row[d + e] = (T)x[e];
  }
}

// ---------------------------------------------------------------- launches
inline int host_ext_bytes(const BaParams& p) { return ext_entries(p.dsat, p.causal) * 4; }
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
constexpr int kLds = 160 * 1024;   // a CU's LDS
inline size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
inline char* align256(void* ws) { return (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255); }

}  // namespace
}  // namespace gt
