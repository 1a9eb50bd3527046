// The step between two blocks of a transformer with norms on both sides of a block, gfx950:
//   out = x + scale gate * N1(y) ,   h = N2(out) ,   N(t) = u w + b ,  u = (t - mean) / sqrt(var + eps)  (layer)
//                                                               u = t / sqrt(mean t^2 + eps)         (rms)
// x the residual stream, y the finished block's output, h the next block's input; statistics over the C channels.
// Bound by memory: the forward reads x and y and writes out and h once, the backward reads x, y, d out, dh and writes
// dx and dy. One group of TPR threads holds a whole row in registers (E channels a thread), so both norms are two-pass
// (mean, then centred squares) without reading anything twice; groups walk their rows with the next row's loads in
// flight and with gate and weights, the same for every row of a batch entry, in registers. bf16, where a copy reaches
// 4.9 TB/s: forward, 4 x 4096 rows of 4096 (537 MB) in 117 us, 4.6 TB/s; backward, 4 x 2048 rows of 2048 (201 MB) in
// 57 us, 3.6 TB/s (156 registers: three waves a SIMD), and 10 us for the column sums. Two rows' loads in flight instead
// of one: the same times. Above 4096 channels a row has 1024 threads, 128 registers each: the backward spills 51 to 91 of
// its values, 4 x 512 rows of 8192 (201 MB) take 142 us in bf16 and 262 in fp32.
#include "rnorm.h"

#include "common.h"

namespace gt {
namespace {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <class T> struct Raw8;
template <> struct Raw8<float> { f32x4 a, b; };
template <> struct Raw8<bf16> { bf16x8 a; };
template <> struct Raw8<f16> { f16x8 a; };
GT_DEV float raw_get(const Raw8<float>& r, int e) { return e < 4 ? r.a[e] : r.b[e - 4]; }
GT_DEV float raw_get(const Raw8<bf16>& r, int e) { return (float)r.a[e]; }
GT_DEV float raw_get(const Raw8<f16>& r, int e) { return (float)r.a[e]; }
GT_DEV void raw_set(Raw8<float>& r, int e, float v) { if (e < 4) r.a[e] = v; else r.b[e - 4] = v; }
GT_DEV void raw_set(Raw8<bf16>& r, int e, bf16 v) { r.a[e] = v; }
GT_DEV void raw_set(Raw8<f16>& r, int e, f16 v) { r.a[e] = v; }
GT_DEV Raw8<float> raw_pack(const float* x, float) { return {{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}}; }
GT_DEV Raw8<bf16> raw_pack(const float* x, bf16) { return {__builtin_bit_cast(bf16x8, f_to_item(x, bf16()))}; }
GT_DEV Raw8<f16> raw_pack(const float* x, f16) {
  return {__builtin_convertvector((f32x8){x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}, f16x8)};
}

// Channels of a thread: VEC: NC groups of eight consecutive ones (16-byte accesses); otherwise (a width or an address
// that breaks the 16-byte grid) single ones TPR apart, so that a wave's accesses still fall on consecutive addresses
template <class T, int TPR, int NC, bool VEC> struct Row {
  static constexpr int E = 8 * NC;
  GT_DEV static int chan(int t, int e) { return VEC ? (t + TPR * (e >> 3)) * 8 + (e & 7) : t + TPR * e; }
  Raw8<T> r[NC];
  GT_DEV void load(const T* p, int t, int C) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (VEC) {
        const int c = (t + TPR * n) * 8;
        if (c < C) r[n] = *(const Raw8<T>*)(p + c);
        else r[n] = __builtin_bit_cast(Raw8<T>, Raw8<T>{});
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw_set(r[n], e, chan(t, 8 * n + e) < C ? p[chan(t, 8 * n + e)] : (T)0.f);
      }
    }
  }
  GT_DEV float get(int e) const { return raw_get(r[e >> 3], e & 7); }
};
template <class T, int TPR, int NC, bool VEC> GT_DEV void row_store(T* p, const float* x, int t, int C) {
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    if (VEC) {
      const int c = (t + TPR * n) * 8;
      if (c < C) *(Raw8<T>*)(p + c) = raw_pack(x + 8 * n, T());
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = t + TPR * (8 * n + e);
        if (c < C) p[c] = (T)x[8 * n + e];
      }
    }
  }
}

// sum over the wave in registers (row rotations, then swaps of 16- and 32-lane rows): no LDS round trip a step
GT_DEV float wave_total(float x) {
  x = row_sum16(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// sums over the TPR threads of a row group; every thread gets them, in one order
template <int TPR, int N> struct RowSum {
  float* s;   // [2][TPR / 64][N] for this group
  int flip;
  GT_DEV void operator()(float (&v)[N], int t) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_total(v[i]);
    if constexpr (TPR > 64) {
      constexpr int NW = TPR / 64;
      float* b = s + flip * NW * N;
      flip ^= 1;   // two buffers: the next sum's writes cannot meet this one's reads
      if ((t & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) b[(t >> 6) * N + i] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float a = b[i];
#pragma unroll
        for (int w = 1; w < NW; ++w) a += b[w * N + i];
        v[i] = a;
      }
    }
  }
};

// rows of one wave share a workgroup with three others; wider groups meet at barriers, so they are workgroups of their own
template <int TPR> constexpr int kThreads = TPR == 64 ? 256 : TPR;

GT_DEV int row_len(const RnParams& p, int b) {
  if (!p.len) return p.T;
  const int64_t n = p.len[b];
  return n < 0 ? 0 : n > p.T ? p.T : (int)n;
}

// rows of group `g` of the launch: batch entry, first row and one past the last
template <int TPR> GT_DEV bool chunk_of(const RnParams& p, int& b, int& t0, int& t1, int& chunk) {
  const long g = (long)blockIdx.x * (kThreads<TPR> / TPR) + threadIdx.x / TPR;
  if (g >= (long)p.B * p.chunks) return false;
  b = (int)(g / p.chunks);
  chunk = (int)(g % p.chunks);
  t0 = chunk * p.rows_per_chunk;
  t1 = min(p.T, t0 + p.rows_per_chunk);
  return true;
}

template <class T, int TPR, int NC, bool VEC>
__global__ __launch_bounds__(kThreads<TPR>) void rn_fwd_kernel(RnParams p) {
  typedef Row<T, TPR, NC, VEC> R;
  constexpr int E = R::E;
  __shared__ float s_sum[TPR > 64 ? 2 * TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  int b, t0, t1, chunk;
  if (!chunk_of<TPR>(p, b, t0, t1, chunk)) return;   // whole groups: blocks of one group do not reach this
  RowSum<TPR, 1> rsum{s_sum, 0};
  auto sum1 = [&](float v) { float a[1] = {v}; rsum(a, t); return a[0]; };
  const float rc = 1.f / (float)p.C;
  float a1[E], c1[E], w2[E], b2[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = R::chan(t, e);
    const bool in = c < p.C;
    const float g = in ? p.scale * (p.gate ? p.gate[(p.gate_batch ? (long)b * p.C : 0) + c] : 1.f) : 0.f;
    a1[e] = in ? g * p.w1[c] : 0.f;
    c1[e] = in && p.b1 ? g * p.b1[c] : 0.f;
    w2[e] = in ? p.w2[c] : 0.f;
    b2[e] = in && p.b2 ? p.b2[c] : 0.f;
  }
  const int live = row_len(p, b);
  const long base = (long)b * p.T;
  R xn, yn;
  if (t0 < min(t1, live)) {
    xn.load((const T*)p.x + (base + t0) * p.C, t, p.C);
    yn.load((const T*)p.y + (base + t0) * p.C, t, p.C);
  }
  for (int row = t0; row < t1; ++row) {
    T* out = (T*)p.out + (base + row) * p.C;
    T* h = (T*)p.h + (base + row) * p.C;
    float o[E], u[E];
    if (row >= live) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
      row_store<T, TPR, NC, VEC>(out, o, t, p.C);
      row_store<T, TPR, NC, VEC>(h, o, t, p.C);
      continue;
    }
    const R x = xn, y = yn;
    if (row + 1 < min(t1, live)) {
      xn.load((const T*)p.x + (base + row + 1) * p.C, t, p.C);
      yn.load((const T*)p.y + (base + row + 1) * p.C, t, p.C);
    }
    auto moments = [&](float (&v)[E], float& mean, float& rstd) {   // v becomes the unit row
      mean = 0.f;
      float a = 0.f;
      if (!p.rms) {
#pragma unroll
        for (int e = 0; e < E; ++e) a += v[e];
        mean = sum1(a) * rc;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = R::chan(t, e) < p.C ? v[e] - mean : 0.f;
        a = 0.f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) a = __builtin_fmaf(v[e], v[e], a);
      rstd = 1.f / sqrtf(sum1(a) * rc + p.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= rstd;
    };
    float m1, r1, m2, r2;
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = y.get(e);
    moments(u, m1, r1);
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = o[e] = x.get(e) + __builtin_fmaf(u[e], a1[e], c1[e]);
    row_store<T, TPR, NC, VEC>(out, o, t, p.C);
    moments(u, m2, r2);
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = __builtin_fmaf(u[e], w2[e], b2[e]);
    row_store<T, TPR, NC, VEC>(h, u, t, p.C);
    if (p.stats && t == 0) *(f32x4*)(p.stats + (base + row) * 4) = (f32x4){m1, r1, m2, r2};
  }
}

// d = d out + N2'(dh):  du2 = dh w2,  d = d out + r2 (du2 - mean(du2) - u2 mean(du2 u2));  dx = d
// dy = N1'(d scale gate w1) likewise with r1, u1.  Column sums over the chunk's rows: d u1, d, dh u2, dh -- from these
// come d gate, d w1, d b1, d w2, d b2 (scale, gate and the weights do not change within a batch entry). out is formed
// again in fp32 from x and y: its rounded copy would cost the same bytes and lose bits.
template <class T, int TPR, int NC, bool VEC>
__global__ __launch_bounds__(kThreads<TPR>) void rn_bwd_kernel(RnParams p) {
  typedef Row<T, TPR, NC, VEC> R;
  constexpr int E = R::E;
  __shared__ float s_sum[TPR > 64 ? 4 * TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  int b, t0, t1, chunk;
  if (!chunk_of<TPR>(p, b, t0, t1, chunk)) return;
  RowSum<TPR, 2> sum2{s_sum, 0};
  const float rc = 1.f / (float)p.C, rcl = p.rms ? 0.f : rc;
  float a1[E], c1[E], w2[E], cd1[E], cd[E], ch2[E], ch[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = R::chan(t, e);
    const bool in = c < p.C;
    const float g = in ? p.scale * (p.gate ? p.gate[(p.gate_batch ? (long)b * p.C : 0) + c] : 1.f) : 0.f;
    a1[e] = in ? g * p.w1[c] : 0.f;
    c1[e] = in && p.b1 ? g * p.b1[c] : 0.f;
    w2[e] = in ? p.w2[c] : 0.f;
    cd1[e] = cd[e] = ch2[e] = ch[e] = 0.f;
  }
  const int live = row_len(p, b);
  const long base = (long)b * p.T;
  R xn, yn, gn, hn;
  f32x4 sn = {0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](int row) {
    const long o = (base + row) * p.C;
    xn.load((const T*)p.x + o, t, p.C);
    yn.load((const T*)p.y + o, t, p.C);
    gn.load((const T*)p.dout + o, t, p.C);
    hn.load((const T*)p.dh + o, t, p.C);
    sn = *(const f32x4*)(p.stats + (base + row) * 4);
  };
  if (t0 < min(t1, live)) fetch(t0);
  for (int row = t0; row < t1; ++row) {
    T* dx = (T*)p.dx + (base + row) * p.C;
    T* dy = (T*)p.dy + (base + row) * p.C;
    float d[E];
    if (row >= live) {
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = 0.f;
      row_store<T, TPR, NC, VEC>(dx, d, t, p.C);
      row_store<T, TPR, NC, VEC>(dy, d, t, p.C);
      continue;
    }
    const R x = xn, y = yn, gr = gn, hr = hn;
    const f32x4 st = sn;
    if (row + 1 < min(t1, live)) fetch(row + 1);
    float u1[E], u2[E], s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = R::chan(t, e) < p.C;
      const float dh = hr.get(e);
      u1[e] = in ? (y.get(e) - st[0]) * st[1] : 0.f;
      u2[e] = in ? (x.get(e) + __builtin_fmaf(u1[e], a1[e], c1[e]) - st[2]) * st[3] : 0.f;
      ch2[e] = __builtin_fmaf(dh, u2[e], ch2[e]);
      ch[e] += dh;
      d[e] = dh * w2[e];
      s[0] += d[e];
      s[1] = __builtin_fmaf(d[e], u2[e], s[1]);
    }
    sum2(s, t);
    s[0] *= rcl;
    s[1] *= rc;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      d[e] = gr.get(e) + st[3] * (d[e] - s[0] - u2[e] * s[1]);
      if (R::chan(t, e) >= p.C) d[e] = 0.f;
      cd1[e] = __builtin_fmaf(d[e], u1[e], cd1[e]);
      cd[e] += d[e];
      u2[e] = d[e] * a1[e];
      q[0] += u2[e];
      q[1] = __builtin_fmaf(u2[e], u1[e], q[1]);
    }
    row_store<T, TPR, NC, VEC>(dx, d, t, p.C);
    sum2(q, t);
    q[0] *= rcl;
    q[1] *= rc;
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = st[1] * (u2[e] - q[0] - u1[e] * q[1]);
    row_store<T, TPR, NC, VEC>(dy, d, t, p.C);
  }
  float* part = p.part + ((long)b * p.chunks + chunk) * 4 * p.C;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = R::chan(t, e);
    if (c >= p.C) continue;
    part[c] = cd1[e];
    part[p.C + c] = cd[e];
    part[2 * p.C + c] = ch2[e];
    part[3 * p.C + c] = ch[e];
  }
}

// Column sums of the chunks in two steps, in a fixed order: 64 channels and a range of one batch entry's chunks a workgroup
// (blockIdx.y: range, blockIdx.z: entry), then all ranges and entries.
__global__ __launch_bounds__(256) void rn_cols_kernel(RnParams p) {
  __shared__ float s[4][4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const int per = (p.chunks + p.ranges - 1) / p.ranges, k0 = blockIdx.y * per, k1 = min(p.chunks, k0 + per);
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C)
    for (int k = k0 + wv; k < k1; k += 4) {
      const float* q = p.part + ((long)blockIdx.z * p.chunks + k) * 4 * p.C + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] += q[(long)i * p.C];
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[wv][i][lane] = a[i];
  __syncthreads();
  // wave i adds up column sum i
  if (c < p.C)
    p.part2[(((long)blockIdx.z * p.ranges + blockIdx.y) * 4 + wv) * p.C + c] = s[0][wv][lane] + s[1][wv][lane] + s[2][wv][lane] + s[3][wv][lane];
}
// sums of d u1, d -> dgate, dw1, db1; of dh u2, dh -> dw2, db2
__global__ __launch_bounds__(1024) void rn_params_kernel(RnParams p) {
  __shared__ float s[5][16][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const bool in = c < p.C;
  const float w1 = in ? p.w1[c] : 0.f, b1 = in && p.b1 ? p.b1[c] : 0.f;
  float t[5] = {0.f, 0.f, 0.f, 0.f, 0.f};   // dw1, db1, dw2, db2, dgate
  if (in)
    for (int b = wv; b < p.B; b += 16) {   // a wave every sixteenth entry
      float a[4] = {0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < p.ranges; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] += p.part2[(((long)b * p.ranges + r) * 4 + i) * p.C + c];
      const float g = p.scale * (p.gate ? p.gate[(p.gate_batch ? (long)b * p.C : 0) + c] : 1.f);
      t[0] = __builtin_fmaf(g, a[0], t[0]);
      t[1] = __builtin_fmaf(g, a[1], t[1]);
      t[2] += a[2];
      t[3] += a[3];
      const float x = p.scale * (w1 * a[0] + b1 * a[1]);
      if (p.dgate && p.gate_batch) p.dgate[(long)b * p.C + c] = x;
      t[4] += x;
    }
#pragma unroll
  for (int i = 0; i < 5; ++i) s[i][wv][lane] = t[i];
  __syncthreads();
  float* out[5] = {p.dw1, p.db1, p.dw2, p.db2, p.gate_batch ? nullptr : p.dgate};
#pragma unroll
  for (int i = 0; i < 5; ++i)
    if (wv == i && in && out[i]) {
      float a = 0.f;
      for (int w = 0; w < 16; ++w) a += s[i][w][lane];
      out[i][c] = a;
    }
}

// ---------------------------------------------------------------- launches
// threads of a row, 8 channels each
int tpr_of(int C) { return C <= 512 ? 64 : C <= 1024 ? 128 : C <= 2048 ? 256 : C <= 4096 ? 512 : 1024; }

// chunks of a batch entry: about 256 CUs x 1024 threads in all, the rows of the backward's column sums too (its 156
// registers leave room for 768), at least 4 rows each
void set_chunks(RnParams& p, bool bwd) {
  const long groups = (bwd ? 196608 : 262144) / tpr_of(p.C), rows = (long)p.B * p.T;
  p.rows_per_chunk = p.chunks = p.ranges = 0;
  if (rows == 0) return;
  long rpc = (rows + groups - 1) / groups;
  if (rpc < 4) rpc = 4;
  if (rpc > p.T) rpc = p.T;
  p.rows_per_chunk = (int)rpc;
  p.chunks = (int)((p.T + rpc - 1) / rpc);
  // ranges: about 512 workgroups of column sums, 8 chunks each at least
  const long blocks = (long)((p.C + 63) / 64) * p.B, want = (512 + blocks - 1) / blocks, most = (p.chunks + 7) / 8;
  p.ranges = (int)(want < most ? want : most);
}

template <class T, int TPR, int NC, bool VEC> hipError_t go(const RnParams& p, bool bwd, hipStream_t s) {
  constexpr int NT = kThreads<TPR>;
  const long groups = (long)p.B * p.chunks, blocks = (groups * TPR + NT - 1) / NT;
  if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
  if (bwd) rn_bwd_kernel<T, TPR, NC, VEC><<<dim3((unsigned)blocks), dim3(NT), 0, s>>>(p);
  else rn_fwd_kernel<T, TPR, NC, VEC><<<dim3((unsigned)blocks), dim3(NT), 0, s>>>(p);
  return hipGetLastError();
}
template <class T, bool VEC> hipError_t go_c(const RnParams& p, bool bwd, hipStream_t s) {
  switch (tpr_of(p.C)) {
    case 64: return go<T, 64, 1, VEC>(p, bwd, s);
    case 128: return go<T, 128, 1, VEC>(p, bwd, s);
    case 256: return go<T, 256, 1, VEC>(p, bwd, s);
    case 512: return go<T, 512, 1, VEC>(p, bwd, s);
    default: return go<T, 1024, 1, VEC>(p, bwd, s);
  }
}
hipError_t go_t(const RnParams& p, int dtype, bool bwd, hipStream_t s) {
  if (dtype == 0) return p.vec ? go_c<float, true>(p, bwd, s) : go_c<float, false>(p, bwd, s);
  if (dtype == 1) return p.vec ? go_c<bf16, true>(p, bwd, s) : go_c<bf16, false>(p, bwd, s);
  return p.vec ? go_c<f16, true>(p, bwd, s) : go_c<f16, false>(p, bwd, s);
}

}  // namespace

size_t rn_backward_ws(const RnParams& p0) {
  RnParams p = p0;
  set_chunks(p, true);
  return (size_t)p.B * (p.chunks + p.ranges) * 4 * p.C * 4 + 256;
}
hipError_t launch_rn_forward(RnParams p, int dtype, hipStream_t s) {
  set_chunks(p, false);
  return p.chunks ? go_t(p, dtype, false, s) : hipSuccess;
}
hipError_t launch_rn_backward(RnParams p, int dtype, void* ws, hipStream_t s) {
  set_chunks(p, true);
  p.part = (float*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
  p.part2 = p.part + (size_t)p.B * p.chunks * 4 * p.C;
  const unsigned cols = (unsigned)((p.C + 63) / 64);
  if (p.chunks) {
    if (p.B > 65535) return hipErrorInvalidValue;   // (block_ops.cpp refuses it)
    if (hipError_t e = go_t(p, dtype, true, s)) return e;
    rn_cols_kernel<<<dim3(cols, (unsigned)p.ranges, (unsigned)p.B), dim3(256), 0, s>>>(p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  rn_params_kernel<<<dim3(cols), dim3(1024), 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace gt
