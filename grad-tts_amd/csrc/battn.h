// Attention with a learned relative position bias by buckets (battn_fwd.hip, battn_bwd.hip): parameter block, launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gt {

constexpr int BA_MAX_D = 128, BA_MAX_BUCKETS = 128, BA_MAX_DISTANCE = 1024;

struct BaStride { long b, t, h; };   // elements; the channels of a head are contiguous

struct BaParams {
  const void *q, *k, *v, *table;
  BaStride qs, ks, vs;
  int B, Tq, Tk, Hq, Hkv, G, D;      // G = Hq / Hkv query heads a key / value head
  int causal, vec;                   // vec: every row starts on 16 bytes and D % 8 == 0
  float c, inv_scale, scale;         // c = scale log2(e)
  // bucket of a distance: itself below `exact`, else exact + #{k : distance >= border[k]}; all distances >= dsat share
  // the last bucket. side = buckets of one direction (bidirectional: offsets > 0 use side .. 2 side - 1)
  int nb, side, exact, nborder, dsat;
  int border[64];                    // the unused ones beyond any distance
  const int64_t *len, *qlen, *qstart;   // [B] or null: all of Tk, all of Tq, 0
  int ntile, pair;                   // tiles of the launch's stationary side; two of them a workgroup
  // forward
  void* out; BaStride os;
  float* lse;                        // [B][Hq][Tq], log2 units; +inf: no visible key
  int gp, qpb;                       // spread form: heads and queries packed into the 32 rows of a block
  int nsplit, split_keys;            // spread form: key ranges of their own workgroups
  float *part, *part_ml;             // [row block][split][32][D]; [row block][split][2][32]
  // backward
  const void *o, *dout; BaStride dos;
  void *dq, *dk, *dv, *dtable; BaStride dqs, dks, dvs;
  float *delta, *tpart;              // [B][Hq][Tq]; [nb][Hq][B workgroups of a head]
  int gsplit;                        // dK dV: groups of heads with workgroups of their own, summed from gpart
  float* gpart;                      // [2][gsplit][B][Tk][Hkv][D]
};

// dtype: 0 fp32, 1 bf16, 2 fp16
size_t ba_forward_ws(const BaParams& p, int dtype);
size_t ba_backward_ws(const BaParams& p, int dtype);
hipError_t launch_ba_forward(BaParams p, int dtype, void* ws, hipStream_t s);
hipError_t launch_ba_backward(BaParams p, int dtype, void* ws, hipStream_t s);

}  // namespace gt
