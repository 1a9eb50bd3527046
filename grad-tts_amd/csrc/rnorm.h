// The residual step between two blocks (rnorm.hip): parameter block and launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gt {

constexpr int RN_MAX_C = 8192;

struct RnParams {
  const void *x, *y;                 // [B][T][C] contiguous
  const float *gate;                 // [C] or [B][C] (gate_batch), null: 1
  const float *w1, *b1, *w2, *b2;    // post / pre weights and biases [C]; biases may be null
  int B, T, C, rms, gate_batch;
  float scale, eps;
  const int64_t* len;                // [B] or null
  void *out, *h;                     // [B][T][C]
  float* stats;                      // [B][T][4]: mean, 1/std of y; mean, 1/std of out (null: not kept)
  int vec;                           // C % 8 == 0 and every tensor on 16 bytes
  // backward
  const void *dout, *dh;
  void *dx, *dy;
  float *dgate, *dw1, *db1, *dw2, *db2;   // dgate [C] or [B][C]; dgate, db1, db2 may be null
  float *part, *part2;               // [B][chunks][4][C]; [B][ranges][4][C]
  int rows_per_chunk, chunks, ranges;   // of one batch entry; ranges of its chunks
};

size_t rn_backward_ws(const RnParams& p);
hipError_t launch_rn_forward(RnParams p, int dtype, hipStream_t s);
hipError_t launch_rn_backward(RnParams p, int dtype, void* ws, hipStream_t s);

}  // namespace gt
