// The gated feed-forward's tensor-core products (ffn_gemm.cu).
#pragma once

#include "dense.cuh"

namespace artlite {

// T token rows, H values a row of x, F features; all operands of one 16-bit type, rows of the matrices and of g, u, dg,
// du consecutive (ld H and F)
struct FfnArgs {
  int dtype, act;
  const void *x, *wg, *wu;  // x: ldx apart
  int64_t ldx;
  void* h;                  // forward: T x F, ldh apart
  int64_t ldh;
  float *g, *u;             // forward: the kept gate and up values (may be null); backward: read
  const void* dh;           // backward: lddh apart
  int64_t lddh;
  void *dg, *du;            // backward: the gradients of the gate and up values
  void* dx;                 // backward (may be null): lddx apart
  int64_t lddx;
  void *dwg, *dwu;          // backward (may be null)
  int64_t T;
  int H, F;
  DevStatus* status;
};
int launch_ffn_forward_gemm(const FfnArgs& a, cudaStream_t st);
int launch_ffn_backward_gemm(const FfnArgs& a, cudaStream_t st);  // dx, or dwg and dwu, or all three

}  // namespace artlite
