// The 4-bit linear's launchers (linear_gemm.cu) and the dense products' host helpers (linear.cu).
#pragma once

#include "dense.cuh"

namespace artlite {

// y = x . W^T (gated: act(x Wg^T) (x Wu^T)) for prompts, on tcgen05 (linear_gemm.cu)
struct LinearGemmArgs {
  int qtype;
  const uint8_t* w0;      // packed tiles
  const uint8_t* w1;      // gated: the up matrix's
  const uint16_t* x;      // fp16 rows, ldx apart (a multiple of 8), 16-byte aligned
  int64_t ldx;
  const int32_t* row_exp; // (may be null) row t of x holds the row's values times 2^-row_exp[t]
  int w_exp0, w_exp1;     // powers of two for the scales: 2^w_exp keeps the matrix inside fp16
  void* y;
  int64_t ldy;
  int out_dtype;          // ARTLITE_BF16 or ARTLITE_F16
  int64_t T;
  int K, N;
  bool gated;
  int act;
  DevStatus* status;
};
int launch_linear_gemm(const LinearGemmArgs& a, cudaStream_t st);

// x (T rows of K bf16, ldx apart) as fp16 rows (K apart), each times 2^-row_exp so that its largest value lies in
// [2^14, 2^15)
int launch_half_rows(const uint16_t* x, int64_t ldx, int64_t T, int K, uint16_t* out, int32_t* row_exp, cudaStream_t st);

// n bytes of device `dev` in stream order, from this library's own pool (inside a capture: the graph's own memory);
// give them back with stream_free on the same stream
int stream_alloc(int dev, size_t n, cudaStream_t st, void** out);
int stream_free(void* p, cudaStream_t st);

}  // namespace artlite
