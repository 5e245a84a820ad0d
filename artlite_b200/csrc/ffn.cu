// The gated feed-forward over a model's own 16-bit matrices (artlite_gated_ffn, artlite_gated_ffn_backward): argument
// checks, the choice of kernel, and the backward pass's elementwise step. No state: every buffer is the caller's.
#include <cuda_runtime.h>

#include "dense_gemm.cuh"
#include "ffn.cuh"
#include "kernels.cuh"
#include "small_batch.cuh"

namespace artlite {
namespace {

// dg = dh u act'(g), du = dh act(g) of eight values a thread, from the fp32 gate and up values; rounded once to 16 bits
// as the two products' operands (each a sum over many of them: the roundings average out under the output's own).
// Bound by HBM: 14 bytes a value, 940 MB of an 8192 x 8192 step in 133 us (7.1 TB/s).
template <class T>
__global__ void gate_grad_kernel(const T* dh, int64_t lddh, const float* g, const float* u, int act, int64_t T_, int F,
                                 T* dg, T* du) {
  const int per = F / 8;
  const int64_t n = T_ * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per;
    const int f = 8 * (int)(i - row * per);
    const uint4 d4 = __ldcs(reinterpret_cast<const uint4*>(dh + row * lddh + f));
    const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w};
    const float4* gp = reinterpret_cast<const float4*>(g + row * F + f);
    const float4* up = reinterpret_cast<const float4*>(u + row * F + f);
    const float4 g0 = __ldcs(gp), g1 = __ldcs(gp + 1), u0 = __ldcs(up), u1 = __ldcs(up + 1);
    const float gv[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
    const float uv[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float2 d = Num<T>::unpack(dw[j]);
      float a0, a1, s0, s1;
      act_and_slope(act, gv[2 * j], &a0, &s0);
      act_and_slope(act, gv[2 * j + 1], &a1, &s1);
      og[j] = Num<T>::pack(d.x * uv[2 * j] * s0, d.y * uv[2 * j + 1] * s1);
      ou[j] = Num<T>::pack(d.x * a0, d.y * a1);
    }
    *reinterpret_cast<uint4*>(dg + row * F + f) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(du + row * F + f) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

template <class T>
int launch_gate_grad(const FfnArgs& a, cudaStream_t st) {
  const int64_t n = a.T * (a.F / 8);
  const unsigned grid = (unsigned)min64(cdiv(n, 256), 1 << 20);
  gate_grad_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T*>(a.dh), a.lddh, a.g, a.u, a.act, a.T, a.F,
                                            static_cast<T*>(a.dg), static_cast<T*>(a.du));
  AL_LAUNCHED();
  return ARTLITE_OK;
}

// tokens up to which the small-batch kernel runs. Measured (us) at 2048 x 6144 bf16 against tensor-core tiles: T = 1
// 12.6 / 23.0, 8 14.1 / 18.7, 16 16.5 / 18.4, 24 20.2 / 18.3
constexpr int64_t kSmallTokens = 16;

int forward(const FfnArgs& a, int dev, cudaStream_t st) {
  if (a.T > kSmallTokens || a.H > sb::kMaxK) return launch_ffn_forward_gemm(a, st);
  sb::Args s{};
  AL_TRY(dg::make_operand_map(&s.map[0], a.wg, a.H, a.F, a.H, 64, kTileRows));
  AL_TRY(dg::make_operand_map(&s.map[1], a.wu, a.H, a.F, a.H, 64, kTileRows));
  s.x = a.x;
  s.y = a.h;
  s.ldx = a.ldx;
  s.ldy = a.ldh;
  s.T = a.T;
  s.K = a.H;
  s.N = a.F;
  s.act = a.act;
  s.vec = 1;
  s.keep_g = a.g;
  s.keep_u = a.u;
  s.status = a.status;
  if (a.dtype == ARTLITE_BF16) return sb::launch<sb::Plain<__nv_bfloat16>, __nv_bfloat16, true>(s, dev, st);
  return sb::launch<sb::Plain<__half>, __half, true>(s, dev, st);
}

// the checks both passes share; *dev: the device of the buffers
int check_common(const char* who, int dtype, int act, int64_t T, int H, int F) {
  AL_CHECK(dtype == ARTLITE_BF16 || dtype == ARTLITE_F16, ARTLITE_EINVAL, "%s: type %d (BF16 or F16)", who, dtype);
  AL_CHECK(act == kActSilu || act == kActGelu, ARTLITE_EINVAL, "%s: activation %d", who, act);
  AL_CHECK(T >= 0 && T <= 0x7FFFFFFF && H >= 8 && F >= 8 && H % 8 == 0 && F % 8 == 0, ARTLITE_EINVAL,
           "%s: T %lld, n_in %d, n_ffn %d (both multiples of 8)", who, (long long)T, H, F);
  return ARTLITE_OK;
}
struct Buf {
  const char* name;
  const void* p;
  int64_t ld, cols;
};
int check_buffers(const char* who, const Buf* b, int n, int* dev) {
  *dev = -1;
  for (int i = 0; i < n; i++) {
    if (!b[i].p) continue;
    AL_CHECK((uintptr_t)b[i].p % 16 == 0 && b[i].ld >= b[i].cols && b[i].ld % 8 == 0, ARTLITE_EINVAL,
             "%s: %s is not 16-byte aligned, or its rows are %lld apart (%lld values, a multiple of 8)", who, b[i].name,
             (long long)b[i].ld, (long long)b[i].cols);
    const int d = device_of(b[i].p);
    AL_CHECK(d >= 0, ARTLITE_EINVAL, "%s: %s is not device memory", who, b[i].name);
    if (*dev < 0) *dev = d;
    AL_CHECK(d == *dev, ARTLITE_EINVAL, "%s: %s is on device %d, the others on device %d", who, b[i].name, d, *dev);
  }
  return ARTLITE_OK;
}

}  // namespace
}  // namespace artlite

using namespace artlite;

extern "C" {
#pragma GCC visibility push(default)

int64_t artlite_gated_ffn_work_bytes(int64_t T, int n_ffn) { return T > 0 && n_ffn > 0 ? 4 * T * n_ffn : 0; }

int artlite_gated_ffn(int dtype, int activation, const void* x, int64_t ldx, const void* w_gate, const void* w_up, void* h,
                      int64_t ldh, float* gate, float* up, int64_t T, int n_in, int n_ffn, void* stream) {
  AL_TRY(check_common("gated_ffn", dtype, activation, T, n_in, n_ffn));
  if (T == 0) return ARTLITE_OK;
  AL_CHECK(x && w_gate && w_up && h, ARTLITE_EINVAL, "gated_ffn: null array");
  AL_CHECK((gate == nullptr) == (up == nullptr), ARTLITE_EINVAL, "gated_ffn: gate and up are kept together or not at all");
  const Buf bufs[] = {{"x", x, ldx, n_in},       {"w_gate", w_gate, n_in, n_in}, {"w_up", w_up, n_in, n_in},
                      {"h", h, ldh, n_ffn},      {"gate", gate, n_ffn, n_ffn},   {"up", up, n_ffn, n_ffn}};
  int dev;
  AL_TRY(check_buffers("gated_ffn", bufs, 6, &dev));
  DeviceScope scope(dev);
  AL_TRY(scope.code);
  AL_TRY(take_dense_status(dev, "gated_ffn"));
  FfnArgs a{};
  a.dtype = dtype;
  a.act = activation;
  a.x = x;
  a.ldx = ldx;
  a.wg = w_gate;
  a.wu = w_up;
  a.h = h;
  a.ldh = ldh;
  a.g = gate;
  a.u = up;
  a.T = T;
  a.H = n_in;
  a.F = n_ffn;
  AL_TRY(dense_status(dev, &a.status));
  const int rc = forward(a, dev, static_cast<cudaStream_t>(stream));
  if (rc == ARTLITE_ECUDA) cudaGetLastError();  // (reported here, not by the next launch)
  return rc;
}

int artlite_gated_ffn_backward(int dtype, int activation, const void* dh, int64_t lddh, const void* x, int64_t ldx,
                               const void* w_gate, const void* w_up, const float* gate, const float* up, void* work, void* dx,
                               int64_t lddx, void* dw_gate, void* dw_up, int64_t T, int n_in, int n_ffn, void* stream) {
  AL_TRY(check_common("gated_ffn_backward", dtype, activation, T, n_in, n_ffn));
  AL_CHECK((dw_gate == nullptr) == (dw_up == nullptr), ARTLITE_EINVAL,
           "gated_ffn_backward: dw_gate and dw_up are computed together or not at all");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // (a sum over no tokens)
    if (!dw_gate) return ARTLITE_OK;
    const Buf outs[] = {{"dw_gate", dw_gate, n_in, n_in}, {"dw_up", dw_up, n_in, n_in}};
    int dev;
    AL_TRY(check_buffers("gated_ffn_backward", outs, 2, &dev));
    DeviceScope scope(dev);
    AL_TRY(scope.code);
    AL_CUDA(cudaMemsetAsync(dw_gate, 0, (size_t)n_in * n_ffn * 2, st));
    AL_CUDA(cudaMemsetAsync(dw_up, 0, (size_t)n_in * n_ffn * 2, st));
    return ARTLITE_OK;
  }
  AL_CHECK(dh && gate && up && work, ARTLITE_EINVAL, "gated_ffn_backward: null array");
  AL_CHECK(!dx || (w_gate && w_up), ARTLITE_EINVAL, "gated_ffn_backward: dx needs the matrices");
  AL_CHECK(!dw_gate || x, ARTLITE_EINVAL, "gated_ffn_backward: dw_gate and dw_up need x");
  const Buf bufs[] = {{"dh", dh, lddh, n_ffn},    {"x", dw_gate ? x : nullptr, ldx, n_in},
                      {"w_gate", dx ? w_gate : nullptr, n_in, n_in}, {"w_up", dx ? w_up : nullptr, n_in, n_in},
                      {"gate", gate, n_ffn, n_ffn}, {"up", up, n_ffn, n_ffn},
                      {"work", work, n_ffn, n_ffn}, {"dx", dx, lddx, n_in},
                      {"dw_gate", dw_gate, n_in, n_in}, {"dw_up", dw_up, n_in, n_in}};
  int dev;
  AL_TRY(check_buffers("gated_ffn_backward", bufs, 10, &dev));
  DeviceScope scope(dev);
  AL_TRY(scope.code);
  AL_TRY(take_dense_status(dev, "gated_ffn_backward"));
  FfnArgs a{};
  a.dtype = dtype;
  a.act = activation;
  a.x = x;
  a.ldx = ldx;
  a.wg = w_gate;
  a.wu = w_up;
  a.g = const_cast<float*>(gate);
  a.u = const_cast<float*>(up);
  a.dh = dh;
  a.lddh = lddh;
  a.dg = work;
  a.du = static_cast<uint16_t*>(work) + T * (int64_t)n_ffn;
  a.dx = dx;
  a.lddx = lddx;
  a.dwg = dw_gate;
  a.dwu = dw_up;
  a.T = T;
  a.H = n_in;
  a.F = n_ffn;
  AL_TRY(dense_status(dev, &a.status));
  if (!dx && !dw_gate) return ARTLITE_OK;
  int rc = dtype == ARTLITE_BF16 ? launch_gate_grad<__nv_bfloat16>(a, st) : launch_gate_grad<__half>(a, st);
  if (rc == ARTLITE_OK) rc = launch_ffn_backward_gemm(a, st);
  if (rc == ARTLITE_ECUDA) cudaGetLastError();
  return rc;
}

#pragma GCC visibility pop
}  // extern "C"
