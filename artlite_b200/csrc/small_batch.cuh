// The small-batch product: y (T x N) = x (T x K) . W^T for a few tokens, W streamed once from HBM straight into
// mma.sync fragments. With T <= 8 a token tile's 8 columns are the MMA's N, so every weight is read once for 8 tokens;
// the bound is the weight bytes.
//
// A CTA owns MT 16-row tiles (linear: 16 MT output rows; gated: tile 0 the gate rows and tile 1 the up rows of the same
// 16 features) and 8 NT tokens; its 8 warps split K chunk by chunk (a chunk is 256 values of 4-bit weights, 64 of
// 16-bit ones, 16 B a lane a load) and their partial sums meet in shared memory in a fixed order, so results do not
// depend on scheduling. A lane's weight loads are 16 consecutive bytes of the fragment it feeds to the MMA: no shared
// memory and no shuffles on the weights' way. The next chunk's weights are in flight while this one is multiplied.
// x is read from L1 / L2 in the same k order (eight consecutive values a lane and 32-value group). fp32 x is cut into three bf16 planes whose
// sum it is exactly (24 bits = 8 + 8 + 8), each multiplied into the same fp32 accumulator.
//
// 4-bit weights: the codes become exact small integers in bf16 / fp16 (128 + q or 1024 + q by one logic operation, the
// offset taken away exactly), their products with x are exact in fp32, a 32-value group's sum is multiplied by the
// group's fp32 scale; the minimum term of Q4_1 / Q4_K is the group's sum of x (an MMA with ones) times the minimum. No
// rounding but the fp32 sums' and the output's.
#pragma once

#include "dense.cuh"

namespace artlite {
namespace sb {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

struct Args {
  const void* w0;  // packed tiles (4-bit), or rows of K values (16-bit)
  const void* w1;  // gated: the up matrix
  const void* x;
  void* y;
  int64_t ldx, ldy;
  int64_t T;
  int K, N;
  int act;
  float scale0, scale1;  // 4-bit: powers of two that undo the packed scales' (first matrix, up matrix)
  float* keep_g;  // gated, 16-bit weights: the fp32 gate and up values (T x N), or null
  float* keep_u;
};

template <class XT>
struct MmaOf {
  using type = XT;
};
template <>
struct MmaOf<float> {
  using type = __nv_bfloat16;
};

template <class B>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(B) == 2 && __is_same(B, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- x

template <class XT>
constexpr int planes() { return sizeof(XT) == 4 ? 3 : 1; }

// values k0 .. k0 + 7 and k0 + 32 .. k0 + 39 of a row (zero at and past K, or for a missing row: row == null) as eight
// MMA pairs a plane
template <class XT, bool VEC>
__device__ __forceinline__ void load_x(const XT* row, int k0, int K, uint32_t (&r)[planes<XT>()][8]) {
  if constexpr (sizeof(XT) == 2) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row && k0 + 32 * j < K) v = __ldg(reinterpret_cast<const uint4*>(row + k0 + 32 * j));
        r[0][4 * j] = v.x, r[0][4 * j + 1] = v.y, r[0][4 * j + 2] = v.z, r[0][4 * j + 3] = v.w;
      }
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int k = k0 + 32 * (i >> 2) + 2 * (i & 3);
        uint32_t lo = 0, hi = 0;
        if (row && k < K) lo = p[k];
        if (row && k + 1 < K) hi = p[k + 1];
        r[0][i] = lo | hi << 16;
      }
    }
  } else {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int k = k0 + 32 * (i >> 3) + (i & 7);
      if constexpr (VEC) {
        float4 f = make_float4(0, 0, 0, 0);
        if (row && k < K) f = __ldg(reinterpret_cast<const float4*>(row + k));
        v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[i + e] = row && k + e < K ? row[k + e] : 0.0f;
      }
    }
    // v = hi + mid + lo, each the upper 16 bits of what is left: 8 significant bits a plane, all 24 kept
#pragma unroll
    for (int j = 0; j < 8; j++) {
      uint32_t a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
#pragma unroll
      for (int pl = 0; pl < 3; pl++) {
        r[pl][j] = __byte_perm(a, b, 0x7632);
        if (pl < 2) {
          a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xFFFF0000u));
          b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
        }
      }
    }
  }
}

// ---------------------------------------------------------------- the code table of IQ4_NL (dequant.cpp:119)

template <class B>
__device__ __forceinline__ uint32_t iq4_pair(int byte) {
  constexpr int8_t v[16] = {-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113};
  return Num<B>::pack((float)v[byte & 15], (float)v[byte >> 4]);
}

// ---------------------------------------------------------------- weight sources
//
// A source has: kChunkK (values a chunk), kGroups (whether sums are scaled by 32-value groups), Frag (a lane's registers
// of one tile's chunk), load(...), and mul(...) which multiplies the chunk into the accumulators.

template <int QT>
struct Quant {
  static constexpr int kChunkK = kTileK;
  static constexpr bool kTable = QT == ARTLITE_IQ4_NL;
  static constexpr bool kMin = QT == ARTLITE_Q4_1 || QT == ARTLITE_Q4_K;
  static constexpr int kRegs = QT == ARTLITE_Q4_1 ? 4 : 2;
  struct Frag {
    uint4 q[kUnits];
    uint32_t s[kRegs];
  };
  // tile `mt`'s chunk ch
  static __device__ __forceinline__ void load(const Args&, const void* w, int mt, int ch, int chunks, int lane, Frag& f) {
    const uint8_t* b = static_cast<const uint8_t*>(w) + ((int64_t)mt * chunks + ch) * tile_bytes(QT);
    const uint4* q = reinterpret_cast<const uint4*>(b) + lane;
#pragma unroll
    for (int u = 0; u < kUnits; u++) f.q[u] = __ldcs(q + 32 * u);
    if constexpr (kRegs == 4) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(b + kCodeBytes) + lane);
      f.s[0] = v.x, f.s[1] = v.y, f.s[2] = v.z, f.s[3] = v.w;
    } else {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(b + kCodeBytes) + lane);
      f.s[0] = v.x, f.s[1] = v.y;
    }
  }

  // a lane's own unit's scales (sc[row][group]) and minima, as fp32; undo: the power of two that undoes the packing's
  static __device__ __forceinline__ void own_scales(const Frag& f, int t, float undo, float (&sc)[4], float (&mn)[4]) {
    if constexpr (QT == ARTLITE_Q4_K) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        uint32_t dd = (f.s[r] >> 24) << (8 * t);  // (d | dmin << 16 from its four lanes' bytes)
        dd |= __shfl_xor_sync(0xFFFFFFFFu, dd, 1);
        dd |= __shfl_xor_sync(0xFFFFFFFFu, dd, 2);
        const float2 d = Num<__half>::unpack(dd);
        const float du = d.x * undo, dm = -d.y * undo;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          sc[2 * r + j] = du * (float)((f.s[r] >> (12 * j)) & 63u);
          mn[2 * r + j] = dm * (float)((f.s[r] >> (12 * j + 6)) & 63u);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const float2 d = Num<__half>::unpack(f.s[r]);
        sc[2 * r] = d.x * undo, sc[2 * r + 1] = d.y * undo;
        if constexpr (kMin) {
          const float2 m = Num<__half>::unpack(f.s[2 + r]);
          mn[2 * r] = m.x * undo, mn[2 * r + 1] = m.y * undo;
        }
      }
    }
  }

  // word w's four A registers: the codes as integers (Q4_0: less 8), or the table's values
  template <class B>
  static __device__ __forceinline__ void unpack(uint32_t w, const uint32_t* table, uint32_t (&a)[4]) {
    if constexpr (kTable) {
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = table[((w >> (8 * i)) & 0xFFu) * 32];
    } else {
      constexpr bool kHalf = __is_same(B, __half);
      constexpr uint32_t kBase = kHalf ? 0x64006400u : 0x43004300u;  // 1024 or 128
      constexpr int kOff = QT == ARTLITE_Q4_0 ? 8 : 0;
      const uint32_t off = kHalf ? 0x64006400u + 0x00010001u * kOff : 0x43004300u + 0x00010001u * kOff;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | kBase;
        if constexpr (kHalf) {
          const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&off));
          a[i] = *reinterpret_cast<const uint32_t*>(&d);
        } else {
          const __nv_bfloat162 d =
              __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
          a[i] = *reinterpret_cast<const uint32_t*>(&d);
        }
      }
    }
  }
};

// rows of K 16-bit values, ld K (K a multiple of 8, 16-byte aligned)
template <class WT>
struct Plain {
  static constexpr int kChunkK = 64;
  static constexpr bool kTable = false;
  struct Frag {
    uint4 v[4];  // row g's eight values of the two 32-value groups, then row g + 8's
  };
  static __device__ __forceinline__ void load(const Args& a, const void* w, int mt, int ch, int, int lane, Frag& f) {
    const int g = lane >> 2, k0 = 64 * ch + 8 * (lane & 3);
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const int64_t row = 16 * (int64_t)mt + g + 8 * r;
      const WT* p = static_cast<const WT*>(w) + row * a.K + k0;
#pragma unroll
      for (int j = 0; j < 2; j++)
        f.v[2 * r + j] = row < a.N && k0 + 32 * j < a.K ? __ldg(reinterpret_cast<const uint4*>(p + 32 * j))
                                                        : make_uint4(0, 0, 0, 0);
    }
  }
};

template <class S>
struct IsPlain {
  static constexpr bool value = false;
};
template <class WT>
struct IsPlain<Plain<WT>> {
  static constexpr bool value = true;
};

// ---------------------------------------------------------------- the kernel

template <int MT, int NT>
struct Shared {
  float red[kWarps][MT * 16][8 * NT + 1];
};
template <class S, int MT, int NT>
constexpr int smem_bytes() { return (int)sizeof(Shared<MT, NT>) + (S::kTable ? 256 * 32 * 4 : 0); }

template <class S, class XT, int MT, int NT, bool GATED, bool VEC>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) small_batch(const Args a) {
  using B = typename MmaOf<XT>::type;
  constexpr int P = planes<XT>();
  static_assert(!GATED || MT == 2, "a gated CTA holds one gate and one up tile");
  extern __shared__ __align__(16) uint8_t smem[];
  Shared<MT, NT>& sh = *reinterpret_cast<Shared<MT, NT>*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t tok0 = (int64_t)blockIdx.y * 8 * NT;
  const int chunks = (a.K + S::kChunkK - 1) / S::kChunkK;
  const uint32_t* table = nullptr;
  if constexpr (S::kTable) {  // a copy of the table for every lane: reads without bank conflicts
    uint32_t* tb = reinterpret_cast<uint32_t*>(smem + sizeof(Shared<MT, NT>));
    for (int i = threadIdx.x; i < 256 * 32; i += kThreads) tb[i] = iq4_pair<B>(i >> 5);
    table = tb + lane;
    __syncthreads();
  }
  const XT* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const int64_t tok = tok0 + 8 * n + g;
    xr[n] = tok < a.T ? static_cast<const XT*>(a.x) + tok * a.ldx : nullptr;
  }
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[m][n][i] = 0.0f;

  typename S::Frag cur[MT], nxt[MT];
  auto fetch = [&](int ch, typename S::Frag(&f)[MT]) {
#pragma unroll
    for (int m = 0; m < MT; m++)
      S::load(a, GATED && m == 1 ? a.w1 : a.w0, GATED ? (int)blockIdx.x : (int)blockIdx.x * MT + m, ch, chunks, lane, f[m]);
  };
  if (warp < chunks) fetch(warp, cur);
  for (int ch = warp; ch < chunks; ch += kWarps) {
    if (ch + kWarps < chunks) fetch(ch + kWarps, nxt);
    if constexpr (IsPlain<S>::value) {
      uint32_t x[NT][P][8];
#pragma unroll
      for (int n = 0; n < NT; n++) load_x<XT, VEC>(xr[n], 64 * ch + 8 * t, a.K, x[n]);
#pragma unroll
      for (int s = 0; s < 4; s++)
#pragma unroll
        for (int m = 0; m < MT; m++) {
          const uint4 lo = cur[m].v[s >> 1], hi = cur[m].v[2 + (s >> 1)];
          const uint32_t A[4] = {s & 1 ? lo.z : lo.x, s & 1 ? hi.z : hi.x, s & 1 ? lo.w : lo.y, s & 1 ? hi.w : hi.y};
#pragma unroll
          for (int n = 0; n < NT; n++) mma16816<B>(acc[m][n], A, x[n][0][2 * s], x[n][0][2 * s + 1]);
        }
    } else {
      float sc[MT][4], mn[MT][4];
#pragma unroll
      for (int m = 0; m < MT; m++) S::own_scales(cur[m], t, GATED && m == 1 ? a.scale1 : a.scale0, sc[m], mn[m]);
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        if (kTileK * ch + 64 * u >= a.K) break;  // (uniform)
        uint32_t x[NT][P][8];
#pragma unroll
        for (int n = 0; n < NT; n++) load_x<XT, VEC>(xr[n], kTileK * ch + 64 * u + 8 * t, a.K, x[n]);
        const int src = (lane & ~3) | u;  // the lane that holds this unit's scales of rows g and g + 8
#pragma unroll
        for (int j = 0; j < 2; j++) {  // the unit's two 32-value groups
          float xs[NT][4];             // (the group's sums of x, columns 2 t and 2 t + 1, in every row)
          if constexpr (S::kMin) {
            constexpr uint32_t kOne = __is_same(B, __half) ? 0x3C003C00u : 0x3F803F80u;
            const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
              for (int i = 0; i < 4; i++) xs[n][i] = 0.0f;
#pragma unroll
              for (int h = 0; h < 2; h++)
#pragma unroll
                for (int pl = 0; pl < P; pl++)
                  mma16816<B>(xs[n], ones, x[n][pl][4 * j + 2 * h], x[n][pl][4 * j + 2 * h + 1]);
            }
          }
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const uint4 q = cur[m].q[u];
            uint32_t A[2][4];
            S::template unpack<B>(j ? q.z : q.x, table, A[0]);
            S::template unpack<B>(j ? q.w : q.y, table, A[1]);
            const float s0 = __shfl_sync(0xFFFFFFFFu, sc[m][j], src), s1 = __shfl_sync(0xFFFFFFFFu, sc[m][2 + j], src);
            float m0 = 0.0f, m1 = 0.0f;
            if constexpr (S::kMin)
              m0 = __shfl_sync(0xFFFFFFFFu, mn[m][j], src), m1 = __shfl_sync(0xFFFFFFFFu, mn[m][2 + j], src);
#pragma unroll
            for (int n = 0; n < NT; n++) {
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int h = 0; h < 2; h++)
#pragma unroll
                for (int pl = 0; pl < P; pl++)
                  mma16816<B>(c, A[h], x[n][pl][4 * j + 2 * h], x[n][pl][4 * j + 2 * h + 1]);
#pragma unroll
              for (int i = 0; i < 4; i++) {
                acc[m][n][i] = fmaf(i < 2 ? s0 : s1, c[i], acc[m][n][i]);
                if constexpr (S::kMin) acc[m][n][i] = fmaf(i < 2 ? m0 : m1, xs[n][i], acc[m][n][i]);
              }
            }
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; m++) cur[m] = nxt[m];
  }
  // the warps' partial sums, added in warp order
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        sh.red[warp][16 * m + g + 8 * (i >> 1)][8 * n + 2 * t + (i & 1)] = acc[m][n][i];
  __syncthreads();
  constexpr int kRows = GATED ? 16 : 16 * MT;
  for (int o = threadIdx.x; o < kRows * 8 * NT; o += kThreads) {
    const int r = o % kRows, c = o / kRows;
    const int64_t row = (int64_t)blockIdx.x * kRows + r, tok = tok0 + c;
    if (row >= a.N || tok >= a.T) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) v += sh.red[w][r][c];
    if constexpr (GATED) {
      float u = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) u += sh.red[w][16 + r][c];
      if (IsPlain<S>::value && a.keep_g) {
        a.keep_g[tok * a.N + row] = v;
        a.keep_u[tok * a.N + row] = u;
      }
      v = act_of<sizeof(XT) == 4>(a.act, v) * u;
    }
    static_cast<XT*>(a.y)[tok * a.ldy + row] = Num<XT>::down(v);
  }
}

template <class S, class XT, int MT, int NT, bool GATED, bool VEC>
int launch_one(const Args& a, cudaStream_t st) {
  constexpr int smem = smem_bytes<S, MT, NT>();
  auto kern = small_batch<S, XT, MT, NT, GATED, VEC>;
  if (smem > 48 * 1024) AL_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int rows = GATED ? 16 : 16 * MT;
  // (the grid's y extent is 16 bits: longer batches go in several launches)
  const int64_t per = (int64_t)8 * NT * 32768;
  for (int64_t t0 = 0; t0 < a.T; t0 += per) {
    Args b = a;
    b.T = min64(per, a.T - t0);
    b.x = static_cast<const XT*>(a.x) + t0 * a.ldx;
    b.y = static_cast<XT*>(a.y) + t0 * a.ldy;
    if (a.keep_g) b.keep_g = a.keep_g + t0 * a.N, b.keep_u = a.keep_u + t0 * a.N;
    kern<<<dim3((unsigned)cdiv(a.N, rows), (unsigned)cdiv(b.T, 8 * NT)), kThreads, smem, st>>>(b);
    AL_LAUNCHED();
  }
  return ARTLITE_OK;
}

// the token tile: 8, 16 or 32 tokens a CTA
template <class S, class XT, bool GATED, bool VEC>
int launch(const Args& a, cudaStream_t st) {
  if (a.T <= 8) return launch_one<S, XT, 2, 1, GATED, VEC>(a, st);
  if (a.T <= 16) return launch_one<S, XT, 2, 2, GATED, VEC>(a, st);
  return launch_one<S, XT, 2, 4, GATED, VEC>(a, st);
}

}  // namespace sb
}  // namespace artlite
