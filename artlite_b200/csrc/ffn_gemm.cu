// The gated feed-forward's products on the 5th-generation tensor cores, for a model's own 16-bit matrices (no packing:
// they change every training step):
//   forward  h = act(x Wg^T) (x Wu^T): both products, the activation and the product in one kernel. A tile's 256
//            columns are 128 gate rows (CTA 0's half of B) and the 128 up rows (CTA 1's half) of the same 128 features.
//   dx       dx = dg Wg + du Wu: one accumulator over both reductions, 2 F values deep. A is K-major (dg rows), B
//            MN-major: the matrices as they lie (rows of H values), no transposed copy.
//   dw       dWg = dg^T x, dWu = du^T x: the reduction is over tokens, so both operands are MN-major as they lie.
// The transposes are the UMMA descriptors': a TMA box of 64 values x 64 k rows lands with its values consecutive, and
// the instruction descriptor's major bits say so. Tiles past an edge read the tensor map's zeros.
//
// Warps (192 threads): 0 TMA, 1 the MMAs (the leader CTA's), 2 - 5 the epilogue, whose results leave by TMA stores. Three
// stages of 64 KB a CTA.
#include <cuda.h>
#include <cuda_runtime.h>

#include "dense_gemm.cuh"
#include "ffn.cuh"

namespace artlite {
namespace {

using namespace dg;

enum { kForward = 0, kDx = 1, kDw = 2 };
constexpr int kEpilogue = 4, kThreads = 64 + 32 * kEpilogue;
constexpr int S = 3, KS = 2 * BK, kStage = 2 * kStageBytes;  // stages, of 128 values of the reduction
constexpr int NS = 2;                                                    // output slots a warp
constexpr int slot_bytes(bool keep) { return keep ? kSlot : kSlot / 2; }  // (fp32 chunks; 16-bit ones)

struct Params {
  CUtensorMap a[2], b[2];  // forward: x; Wg, Wu. dx: dg, du; Wg, Wu. dw: dg, du; x
  CUtensorMap out[2];      // forward: h. dx: dx. dw: dWg, dWu
  CUtensorMap g, u;        // forward: the kept values
  int rows, cols;          // of the output
  int ksteps;              // stages a reduction (dx: of one of its two)
  int act;
  TileOrder order;
  DevStatus* status;
};

struct Smem {
  uint64_t full[S], empty[S], tfull[2], tempty[2];
  uint32_t tmem_base;
  int abort;
};
template <bool KEEP>
constexpr size_t smem_bytes() {
  return 1024 + 2 * (size_t)S * kStage + kEpilogue * NS * (size_t)slot_bytes(KEEP) + sizeof(Smem) + 64;
}

template <int MODE, class T, bool KEEP>
__global__ void __launch_bounds__(kThreads, 1) ffn_gemm(const __grid_constant__ Params p) {
  constexpr int SLOT = slot_bytes(KEEP);
  constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
  constexpr bool kAmn = MODE == kDw, kBmn = MODE != kForward;
  constexpr int kMats = MODE == kDw ? 2 : 1, kSegs = MODE == kDx ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = base;
  uint8_t* sB = sA + S * kStage;
  uint8_t* sOut = sB + S * kStage;
  Smem* sm = reinterpret_cast<Smem*>(sOut + kEpilogue * NS * SLOT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = tc::cluster_rank();
  const int per = p.order.tm * p.order.tn, total = per * kMats, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  griddep_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; i++) {
      tc::mbar_init(&sm->full[i], 1);
      tc::mbar_init(&sm->empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&sm->tfull[i], 1);
      tc::mbar_init(&sm->tempty[i], 2 * kEpilogue);
    }
    sm->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc_pair(&sm->tmem_base);
  tc::fence_before();
  tc::cluster_sync();
  tc::fence_after();
  const uint32_t tmem = sm->tmem_base;
  griddep_wait();

  if (warp == 0 && lane == 0) {
    // ---------------- TMA: this CTA's halves of A and B
    int s = 0, ph = 0;
    for (int id = pair; id < total; id += pairs) {
      int m, n;
      const int mat = id / per;
      tile_at(p.order, id - mat * per, &m, &n);
      const int row = m * TILE + HALF * (int)crank;
      for (int ks = 0; ks < kSegs * p.ksteps; ks++) {
        if (!tc::wait(&sm->abort, &sm->empty[s], ph ^ 1, p.status, 60)) goto out;
        if (crank == 0)
          tc::mbar_expect_tx(&sm->full[s], 4 * kStage);
        const uint32_t bar = tc::peer_addr(&sm->full[s], 0);
        const int seg = kSegs == 2 && ks >= p.ksteps ? 1 : 0;
        for (int h = 0; h < 2; h++) {
          const int k = (ks - seg * p.ksteps) * KS + h * BK;
          uint8_t *da = sA + s * kStage + h * kStageBytes, *db = sB + s * kStage + h * kStageBytes;
          if constexpr (MODE == kForward) {
            tc::tma_load_2d_pair(da, &p.a[0], bar, k, row);
            tc::tma_load_2d_pair(db, &p.b[crank], bar, k, n * HALF);
          } else {
            const int col = n * TILE + HALF * (int)crank;
            if constexpr (MODE == kDx) {
              tc::tma_load_2d_pair(da, &p.a[seg], bar, k, row);
            } else {
              tc::tma_load_2d_pair(da, &p.a[mat], bar, row, k);
              tc::tma_load_2d_pair(da + kStageBytes / 2, &p.a[mat], bar, row + 64, k);
            }
            tc::tma_load_2d_pair(db, &p.b[seg], bar, col, k);
            tc::tma_load_2d_pair(db + kStageBytes / 2, &p.b[seg], bar, col + 64, k);
          }
        }
        if (++s == S) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 1 && lane == 0 && crank == 0) {
    // ---------------- the MMAs
    int s = 0, ph = 0, acc = 0, aph = 0;
    const uint32_t id_mma = tc::idesc_of(kBf16, kAmn, kBmn, TILE, TILE);
    // a K step of 16: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
    constexpr uint64_t kStepA = kAmn ? 2048 >> 4 : 32 >> 4, kStepB = kBmn ? 2048 >> 4 : 32 >> 4;
    for (int id = pair; id < total; id += pairs) {
      if (!tc::wait_cluster(&sm->abort, &sm->tempty[acc], aph ^ 1, p.status, 61)) goto out;
      tc::fence_after();
      const uint32_t d = tmem + acc * TILE;
      for (int ks = 0; ks < kSegs * p.ksteps; ks++) {
        if (!tc::wait_cluster(&sm->abort, &sm->full[s], ph, p.status, 62)) goto out;
        tc::fence_after();
        const uint32_t aa = tc::smem_u32(sA + s * kStage), ab = tc::smem_u32(sB + s * kStage);
        const uint64_t da = kAmn ? tc::sdesc_mn(aa, kStageBytes / 2) : tc::sdesc(aa);
        const uint64_t db = kBmn ? tc::sdesc_mn(ab, kStageBytes / 2) : tc::sdesc(ab);
#pragma unroll
        for (int k = 0; k < KS / 16; k++) {
          const uint64_t box = (k / 4) * (kStageBytes >> 4);
          tc::mma_pair(d, da + box + (k % 4) * kStepA, db + box + (k % 4) * kStepB, id_mma, (ks | k) != 0);
        }
        tc::commit_pair(&sm->empty[s]);
        if (++s == S) s = 0, ph ^= 1;
      }
      tc::commit_pair(&sm->tfull[acc]);
      if (++acc == 2) acc = 0, aph ^= 1;
    }
  } else if (warp >= 2) {
    // ---------------- the epilogue: TMEM lanes 32 q .. + 31, an output row each
    const int q = warp & 3;
    int acc = 0, aph = 0, slot = 0;
    uint8_t* mine = sOut + (warp - 2) * NS * SLOT;
    const uint32_t tempty0 = tc::peer_addr(&sm->tempty[0], 0);
    for (int id = pair; id < total; id += pairs) {
      int m, n;
      const int mat = id / per;
      tile_at(p.order, id - mat * per, &m, &n);
      if (!tc::wait(&sm->abort, &sm->tfull[acc], aph, p.status, 63)) goto out;
      tc::fence_after();
      const uint32_t col0 = tmem + ((uint32_t)(32 * q) << 16) + acc * TILE;
      const int row = m * TILE + HALF * (int)crank + 32 * q;
      constexpr int cols = MODE == kForward ? HALF : TILE;
      for (int c = 0; c < cols; c += 32) {
        const int f = n * cols + c;
        if (f >= p.cols || row >= p.rows) break;  // (uniform: nothing of the box is inside)
        uint32_t v[32];
        float o[32];
        tc::tmem_ld32(col0 + c, v);
        if constexpr (MODE == kForward) {
          uint32_t w[32];
          tc::tmem_ld32(col0 + HALF + c, w);
          tc::tmem_wait32(v);
          tc::tmem_wait32(w);
          if constexpr (KEEP) {
            store_wait<NS - 1>(lane);
            store_chunk<float>(mine + slot * SLOT, &p.g, f, row, reinterpret_cast<const float(&)[32]>(v), lane);
            slot = (slot + 1) & (NS - 1);
            store_wait<NS - 1>(lane);
            store_chunk<float>(mine + slot * SLOT, &p.u, f, row, reinterpret_cast<const float(&)[32]>(w), lane);
            slot = (slot + 1) & (NS - 1);
          }
#pragma unroll
          for (int j = 0; j < 32; j++)
            o[j] = act_of<false>(p.act, __uint_as_float(v[j])) * __uint_as_float(w[j]);
        } else {
          tc::tmem_wait32(v);
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = __uint_as_float(v[j]);
        }
        store_wait<NS - 1>(lane);
        store_chunk<T>(mine + slot * SLOT, &p.out[mat], f, row, o, lane);
        slot = (slot + 1) & (NS - 1);
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        if (crank != 0) tc::arrive_cluster(tempty0 + acc * (uint32_t)sizeof(uint64_t));
        else tc::mbar_arrive(&sm->tempty[acc]);
      }
      if (++acc == 2) acc = 0, aph ^= 1;
    }
    store_finish(lane);
  }
out:
  __syncwarp();
  __syncthreads();
  if (*(volatile int*)&sm->abort && threadIdx.x == 0) {  // let issued copies and MMAs land before TMEM is freed
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000LL) {
    }
  }
  tc::cluster_sync();  // (the leader's MMAs read the peer's shared memory until here)
  if (warp == 0) {
    tc::fence_after();
    tmem_free_pair(tmem);
  }
}

template <int MODE, bool KEEP = false>
int go(const Params& p, int dtype, int mats, int pairs, cudaStream_t st) {
  const int64_t total = (int64_t)p.order.tm * p.order.tn * mats;
  AL_CHECK(total < (1ll << 31), ARTLITE_EUNSUPPORTED, "gated_ffn: %lld tiles", (long long)total);
  const int n = total < pairs ? (int)total : pairs;
  return dtype == ARTLITE_BF16 ? launch_pairs(ffn_gemm<MODE, __nv_bfloat16, KEEP>, p, n, kThreads, smem_bytes<KEEP>(), st)
                               : launch_pairs(ffn_gemm<MODE, __half, KEEP>, p, n, kThreads, smem_bytes<KEEP>(), st);
}

int card_pairs(int* out) {
  int dev, sms;
  AL_CUDA(cudaGetDevice(&dev));
  AL_TRY(sm_count(dev, &sms));
  *out = sms / 2;
  return ARTLITE_OK;
}

}  // namespace

int launch_ffn_forward_gemm(const FfnArgs& a, cudaStream_t st) {
  Params p{};
  int pairs;
  AL_TRY(card_pairs(&pairs));
  p.ksteps = (int)cdiv(a.H, KS);
  AL_TRY(make_operand_map(&p.a[0], a.x, a.H, a.T, a.ldx, BK, HALF));
  AL_TRY(make_operand_map(&p.b[0], a.wg, a.H, a.F, a.H, BK, HALF));
  AL_TRY(make_operand_map(&p.b[1], a.wu, a.H, a.F, a.H, BK, HALF));
  AL_TRY(make_operand_map(&p.out[0], a.h, a.F, a.T, a.ldh, 32, 32));
  if (a.g) {
    AL_TRY(make_tile_map(&p.g, a.g, true, a.F, a.T, a.F, 32, 32));
    AL_TRY(make_tile_map(&p.u, a.u, true, a.F, a.T, a.F, 32, 32));
  }
  p.rows = (int)a.T;
  p.cols = a.F;
  p.act = a.act;
  p.order = {(int)cdiv(a.T, TILE), (int)cdiv(a.F, HALF)};
  p.status = a.status;
  return a.g ? go<kForward, true>(p, a.dtype, 1, pairs, st) : go<kForward>(p, a.dtype, 1, pairs, st);
}

int launch_ffn_dx_gemm(const FfnArgs& a, cudaStream_t st) {
  Params p{};
  int pairs;
  AL_TRY(card_pairs(&pairs));
  p.ksteps = (int)cdiv(a.F, KS);
  AL_TRY(make_operand_map(&p.a[0], a.dg, a.F, a.T, a.F, BK, HALF));
  AL_TRY(make_operand_map(&p.a[1], a.du, a.F, a.T, a.F, BK, HALF));
  AL_TRY(make_operand_map(&p.b[0], a.wg, a.H, a.F, a.H, 64, BK));
  AL_TRY(make_operand_map(&p.b[1], a.wu, a.H, a.F, a.H, 64, BK));
  AL_TRY(make_operand_map(&p.out[0], a.dx, a.H, a.T, a.lddx, 32, 32));
  p.rows = (int)a.T;
  p.cols = a.H;
  p.order = {(int)cdiv(a.T, TILE), (int)cdiv(a.H, TILE)};
  p.status = a.status;
  return go<kDx>(p, a.dtype, 1, pairs, st);
}

int launch_ffn_dw_gemm(const FfnArgs& a, cudaStream_t st) {
  Params p{};
  int pairs;
  AL_TRY(card_pairs(&pairs));
  p.ksteps = (int)cdiv(a.T, KS);
  AL_TRY(make_operand_map(&p.a[0], a.dg, a.F, a.T, a.F, 64, BK));
  AL_TRY(make_operand_map(&p.a[1], a.du, a.F, a.T, a.F, 64, BK));
  AL_TRY(make_operand_map(&p.b[0], a.x, a.H, a.T, a.ldx, 64, BK));
  AL_TRY(make_operand_map(&p.out[0], a.dwg, a.H, a.F, a.H, 32, 32));
  AL_TRY(make_operand_map(&p.out[1], a.dwu, a.H, a.F, a.H, 32, 32));
  p.rows = a.F;
  p.cols = a.H;
  p.order = {(int)cdiv(a.F, TILE), (int)cdiv(a.H, TILE)};
  p.status = a.status;
  return go<kDw>(p, a.dtype, 2, pairs, st);
}

}  // namespace artlite
