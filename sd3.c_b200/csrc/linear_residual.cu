// out = act(x w^T + bias) + add for the sizes that the CTA-pair GEMM does not cover or would leave most SMs idle with:
// few rows, odd widths, outputs whose rows no TMA store can write.
//
//   acc[m, n] = sum_k x[m, k] w[n, k],   out = act(acc + bias[n]) + add[m, n]
//
// For few rows the weights are all there is to read (one row, K 1536, N 6144: 18.9 MB, 2.9 us at the copy rate), so the
// kernel is built to have every SM read its share of them at once: a tile is 128 rows by BN columns, and a cluster of up to
// eight CTAs shares its K.  Each CTA runs an ordinary TMA ring and tcgen05.mma over its K blocks (a lone tile of rows
// loads only the rows there are) and leaves the accumulator in the shared memory of the CTAs of its cluster: CTA r gets
// the columns r of the cluster's split of the tile from everyone.  It adds the partial sums in the CTAs' order (the same
// bits every time), applies bias, activation and residual and writes its columns, neighbouring threads neighbouring
// columns: coalesced whatever the row pitch, element by element where rows are not aligned.
#include <cuda.h>

#include <mutex>

#include "gemm_epilogue.cuh"
#include "kernels.h"
#include "launch_rules.h"
#include "ptx.cuh"

namespace sd3 {

int encode_tmap_2d(CUtensorMap* map, const void* base, int elem_bytes, uint64_t inner, uint64_t outer, uint64_t ld_bytes,
                   uint32_t box_inner, uint32_t box_outer);
int device_sm_count();
bool gemm_pair_supported(int operand_dtype, int M, int N, int K, const GemmEpilogue& epi);
int launch_gemm_pair(const GemmProblem* q, int n, int operand_dtype, int N, int K, int* dev_status, cudaStream_t stream);

namespace {

using namespace gemm_detail;

constexpr int LR_BM = 128;
constexpr int LR_KBYTES = 128;  // bytes of K per stage row: 64 bf16
constexpr int LR_MAX_STAGES = 12;
constexpr int LR_MAX_SPLIT = 8;
constexpr int LR_THREADS = 64 + 32 * EPI_WARPS;
constexpr int LR_SMEM = 227 * 1024;

struct LinearArgs {
  int M, N, k_blocks, tiles_m, tiles_n;
  int split;        // CTAs of a cluster, each with its share of the K blocks
  int cols;         // columns that a CTA of the cluster finishes, a multiple of 4
  int a_rows;       // rows of x that a stage loads
  int stages, stage_bytes;
  int vec_store;    // groups of four columns of out and add are aligned
  GemmEpilogue epi;
  int* status;
};

// room for the partial sums of `cols` columns from `split` CTAs; rows 4 floats longer than the columns need, so that the
// 16-byte writes of eight consecutive rows fall into different banks
__host__ __device__ inline int partial_bytes(int split, int cols) { return split * LR_BM * (cols + 4) * 4; }

template <bool OUT_F32>
__device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, const float4& acc) {
  const GemmEpilogue& e = a.epi;
  float v[4] = {acc.x, acc.y, acc.z, acc.w};
  const bool whole = a.vec_store != 0 && n + 4 <= a.N;
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < a.N) v[j] += e.bias[n + j];
  }
  activate_chunk(v, e.act);
  const long at = static_cast<long>(m) * e.ldo + n, from = static_cast<long>(m) * e.ld_add + n;
  if constexpr (OUT_F32) {
    float* out = static_cast<float*>(e.out) + at;
    const float* add = static_cast<const float*>(e.add) + from;
    if (whole) {
      if (e.add) {
        const float4 r = *reinterpret_cast<const float4*>(add);
        v[0] += r.x; v[1] += r.y; v[2] += r.z; v[3] += r.w;
      }
      *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) out[j] = e.add ? v[j] + add[j] : v[j];
    }
  } else {
    bf16* out = static_cast<bf16*>(e.out) + at;
    const bf16* add = static_cast<const bf16*>(e.add) + from;
    if (whole) {
      if (e.add) {
        const uint2 r = *reinterpret_cast<const uint2*>(add);
        v[0] += __uint_as_float(r.x << 16);
        v[1] += __uint_as_float(r.x & 0xffff0000u);
        v[2] += __uint_as_float(r.y << 16);
        v[3] += __uint_as_float(r.y & 0xffff0000u);
      }
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) out[j] = __float2bfloat16_rn(e.add ? v[j] + __bfloat162float(add[j]) : v[j]);
    }
  }
}

template <int BN, bool OUT_F32>
__global__ void __launch_bounds__(LR_THREADS, 1)
linear_residual_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ LinearArgs a) {
  constexpr uint32_t IDESC = make_idesc(1, 1, LR_BM, BN, 0, 0);
  constexpr int W_BYTES = BN * LR_KBYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // a stage: the W tile, then the rows of x (an MMA reads 128 of them: what lies behind the loaded ones gives accumulator
  // rows that nobody stores; the last stage is followed by the partial sums, which are at least 16 KiB)
  float* partial = reinterpret_cast<float*>(smem + a.stages * a.stage_bytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + a.stages * a.stage_bytes + partial_bytes(a.split, a.cols));
  uint64_t* empty_bar = full_bar + LR_MAX_STAGES;
  uint64_t* tfull_bar = empty_bar + LR_MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull_bar + 1);
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // known uniform
  const int lane = threadIdx.x & 31;
  const int rank = a.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = blockIdx.x / a.split;
  const int m0 = (tile / a.tiles_n) * LR_BM, n0 = (tile % a.tiles_n) * BN;
  const int kb0 = static_cast<int>(static_cast<long>(a.k_blocks) * rank / a.split);
  const int KB = static_cast<int>(static_cast<long>(a.k_blocks) * (rank + 1) / a.split) - kb0;  // at least one

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tfull_bar, 1);
    *s_abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, BN);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_dep_wait();
  grid_dep_launch();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const WaitCtx wc{s_abort, a.status};
  if (a.split > 1) cluster_sync_all();  // every CTA of the cluster runs before its shared memory is written to

  if (warp == 0) {
    // ------------------------------ TMA producer (a converged warp, one lane issues) ------
    const bool issuer = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = 0; kb < KB; ++kb) {
      if (!mbar_wait_all(&empty_bar[stage], phase ^ 1, wc, DEV_TIMEOUT_EMPTY)) break;
      if (issuer) {
        uint8_t* st = smem + stage * a.stage_bytes;
        mbar_expect_tx(&full_bar[stage], W_BYTES + a.a_rows * LR_KBYTES);
        tma_load_2d(st, &tmW, &full_bar[stage], (kb0 + kb) * (LR_KBYTES / 2), n0);
        tma_load_2d(st + W_BYTES, &tmA, &full_bar[stage], (kb0 + kb) * (LR_KBYTES / 2), m0);
      }
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (a converged warp, one lane issues) ------
    const bool issuer = elect_one();
    const uint64_t desc0 = make_smem_desc_sw128(smem_u32(smem), 16, 1024);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = 0; kb < KB; ++kb) {
      if (!mbar_wait_all(&full_bar[stage], phase, wc, DEV_TIMEOUT_FULL)) break;
      tc_fence_after_sync();
      if (issuer) {
        const uint64_t w_desc = desc0 + static_cast<uint32_t>(stage * (a.stage_bytes >> 4));
        const uint64_t a_desc = w_desc + (W_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < LR_KBYTES / 32; ++k)
          mma_f16_ss(tmem_base, a_desc + 2 * k, w_desc + 2 * k, IDESC, (kb | k) != 0);
        mma_commit(&empty_bar[stage]);
        if (kb == KB - 1) mma_commit(tfull_bar);
      }
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
    }
  } else {
    // ------------------------------ accumulator -> partial sums of the cluster's CTAs ------
    // warp w may read TMEM lanes [32 (w % 4), +32); warps 2-5 take the first half of the columns, warps 6-9 the second
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row = quad * 32 + lane;
    // bring this CTA's columns of add into L2 while the products run
    if (a.epi.add) {
      const int threads = 32 * EPI_WARPS, t = threadIdx.x - 64, esz = OUT_F32 ? 4 : 2;
      const int m = m0 + t % LR_BM;
      if (m < a.M)
        for (int c = (t / LR_BM) * 32; c < a.cols; c += threads / LR_BM * 32) {
          const int n = n0 + rank * a.cols + c;
          if (n < a.N && rank * a.cols + c < BN)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.epi.add) +
                                                           (static_cast<long>(m) * a.epi.ld_add + n) * esz));
        }
    }
    if (m0 + quad * 32 < a.M && mbar_wait_warp(tfull_bar, 0, wc, DEV_TIMEOUT_TMEM_FULL)) {
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
      const bool live = m0 + row < a.M;
#pragma unroll 1
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c, r);
        tmem_wait_ld();
        if (live) {
          int owner = c / a.cols, col = c - owner * a.cols;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float* dst = partial + (rank * LR_BM + row) * (a.cols + 4) + col;
            if (a.split > 1)
              st_cluster_v4(map_to_cta(smem_u32(dst), owner), __uint_as_float(r[j]), __uint_as_float(r[j + 1]),
                            __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
            else
              *reinterpret_cast<float4*>(dst) = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]),
                                                            __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
            col += 4;
            if (col == a.cols) { col = 0; ++owner; }
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncwarp();
  if (a.split > 1) cluster_sync_all();  // the partial sums are complete; no CTA is written to after this
  else __syncthreads();
  if (*s_abort) drain_after_abort();
  // ------------------------------ sum, bias, activation, residual, store: all threads ------
  const int rows = min(LR_BM, a.M - m0);
  const int quads = max(0, min(a.cols, BN - rank * a.cols)) / 4;
  const int pitch = (a.cols + 4) / 4;
  const float4* p4 = reinterpret_cast<const float4*>(partial);
  for (int i = threadIdx.x; i < rows * quads; i += LR_THREADS) {
    const int r = i / quads, q = i - r * quads;
    const int n = n0 + rank * a.cols + 4 * q;
    if (n >= a.N) continue;
    float4 v = p4[r * pitch + q];
    for (int s = 1; s < a.split; ++s) {
      const float4 u = p4[(s * LR_BM + r) * pitch + q];
      v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    finish4<OUT_F32>(a, m0 + r, n, v);
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, BN);
  }
}

template <int BN, bool OUT_F32>
int launch_inst(const CUtensorMap& tmA, const CUtensorMap& tmW, const LinearArgs& a, int smem, cudaStream_t stream) {
  auto kern = linear_residual_kernel<BN, OUT_F32>;
  static std::mutex attr_mutex;
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64) {
    std::lock_guard<std::mutex> lock(attr_mutex);
    if (!attr_done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, LR_SMEM);
      if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(linear_residual)");
      attr_done[dev] = true;
    }
  }
  launch_dependent_cluster(kern, static_cast<unsigned>(a.tiles_m) * a.tiles_n * a.split, a.split, LR_THREADS, smem, stream,
                           tmA, tmW, a);
  return after_launch("linear_residual_kernel");
}

}  // namespace

int launch_linear_residual(const bf16* x, long lda, const bf16* w, long ldw, int M, int N, int K, const GemmEpilogue& epi,
                           int* dev_status, cudaStream_t stream) {
  const long esz = epi.out_f32 ? 4 : 2;
  const bool tma_out = (epi.ldo * esz) % 16 == 0 && (reinterpret_cast<uintptr_t>(epi.out) & 15) == 0 &&
                       (!epi.add || ((epi.ld_add * esz) % 16 == 0 && (reinterpret_cast<uintptr_t>(epi.add) & 15) == 0));
  const int sms = device_sm_count();
  const int k_blocks = (K + 63) / 64;
  const LinearPlan plan = linear_plan(M, N, k_blocks, tma_out, sms);
  if (plan.pair) {
    GemmProblem q;
    q.A = x; q.lda = lda; q.W = w; q.ldw = ldw; q.M = M; q.epi = epi;
    return launch_gemm_pair(&q, 1, OPERAND_BF16, N, K, dev_status, stream);
  }
  LinearArgs a;
  a.M = M; a.N = N;
  a.k_blocks = k_blocks;
  a.tiles_m = (M + LR_BM - 1) / LR_BM;
  a.tiles_n = (N + plan.bn - 1) / plan.bn;
  a.split = plan.split;
  a.cols = (plan.bn / 4 + a.split - 1) / a.split * 4;
  a.a_rows = M < LR_BM ? (M + 7) / 8 * 8 : LR_BM;
  a.stage_bytes = (plan.bn + a.a_rows) * LR_KBYTES;
  const int bars = (2 * LR_MAX_STAGES + 1) * 8 + 8;
  const int room = LR_SMEM - 1024 - bars - partial_bytes(a.split, a.cols);
  a.stages = room / a.stage_bytes;
  if (a.stages > LR_MAX_STAGES) a.stages = LR_MAX_STAGES;
  const int most = (k_blocks + a.split - 1) / a.split;
  if (a.stages > most) a.stages = most;
  a.vec_store = (epi.ldo * esz) % (4 * esz) == 0 && (reinterpret_cast<uintptr_t>(epi.out) % (4 * esz)) == 0 &&
                (!epi.add || ((epi.ld_add * esz) % (4 * esz) == 0 && (reinterpret_cast<uintptr_t>(epi.add) % (4 * esz)) == 0));
  a.epi = epi;
  a.status = dev_status;
  CUtensorMap tmA, tmW;
  int rc = encode_tmap_2d(&tmA, x, 2, (uint64_t)K, (uint64_t)M, (uint64_t)lda * 2, 64, a.a_rows);
  if (rc) return rc;
  rc = encode_tmap_2d(&tmW, w, 2, (uint64_t)K, (uint64_t)N, (uint64_t)ldw * 2, 64, plan.bn);
  if (rc) return rc;
  const int smem = 1024 + a.stages * a.stage_bytes + partial_bytes(a.split, a.cols) + bars;
  if (plan.bn == 64)
    return epi.out_f32 ? launch_inst<64, true>(tmA, tmW, a, smem, stream) : launch_inst<64, false>(tmA, tmW, a, smem, stream);
  return epi.out_f32 ? launch_inst<128, true>(tmA, tmW, a, smem, stream) : launch_inst<128, false>(tmA, tmW, a, smem, stream);
}

}  // namespace sd3
