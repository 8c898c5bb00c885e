// Linear layers in 8-bit floating point for many rows: a pair of SMs (tcgen05.mma.cta_group::2)
// multiplies a tile of 256 rows by 256 weight rows.  Each CTA loads 128 rows of either operand per
// block of 128 channels (32 KB; a single CTA's 128 x 256 tile would take 48 KB for the same work) and
// holds 128 rows x 256 columns of the block's sums in its tensor memory.
//
// Every block of 128 channels has scales of its own, so its sums cannot stay in tensor memory: eight
// epilogue warps drain them while the next block is multiplied into the other of two buffers, and add
// s_x s_w times them to fp32 registers (a lane is a row; the 128 columns of a warp share one weight
// scale), two columns per instruction.  The rows' scales of eight blocks come as one 128 x 8 box; results
// leave through shared memory as 128-byte rows of a bulk store, so that the warps are back at the next
// tile's blocks at once.
//
// About 1000 cycles a block, of which the tensor pipe works 512 and the additions issue for 256: neither is the
// limit, the epilogue warps' chain of waits and tensor-memory loads, one after the other, is.  16384 x 5120 -> 5120,
// codes to bf16: 376 us, 2.3 PFLOP/s.  What it took: cluster-scope release / acquire on the barriers between the
// two CTAs 1001 us, default scope 430 (nothing but tensor memory passes through them, which tcgen05's own
// fences order); scales through shared memory, bulk store 407; eight warps of 128 columns with 224
// registers, loads and additions overlapped 389, with the present ring and register split 376.  Not better: sixteen warps of 64 columns (407), four
// buffers of 128 columns (442), one CTA per 128 x 256 tile (410).
#include "fp8.cuh"

namespace modiff {

int read_device_status_fp8_pair(int* status, int reset) { return read_status_this_unit(status, reset); }

namespace {

constexpr int kTile = 256;                  // rows and weight rows of a pair's tile
constexpr int kHalfTile = 128 * kFp8Block;  // bytes one CTA loads of one operand per block
constexpr int kStageBytes = 2 * kHalfTile;
constexpr int kStages = 5;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;                // warps 0, 1: copies, MMAs; 2: scales; 3: none
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
constexpr int kWarpCols = 128;              // columns an epilogue warp owns
constexpr int kScaleBlocks = 8;             // channel blocks of one copy of scales
constexpr int kScaleBytes = 128 * kScaleBlocks * 4;
constexpr int kStaging = 32 * 128;          // bytes a warp stores at once: 32 rows of 128 bytes
// Registers: 168 a thread at launch; the four warps without accumulators hand theirs to the eight that
// have 128 of them.
constexpr int kRegsAtLaunch = 168, kRegsCopy = 56, kRegsEpi = 224;
static_assert(kRegsAtLaunch * kThreads >= 32 * (kFirstEpi * kRegsCopy + kEpiWarps * kRegsEpi), "register split");
constexpr int kSmem = kStages * kStageBytes + 2 * kScaleBytes + kEpiWarps * kStaging;
constexpr int kGroup = 8;                   // row tiles that neighbouring pairs share weights over

__device__ inline void tc_mma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                      uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ inline void tc_commit_pair(uint32_t bar) {
  const uint16_t mask = 3;
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar), "h"(mask)
      : "memory");
}
// copy into this CTA's shared memory whose bytes count on a barrier of the pair's leader
__device__ inline void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(leader_bar), "r"(c0), "r"(c1)
      : "memory");
}

// arrival on a barrier of the leader (or of this CTA); nothing in ordinary memory is handed over
__device__ inline void mbar_arrive_leader(uint32_t leader_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_bar) : "memory");
}
struct PairParams {
  Fp8Params p;
  int m_tiles, n_tiles, total;
  int store;                                // rows of y start and end on 16 bytes (bulk stores): 0; start on 4: 1; else 2
};

__device__ inline void tile_at(const PairParams& q, int tile, int& mt, int& nt) {
  const int group = tile / (kGroup * q.n_tiles);
  const int first = group * kGroup;
  const int height = min(kGroup, q.m_tiles - first);
  const int rem = tile - group * kGroup * q.n_tiles;
  mt = first + rem % height;
  nt = rem / height;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
fp8_linear_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_y,
                       const __grid_constant__ PairParams q) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kStages], bar_empty[kStages], bar_acc_full[2], bar_acc_empty[2];
  __shared__ __align__(8) uint64_t bar_sc_full[2], bar_sc_empty[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const Fp8Params& p = q.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_sh;
  const uint32_t ring = smem_u32(smem_raw);
  const uint32_t scales = ring + kStages * kStageBytes;
  const uint32_t rank = cluster_ctarank();
  const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);        // the leader's: bytes of both CTAs
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), 2 * kEpiWarps);   // the leader's: both CTAs' epilogue warps
      mbar_init(smem_u32(&bar_sc_full[b]), 1);
      mbar_init(smem_u32(&bar_sc_empty[b]), kEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();        // both CTAs' barriers and tensor memory exist before any signal
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;

  if (warp < kFirstEpi) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ------------------------------------------------------------ operand copies
      if (lane == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");       // the rows' codes
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair; tile < q.total && ok; tile += pairs) {
          int mt, nt;
          tile_at(q, tile, mt, nt);
          const int x0 = mt * kTile + (int)rank * 128, w0 = nt * kTile + (int)rank * 128;
          for (int kb = 0; kb < p.kb; ++kb) {
            ok = mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, abort_flag);
            if (!ok) break;
            const uint32_t full = map_to_cta(smem_u32(&bar_full[stage]), 0);
            if (rank == 0) mbar_arrive_expect_tx(smem_u32(&bar_full[stage]), 2 * kStageBytes);
            const uint32_t dst = ring + stage * kStageBytes;
            tma_load_2d_pair(dst, &map_x, full, kb * kFp8Block, x0);
            tma_load_2d_pair(dst + kHalfTile, &map_w, full, kb * kFp8Block, w0);
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMAs, issued by the leader
      if (rank == 0) {
        const uint32_t idesc = make_idesc_e4m3(256, 256);
        int stage = 0, buf = 0;
        uint32_t phase = 0, bphase = 0;
        bool ok = true;
        for (int tile = pair; tile < q.total && ok; tile += pairs) {
          for (int kb = 0; kb < p.kb; ++kb) {
            ok = mbar_wait(smem_u32(&bar_acc_empty[buf]), bphase ^ 1u, abort_flag) &&
                 mbar_wait(smem_u32(&bar_full[stage]), phase, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint64_t adesc = make_smem_desc(ring + stage * kStageBytes);
            const uint64_t bdesc = make_smem_desc(ring + stage * kStageBytes + kHalfTile);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kFp8Block / 32; ++k)
                tc_mma_f8_pair(tmem_base + (uint32_t)(buf * 256), adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k),
                               idesc, k > 0 ? 1u : 0u);
              tc_commit_pair(smem_u32(&bar_empty[stage]));
              tc_commit_pair(smem_u32(&bar_acc_full[buf]));
            }
            __syncwarp();
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
            if (++buf == 2) { buf = 0; bphase ^= 1u; }
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------ the rows' scales, eight blocks at a time
      if (lane == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int buf = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair; tile < q.total && ok; tile += pairs) {
          int mt, nt;
          tile_at(q, tile, mt, nt);
          for (int kb = 0; kb < p.kb; kb += kScaleBlocks) {
            ok = mbar_wait(smem_u32(&bar_sc_empty[buf]), phase ^ 1u, abort_flag);
            if (!ok) break;
            const uint32_t full = smem_u32(&bar_sc_full[buf]);
            mbar_arrive_expect_tx(full, kScaleBytes);
            tma_load_2d(scales + buf * kScaleBytes, &map_s, full, mt * kTile + (int)rank * 128, kb);
            if (++buf == 2) { buf = 0; phase ^= 1u; }
          }
        }
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ------------------------------------------------------------ scaling, sums, output
    const int quarter = warp & 3, cols = ((warp - kFirstEpi) >> 2) * kWarpCols;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)cols;
    const uint32_t empty0 = map_to_cta(smem_u32(&bar_acc_empty[0]), 0);
    const float* sc = reinterpret_cast<const float*>(smem_raw + kStages * kStageBytes) + quarter * 32 + lane;
    uint8_t* staging = smem_raw + kStages * kStageBytes + 2 * kScaleBytes + (warp - kFirstEpi) * kStaging;
    int buf = 0, sbuf = 0;
    uint32_t bphase = 0, sphase = 0;
    bool ok = true;
    for (int tile = pair; tile < q.total && ok; tile += pairs) {
      int mt, nt;
      tile_at(q, tile, mt, nt);
      const int m0 = mt * kTile + (int)rank * 128 + quarter * 32;
      const int n0 = nt * kTile + cols;
      const float* sw = p.sw + (int64_t)(min(n0, p.n - 1) / kFp8Block) * p.sw_pitch;
      uint64_t acc2[kWarpCols / 2];
#pragma unroll
      for (int j = 0; j < kWarpCols / 2; ++j) acc2[j] = 0ull;
      float w_next = lane < p.kb ? __ldg(sw + lane) : 0.0f, w_here = 0.0f;   // 32 blocks' weight scales, one a lane
      for (int kb = 0; kb < p.kb; ++kb) {
        if ((kb & 31) == 0) {
          w_here = w_next;
          w_next = kb + 32 + lane < p.kb ? __ldg(sw + kb + 32 + lane) : 0.0f;
        }
        const int si = kb % kScaleBlocks;
        if (si == 0) {
          ok = mbar_wait(smem_u32(&bar_sc_full[sbuf]), sphase, abort_flag);
          if (!ok) break;
        }
        const float s = sc[(sbuf * kScaleBlocks + si) * 128] * __shfl_sync(0xffffffffu, w_here, kb & 31);
        ok = mbar_wait(smem_u32(&bar_acc_full[buf]), bphase, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_acc = t_lane + (uint32_t)(buf * 256);
        uint64_t s2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
        int v[2][32];
        tc_ld32(t_acc, v[0]);
#pragma unroll
        for (int c = 0; c < kWarpCols / 32; ++c) {
          tc_wait_ld();
          if (c + 1 < kWarpCols / 32) {
            tc_ld32(t_acc + 32 * (c + 1), v[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(empty0 + 8 * buf);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) fma_pair(acc2[16 * c + j / 2], v[c & 1][j], v[c & 1][j + 1], s2);
        }
        if (++buf == 2) { buf = 0; bphase ^= 1u; }
        if (si == kScaleBlocks - 1 || kb == p.kb - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_sc_empty[sbuf]));
          if (++sbuf == 2) { sbuf = 0; sphase ^= 1u; }
        }
      }
      if (!ok) break;
      float acc[kWarpCols];
#pragma unroll
      for (int j = 0; j < kWarpCols / 2; ++j) asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * j]), "=f"(acc[2 * j + 1]) : "l"(acc2[j]));
      if (m0 >= p.rows || n0 >= p.n) continue;
      if (p.bias) {
        const T* bias = static_cast<const T*>(p.bias) + n0;
#pragma unroll
        for (int j = 0; j < kWarpCols; ++j)
          if (n0 + j < p.n) acc[j] += to_f32<T>(bias[j]);
      }
      constexpr int kPass = 128 / (int)sizeof(T);              // columns of one 128-byte row
      const bool bulk = q.store == 0;
#pragma unroll
      for (int c0 = 0; c0 < kWarpCols; c0 += kPass) {
        // the store that used this memory before has read it
        if (bulk && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {                          // 16-byte pieces, 128-byte swizzle
          Pack<T, 16 / sizeof(T)> w;
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T); ++e) w.v[e] = from_f32<T>(acc[c0 + i * (16 / (int)sizeof(T)) + e]);
          *reinterpret_cast<Pack<T, 16 / sizeof(T)>*>(staging + lane * 128 + ((i ^ (lane & 7)) << 4)) = w;
        }
        if (bulk) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (bulk) {
          if (lane == 0 && n0 + c0 < p.n) {
            tma_store_2d(&map_y, smem_u32(staging), n0 + c0, m0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          // rows that are not whole 16 bytes: a row at a time, neighbouring lanes next to each other, in words
          // of 4 bytes where rows start on them (2955 x 2665 -> 6177, fp16: 250 us with a row a lane, 73 so)
          const int here = min(32, p.rows - m0), cols_here = p.n - n0 - c0;
          T* y = static_cast<T*>(p.y) + (int64_t)m0 * p.y_pitch + n0 + c0;
          if (q.store == 1) {
            constexpr int kPer = 4 / (int)sizeof(T);
#pragma unroll 4
            for (int r = 0; r < here; ++r) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(staging + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3));
              const T* e = reinterpret_cast<const T*>(&w);
              if (kPer * lane + kPer <= cols_here) *reinterpret_cast<uint32_t*>(y + r * p.y_pitch + kPer * lane) = w;
              else if (kPer * lane < cols_here) y[r * p.y_pitch + kPer * lane] = e[0];
            }
          } else {
#pragma unroll 4
            for (int r = 0; r < here; ++r)
#pragma unroll
              for (int c = lane; c < kPass; c += 32) {
                const int at = c * (int)sizeof(T);
                const T v = *reinterpret_cast<const T*>(staging + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
                if (c < cols_here) y[r * p.y_pitch + c] = v;
              }
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // ---------------------------------------------------------------- teardown
  __syncwarp();
  if (abort_sh) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);            // let copies in flight land
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();        // the peer may still be read by / signalling this CTA
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

template <typename T>
int launch(const Fp8Operands& o, const Fp8Params& p, cudaStream_t s) {
  EncodeTiledFn encode = get_encode_fn();
  if (!encode) return set_error(MODIFF_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
  PairParams q;
  q.p = p;
  q.m_tiles = ceil_div(p.rows, kTile);
  q.n_tiles = ceil_div(p.n, kTile);
  MODIFF_CHECK_ARG((int64_t)q.m_tiles * q.n_tiles < 0x7fffffff / 2, "too many tiles");
  q.total = q.m_tiles * q.n_tiles;
  const uintptr_t starts = (uintptr_t)p.y | (uintptr_t)(p.y_pitch * (int64_t)sizeof(T));
  // a bulk store ends its rows on 16 bytes as well: what lies behind a shorter one would be zeroed
  const bool bulk = ((starts | (uintptr_t)p.n * sizeof(T)) & 15) == 0;
  q.store = bulk ? 0 : ((starts & 3) == 0 ? 1 : 2);
  CUtensorMap mx, mw, ms, my;
  CUresult r = fp8_map(encode, &mx, o.x, o.k, p.rows, o.x_pitch, 128);
  if (r == CUDA_SUCCESS) r = fp8_map(encode, &mw, o.w, o.k, p.n, o.w_pitch, 128);
  auto plain = [&](CUtensorMap* m, CUtensorMapDataType type, const void* base, int inner, int rows, int64_t pitch,
                   cuuint32_t box_inner, cuuint32_t box_rows, CUtensorMapSwizzle swizzle) {
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)pitch};
    cuuint32_t box[2] = {box_inner, box_rows}, estr[2] = {1, 1};
    return encode(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  if (r == CUDA_SUCCESS)
    r = plain(&ms, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, p.sx, p.rows, p.kb, 4 * p.sx_pitch, 128, kScaleBlocks,
              CU_TENSOR_MAP_SWIZZLE_NONE);
  constexpr CUtensorMapDataType kType = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  my = ms;
  if (r == CUDA_SUCCESS && q.store == 0)
    r = plain(&my, kType, p.y, p.n, p.rows, (int64_t)sizeof(T) * p.y_pitch, 128 / sizeof(T), 32,
              CU_TENSOR_MAP_SWIZZLE_128B);
  if (r != CUDA_SUCCESS) return set_error(MODIFF_ERR_CUDA, "cuTensorMapEncodeTiled(fp8 operands) failed: %d", (int)r);
  static SmemLimit limit;
  MODIFF_CUDA(raise_smem_limit(fp8_linear_pair_kernel<T>, kSmem, limit));
  // the split waits for registers: they have to be there from the launch on
  static const int regs = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, fp8_linear_pair_kernel<T>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kRegsAtLaunch) return set_error(MODIFF_ERR_UNSUPPORTED, "kernel built with %d registers", regs);
  const int pairs = device_sms() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (q.total < pairs ? q.total : pairs)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.x ? 2 : 1;
  MODIFF_CUDA(cudaLaunchKernelEx(&cfg, fp8_linear_pair_kernel<T>, mx, mw, ms, my, q));
  return MODIFF_OK;
}

}  // namespace

// Above 64 rows, once tiles of 128 x 128 fill more than half of the SMs: below that the other kernel splits the
// channels (us, this kernel : that one; 256 x 4096 x 4096 19.2 : 15.7, 1000 x 8192 x 1000 32.0 : 23.8), above it
// cannot as much (200 x 8192 x 8192 33.1 : 38.0, 4096 x 512 x 512 7.9 : 8.1).  Up to 64 rows that one's narrow tiles
// are faster whatever the weights' size is (64 x 5120 x 25600 41.7 : 28.3, 8 x 1024 x 40000 19.1 : 8.5).
bool fp8_pair_wanted(int rows, int n) {
  return rows > 64 && 2 * (int64_t)ceil_div(rows, 128) * ceil_div(n, 128) > device_sms();
}

int fp8_launch_pair(const Fp8Operands& o, const Fp8Params& p, int dtype, cudaStream_t s) {
  return with_dtype(dtype, [&](auto tag) { return launch<decltype(tag)>(o, p, s); });
}

}  // namespace modiff
