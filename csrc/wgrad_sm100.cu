// Weight gradients (sm_100a: tcgen05 + TMEM + TMA):  dW[n, k] = sum_l dY[l, n] * X[l, k].
//
// The sum runs over the rows of a batch, the long axis, while dW is often a few tiles: so the tiles of the last,
// partial wave are split over the rows.  CTA pairs (cta_group::2) own 256 x 256 tiles and walk the rows 64 at a time, both
// operands MN-major as they lie in memory; each CTA holds 128 columns of dY and 128 columns of X.  Warps of a CTA:
//   0      TMA producer, both CTAs' bytes count on the pair leader's `full`
//   1      MMA issuer (one lane of the leader), commits to `empty` of both CTAs
//   2..5   epilogue: TMEM -> registers -> swizzled staging -> TMA store, one accumulator while the other fills
// Whole tiles fill the GPU's 74 pairs wave by wave.  The tiles left over are cut into pieces of rows so that the pairs that
// would idle take part; the pieces' fp32 tiles go to scratch and a second kernel adds them in a fixed order (no atomics: the
// same bits every time).  A small dW of many rows is all last wave.  Bound: the tensor core for wide dW (4096 rows, 12288 x 4096: 285 us,
// 1.45 PFLOP/s, 94 % of the tensor pipe's cycles), the join and the ramp of short pieces for small ones (4096 x 4096: 120 us, 1.15).
//
// The kept activations reach this kernel as bf16 rows that restore8 wrote just before (their values are exact in
// bf16).  Decoding inside the kernel was built and measured: decoder warps turned codes into the swizzled operand tile, the
// codes coming by TMA or straight to registers.  Its best was 960 TFLOP/s where the dense form ran at 1420 (4096 rows, 12288 x 4096): the tile
// handover alone cost 15 %, and the decoders' shared-memory stores another 20 %, since the operands' writes and reads
// already fill the 128 bytes a cycle; the reload it saves takes 12 us of 300.
// Every wait is bounded (4 s): a kernel that gives up records an error code and unwinds.
#include "common.cuh"
#include "gemm_host.h"
#include "kept8.cuh"
#include "launchers.h"
#include "sm100.cuh"
#include "smem_opt_in.h"

namespace pan {
namespace wgrad {
using namespace sm100;

constexpr int TILE = 256;      // dW rows and columns of a pair's tile
constexpr int HALF = 128;      // ... of one CTA's operands
constexpr int STEP = 64;       // rows l of a stage
constexpr int STAGES = 6;
constexpr int A_STAGE = HALF * STEP * 2, B_STAGE = HALF * STEP * 2;
constexpr int EPI_SLOT = 4096, EPI_BYTES = 4 * 2 * EPI_SLOT;
constexpr int kThreads = 192;
constexpr int SMEM_BYTES = STAGES * (A_STAGE + B_STAGE) + EPI_BYTES + 1024 /*align*/ + 256 /*barriers*/;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");

struct Params {
  int n, k;                  // dW is [n, k]
  int n_tiles, k_tiles;
  int whole, split;          // whole tiles; pieces of each later tile
  int items;                 // whole + pieces
  int steps;                 // stages over all rows
  int d_fp32, add;           // add: dW += (fp32)
};

struct Maps {
  CUtensorMap dy, x, d, part;
};

struct Item {
  int nt, kt;       // tile
  int s0, s1;       // stages of the rows
  int piece;        // index of the partial tile, -1: a whole tile
};

// Tiles in bands of 8 columns with the dW row outer: tiles that run together share dY and X through L2.
__device__ __forceinline__ Item item_of(const Params& p, int w) {
  Item it;
  int tile = w;
  it.piece = -1;
  it.s0 = 0;
  it.s1 = p.steps;
  if (w >= p.whole && p.split > 1) {
    it.piece = w - p.whole;
    tile = p.whole + it.piece / p.split;
    const int q = it.piece % p.split;
    it.s0 = (int)((long long)p.steps * q / p.split);
    it.s1 = (int)((long long)p.steps * (q + 1) / p.split);
  }
  const int band = tile / (p.n_tiles * 8);
  const int width = min(8, p.k_tiles - band * 8);
  const int idx = tile - band * p.n_tiles * 8;
  it.nt = idx / width;
  it.kt = band * 8 + idx % width;
  return it;
}

__global__ void __launch_bounds__(kThreads, 1)
wgrad_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem_a + STAGES * A_STAGE;
  uint8_t* smem_epi = smem_b + STAGES * B_STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_epi + EPI_BYTES);
  // full[S], empty[S], tmem_full[2], tmem_empty[2]; then the TMEM base address and the abort flag
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int& s_abort = *reinterpret_cast<volatile int*>(bars + 2 * STAGES + 5);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int crank = (int)cluster_ctarank();
  const int item0 = (int)cluster_id_x(), item_step = (int)nclusters_x();
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + STAGES + s); };
  auto tfull_bar = [&](int a) { return smem_u32(bars + 2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return smem_u32(bars + 2 * STAGES + 2 + a); };

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 8);  // one arrival per epilogue warp of both CTAs
    }
    fence_barrier_init();
    prefetch_tmap(&maps.dy);
    prefetch_tmap(&maps.x);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist and its TMEM is allocated before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int w = item0; w < p.items && !s_abort; w += item_step) {
        const Item it = item_of(p, w);
        const int n0 = it.nt * TILE + crank * HALF, k0 = it.kt * TILE + crank * HALF;
        for (int st = it.s0; st < it.s1 && !s_abort; ++st) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, 61)) { s_abort = 1; break; }
          const uint32_t fb = mapa_shared(full_bar(stage), 0);
          if (crank == 0) mbar_expect_tx(full_bar(stage), 2 * (A_STAGE + B_STAGE));
          const uint32_t sa = smem_u32(smem_a + stage * A_STAGE), sb = smem_u32(smem_b + stage * B_STAGE);
          tma_load_3d_pair(sa, &maps.dy, fb, n0, st * STEP, 0);
          tma_load_3d_pair(sa + 8192, &maps.dy, fb, n0 + 64, st * STEP, 0);
          tma_load_3d_pair(sb, &maps.x, fb, k0, st * STEP, 0);
          tma_load_3d_pair(sb + 8192, &maps.x, fb, k0 + 64, st * STEP, 0);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (pair leader)
    if (lane == 0 && crank == 0) {
      const uint32_t idesc = idesc_bf16_f32(TILE, TILE, 1, 1);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int w = item0; w < p.items && !s_abort; w += item_step) {
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1, 62)) { s_abort = 1; break; }
        tc_fence_after();
        const Item it = item_of(p, w);
        const uint32_t d_tmem = tmem_base + acc * TILE;
        bool ok = true;
        for (int st = it.s0; st < it.s1; ++st) {
          if (!mbar_wait(full_bar(stage), phase, 63)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem_a + stage * A_STAGE), sb = smem_u32(smem_b + stage * B_STAGE);
#pragma unroll
          for (int kk = 0; kk < STEP / 16; ++kk)  // MN-major: next 64 columns 8 KB on, next 8 rows 1 KB on
            mma_bf16_ss_pair(d_tmem, smem_desc_sw128(sa + kk * 2048, 8192, 1024),
                             smem_desc_sw128(sb + kk * 2048, 8192, 1024), idesc, st != it.s0 || kk != 0);
          mma_commit_pair(empty_bar(stage), 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) { s_abort = 1; break; }
        mma_commit_pair(tfull_bar(acc), 0x3);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    uint8_t* slots = smem_epi + q * 2 * EPI_SLOT;
    int n_used = 0;
    auto acquire = [&]() -> uint8_t* {  // the store that last read the slot (two stores ago) must be done with it
      uint8_t* b = slots + (n_used & 1) * EPI_SLOT;
      if (n_used >= 2 && lane == 0) bulk_wait_read<1>();
      __syncwarp();
      ++n_used;
      return b;
    };
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int w = item0; w < p.items && !s_abort; w += item_step) {
      if (!mbar_wait(tfull_bar(acc), acc_phase, 64)) { s_abort = 1; break; }
      tc_fence_after();
      const Item it = item_of(p, w);
      const bool fp32 = it.piece >= 0 || p.d_fp32;
      const int row = crank * HALF + q * 32;
      const uint32_t t_row = tmem_base + acc * TILE + ((uint32_t)(q * 32) << 16);
      for (int ch = 0; ch < TILE / 32; ++ch) {
        uint32_t r[32];
        tmem_ld32(t_row + ch * 32, r);
        tmem_ld_wait();
        const int col = it.kt * TILE + ch * 32;
        if (it.nt * TILE + row >= p.n || col >= p.k) continue;  // also of a partial tile: never read
        uint8_t* b = acquire();
        if (fp32) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(b + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 o;
            uint32_t* ow = &o.x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ow[e] = pack_bf16(__uint_as_float(r[8 * j + 2 * e]), __uint_as_float(r[8 * j + 2 * e + 1]));
            *reinterpret_cast<uint4*>(b + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = o;
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          if (it.piece >= 0) tma_store_3d(&maps.part, smem_u32(b), ch * 32, it.piece * TILE + row, 0);
          else if (p.add) tma_reduce_add_3d(&maps.d, smem_u32(b), col, it.nt * TILE + row, 0);
          else tma_store_3d(&maps.d, smem_u32(b), col, it.nt * TILE + row, 0);
          bulk_commit();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(tempty_bar(acc), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's MMAs and arrivals target this CTA until both are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// dW of the split tiles: the pieces' fp32 tiles added in order, eight columns a thread.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p, const float* __restrict__ part,
                                                   T* __restrict__ d, long long ldd) {
  const int tile = blockIdx.x >> 5;
  const int e = ((blockIdx.x & 31) * 256 + threadIdx.x) * 8, r = e / TILE, c = e % TILE;
  const Item it = item_of(p, p.whole + tile * p.split);
  const int row = it.nt * TILE + r, col = it.kt * TILE + c;
  if (row >= p.n || col >= p.k) return;
  const float* src = part + ((long long)tile * p.split * TILE + r) * TILE + c;
  float v[8];
  load_v<float, 8>(src, v);
  for (int q = 1; q < p.split; ++q) {
    float u[8];
    load_v<float, 8>(src + (long long)q * TILE * TILE, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += u[i];
  }
  T* at = d + (long long)row * ldd + col;  // ldd holds k rounded up to 8
  if (p.add) {
    float u[8];
    load_v<T, 8>(at, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += u[i];
  }
  store_v<T, 8>(at, v);
}

}  // namespace wgrad

WgradPlan wgrad_plan(long long rows, int n, int k) {
  using namespace wgrad;
  WgradPlan pl;
  const int pairs = gemm::num_sms() / 2;
  const int tiles = ((n + TILE - 1) / TILE) * ((k + TILE - 1) / TILE);
  const int steps = (int)((rows + STEP - 1) / STEP);
  const int tail = tiles % pairs;
  // Pieces of at least 8 stages (512 rows), and only where the last wave gets at least 16 stages shorter: joining costs a
  // launch and a pass over the pieces, 4 us and more, a stage 0.3 us.  Measured, whole against split: 16384 rows, 1024 x 1024
  // (16 tiles, 4 pieces) 82 / 37 us; 32768 rows, 256 x 256 (1 tile, 64 pieces) 151 / 27, 24 with 32 pieces; 2048 rows, 1024 x
  // 1024 17.6 / 16.7; 256 rows 9.0 / 15.1 (not split).
  int split = tail > 0 ? pairs / tail : 1;
  if (split > steps / 8) split = steps / 8;
  if (split < 2 || steps - steps / split < 16) split = 1;
  pl.split = split;
  pl.whole = split > 1 ? tiles - tail : tiles;
  pl.pieces = split > 1 ? tail * split : 0;
  pl.part_floats = (long long)pl.pieces * TILE * TILE;
  return pl;
}

const char* launch_wgrad(const WgradPlan& pl, const void* dy, long long lddy, const void* x, long long ldx, long long rows,
                         int n, int k, void* d, long long ldd, bool d_fp32, bool add, float* part, cudaStream_t s) {
  using namespace wgrad;
  if (rows <= 0) return "wgrad: no rows";
  if (lddy % 8 != 0 || ldx % 8 != 0 || ldd % 8 != 0) return "wgrad: row strides must be multiples of 8 elements";
  if (add && !d_fp32) return "wgrad: only an fp32 result is added to";
  Params p{};
  p.n = n;
  p.k = k;
  p.n_tiles = (n + TILE - 1) / TILE;
  p.k_tiles = (k + TILE - 1) / TILE;
  p.whole = pl.whole;
  p.split = pl.split;
  p.items = pl.whole + pl.pieces;
  p.steps = (int)((rows + STEP - 1) / STEP);
  p.d_fp32 = d_fp32;
  p.add = add;
  Maps maps;
  const char* err = gemm::make_map(&maps.dy, dy, rows, n, lddy, STEP, 64, 1, 0, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                   CU_TENSOR_MAP_SWIZZLE_128B);
  if (err == nullptr)
    err = gemm::make_map(&maps.x, x, rows, k, ldx, STEP, 64, 1, 0, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                         CU_TENSOR_MAP_SWIZZLE_128B);
  if (err == nullptr) err = gemm::make_out_map(&maps.d, d, n, k, ldd, d_fp32, 1, 0);
  if (err == nullptr) {
    if (pl.pieces > 0) err = gemm::make_out_map(&maps.part, part, pl.pieces * TILE, TILE, TILE, true, 1, 0);
    else maps.part = maps.d;
  }
  if (err != nullptr) return err;
  static SmemOptIn opted;
  if (!allow_smem(opted, wgrad_kernel, SMEM_BYTES)) return "wgrad: cannot set the dynamic shared memory size";
  const int pairs = gemm::num_sms() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (p.items < pairs ? p.items : pairs), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, wgrad_kernel, p, maps) != cudaSuccess) return "wgrad: launch failed";
  if (pl.pieces > 0) {
    const int grid = pl.pieces / pl.split * 32;
    if (d_fp32) join_kernel<float><<<grid, 256, 0, s>>>(p, part, (float*)d, ldd);
    else join_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p, part, (__nv_bfloat16*)d, ldd);
  }
  return cudaGetLastError() == cudaSuccess ? nullptr : "wgrad: launch failed";
}

int wgrad_error_flag(bool reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, sm100::g_error_flag, sizeof(int));
  if (reset) {
    int z = 0;
    cudaMemcpyToSymbol(sm100::g_error_flag, &z, sizeof(int));
  }
  return v;
}

}  // namespace pan
