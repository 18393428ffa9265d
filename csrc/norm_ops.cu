// Layer norm and RMS norm with learned weight and bias, forward and backward (sm_100a).
//
//   n = (x - mean) * rstd,  y = n * w + b                (RMS norm: mean = 0, no b)
//   g = dy * w,  dx = rstd * (g - mean_c(g) - n * mean_c(g n))      (RMS norm without mean_c(g))
//   dw = sum_rows dy * n,  db = sum_rows dy
//
// Statistics are fp32 and two-pass (mean first, then the centred squares), so a large common offset
// does not cancel the variance away.  The backward reads x either as it was or from its 8-bit codes
// (kept8.cuh); mean and rstd are always those of the exact x.
//
// Both directions are DRAM-bound, so every tensor is read and written once.  A group of G threads owns the
// columns of a row for all the rows that its CTA walks: weight, bias and the growing dw / db stay in
// registers, and one partial row of dw / db per CTA goes to scratch, which a second kernel adds up in order (no
// atomics: the same bits every time).  Four forms:
//   staged   (C % 8 == 0, 16-byte aligned rows, C <= 16384)  8-column fragments through rings in shared memory
//   flat     (contiguous rows of other widths)               batches of rows as runs of bytes (flat.cuh): groups, or warps (long rows);
//                                                            backward to 8192 columns, forward while two stages fit (14065 fp32, 18753 bf16)
//   single   (other views, C <= 8192)                        one column at a time, straight from memory
//   wide     (wider rows)                                    CTA per row, the row swept from memory: 6000 x 16001 backward 0.1 (bf16,
//                                                            kept) to 0.26 (fp32) of the copy rate
// Groups of up to a warp reduce by shuffles, larger ones through shared memory.
#include "flat.cuh"
#include "kept8.cuh"
#include "launchers.h"
#include "smem_opt_in.h"

namespace pan {
namespace {

constexpr int kThreads = 256;
constexpr int threads_of(int G) { return G > kThreads ? G : kThreads; }

struct Kept {
  int8_t* codes;
  uint8_t* scales;
  int Cp, nb, nbp;
};

struct Vectors {  // learned weight and bias, bf16 or fp32, either may be missing
  const void* w;
  const void* b;
  bool fp32;
};

template <int V>
__device__ __forceinline__ void load_vec(const void* p, bool fp32, int c, float missing, float (&v)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = missing;
  } else if (fp32) {
    load_v<float, V>(reinterpret_cast<const float*>(p) + c, v);
  } else {
    load_v<__nv_bfloat16, V>(reinterpret_cast<const __nv_bfloat16*>(p) + c, v);
  }
}

__device__ __forceinline__ float vec_at(const void* p, bool fp32, int c, float missing) {
  float v[1];
  load_vec<1>(p, fp32, c, missing, v);
  return v[0];
}

// Eight columns from c on, `missing` past the row's end.
__device__ __forceinline__ void load_pairs(const void* p, bool fp32, int c, int C, float missing, float2 (&v)[4]) {
  float f[8];
  load_vec<8>(c < C ? p : nullptr, fp32, c, missing, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
}

template <typename W>
__device__ __forceinline__ void store_out(void* out, int c, float v) {
  if (out != nullptr) reinterpret_cast<W*>(out)[c] = from_f32<W>(v);
}

// ---------------------------------------------------------------- reductions
// Sums of N values over each group of G threads; every thread of the group gets them.  `ws`, 16-byte aligned, holds
// N floats a warp; calls that may overlap use different ones.  Inside a warp two values share each
// exchange while there are two: a lane keeps one of a pair and hands over the other, so N values cost
// N - 1 + log2(G) - log2(N) exchanges in place of N log2(G).
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* ws) {
  constexpr int L = G < 32 ? G : 32;
  constexpr bool kPair = N == 2 && L >= 2;
  const int lane = threadIdx.x & 31;
  if constexpr (kPair) {
    const bool odd = lane & 1;
    float mine = odd ? v[1] : v[0];
    mine += __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
#pragma unroll
    for (int o = L / 2; o > 1; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if constexpr (G <= 32) {
      const float other = __shfl_xor_sync(0xffffffffu, mine, 1);
      v[0] = odd ? other : mine;
      v[1] = odd ? mine : other;
    } else {
      v[0] = mine;  // even lanes: the first sum, odd lanes: the second
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if constexpr (G > 32) {
    constexpr int W = G / 32;  // warps of a group: their sums lie together, value by value
    const int warp = threadIdx.x >> 5;
    float* g = ws + warp / W * W * N;
    if constexpr (kPair) {
      if (lane < 2) g[lane * W + warp % W] = v[0];
    } else if (lane == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) g[k * W + warp % W] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
      if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const float4 q = *reinterpret_cast<const float4*>(g + k * W + i);
          v[k] += (q.x + q.y) + (q.z + q.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[k] += g[k * W + i];
      }
    }
  }
}

// ---------------------------------------------------------------- staged form
// Each thread copies its own fragments DEPTH - 1 row batches ahead with asynchronous copies and waits
// for its own copies only, so loads stay in flight across the reductions without holding registers and
// without barriers between copying and using.  Slots of columns past the row's end are zeroed once.
// L1: through the first-level cache, which copies of under 16 bytes take anyway.
template <int BYTES, bool L1 = BYTES != 16>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (!L1) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One ring of fragments: SLOTS of every thread a stage, Q 16-byte pieces a fragment (bf16 1, fp32 2).  The two halves of a 32-byte
// sector of fp32 are two copies, so those go through L1: past it each sector crossed from L2 twice (layer norm of 24414 x 2048,
// forward 99 and 69 us, backward 173 and 135).
template <typename T, int NT, int SLOTS>
struct Ring {
  static constexpr int Q = sizeof(T) / 2, PIECE = NT * 16, STAGE = SLOTS * Q * PIECE;
  __device__ __forceinline__ static void fetch(uint32_t stage, int slot, const T* p) {
#pragma unroll
    for (int h = 0; h < Q; ++h)
      copy_async<16, Q == 2>(stage + (slot * Q + h) * PIECE + threadIdx.x * 16, reinterpret_cast<const uint4*>(p) + h);
  }
  __device__ __forceinline__ static void get(const uint8_t* stage, int slot, Frag<T>& f) {
    const uint8_t* at = stage + slot * Q * PIECE + threadIdx.x * 16;
    if constexpr (Q == 1) {
      f.raw = *reinterpret_cast<const uint4*>(at);
    } else {
      f.raw[0] = *reinterpret_cast<const float4*>(at);
      f.raw[1] = *reinterpret_cast<const float4*>(at + PIECE);
    }
  }
};
// The same for codes: 8 bytes a fragment, then the 4-byte word of scales that holds its block's.
template <int NT, int SLOTS>
struct CodeRing {
  static constexpr int STAGE = SLOTS * NT * 12, SCALES = SLOTS * NT * 8;
  __device__ __forceinline__ static void fetch(uint32_t stage, int slot, const int8_t* codes, const uint8_t* scales, int c) {
    copy_async<8>(stage + (slot * NT + threadIdx.x) * 8, codes + c);
    copy_async<4>(stage + SCALES + (slot * NT + threadIdx.x) * 4, scales + c / kKeptBlock / 4 * 4);
  }
  // the codes as numbers, and their step
  __device__ __forceinline__ static float get(const uint8_t* stage, int slot, int c, float2 (&v)[4]) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(stage + SCALES + (slot * NT + threadIdx.x) * 4);
    const uint32_t b = (word >> (c / kKeptBlock % 4 * 8)) & 0xffu;  // 0 in a slot past the row's end, where codes are 0
    kept8_numbers(*reinterpret_cast<const uint2*>(stage + (slot * NT + threadIdx.x) * 8), v);
    return kept8_step(b);
  }
};

__device__ __forceinline__ void zero_ring(uint8_t* ring, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
}

// R rows a group a turn.  x is read once: into the ring, from there into registers, which the mean, the centred squares, the
// codes and y all use.  Bound by DRAM: layer norm of 94960 x 4096 bf16 255 us (6.1 TB/s), kept 366 us (5.3 TB/s: the codes'
// arithmetic shares the issue slots); 16384 x 32 x 128 RMS 52 us (5.2 TB/s).
template <typename T, int G, int UPT, int R, int DEPTH, int CTAS, bool LAYER>
__global__ void __launch_bounds__(threads_of(G), CTAS)
    norm_fwd_staged_kernel(RowView x, uint32_t rows, int C, Vectors vec, float eps, T* __restrict__ y,
                           float* __restrict__ stats, Kept k) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  using X = Ring<T, NT, R * UPT>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float ws[2][2][NT / 32 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  const uint64_t step = (uint64_t)gridDim.x * (GROUPS * R);
  const uint32_t first = blockIdx.x * (GROUPS * R);
  if (C < G * UPT * 8) zero_ring(ring, DEPTH * X::STAGE);

  auto fetch = [&](uint64_t r0, int stage) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      if (r >= rows) continue;
      const T* p = row_ptr<T>(x, (uint32_t)r);
#pragma unroll
      for (int i = 0; i < UPT; ++i)
        if ((t + i * G) * 8 < C) X::fetch(ring0 + stage * X::STAGE, q * UPT + i, p + (t + i * G) * 8);
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    fetch(first + d * step, d);
    copy_commit();
  }
  float2 w[UPT][4], b[LAYER ? UPT : 1][4];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    load_pairs(vec.w, vec.fp32, (t + i * G) * 8, C, 1.f, w[i]);
    if (LAYER) load_pairs(vec.b, vec.fp32, (t + i * G) * 8, C, 0.f, b[i]);
  }
  const float inv_c = 1.f / C;
  int stage = 0, flip = 0;
  for (uint64_t r0 = first; r0 < rows; r0 += step) {
    fetch(r0 + (DEPTH - 1) * step, stage == 0 ? DEPTH - 1 : stage - 1);  // into the stage of the last turn
    copy_commit();
    copy_wait<DEPTH - 1>();
    Frag<T> f[R][UPT];
    float mean[R], var[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      float2 s = twice(0.f);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        X::get(ring + stage * X::STAGE, q * UPT + i, f[q][i]);
        if (LAYER) {
          float2 v[4];
          f[q][i].get(v);
          s = add2(s, add2(add2(v[0], v[1]), add2(v[2], v[3])));
        }
      }
      mean[q] = s.x + s.y;
    }
    if (LAYER) group_sum<G, R>(mean, ws[flip][0]);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = LAYER ? mean[q] * inv_c : 0.f;
      float2 s = twice(0.f);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        if ((t + i * G) * 8 >= C) continue;
        float2 v[4];
        f[q][i].get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (LAYER) v[j] = add2(v[j], twice(-mean[q]));
          s = fma2(v[j], v[j], s);
        }
      }
      var[q] = s.x + s.y;
    }
    group_sum<G, R>(var, ws[flip][1]);
    flip ^= 1;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      const bool in = r < rows;
      const float rstd = rsqrtf(var[q] * inv_c + eps);
      if (in && t == 0 && stats != nullptr) *reinterpret_cast<float2*>(stats + 2 * r) = make_float2(mean[q], rstd);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * 8;
        if (k.codes != nullptr) {  // all lanes: a block is four of them, zeros past the row's end
          uint32_t sb;
          uint2 codes;
          kept8_encode(f[q][i], sb, codes);
          if (in && c < k.Cp) {
            *reinterpret_cast<uint2*>(k.codes + (long long)r * k.Cp + c) = codes;
            if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, sb);
          }
        }
        if (!in || c >= C) continue;
        float2 v[4];
        f[q][i].get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (LAYER) v[j] = fma2(mul2(add2(v[j], twice(-mean[q])), twice(rstd)), w[i][j], b[LAYER ? i : 0][j]);
          else v[j] = mul2(mul2(v[j], twice(rstd)), w[i][j]);
        }
        store_pairs(y + (long long)r * C + c, v);
      }
    }
    stage = stage == DEPTH - 1 ? 0 : stage + 1;
  }
  copy_wait<0>();
}

// The CTA's groups hold the same columns: add them up, in a fixed order, into the first group.  P values a thread.
template <int G, int GROUPS, int P>
__device__ __forceinline__ void join_groups(float (&acc)[P], int t, int group) {
  if constexpr (GROUPS > 1) {
    __shared__ float cs[GROUPS / 2 * G * 4];
#pragma unroll
    for (int i = 0; i < P; i += 4) {
#pragma unroll
      for (int h = GROUPS / 2; h > 0; h >>= 1) {
        __syncthreads();
        if (group >= h && group < 2 * h) {
#pragma unroll
          for (int j = 0; j < 4; ++j) cs[((group - h) * 4 + j) * G + t] = acc[i + j];
        }
        __syncthreads();
        if (group < h) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i + j] += cs[(group * 4 + j) * G + t];
        }
      }
    }
  }
}

// Column c of the CTA's partial row; a lone CTA's is the result.
__device__ __forceinline__ void store_partial(float v, int c, int C, int which, bool fp32, float* part, void* out) {
  if (gridDim.x > 1) part[((long long)blockIdx.x * 2 + which) * C + c] = v;
  else if (fp32) store_out<float>(out, c, v);
  else store_out<__nv_bfloat16>(out, c, v);
}

// One row a group a turn.  Between the sums and dx a thread holds its g' and x - mean as fp32 (UPT = 2: 32
// registers); with more columns, where dw and db take the registers, it reads the ring a second time.  Bound by DRAM: layer
// norm of 94960 x 4096 bf16 390 us (6.0 TB/s), from the codes 389 us (5.0 TB/s; decoding shares the issue slots; three
// CTAs an SM that hold nothing took 144 us for 24414 rows against 119).
template <typename T, int G, int UPT, int DEPTH, int CTAS, bool LAYER, bool KEPT>
__global__ void __launch_bounds__(threads_of(G), CTAS)
    norm_bwd_staged_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C, Vectors vec,
                           const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw,
                           void* db) {
  constexpr int NT = threads_of(G), GROUPS = NT / G, N = LAYER ? 2 : 1;
  using D = Ring<T, NT, UPT>;
  using X = Ring<T, NT, UPT>;
  using XK = CodeRing<NT, UPT>;
  constexpr int STAGE = D::STAGE + (KEPT ? XK::STAGE : X::STAGE);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float ws[2][NT / 32 * N];
  constexpr bool HOLD = UPT <= 2;
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  const uint64_t step = (uint64_t)gridDim.x * (GROUPS);
  const uint32_t first = blockIdx.x * (GROUPS);
  if (C < G * UPT * 8) zero_ring(ring, DEPTH * STAGE);

  auto fetch = [&](uint64_t r0, int stage) {
    const uint64_t r = r0 + group;
    if (r >= rows) return;
    const uint32_t at = ring0 + stage * STAGE;
    const T* gr = row_ptr<T>(dy, (uint32_t)r);
    const T* xr = KEPT ? nullptr : row_ptr<T>(x, (uint32_t)r);
    const int8_t* codes = KEPT ? k.codes + (long long)r * k.Cp : nullptr;
    const uint8_t* scales = KEPT ? k.scales + (long long)r * k.nbp : nullptr;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int c = (t + i * G) * 8;
      if (c >= C) continue;
      D::fetch(at, i, gr + c);
      if constexpr (KEPT) XK::fetch(at + D::STAGE, i, codes, scales, c);
      else X::fetch(at + D::STAGE, i, xr + c);
    }
  };
  // dy, and v with (x - mean) = v * unit: a layer norm subtracts the mean here (unit 1), an RMS norm leaves codes as they
  // are and passes their step on
  auto get = [&](int stage, int slot, int c, float mean, float2 (&g)[4], float2 (&v)[4]) -> float {
    const uint8_t* at = ring + stage * STAGE;
    Frag<T> f;
    D::get(at, slot, f);
    f.get(g);
    float unit = 1.f;
    if constexpr (KEPT) {
      unit = XK::get(at + D::STAGE, slot, c, v);
    } else {
      X::get(at + D::STAGE, slot, f);
      f.get(v);
    }
    if constexpr (LAYER) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = KEPT ? fma2(v[j], twice(unit), twice(-mean)) : add2(v[j], twice(-mean));
      unit = 1.f;
    }
    return unit;
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    fetch(first + d * step, d);
    copy_commit();
  }
  float2 w[UPT][4], aw[UPT][4], ab[LAYER ? UPT : 1][4];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    load_pairs(vec.w, vec.fp32, (t + i * G) * 8, C, 1.f, w[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      aw[i][j] = twice(0.f);
      if (LAYER) ab[i][j] = twice(0.f);
    }
  }
  const float inv_c = 1.f / C;
  auto stats_of = [&](uint64_t r0) {
    const uint64_t r = r0 + group;
    return r < rows ? *reinterpret_cast<const float2*>(stats + 2 * r) : make_float2(0.f, 0.f);
  };
  float2 next = stats_of(first);
  int stage = 0, flip = 0;
  for (uint64_t r0 = first; r0 < rows; r0 += step) {
    const float2 st = next;
    fetch(r0 + (DEPTH - 1) * step, stage == 0 ? DEPTH - 1 : stage - 1);  // into the stage of the last turn
    copy_commit();
    next = stats_of(r0 + step);
    copy_wait<DEPTH - 1>();
    // with d = x - mean and g' = dy w rstd:  s = (sum g' d, sum g'),  dw += dy rstd d,  db += dy
    float2 gw[HOLD ? UPT : 1][4], v[HOLD ? UPT : 1][4];
    float unit[HOLD ? UPT : 1];
    const uint64_t r = r0 + group;
    const bool in = r < rows;  // a slot without a row holds another row's values
    float2 sn = twice(0.f), sg = twice(0.f);
    if (in) {
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int h = HOLD ? i : 0;
        float2 g[4];
        unit[h] = get(stage, i, (t + i * G) * 8, st.x, g, v[h]);
        float2 part_n = twice(0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 gr = mul2(g[j], twice(st.y));
          gw[h][j] = mul2(gr, w[i][j]);
          if constexpr (LAYER || !KEPT) {
            sn = fma2(gw[h][j], v[h][j], sn);
            aw[i][j] = fma2(gr, v[h][j], aw[i][j]);
          } else {
            part_n = fma2(gw[h][j], v[h][j], part_n);
            aw[i][j] = fma2(mul2(gr, twice(unit[h])), v[h][j], aw[i][j]);
          }
          if (LAYER) {
            sg = add2(sg, gw[h][j]);
            ab[i][j] = add2(ab[i][j], g[j]);
          }
        }
        if constexpr (!LAYER && KEPT) sn = fma2(part_n, twice(unit[h]), sn);
      }
    }
    if (dx != nullptr) {
      float s[N];
      s[0] = sn.x + sn.y;
      if (LAYER) s[N - 1] = sg.x + sg.y;
      group_sum<G, N>(s, ws[flip]);
      flip ^= 1;
      if (in) {
        // dx = g' - mean_c(g') - d rstd^2 mean_c(g' d)
        const float2 a = twice(LAYER ? -s[N - 1] * inv_c : 0.f);
        const float b = -s[0] * inv_c * st.y * st.y;
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
          const int h = HOLD ? i : 0, c = (t + i * G) * 8;
          if (c >= C) continue;
          if constexpr (!HOLD) {
            float2 g[4];
            unit[h] = get(stage, i, c, st.x, g, v[h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) gw[h][j] = mul2(mul2(g[j], twice(st.y)), w[i][j]);
          }
          float2 o[4];
          const float2 bu = twice(b * unit[h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = fma2(v[h][j], bu, LAYER ? add2(gw[h][j], a) : gw[h][j]);
          store_pairs(dx + (long long)r * C + c, o);
        }
      }
    }
    stage = stage == DEPTH - 1 ? 0 : stage + 1;
  }
  copy_wait<0>();
  if (part == nullptr) return;
#pragma unroll
  for (int which = 0; which < N; ++which) {
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      float acc[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = which == 0 ? aw[i][j] : ab[LAYER ? i : 0][j];
        acc[2 * j] = v.x;
        acc[2 * j + 1] = v.y;
      }
      join_groups<G, GROUPS>(acc, t, group);
      const int c = (t + i * G) * 8;
      if (group != 0 || c >= C) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) store_partial(acc[j], c + j, C, which, vec.fp32, part, which == 0 ? dw : db);
    }
  }
}

// ---------------------------------------------------------------- flat form
// A batch is GROUPS * R neighbouring rows, one run of bytes; the next two arrive while one is worked on (with one, the kernel
// waited for memory at 35 % of its bandwidth).  Fragment i of thread t are the 4 columns from 4 (t + i G) on: eight lanes
// hold a block of the codes.  Results take the place of the input and leave as one run.  What bounds it is instruction
// issue: single elements are read, converted and masked (50 instructions an element in the kept forward of width 631), so
// bf16 groups are sized for few idle lanes: 100 M elements, layer norm, kept forward / kept backward, two fragments of
// twice the threads and then three a thread: width 333 269 / 250 and 210 / 182 us, 631 268 / 272 and 215 / 192, 77 291 / 249
// and 213 / 191.  Packed fp32 pairs cost more in moves than they save here (631: 226 / 217), and so does a branch for
// whole fragments (230 / 225).
constexpr int group_ctas(int G) { return G > kThreads ? 1 : 2; }
constexpr int kGroupDepth = 3;

template <typename T, int G, int UPT, int R>
struct FlatBatch {
  static constexpr int NT = threads_of(G), GROUPS = NT / G, ROWS = GROUPS * R, WIDTH = G * UPT * 4;
  static constexpr uint32_t ROOM = FlatRun<T>::room(ROWS * WIDTH);
  static constexpr uint32_t CODES = FlatRun<int8_t>::room(ROWS * WIDTH);
  static constexpr uint32_t SCALES = FlatRun<uint8_t>::room(ROWS * ((WIDTH / kKeptBlock + 3) / 4 * 4));
};

// `n` of the four elements from p on, zeros for the others.
template <typename T>
__device__ __forceinline__ void read4(const T* p, int n, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = j < n ? to_f32(p[j]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void write4(T* p, int n, const float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) p[j] = from_f32<T>(v[j]);
}

template <typename T, int G, int UPT, int R>
__global__ void __launch_bounds__(threads_of(G), group_ctas(G))
    norm_fwd_flat_kernel(const T* x, uint32_t rows, int C, Vectors vec, float eps, bool layer, T* __restrict__ y,
                         float* __restrict__ stats, Kept k) {
  using B = FlatBatch<T, G, UPT, R>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float ws[2][2][B::NT / 32 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  auto run_of = [&](const T* p, uint64_t r0) {
    return FlatRun<T>(p, (long long)r0 * C, (uint32_t)min((uint64_t)B::ROWS, rows - r0) * C);
  };
  const uint64_t step = (uint64_t)gridDim.x * B::ROWS;
  uint64_t r0 = (uint64_t)blockIdx.x * B::ROWS;
  constexpr int DEPTH = kGroupDepth;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    if (r0 + d * step < rows) run_of(x, r0 + d * step).fetch(ring + d * B::ROOM);
    copy_commit();
  }
  float w[UPT][4], b[UPT][4];
  int n[UPT];  // columns of the fragment inside the row
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int c = (t + i * G) * 4;
    n[i] = max(0, min(4, C - c));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[i][j] = j < n[i] ? vec_at(vec.w, vec.fp32, c + j, 1.f) : 0.f;
      b[i][j] = j < n[i] ? vec_at(vec.b, vec.fp32, c + j, 0.f) : 0.f;
    }
  }
  const float inv_c = 1.f / C;
  int stage = 0, flip = 0;
  for (; r0 < rows; r0 += step, stage = stage == DEPTH - 1 ? 0 : stage + 1, flip ^= 1) {
    const uint64_t ahead = r0 + (DEPTH - 1) * step;
    if (ahead < rows) run_of(x, ahead).fetch(ring + (stage == 0 ? DEPTH - 1 : stage - 1) * B::ROOM);
    copy_commit();
    copy_wait<DEPTH - 1>();
    __syncthreads();
    T* tile = reinterpret_cast<T*>(ring + stage * B::ROOM + run_of(x, r0).head);
    float v[R][UPT][4], mean[R], var[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int row = q * B::GROUPS + group;
      const bool in = r0 + row < rows;
      mean[q] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        read4(tile + row * C + (t + i * G) * 4, in ? n[i] : 0, v[q][i]);
        mean[q] += (v[q][i][0] + v[q][i][1]) + (v[q][i][2] + v[q][i][3]);
      }
    }
    if (layer) group_sum<G, R>(mean, ws[flip][0]);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = layer ? mean[q] * inv_c : 0.f;
      var[q] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float d = j < n[i] ? v[q][i][j] - mean[q] : 0.f;
          var[q] = fmaf(d, d, var[q]);
        }
    }
    group_sum<G, R>(var, ws[flip][1]);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int row = q * B::GROUPS + group;
      const uint64_t r = r0 + row;
      const bool in = r < rows;
      const float rstd = rsqrtf(var[q] * inv_c + eps);
      if (in && t == 0 && stats != nullptr) *reinterpret_cast<float2*>(stats + 2 * r) = make_float2(mean[q], rstd);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * 4;
        if (k.codes != nullptr) {  // all lanes
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[q][i][j]) & 0x7fffffffu);
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const uint32_t sb = kept8_byte(m);
          if (in && c < k.Cp) {
            const float inv = kept8_inv_step(sb);
            *reinterpret_cast<uint32_t*>(k.codes + (long long)r * k.Cp + c) =
                pack4_low_bytes(kept8_code(v[q][i][0], inv), kept8_code(v[q][i][1], inv), kept8_code(v[q][i][2], inv),
                                kept8_code(v[q][i][3], inv));
            if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, sb);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[q][i][j] = fmaf((v[q][i][j] - mean[q]) * rstd, w[i][j], b[i][j]);
        write4(tile + row * C + c, in ? n[i] : 0, v[q][i]);
      }
    }
    __syncthreads();
    run_of(y, r0).store(ring + stage * B::ROOM);  // y is aligned as x is: the same offsets
    __syncthreads();
  }
}

template <typename T, int G, int UPT, int R, bool KEPT>
__global__ void __launch_bounds__(threads_of(G), group_ctas(G))
    norm_bwd_flat_kernel(const T* dy, const T* x, Kept k, uint32_t rows, int C, Vectors vec, bool layer,
                         const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw,
                         void* db) {
  using B = FlatBatch<T, G, UPT, R>;
  constexpr uint32_t X0 = B::ROOM, S0 = X0 + (KEPT ? B::CODES : B::ROOM), STAGE = S0 + (KEPT ? B::SCALES : 0);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float ws[2][B::NT / 32 * 2 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  auto count = [&](uint64_t r0) { return (uint32_t)min((uint64_t)B::ROWS, rows - r0); };
  auto fetch = [&](uint64_t r0, uint8_t* at) {
    FlatRun<T>(dy, (long long)r0 * C, count(r0) * C).fetch(at);
    if constexpr (KEPT) {
      FlatRun<int8_t>(k.codes, (long long)r0 * k.Cp, count(r0) * k.Cp).fetch(at + X0);
      FlatRun<uint8_t>(k.scales, (long long)r0 * k.nbp, count(r0) * k.nbp).fetch(at + S0);
    } else {
      FlatRun<T>(x, (long long)r0 * C, count(r0) * C).fetch(at + X0);
    }
  };
  const uint64_t step = (uint64_t)gridDim.x * B::ROWS;
  uint64_t r0 = (uint64_t)blockIdx.x * B::ROWS;
  constexpr int DEPTH = kGroupDepth;
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    if (r0 + d * step < rows) fetch(r0 + d * step, ring + d * STAGE);
    copy_commit();
  }
  float w[UPT][4], aw[UPT * 4], ab[UPT * 4];
  int n[UPT];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int c = (t + i * G) * 4;
    n[i] = max(0, min(4, C - c));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[i][j] = j < n[i] ? vec_at(vec.w, vec.fp32, c + j, 1.f) : 0.f;
      aw[i * 4 + j] = ab[i * 4 + j] = 0.f;
    }
  }
  const float inv_c = 1.f / C;
  int stage = 0, flip = 0;
  for (; r0 < rows; r0 += step, stage = stage == DEPTH - 1 ? 0 : stage + 1, flip ^= 1) {
    const uint64_t ahead = r0 + (DEPTH - 1) * step;
    if (ahead < rows) fetch(ahead, ring + (stage == 0 ? DEPTH - 1 : stage - 1) * STAGE);
    copy_commit();
    copy_wait<DEPTH - 1>();
    float2 st[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * B::GROUPS + group;
      st[q] = r < rows ? *reinterpret_cast<const float2*>(stats + 2 * r) : make_float2(0.f, 0.f);
    }
    __syncthreads();
    uint8_t* at = ring + stage * STAGE;
    const uint32_t head = FlatRun<T>(dy, (long long)r0 * C, 0).head;
    T* gt = reinterpret_cast<T*>(at + head);
    const T* xt = reinterpret_cast<const T*>(at + X0 + head);
    const uint8_t* ct = at + X0;
    const uint8_t* bt = at + S0 + (r0 * k.nbp & 15);
    float gw[R][UPT][4], d[R][UPT][4], s[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int row = q * B::GROUPS + group;
      const bool in = r0 + row < rows;
      s[2 * q] = s[2 * q + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * 4, m = in ? n[i] : 0;
        float g[4];
        read4(gt + row * C + c, m, g);
        if constexpr (KEPT) {
          const uint32_t u = m > 0 ? *reinterpret_cast<const uint32_t*>(ct + row * k.Cp + c) ^ 0x80808080u : 0x80808080u;
          const float unit = m > 0 ? kept8_step(bt[row * k.nbp + c / kKeptBlock]) : 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            d[q][i][j] = fmaf(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + j)) - 8388736.f, unit, -st[q].x);
        } else {
          read4(xt + row * C + c, m, d[q][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) d[q][i][j] -= st[q].x;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // past the row's end g is zero and d some finite number unless the row is not
          const float gr = g[j] * st[q].y;
          gw[q][i][j] = gr * w[i][j];
          s[2 * q] = fmaf(gw[q][i][j], d[q][i][j], s[2 * q]);
          s[2 * q + 1] += gw[q][i][j];
          aw[i * 4 + j] = fmaf(gr, d[q][i][j], aw[i * 4 + j]);
          ab[i * 4 + j] += g[j];
        }
      }
    }
    if (dx != nullptr) {
      group_sum<G, 2 * R>(s, ws[flip]);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int row = q * B::GROUPS + group;
        if (r0 + row >= rows) continue;
        const float a = layer ? s[2 * q + 1] * inv_c : 0.f, b = -s[2 * q] * inv_c * st[q].y * st[q].y;
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) d[q][i][j] = fmaf(d[q][i][j], b, gw[q][i][j] - a);
          write4(gt + row * C + (t + i * G) * 4, n[i], d[q][i]);
        }
      }
      __syncthreads();
      FlatRun<T>(dx, (long long)r0 * C, count(r0) * C).store(at);  // dx is aligned as dy is: the same offsets
    }
    __syncthreads();
  }
  if (part == nullptr) return;
  join_groups<G, B::GROUPS>(aw, t, group);
  join_groups<G, B::GROUPS>(ab, t, group);
  if (group != 0) return;
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= n[i]) continue;
      store_partial(aw[i * 4 + j], (t + i * G) * 4 + j, C, 0, vec.fp32, part, dw);
      store_partial(ab[i * 4 + j], (t + i * G) * 4 + j, C, 1, vec.fp32, part, db);
    }
  }
}

// ---------------------------------------------------------------- flat form, long rows
// Row sums are taken by whole warps, a row each (or `segs` warps a row where few rows fit): no barrier and no idle threads
// per row.  Lanes read neighbouring columns, so odd widths cost no bank conflicts, and a warp's 32 columns are one block of
// the codes; but each element is read from shared memory once a pass instead of being held.  For widths where groups do
// not fit, or leave too much idle: fp32 1025 to 1536 and past 2048, bf16 past 6144.  100 M bf16 elements, kept forward / backward,
// this form and then groups: width 1501 314 / 261 and 208 / 179 us, 2901 328 / 307 and 207 / 186, 5001 329 / 399 and 255 / 230; 50 M fp32:
// 1101 171 / 186 and 203 / 187, 2047 185 / 179 and 132 / 139.
constexpr int kFlatDepth = 2;
struct FlatPlan {
  int rows, segs;          // rows of a batch; warps a row
  uint32_t room, codes, scales;  // bytes of a stage for a tensor, the codes, the scales
  uint32_t stage, vectors; // bytes of a stage; offset of the fp32 weight (and bias)
};

// Sum over a row's columns [c0, c1) of f(c), by one warp; every lane gets it.
template <typename F>
__device__ __forceinline__ float row_sum(int c0, int c1, F&& f) {
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int lane = threadIdx.x & 31;
  int c = c0 + lane;
  for (; c + 96 < c1; c += 128) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += f(c + 32 * j);
  }
  for (; c < c1; c += 32) acc[0] += f(c);
  return warp_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
}

// Sum of the row's segments; `part` holds segs values of the row, written by their warps.
__device__ __forceinline__ float join_segs(float v, float* part, int seg, int segs) {
  if (segs == 1) return v;
  if ((threadIdx.x & 31) == 0) part[seg] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < segs; ++i) v += part[i];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    norm_fwd_long_kernel(const T* x, uint32_t rows, int C, Vectors vec, float eps, bool layer, T* __restrict__ y,
                         float* __restrict__ stats, Kept k, FlatPlan pl) {
  constexpr int WARPS = kThreads / 32;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float parts[2][WARPS];
  float* w = reinterpret_cast<float*>(ring + pl.vectors);
  float* b = w + C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto run_of = [&](const T* p, uint64_t r0) {
    return FlatRun<T>(p, (long long)r0 * C, (uint32_t)min((uint64_t)pl.rows, rows - r0) * C);
  };
  const uint64_t step = (uint64_t)gridDim.x * pl.rows;
  uint64_t r0 = (uint64_t)blockIdx.x * pl.rows;
  if (r0 < rows) run_of(x, r0).fetch(ring);
  copy_commit();
  for (int c = threadIdx.x; c < C; c += kThreads) {
    w[c] = vec_at(vec.w, vec.fp32, c, 1.f);
    b[c] = vec_at(vec.b, vec.fp32, c, 0.f);
  }
  const float inv_c = 1.f / C;
  const int width = pl.segs == 1 ? C : ((C + pl.segs - 1) / pl.segs + 31) / 32 * 32;  // columns of a segment, whole blocks
  for (int stage = 0; r0 < rows; r0 += step, stage ^= 1) {
    if (r0 + step < rows) run_of(x, r0 + step).fetch(ring + (stage ^ 1) * pl.stage);
    copy_commit();
    copy_wait<1>();
    __syncthreads();
    uint8_t* at = ring + stage * pl.stage;
    T* tile = reinterpret_cast<T*>(at + run_of(x, r0).head);
    // with segments every warp has one unit, so that all take the barriers
    for (int u = warp; u < pl.rows * pl.segs; u += WARPS) {
      const int row = u / pl.segs, seg = u % pl.segs;
      const bool in = r0 + row < rows;
      if (!in && pl.segs == 1) break;
      T* xr = tile + row * C;
      const int c0 = min(C, seg * width), c1 = in ? min(C, c0 + width) : c0;
      float mean = 0.f;
      if (layer)
        mean = join_segs(row_sum(c0, c1, [&](int c) { return to_f32(xr[c]); }), &parts[0][row * pl.segs], seg, pl.segs) * inv_c;
      const float var = join_segs(row_sum(c0, c1, [&](int c) {
        const float d = to_f32(xr[c]) - mean;
        return d * d;
      }), &parts[1][row * pl.segs], seg, pl.segs);
      if (!in) continue;
      const uint64_t r = r0 + row;
      const float rstd = rsqrtf(var * inv_c + eps);
      if (lane == 0 && seg == 0 && stats != nullptr) *reinterpret_cast<float2*>(stats + 2 * r) = make_float2(mean, rstd);
      int8_t* codes = k.codes + (long long)r * k.Cp;
      uint8_t* scales = k.scales + (long long)r * k.nbp;
#pragma unroll 4
      for (int cb = c0; cb < c1; cb += 32) {
        const int c = cb + lane;
        const float v[1] = {c < c1 ? to_f32(xr[c]) : 0.f};
        if (k.codes != nullptr) {
          const uint32_t sb = kept8_byte(kept8_amax<1>(v));
          kept8_store_code(codes + c, v[0], sb);
          if (lane == 0) kept8_store_byte(scales, cb / kKeptBlock, k.nb, k.nbp, sb);
        }
        if (c < c1) xr[c] = from_f32<T>(fmaf((v[0] - mean) * rstd, w[c], b[c]));
      }
    }
    __syncthreads();
    run_of(y, r0).store(at);  // y is aligned as x is: the same offsets
    __syncthreads();
  }
}

// Phase 1, warps: the sums of each row.  Phase 2, threads: columns t + i NT of all rows, dw and db in registers, dx over dy.
template <typename T, int NT, int E, bool KEPT>
__global__ void __launch_bounds__(NT, NT == 256 ? 2 : 1)
    norm_bwd_long_kernel(const T* dy, const T* x, Kept k, uint32_t rows, int C, Vectors vec, bool layer,
                         const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw,
                         void* db, FlatPlan pl) {
  constexpr int WARPS = NT / 32;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float parts[2][WARPS];
  float* w = reinterpret_cast<float*>(ring + pl.vectors);
  float4* row_of = reinterpret_cast<float4*>(w + (C + 3) / 4 * 4);  // (mean, rstd, a, b) of each row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t X0 = pl.room, S0 = X0 + (KEPT ? pl.codes : pl.room);
  auto count = [&](uint64_t r0) { return (uint32_t)min((uint64_t)pl.rows, rows - r0); };
  auto fetch = [&](uint64_t r0, uint8_t* at) {
    FlatRun<T>(dy, (long long)r0 * C, count(r0) * C).fetch(at);
    if constexpr (KEPT) {
      FlatRun<int8_t>(k.codes, (long long)r0 * k.Cp, count(r0) * k.Cp).fetch(at + X0);
      FlatRun<uint8_t>(k.scales, (long long)r0 * k.nbp, count(r0) * k.nbp).fetch(at + S0);
    } else {
      FlatRun<T>(x, (long long)r0 * C, count(r0) * C).fetch(at + X0);
    }
  };
  const uint64_t step = (uint64_t)gridDim.x * pl.rows;
  uint64_t r0 = (uint64_t)blockIdx.x * pl.rows;
  if (r0 < rows) fetch(r0, ring);
  copy_commit();
  for (int c = threadIdx.x; c < C; c += NT) w[c] = vec_at(vec.w, vec.fp32, c, 1.f);
  const int t = threadIdx.x;
  float aw[E], ab[E];
#pragma unroll
  for (int i = 0; i < E; ++i) aw[i] = ab[i] = 0.f;
  const float inv_c = 1.f / C;
  const int width = pl.segs == 1 ? C : ((C + pl.segs - 1) / pl.segs + 31) / 32 * 32;
  for (int stage = 0; r0 < rows; r0 += step, stage ^= 1) {
    if (r0 + step < rows) fetch(r0 + step, ring + (stage ^ 1) * pl.stage);
    copy_commit();
    copy_wait<1>();
    __syncthreads();
    uint8_t* at = ring + stage * pl.stage;
    const uint32_t head = FlatRun<T>(dy, (long long)r0 * C, 0).head;
    T* gt = reinterpret_cast<T*>(at + head);
    const T* xt = reinterpret_cast<const T*>(at + X0 + head);
    const int8_t* ct = reinterpret_cast<const int8_t*>(at + X0);
    const uint8_t* bt = at + S0 + (r0 * k.nbp & 15);
    auto x_of = [&](int row, int c) -> float {
      if constexpr (KEPT) return kept8_number(ct[row * k.Cp + c]) * kept8_step(bt[row * k.nbp + c / kKeptBlock]);
      else return to_f32(xt[row * C + c]);
    };
    // with d = x - mean and g' = dy w rstd:  a = mean_c(g'),  b = rstd^2 mean_c(g' d)
    for (int u = warp; u < pl.rows * pl.segs; u += WARPS) {
      const int row = u / pl.segs, seg = u % pl.segs;
      const bool in = r0 + row < rows;
      if (!in && pl.segs == 1) break;
      const int c0 = min(C, seg * width), c1 = in ? min(C, c0 + width) : c0;
      const float2 st = in ? *reinterpret_cast<const float2*>(stats + 2 * (r0 + row)) : make_float2(0.f, 0.f);
      float sg = 0.f, sn = 0.f;
      if (dx != nullptr) {
        float gs[2] = {0.f, 0.f}, ns[2] = {0.f, 0.f};
        int c = c0 + lane;
        for (; c + 32 < c1; c += 64) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float gw = to_f32(gt[row * C + c + 32 * j]) * st.y * w[c + 32 * j];
            gs[j] += gw;
            ns[j] = fmaf(gw, x_of(row, c + 32 * j) - st.x, ns[j]);
          }
        }
        if (c < c1) {
          const float gw = to_f32(gt[row * C + c]) * st.y * w[c];
          gs[0] += gw;
          ns[0] = fmaf(gw, x_of(row, c) - st.x, ns[0]);
        }
        sg = join_segs(warp_sum(gs[0] + gs[1]), &parts[0][row * pl.segs], seg, pl.segs);
        sn = join_segs(warp_sum(ns[0] + ns[1]), &parts[1][row * pl.segs], seg, pl.segs);
      }
      if (lane == 0 && seg == 0)
        row_of[row] = make_float4(st.x, st.y, layer ? sg * inv_c : 0.f, sn * inv_c * st.y * st.y);
    }
    __syncthreads();
    const int n = (int)count(r0);
    for (int row = 0; row < n; ++row) {
      const float4 q = row_of[row];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = t + i * NT;
        if (c >= C) continue;
        const float g = to_f32(gt[row * C + c]), d = x_of(row, c) - q.x, gr = g * q.y;
        aw[i] = fmaf(gr, d, aw[i]);
        ab[i] += g;
        // the product rounded as in phase 1, so that equal terms cancel
        if (dx != nullptr) gt[row * C + c] = from_f32<T>(fmaf(-d, q.w, __fmul_rn(gr, w[c]) - q.z));
      }
    }
    __syncthreads();
    if (dx != nullptr) {
      FlatRun<T>(dx, (long long)r0 * C, count(r0) * C).store(at);  // dx is aligned as dy is: the same offsets
      __syncthreads();
    }
  }
  copy_wait<0>();
  if (part == nullptr) return;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int c = t + i * NT;
    if (c >= C) continue;
    store_partial(aw[i], c, C, 0, vec.fp32, part, dw);
    store_partial(ab[i], c, C, 1, vec.fp32, part, db);
  }
}

// ---------------------------------------------------------------- single-column form
// Views that are neither (odd column slices, odd offsets), read where they lie: thread t of a group of whole warps holds
// columns t + i G, so a warp's 32 neighbouring columns are one block of the codes.
constexpr int single_ctas(int G) { return threads_of(G) <= 256 ? 2 : 1; }
template <typename T, int G, int E, int R>
__global__ void __launch_bounds__(threads_of(G), single_ctas(G))
    norm_fwd_single_kernel(RowView x, uint32_t rows, int C, Vectors vec, float eps, bool layer, T* __restrict__ y,
                           float* __restrict__ stats, Kept k) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  __shared__ __align__(16) float ws[2][2][NT / 32 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  float w[E], b[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    w[i] = t + i * G < C ? vec_at(vec.w, vec.fp32, t + i * G, 1.f) : 0.f;
    b[i] = t + i * G < C ? vec_at(vec.b, vec.fp32, t + i * G, 0.f) : 0.f;
  }
  const float inv_c = 1.f / C;
  int flip = 0;
  for (uint64_t r0 = (uint64_t)blockIdx.x * (GROUPS * R); r0 < rows; r0 += (uint64_t)gridDim.x * (GROUPS * R)) {
    float v[R][E], mean[R], var[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      const T* xr = row_ptr<T>(x, r < rows ? (uint32_t)r : 0);
#pragma unroll
      for (int i = 0; i < E; ++i) v[q][i] = r < rows && t + i * G < C ? to_f32(xr[t + i * G]) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = var[q] = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) mean[q] += v[q][i];
    }
    if (layer) group_sum<G, R>(mean, ws[flip][0]);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = layer ? mean[q] * inv_c : 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float d = t + i * G < C ? v[q][i] - mean[q] : 0.f;
        var[q] += d * d;
      }
    }
    group_sum<G, R>(var, ws[flip][1]);
    flip ^= 1;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      const bool in = r < rows;
      const float rstd = rsqrtf(var[q] * inv_c + eps);
      if (in && t == 0 && stats != nullptr) *reinterpret_cast<float2*>(stats + 2 * r) = make_float2(mean[q], rstd);
      T* yr = y + (long long)r * C;
      int8_t* codes = k.codes + (long long)r * k.Cp;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = t + i * G;
        if (k.codes != nullptr && c - (int)(threadIdx.x & 31) < C) {  // whole warps: blocks that the row reaches
          const float one[1] = {v[q][i]};
          const uint32_t sb = kept8_byte(kept8_amax<1>(one));
          if (in) {
            kept8_store_code(codes + c, one[0], sb);
            if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, sb);
          }
        }
        if (in && c < C) yr[c] = from_f32<T>((v[q][i] - mean[q]) * rstd * w[i] + b[i]);
      }
    }
  }
}

template <typename T, int G, int E, int R, bool KEPT>
__global__ void __launch_bounds__(threads_of(G), single_ctas(G))
    norm_bwd_single_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C, Vectors vec, bool layer,
                           const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw,
                           void* db) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  __shared__ __align__(16) float ws[2][NT / 32 * 2 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G, lane = threadIdx.x & 31;
  float w[E], aw[E], ab[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    w[i] = t + i * G < C ? vec_at(vec.w, vec.fp32, t + i * G, 1.f) : 0.f;
    aw[i] = ab[i] = 0.f;
  }
  const float inv_c = 1.f / C;
  int flip = 0;
  for (uint64_t r0 = (uint64_t)blockIdx.x * (GROUPS * R); r0 < rows; r0 += (uint64_t)gridDim.x * (GROUPS * R)) {
    float g[R][E], v[R][E], s[2 * R], step[R];
    float2 st[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      const bool in = r < rows;
      const uint32_t rr = in ? (uint32_t)r : 0;
      const T* gr = row_ptr<T>(dy, rr);
      const T* xr = KEPT ? nullptr : row_ptr<T>(x, rr);
      const int8_t* codes = KEPT ? k.codes + (long long)rr * k.Cp : nullptr;
      st[q] = in ? *reinterpret_cast<const float2*>(stats + 2 * (size_t)rr) : make_float2(0.f, 0.f);
      if (KEPT) {  // lane i reads the scale of the warp's i-th block of this row
        const int blk = (t - lane + lane * G) / kKeptBlock;
        step[q] = in && lane < E && blk < k.nb ? kept8_step(k.scales[(long long)rr * k.nbp + blk]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool at = in && t + i * G < C;
        g[q][i] = at ? to_f32(gr[t + i * G]) : 0.f;
        v[q][i] = !at ? 0.f : KEPT ? kept8_number(codes[t + i * G]) : to_f32(xr[t + i * G]);
      }
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      s[2 * q] = s[2 * q + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (KEPT) v[q][i] *= __shfl_sync(0xffffffffu, step[q], i);
        v[q][i] = (v[q][i] - st[q].x) * st[q].y;  // n; columns past the row have g = 0
        const float gw = g[q][i] * w[i];
        s[2 * q] += gw;
        s[2 * q + 1] += t + i * G < C ? gw * v[q][i] : 0.f;
        aw[i] += g[q][i] * v[q][i];
        ab[i] += g[q][i];
      }
    }
    if (dx == nullptr) continue;
    group_sum<G, 2 * R>(s, ws[flip]);
    flip ^= 1;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint64_t r = r0 + q * GROUPS + group;
      if (r >= rows) continue;
      const float a = layer ? s[2 * q] * inv_c : 0.f, b = s[2 * q + 1] * inv_c;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (t + i * G < C) dx[(long long)r * C + t + i * G] = from_f32<T>(st[q].y * (g[q][i] * w[i] - a - v[q][i] * b));
    }
  }
  if (part == nullptr) return;
  join_groups<G, GROUPS>(aw, t, group);
  join_groups<G, GROUPS>(ab, t, group);
  if (group != 0) return;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (t + i * G >= C) continue;
    store_partial(aw[i], t + i * G, C, 0, vec.fp32, part, dw);
    store_partial(ab[i], t + i * G, C, 1, vec.fp32, part, db);
  }
}

// dw[c], db[c] from the partial rows: 32 columns a CTA, 8 interleaved chains a column, joined in order.
constexpr int kFinalChains = 8;
__global__ void __launch_bounds__(32 * kFinalChains) norm_bwd_final_kernel(const float* __restrict__ part, int parts,
                                                                           int C, bool fp32, void* dw, void* db) {
  __shared__ float sum[kFinalChains][32];
  const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  void* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  float acc = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int p = chain; p < parts; p += kFinalChains) acc += part[((long long)p * 2 + blockIdx.y) * C + c];
  }
  sum[chain][lane] = acc;
  __syncthreads();
  if (chain != 0 || c >= C) return;
#pragma unroll
  for (int i = 1; i < kFinalChains; ++i) acc += sum[i][lane];
  if (fp32) store_out<float>(out, c, acc);
  else store_out<__nv_bfloat16>(out, c, acc);
}

// ---------------------------------------------------------------- rows too wide for registers
__device__ __forceinline__ float cta_sum(float v) {
  __shared__ __align__(16) float ws[kThreads / 32];
  __syncthreads();
  float s[1] = {v};
  group_sum<kThreads, 1>(s, ws);
  return s[0];
}

// One CTA per row, three sweeps over it (mean, variance, output).
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_fwd_wide_kernel(RowView x, uint32_t rows, int C, Vectors vec,
                                                                 float eps, bool layer, T* __restrict__ y,
                                                                 float* __restrict__ stats, Kept k) {
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = row_ptr<T>(x, r);
    float mean = 0.f;
    if (layer) {
      for (int c = threadIdx.x; c < C; c += kThreads) mean += to_f32(xr[c]);
      mean = cta_sum(mean) / C;
    }
    float var = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float d = to_f32(xr[c]) - mean;
      var += d * d;
    }
    const float rstd = rsqrtf(cta_sum(var) / C + eps);
    if (threadIdx.x == 0 && stats != nullptr) *reinterpret_cast<float2*>(stats + 2 * (size_t)r) = make_float2(mean, rstd);
    T* yr = y + (long long)r * C;
    for (int c = threadIdx.x; c < (k.codes != nullptr ? k.Cp : C); c += kThreads) {
      float v[1] = {c < C ? to_f32(xr[c]) : 0.f};
      if (k.codes != nullptr) {  // Cp % 32 == 0: warps stay whole
        const uint32_t sb = kept8_byte(kept8_amax<1>(v));
        kept8_store_code(k.codes + (long long)r * k.Cp + c, v[0], sb);
        if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, sb);
      }
      if (c < C) yr[c] = from_f32<T>((v[0] - mean) * rstd * vec_at(vec.w, vec.fp32, c, 1.f) + vec_at(vec.b, vec.fp32, c, 0.f));
    }
  }
}

// x of (row, c), from the tensor or from its codes.
template <typename T>
__device__ __forceinline__ float x_at(const T* xr, const Kept& k, uint32_t r, int c) {
  if (k.codes == nullptr) return to_f32(xr[c]);
  return (float)k.codes[(long long)r * k.Cp + c] * kept8_step(k.scales[(long long)r * k.nbp + c / kKeptBlock]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_bwd_wide_dx_kernel(RowView dy, RowView x, Kept k, uint32_t rows,
                                                                    int C, Vectors vec, bool layer,
                                                                    const float* __restrict__ stats,
                                                                    T* __restrict__ dx) {
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* gr = row_ptr<T>(dy, r);
    const T* xr = k.codes == nullptr ? row_ptr<T>(x, r) : nullptr;
    const float2 st = *reinterpret_cast<const float2*>(stats + 2 * (size_t)r);
    float a = 0.f, b = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float g = to_f32(gr[c]) * vec_at(vec.w, vec.fp32, c, 1.f);
      a += g;
      b += g * (x_at(xr, k, r, c) - st.x) * st.y;
    }
    a = layer ? cta_sum(a) / C : 0.f;
    b = cta_sum(b) / C;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float g = to_f32(gr[c]) * vec_at(vec.w, vec.fp32, c, 1.f);
      const float n = (x_at(xr, k, r, c) - st.x) * st.y;
      dx[(long long)r * C + c] = from_f32<T>(st.y * (g - a - n * b));
    }
  }
}

// part[chunk, 0, c] = sum of dy * n, part[chunk, 1, c] = sum of dy over a chunk of rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_bwd_wide_partial_kernel(RowView dy, RowView x, Kept k, uint32_t rows,
                                                                         int C, const float* __restrict__ stats,
                                                                         uint32_t chunk, float* __restrict__ part) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= C) return;
  const uint32_t r1 = min(rows, (blockIdx.y + 1) * chunk);
  float aw = 0.f, ab = 0.f;
  for (uint32_t r = blockIdx.y * chunk; r < r1; ++r) {
    const float g = to_f32(row_ptr<T>(dy, r)[c]);
    const float2 st = *reinterpret_cast<const float2*>(stats + 2 * (size_t)r);
    aw += g * (x_at(k.codes == nullptr ? row_ptr<T>(x, r) : nullptr, k, r, c) - st.x) * st.y;
    ab += g;
  }
  part[((long long)blockIdx.y * 2 + 0) * C + c] = aw;
  part[((long long)blockIdx.y * 2 + 1) * C + c] = ab;
}

// ---------------------------------------------------------------- host
RowView view_of(const RowsArg& a) {
  return RowView{a.p, a.outer_stride, a.inner_stride, FastDiv((uint32_t)a.inner)};
}

Kept kept_of(const Kept8Buf& b) {
  Kept k;
  k.codes = (int8_t*)b.codes;
  k.scales = (uint8_t*)b.scales;
  k.Cp = (b.C + kKeptBlock - 1) / kKeptBlock * kKeptBlock;
  k.nb = k.Cp / kKeptBlock;
  k.nbp = (k.nb + 3) / 4 * 4;
  return k;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool rows_aligned16(const RowsArg& a, bool fp32) {
  const int e = fp32 ? 4 : 2;
  return aligned16(a.p) && a.outer_stride * e % 16 == 0 && a.inner_stride * e % 16 == 0;
}

// Whether `a` is a contiguous, 16-byte aligned tensor of rows of C.
bool contiguous_rows(const RowsArg& a, int C) { return a.inner == 1 && a.outer_stride == C && aligned16(a.p); }

int sm_count() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

// CTAs for `rows` in batches of `batch`, at most `ctas` on every SM.
int grid_for(long long rows, int batch, int ctas) {
  const long long want = (rows + batch - 1) / batch, most = (long long)sm_count() * ctas;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

uint32_t wide_grid(long long rows) { return (uint32_t)(rows < 148 * 64 ? rows : 148 * 64); }

constexpr int kRingBudget = 220 * 1024;  // rings of all resident CTAs of an SM

struct FwdCall {
  const NormArgs& a;
  const RowsArg& x;
  void* y;
  float* stats;
  const Kept8Buf& k;
  cudaStream_t s;
  Vectors vec() const { return Vectors{a.w, a.b, a.w_fp32}; }
};

template <typename T, int G, int UPT, int R, int DEPTH, int CTAS, bool LAYER>
void fwd_staged(const FwdCall& f) {
  constexpr int NT = threads_of(G), GROUPS = NT / G, BYTES = DEPTH * Ring<T, NT, R * UPT>::STAGE;
  static_assert(BYTES * CTAS <= kRingBudget, "the rings of an SM's CTAs do not fit its shared memory");
  const auto kernel = norm_fwd_staged_kernel<T, G, UPT, R, DEPTH, CTAS, LAYER>;
  static SmemOptIn opted;
  allow_smem(opted, kernel, BYTES);
  kernel<<<grid_for(f.a.rows, GROUPS * R, CTAS), NT, BYTES, f.s>>>(view_of(f.x), (uint32_t)f.a.rows, f.a.C, f.vec(),
                                                                   f.a.eps, (T*)f.y, f.stats, kept_of(f.k));
}

template <typename T, int G, int E, int R>
void fwd_single(const FwdCall& f) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  norm_fwd_single_kernel<T, G, E, R><<<grid_for(f.a.rows, GROUPS * R, single_ctas(G)), NT, 0, f.s>>>(
      view_of(f.x), (uint32_t)f.a.rows, f.a.C, f.vec(), f.a.eps, f.a.layer, (T*)f.y, f.stats, kept_of(f.k));
}

template <typename T, int G, int UPT, int R>
void fwd_group(const FwdCall& f) {
  using B = FlatBatch<T, G, UPT, R>;
  constexpr int BYTES = kGroupDepth * B::ROOM;
  static_assert(BYTES * group_ctas(G) <= kRingBudget, "the batches of an SM's CTAs do not fit its shared memory");
  const auto kernel = norm_fwd_flat_kernel<T, G, UPT, R>;
  static SmemOptIn opted;
  allow_smem(opted, kernel, BYTES);
  kernel<<<grid_for(f.a.rows, B::ROWS, group_ctas(G)), B::NT, BYTES, f.s>>>((const T*)f.x.p, (uint32_t)f.a.rows, f.a.C,
                                                                           f.vec(), f.a.eps, f.a.layer, (T*)f.y,
                                                                           f.stats, kept_of(f.k));
}

// Batches whose two stages and vectors fit half an SM's shared memory (two CTAs): as many rows as give 32 KB, a multiple of
// the warps, or fewer where rows are long; then several warps share a row.  rows == 0: not even one row fits an SM.
FlatPlan flat_plan(int C, int esize, int tensors, bool kept, int vectors, int warps) {
  FlatPlan p{};
  const long long Cp = (C + kKeptBlock - 1) / kKeptBlock * kKeptBlock, nbp = (Cp / kKeptBlock + 3) / 4 * 4;
  const long long row = (long long)tensors * C * esize + (kept ? Cp + nbp : 0), fixed = (long long)vectors * C * 4 + 32;
  auto fits = [&](long long rows, long long budget) {
    return kFlatDepth * (rows * row + 96) + fixed + rows * 16 <= budget;
  };
  const long long half = kRingBudget / 2;
  long long rows = 32 * 1024 / row / warps * warps;
  if (rows > 256) rows = 256;
  if (rows < warps || !fits(rows, half)) {
    rows = warps;
    while (rows > 1 && !fits(rows, half)) rows /= 2;
    if (!fits(rows, kRingBudget)) return p;
  }
  p.rows = (int)rows;
  p.segs = rows < warps ? (int)(warps / rows) : 1;
  auto room = [](long long bytes) { return (uint32_t)((bytes + 30) / 16 * 16); };
  p.room = room(rows * C * esize);
  p.codes = kept ? room(rows * Cp) : 0;
  p.scales = kept ? room(rows * nbp) : 0;
  p.stage = tensors * p.room + p.codes + p.scales;
  p.vectors = kFlatDepth * p.stage;
  return p;
}
int flat_bytes(const FlatPlan& p, int C, int vectors) { return (int)(p.vectors + ((size_t)vectors * C + 4) * 4 + p.rows * 16); }

template <typename T>
bool fwd_flat(const FwdCall& f) {
  const int C = f.a.C;
  constexpr bool B16 = sizeof(T) == 2;
  constexpr int R = B16 ? 4 : 2;  // batches of about 16 KB
#define GROUP(G) return fwd_group<T, G, 2, R>(f), true
#define THIRDS(G) if constexpr (B16) if (C <= G * 12) return fwd_group<T, G, 3, 2>(f), true
  if (C <= 64) GROUP(8);
  THIRDS(8);
  if (C <= 128) GROUP(16);
  THIRDS(16);
  if (C <= 256) GROUP(32);
  THIRDS(32);
  if (C <= 512) GROUP(64);
  THIRDS(64);
  if (C <= 1024) GROUP(128);
  THIRDS(128);
  if (C <= 2048 && (B16 || C > 1536)) GROUP(256);
  THIRDS(256);
  if constexpr (B16) if (C <= 4096) GROUP(512);
  THIRDS(512);
#undef THIRDS
#undef GROUP
  const FlatPlan pl = flat_plan(f.a.C, sizeof(T), 1, false, 2, kThreads / 32);
  if (pl.rows == 0) return false;
  const int bytes = flat_bytes(pl, f.a.C, 2);
  static SmemOptIn opted;
  allow_smem(opted, norm_fwd_long_kernel<T>, kRingBudget);
  norm_fwd_long_kernel<T><<<grid_for(f.a.rows, pl.rows, 2), kThreads, bytes, f.s>>>(
      (const T*)f.x.p, (uint32_t)f.a.rows, f.a.C, f.vec(), f.a.eps, f.a.layer, (T*)f.y, f.stats, kept_of(f.k), pl);
  return true;
}

// A group holds 16 G columns; rows of up to three quarters of that take groups of half the threads with three fragments a
// thread (THIRDS), which leaves fewer idle.  100 M bf16 elements, layer norm, kept forward / kept backward, 16 G and then
// 24 G / 2: width 384 124 / 129 and 89 / 110 us, 768 125 / 136 and 92 / 112, 1536 130 / 141 and 101 / 121, 6144 130 / 156 and 101 / 134.
// 50 M fp32, kept forward: width 264 101 and 82 us, 1280 85 and 74, 5120 105 and 76; the fp32 backward, whose rings of three
// fragments hold two batches only, keeps 16 G (1280 104 us against 117).
template <typename T, bool LAYER>
void fwd_staged_any(const FwdCall& f) {
  const int C = f.a.C;
  constexpr bool B16 = sizeof(T) == 2;
  constexpr int R = B16 ? 2 : 1, CTAS = B16 ? 2 : 3, DEPTH = CTAS == 2 ? 6 : 4;
#define STAGED(G) return fwd_staged<T, G, 2, R, DEPTH, CTAS, LAYER>(f)
#define THIRDS(G) if (C <= G * 24) return fwd_staged<T, G, 3, 1, B16 ? 8 : 4, 2, LAYER>(f)
  if (C <= 64) STAGED(4);
  if (C <= 128) STAGED(8);
  if (C <= 256) STAGED(16);
  THIRDS(16);
  if (C <= 512) STAGED(32);
  THIRDS(32);
  if (C <= 1024) STAGED(64);
  THIRDS(64);
  if (C <= 2048) STAGED(128);
  THIRDS(128);
  if (C <= 4096) STAGED(256);
  THIRDS(256);
#undef THIRDS
#undef STAGED
  if (C <= 8192) return fwd_staged<T, 512, 2, R, 4, 1, LAYER>(f);
  fwd_staged<T, 512, 4, 1, sizeof(T) == 2 ? 4 : 3, 1, LAYER>(f);
}

template <typename T>
void fwd(const FwdCall& f) {
  const int C = f.a.C;
  if (C % 8 == 0 && C <= 16384 && rows_aligned16(f.x, f.a.fp32) && aligned16(f.a.w) && aligned16(f.a.b))
    return f.a.layer ? fwd_staged_any<T, true>(f) : fwd_staged_any<T, false>(f);
  if (contiguous_rows(f.x, C) && fwd_flat<T>(f)) return;
  if (C <= 256) return fwd_single<T, 32, 8, 2>(f);
  if (C <= 2048) return fwd_single<T, 256, 8, 2>(f);
  if (C <= 8192) return fwd_single<T, 512, 16, 1>(f);
  norm_fwd_wide_kernel<T><<<wide_grid(f.a.rows), kThreads, 0, f.s>>>(view_of(f.x), (uint32_t)f.a.rows, C, f.vec(),
                                                                     f.a.eps, f.a.layer, (T*)f.y, f.stats,
                                                                     kept_of(f.k));
}

struct BwdCall {
  const NormArgs& a;
  const RowsArg &dy, &x;
  const Kept8Buf& k;
  const float* stats;
  void* dx;
  float* part;
  void *dw, *db;
  cudaStream_t s;
  int* parts;  // when not null: only the number of partial rows is wanted
  Vectors vec() const { return Vectors{a.w, nullptr, a.w_fp32}; }
  void finish(int grid) const {
    if (part != nullptr && grid > 1)
      norm_bwd_final_kernel<<<dim3((a.C + 31) / 32, 2), 32 * kFinalChains, 0, s>>>(part, grid, a.C, a.w_fp32, dw, db);
  }
};

template <typename T, int G, int UPT, int DEPTH, int CTAS, bool LAYER, bool KEPT>
void bwd_staged(const BwdCall& b) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  using D = Ring<T, NT, UPT>;
  constexpr int BYTES = DEPTH * (D::STAGE + (KEPT ? CodeRing<NT, UPT>::STAGE : D::STAGE));
  static_assert(BYTES * CTAS <= kRingBudget, "the rings of an SM's CTAs do not fit its shared memory");
  const int grid = grid_for(b.a.rows, GROUPS, CTAS);
  if (b.parts != nullptr) {
    *b.parts = grid;
    return;
  }
  const auto kernel = norm_bwd_staged_kernel<T, G, UPT, DEPTH, CTAS, LAYER, KEPT>;
  static SmemOptIn opted;
  allow_smem(opted, kernel, BYTES);
  kernel<<<grid, NT, BYTES, b.s>>>(view_of(b.dy), view_of(b.x), kept_of(b.k), (uint32_t)b.a.rows, b.a.C, b.vec(),
                                   b.stats, (T*)b.dx, b.part, b.dw, b.db);
  b.finish(grid);
}

template <typename T, int G, int E, int R, bool KEPT>
void bwd_single(const BwdCall& b) {
  constexpr int NT = threads_of(G), GROUPS = NT / G;
  const int grid = grid_for(b.a.rows, GROUPS * R, single_ctas(G));
  if (b.parts != nullptr) {
    *b.parts = grid;
    return;
  }
  norm_bwd_single_kernel<T, G, E, R, KEPT><<<grid, NT, 0, b.s>>>(view_of(b.dy), view_of(b.x), kept_of(b.k),
                                                                 (uint32_t)b.a.rows, b.a.C, b.vec(), b.a.layer,
                                                                 b.stats, (T*)b.dx, b.part, b.dw, b.db);
  b.finish(grid);
}

template <typename T, int G, int UPT, int R, bool KEPT>
void bwd_group(const BwdCall& b) {
  using B = FlatBatch<T, G, UPT, R>;
  constexpr int BYTES = kGroupDepth * (B::ROOM + (KEPT ? B::CODES + B::SCALES : B::ROOM));
  static_assert(BYTES * group_ctas(G) <= kRingBudget, "the batches of an SM's CTAs do not fit its shared memory");
  const int grid = grid_for(b.a.rows, B::ROWS, group_ctas(G));
  if (b.parts != nullptr) {
    *b.parts = grid;
    return;
  }
  const auto kernel = norm_bwd_flat_kernel<T, G, UPT, R, KEPT>;
  static SmemOptIn opted;
  allow_smem(opted, kernel, BYTES);
  kernel<<<grid, B::NT, BYTES, b.s>>>((const T*)b.dy.p, (const T*)b.x.p, kept_of(b.k), (uint32_t)b.a.rows, b.a.C,
                                      b.vec(), b.a.layer, b.stats, (T*)b.dx, b.part, b.dw, b.db);
  b.finish(grid);
}

template <typename T, int NT, int E, bool KEPT>
bool bwd_long(const BwdCall& b) {
  const FlatPlan pl = flat_plan(b.a.C, sizeof(T), KEPT ? 1 : 2, KEPT, 1, NT / 32);
  if (pl.rows == 0) return false;
  const int grid = grid_for(b.a.rows, pl.rows, NT == 256 ? 2 : 1);
  if (b.parts != nullptr) {
    *b.parts = grid;
    return true;
  }
  const int bytes = flat_bytes(pl, b.a.C, 1);
  static SmemOptIn opted;
  allow_smem(opted, norm_bwd_long_kernel<T, NT, E, KEPT>, kRingBudget);
  norm_bwd_long_kernel<T, NT, E, KEPT><<<grid, NT, bytes, b.s>>>(
      (const T*)b.dy.p, (const T*)b.x.p, kept_of(b.k), (uint32_t)b.a.rows, b.a.C, b.vec(), b.a.layer, b.stats, (T*)b.dx,
      b.part, b.dw, b.db, pl);
  b.finish(grid);
  return true;
}

template <typename T, bool KEPT>
bool bwd_flat_any(const BwdCall& b) {
  const int C = b.a.C;
  constexpr bool B16 = sizeof(T) == 2;
#define GROUP(G) return bwd_group<T, G, 2, 2, KEPT>(b), true
#define THIRDS(G) if constexpr (B16) if (C <= G * 12) return bwd_group<T, G, 3, 2, KEPT>(b), true
  if (C <= 64) GROUP(8);
  THIRDS(8);
  if (C <= 128) GROUP(16);
  THIRDS(16);
  if (C <= 256) GROUP(32);
  THIRDS(32);
  if (C <= 512) GROUP(64);
  THIRDS(64);
  if (C <= 1024) GROUP(128);
  THIRDS(128);
  if (C <= 2048 && (B16 || C > 1536)) GROUP(256);
  THIRDS(256);
  if constexpr (B16) if (C <= 4096) GROUP(512);
  THIRDS(512);
#undef THIRDS
#undef GROUP
  if constexpr (!B16) {
    if (C <= 1536) return bwd_long<T, 256, 6, KEPT>(b);
    if (C <= 4096) return bwd_long<T, 256, 16, KEPT>(b);
  }
  if (C <= 8192) return bwd_long<T, 512, 16, KEPT>(b);
  return false;
}

template <typename T>
void bwd_wide(const BwdCall& b) {
  const NormArgs& a = b.a;
  const int parts = (int)(a.rows < 128 ? 2 : a.rows > 1024 * 128 ? 1024 : (a.rows + 127) / 128 + 1);
  if (b.parts != nullptr) {
    *b.parts = parts;
    return;
  }
  if (b.dx != nullptr && a.rows > 0)
    norm_bwd_wide_dx_kernel<T><<<wide_grid(a.rows), kThreads, 0, b.s>>>(
        view_of(b.dy), view_of(b.x), kept_of(b.k), (uint32_t)a.rows, a.C, b.vec(), a.layer, b.stats, (T*)b.dx);
  if (b.part == nullptr) return;
  norm_bwd_wide_partial_kernel<T><<<dim3((a.C + kThreads - 1) / kThreads, parts), kThreads, 0, b.s>>>(
      view_of(b.dy), view_of(b.x), kept_of(b.k), (uint32_t)a.rows, a.C, b.stats,
      (uint32_t)((a.rows + parts - 1) / parts), b.part);
  b.finish(parts);
}

// THIRDS as in the forward, bf16 only.  Fp32 rows past 8192 columns leave room for one stage beside an exact input, so nothing is
// copied ahead (6000 x 16384 265 us, 0.69 of the copy rate), and for two beside codes (241 us, 0.57).
template <typename T, bool LAYER, bool KEPT>
void bwd_staged_any(const BwdCall& b) {
  const int C = b.a.C;
  constexpr bool B16 = sizeof(T) == 2;
  constexpr int DEPTH = B16 ? 6 : 3;
#define STAGED(G) return bwd_staged<T, G, 2, DEPTH, 2, LAYER, KEPT>(b)
#define THIRDS(G) if constexpr (B16) if (C <= G * 24) return bwd_staged<T, G, 3, KEPT ? 5 : 4, 2, LAYER, KEPT>(b)
  if (C <= 64) STAGED(4);
  if (C <= 128) STAGED(8);
  if (C <= 256) STAGED(16);
  THIRDS(16);
  if (C <= 512) STAGED(32);
  THIRDS(32);
  if (C <= 1024) STAGED(64);
  THIRDS(64);
  if (C <= 2048) STAGED(128);
  THIRDS(128);
  if (C <= 4096) STAGED(256);
  THIRDS(256);
#undef THIRDS
#undef STAGED
  if (C <= 8192) return bwd_staged<T, 512, 2, DEPTH, 1, LAYER, KEPT>(b);
  bwd_staged<T, 512, 4, sizeof(T) == 2 ? 3 : KEPT ? 2 : 1, 1, LAYER, KEPT>(b);
}

template <typename T, bool KEPT>
void bwd(const BwdCall& b) {
  const int C = b.a.C;
  const bool fp32 = sizeof(T) == 4;
  if (C % 8 == 0 && C <= 16384 && rows_aligned16(b.dy, fp32) && (KEPT || rows_aligned16(b.x, fp32)) && aligned16(b.a.w))
    return b.a.layer ? bwd_staged_any<T, true, KEPT>(b) : bwd_staged_any<T, false, KEPT>(b);
  if (contiguous_rows(b.dy, C) && (KEPT || contiguous_rows(b.x, C)) && bwd_flat_any<T, KEPT>(b)) return;
  if (C <= 256) return bwd_single<T, 32, 8, 2, KEPT>(b);
  if (C <= 2048) return bwd_single<T, 256, 8, 2, KEPT>(b);
  if (C <= 8192) return bwd_single<T, 1024, 8, 1, KEPT>(b);
  bwd_wide<T>(b);
}

void bwd_any(const BwdCall& b) {
  if (b.a.fp32) b.k.codes != nullptr ? bwd<float, true>(b) : bwd<float, false>(b);
  else b.k.codes != nullptr ? bwd<__nv_bfloat16, true>(b) : bwd<__nv_bfloat16, false>(b);
}

}  // namespace

void launch_norm_fwd(const NormArgs& a, const RowsArg& x, void* y, float* stats, const Kept8Buf& k, cudaStream_t s) {
  if (a.rows <= 0) return;
  const FwdCall f{a, x, y, stats, k, s};
  a.fp32 ? fwd<float>(f) : fwd<__nv_bfloat16>(f);
}

int norm_bwd_parts(const NormArgs& a, const RowsArg& dy, const RowsArg& x, const Kept8Buf& k) {
  int parts = 1;
  bwd_any(BwdCall{a, dy, x, k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, &parts});
  return parts;
}

void launch_norm_bwd(const NormArgs& a, const RowsArg& dy, const RowsArg& x, const Kept8Buf& k, const float* stats,
                     void* dx, float* part, void* dw, void* db, cudaStream_t s) {
  bwd_any(BwdCall{a, dy, x, k, stats, dx, part, dw, db, s, nullptr});
}

}  // namespace pan
