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
// Both directions are DRAM-bound, so every tensor is read and written once.  A group of G threads
// holds a whole row in registers in fragments of V elements (V = 8: 16-byte accesses, for rows whose
// width and alignment allow; V = 1 otherwise; fragment i of thread t starts at column (t + i G) V).
// Groups of up to a warp reduce by shuffles, larger ones through shared memory.  The
// backward's threads own their columns for all the rows that their CTA walks, so dw and db grow in
// registers beside the dx of each row; one partial row per CTA goes to scratch and a second kernel adds those up
// in order (no atomics: the same bits every time).  Rows too wide for registers take the *_wide
// kernels, which sweep the row from memory.
#include "kept8.cuh"
#include "launchers.h"

namespace pan {
namespace {

constexpr int kThreads = 256;

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

// ---------------------------------------------------------------- fragments
// V elements as they lie in memory.
template <typename T, int V>
struct Pack {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void zero() { raw = from_f32<T>(0.f); }
  __device__ __forceinline__ void get(float (&v)[V]) const { v[0] = to_f32(raw); }
};
template <>
struct Pack<__nv_bfloat16, 8> {
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};
template <>
struct Pack<float, 8> {
  float4 raw[2];
  __device__ __forceinline__ void load(const float* p) {
    raw[0] = reinterpret_cast<const float4*>(p)[0];
    raw[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { raw[0] = raw[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = raw[0].x; v[1] = raw[0].y; v[2] = raw[0].z; v[3] = raw[0].w;
    v[4] = raw[1].x; v[5] = raw[1].y; v[6] = raw[1].z; v[7] = raw[1].w;
  }
};

// V codes and their scale byte.
template <int V>
struct CodePack {
  uint2 raw;
  uint32_t b;
  __device__ __forceinline__ void load(const int8_t* p, uint32_t byte) {
    if constexpr (V == 8) raw = *reinterpret_cast<const uint2*>(p);
    else raw.x = (uint8_t)*p;
    b = byte;
  }
  __device__ __forceinline__ void zero() { raw = make_uint2(0, 0), b = kKeptPadByte; }
  __device__ __forceinline__ void get(float (&v)[V]) const {
    const float step = kept8_step(b);
    if constexpr (V == 8) kept8_values(raw, step, v);
    else v[0] = (float)(int8_t)raw.x * step;
  }
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

// ---------------------------------------------------------------- reductions
// Sums of N values over each group of G threads; every thread of the group gets them.  `ws` holds
// N floats a warp; calls that may overlap use different ones.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* ws) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (G > 32) {
    constexpr int W = G / 32;  // warps of a group
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) ws[warp * N + k] = v[k];
    }
    __syncthreads();
    const float* g = ws + warp / W * W * N;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += g[i * N + k];
    }
  }
}

// ---------------------------------------------------------------- forward
// The row lives in registers between its one read and its one write, so the mean, the centred squares, the
// codes and y all come from it.  Up to a warp a row needs no barrier and several rows are in flight a CTA.
template <typename T, int V, int G, int UPT>
__global__ void __launch_bounds__(G > kThreads ? G : kThreads)
    norm_fwd_kernel(RowView x, uint32_t rows, int C, Vectors vec, float eps, bool layer, T* __restrict__ y,
                    float* __restrict__ stats, Kept k) {
  constexpr int NT = G > kThreads ? G : kThreads, GROUPS = NT / G;
  __shared__ float ws[2][NT / 32];
  const int t = threadIdx.x % G;
  const uint32_t r = blockIdx.x * GROUPS + threadIdx.x / G;
  const bool in = r < rows;
  const T* xr = row_ptr<T>(x, in ? r : 0);
  Pack<T, V> raw[UPT];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int c = (t + i * G) * V;
    if (in && c < C) raw[i].load(xr + c);
    else raw[i].zero();
  }
  float mean = 0.f;
  const float inv_c = 1.f / C;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      float v[V];
      raw[i].get(v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[j];
    }
    group_sum<G, 1>(s, ws[0]);
    mean = s[0] * inv_c;
  }
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    if ((t + i * G) * V >= C) continue;
    float v[V];
    raw[i].get(v);
#pragma unroll
    for (int j = 0; j < V; ++j) s[0] += (v[j] - mean) * (v[j] - mean);
  }
  group_sum<G, 1>(s, ws[1]);
  const float rstd = rsqrtf(s[0] * inv_c + eps);
  if (in && t == 0) *reinterpret_cast<float2*>(stats + 2 * (size_t)r) = make_float2(mean, rstd);
  T* yr = y + (long long)r * C;
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int c = (t + i * G) * V;
    float v[V];
    raw[i].get(v);
    if (k.codes != nullptr) {  // whole blocks of 32 / V neighbouring lanes, with zeros past the row's end
      const uint32_t b = kept8_byte(kept8_amax<V>(v));
      if (in && c < k.Cp) {
        kept8_store_codes<V>(k.codes + (long long)r * k.Cp + c, v, b);
        if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, b);
      }
    }
    if (!in || c >= C) continue;
    float w[V], b[V];
    load_vec<V>(vec.w, vec.fp32, c, 1.f, w);
    load_vec<V>(vec.b, vec.fp32, c, 0.f, b);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * w[j] + b[j];
    store_v<T, V>(yr + c, v);
  }
}

// ---------------------------------------------------------------- backward
// x of a fragment comes from the tensor or from the codes (KEPT).
template <typename T, int V, bool KEPT>
struct XPack : Pack<T, V> {
  __device__ __forceinline__ void load(const RowView& x, const Kept&, uint32_t r, int c) {
    Pack<T, V>::load(row_ptr<T>(x, r) + c);
  }
};
template <typename T, int V>
struct XPack<T, V, true> : CodePack<V> {
  __device__ __forceinline__ void load(const RowView&, const Kept& k, uint32_t r, int c) {
    CodePack<V>::load(k.codes + (long long)r * k.Cp + c, k.scales[(long long)r * k.nbp + c / kKeptBlock]);
  }
};

template <typename W>
__device__ __forceinline__ void store_out(void* out, int c, float v) {
  if (out != nullptr) reinterpret_cast<W*>(out)[c] = from_f32<W>(v);
}

// The CTA's groups hold the same columns: add them up, in a fixed order, into the first group.
template <int V, int G, int GROUPS, int UPT, bool BOTH>
__device__ __forceinline__ void join_groups(float* aw, float* ab, int t, int group) {
  if constexpr (GROUPS > 1) {
    __shared__ float cs[GROUPS / 2 * G * V];
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
#pragma unroll
      for (int which = 0; which < (BOTH ? 2 : 1); ++which) {
        float* acc = (which ? ab : aw) + i * V;
#pragma unroll
        for (int h = GROUPS / 2; h > 0; h >>= 1) {
          __syncthreads();
          if (group >= h && group < 2 * h) {
#pragma unroll
            for (int j = 0; j < V; ++j) cs[((group - h) * V + j) * G + t] = acc[j];
          }
          __syncthreads();
          if (group < h) {
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += cs[(group * V + j) * G + t];
          }
        }
      }
    }
  }
}

// The CTA's partial row; a lone CTA's is the result.
template <int V, int G, int UPT, bool BOTH>
__device__ __forceinline__ void store_partial(const float* aw, const float* ab, int t, int C, bool fp32, float* part,
                                              void* dw, void* db) {
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int c = (t + i * G) * V;
    if (c >= C) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (gridDim.x == 1) {
        if (fp32) store_out<float>(dw, c + j, aw[i * V + j]);
        else store_out<__nv_bfloat16>(dw, c + j, aw[i * V + j]);
        if (BOTH && fp32) store_out<float>(db, c + j, ab[i * V + j]);
        else if (BOTH) store_out<__nv_bfloat16>(db, c + j, ab[i * V + j]);
      } else {
        part[(long long)blockIdx.x * 2 * C + c + j] = aw[i * V + j];
        if (BOTH) part[((long long)blockIdx.x * 2 + 1) * C + c + j] = ab[i * V + j];
      }
    }
  }
}

// ---- register form (rows that 16-byte copies cannot address): R rows a group at a time, all their loads issued
// before the first reduction
template <typename T, int V, int G, int UPT, int R, bool KEPT>
__global__ void __launch_bounds__(G > kThreads ? G : kThreads, G > kThreads ? 1 : 2)
    norm_bwd_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C, Vectors vec, bool layer,
                    const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw, void* db) {
  constexpr int NT = G > kThreads ? G : kThreads, GROUPS = NT / G, E = UPT * V;
  __shared__ float ws[2][NT / 32 * 2 * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  float w[E], aw[E], ab[E];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    float v[V];
    const int c = (t + i * G) * V;
    load_vec<V>(c < C ? vec.w : nullptr, vec.fp32, c, 1.f, v);
#pragma unroll
    for (int j = 0; j < V; ++j) w[i * V + j] = v[j], aw[i * V + j] = ab[i * V + j] = 0.f;
  }
  const float inv_c = 1.f / C;
  int flip = 0;
  for (uint32_t r0 = blockIdx.x * (GROUPS * R); r0 < rows; r0 += gridDim.x * (GROUPS * R)) {
    Pack<T, V> gp[R][UPT];
    XPack<T, V, KEPT> xp[R][UPT];
    float2 st[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint32_t r = r0 + q * GROUPS + group;
      const bool in = r < rows;
      const T* gr = row_ptr<T>(dy, in ? r : 0);
      st[q] = in ? *reinterpret_cast<const float2*>(stats + 2 * (size_t)r) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * V;
        if (in && c < C) {
          gp[q][i].load(gr + c);
          xp[q][i].load(x, k, r, c);
        } else {
          gp[q][i].zero();
          xp[q][i].zero();
        }
      }
    }
    float s[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      s[2 * q] = s[2 * q + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        float g[V], v[V];
        gp[q][i].get(g);
        xp[q][i].get(v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float n = (v[j] - st[q].x) * st[q].y;
          const float gw = g[j] * w[i * V + j];
          s[2 * q] += gw;
          s[2 * q + 1] += gw * n;
          aw[i * V + j] += g[j] * n;
          ab[i * V + j] += g[j];
        }
      }
    }
    if (dx == nullptr) continue;
    group_sum<G, 2 * R>(s, ws[flip]);
    flip ^= 1;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint32_t r = r0 + q * GROUPS + group;
      if (r >= rows) continue;
      const float a = layer ? s[2 * q] * inv_c : 0.f, b = s[2 * q + 1] * inv_c;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * V;
        if (c >= C) continue;
        float g[V], v[V];
        gp[q][i].get(g);
        xp[q][i].get(v);
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[j] = st[q].y * (g[j] * w[i * V + j] - a - (v[j] - st[q].x) * st[q].y * b);
        store_v<T, V>(dx + (long long)r * C + c, v);
      }
    }
  }
  if (part == nullptr) return;
  join_groups<V, G, GROUPS, UPT, true>(aw, ab, t, group);
  if (group == 0) store_partial<V, G, UPT, true>(aw, ab, t, C, vec.fp32, part, dw, db);
}

// ---- staged form: 16-byte fragments through a ring in shared memory
// Each thread copies its own fragments (dy, x or its codes and scale word) DEPTH - 1 row batches ahead
// with asynchronous copies and waits for its own copies only, so loads stay in flight across the
// reductions without holding registers; the second use of a fragment (dx, after the reduction) reads it from the ring again.
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes, bool in) {
  const int n = in ? bytes : 0;  // 0: the destination is zero-filled, the source is not read
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int G, int UPT, int R, int DEPTH, bool KEPT>
struct Staged {
  static constexpr int NT = G > kThreads ? G : kThreads, GROUPS = NT / G;
  static constexpr int Q = sizeof(T) / 2;                 // 16-byte pieces of a fragment of T
  static constexpr int PIECE = NT * 16, SLOTS = R * UPT;  // one piece of every thread; fragments of a stage
  static constexpr int STAGE = SLOTS * (Q * PIECE + (KEPT ? NT * 12 : Q * PIECE));
  static constexpr int BYTES = DEPTH * STAGE;
};

template <typename T, int G, int UPT, int R, int DEPTH, int CTAS, bool LAYER, bool KEPT>
__global__ void __launch_bounds__(G > kThreads ? G : kThreads, CTAS)
    norm_bwd_staged_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C, Vectors vec,
                           const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, void* dw,
                           void* db) {
  using S = Staged<T, G, UPT, R, DEPTH, KEPT>;
  constexpr int V = 8, NT = S::NT, GROUPS = S::GROUPS, E = UPT * V, N = LAYER ? 2 : 1;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float ws[2][NT / 32 * N * R];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  // byte offsets inside a stage: dy pieces, then x pieces or codes and scale words
  constexpr int X0 = S::SLOTS * S::Q * S::PIECE, SC0 = X0 + S::SLOTS * NT * 8;
  const uint32_t step = gridDim.x * (GROUPS * R);

  auto fetch = [&](uint32_t r0, int stage) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint32_t r = r0 + q * GROUPS + group;
      const bool row_in = r >= r0 && r < rows;  // r0 past the rows (or wrapped around): zeros
      const uint32_t rr = row_in ? r : 0;
      const T* gr = row_ptr<T>(dy, rr);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int c = (t + i * G) * V, slot = q * UPT + i;
        const bool in = row_in && c < C;
        const int cc = in ? c : 0;
        const uint32_t at = ring0 + stage * S::STAGE;
#pragma unroll
        for (int h = 0; h < S::Q; ++h)
          copy_async(at + (slot * S::Q + h) * S::PIECE + threadIdx.x * 16, reinterpret_cast<const uint4*>(gr + cc) + h, 16, in);
        if constexpr (KEPT) {
          copy_async(at + X0 + (slot * NT + threadIdx.x) * 8, k.codes + (long long)rr * k.Cp + cc, 8, in);
          copy_async(at + SC0 + (slot * NT + threadIdx.x) * 4,
                     k.scales + (long long)rr * k.nbp + cc / kKeptBlock / 4 * 4, 4, in);
        } else {
          const T* xr = row_ptr<T>(x, rr);
#pragma unroll
          for (int h = 0; h < S::Q; ++h)
            copy_async(at + X0 + (slot * S::Q + h) * S::PIECE + threadIdx.x * 16, reinterpret_cast<const uint4*>(xr + cc) + h, 16, in);
        }
      }
    }
  };
  auto dy_of = [&](int stage, int slot, float (&v)[V]) {
    Pack<T, V> p;
    const uint8_t* at = ring + stage * S::STAGE + slot * S::Q * S::PIECE + threadIdx.x * 16;
    if constexpr (sizeof(T) == 2) {
      p.raw = *reinterpret_cast<const uint4*>(at);
    } else {
      p.raw[0] = *reinterpret_cast<const float4*>(at);
      p.raw[1] = *reinterpret_cast<const float4*>(at + S::PIECE);
    }
    p.get(v);
  };
  auto x_of = [&](int stage, int slot, int c, float (&v)[V]) {
    const uint8_t* at = ring + stage * S::STAGE;
    if constexpr (KEPT) {
      const uint32_t word = *reinterpret_cast<const uint32_t*>(at + SC0 + (slot * NT + threadIdx.x) * 4);
      // a zero word (nothing copied) is no scale; its codes are zero
      const uint32_t b = word == 0 ? kKeptPadByte : (word >> (c / kKeptBlock % 4 * 8)) & 0xffu;
      kept8_values(*reinterpret_cast<const uint2*>(at + X0 + (slot * NT + threadIdx.x) * 8), kept8_step(b), v);
    } else {
      Pack<T, V> p;
      at += X0 + slot * S::Q * S::PIECE + threadIdx.x * 16;
      if constexpr (sizeof(T) == 2) {
        p.raw = *reinterpret_cast<const uint4*>(at);
      } else {
        p.raw[0] = *reinterpret_cast<const float4*>(at);
        p.raw[1] = *reinterpret_cast<const float4*>(at + S::PIECE);
      }
      p.get(v);
    }
  };

  const uint32_t first = blockIdx.x * (GROUPS * R);
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) {
    fetch((uint64_t)first + (uint64_t)d * step < rows ? first + d * step : rows, d);
    copy_commit();
  }
  float w[E], aw[E], ab[LAYER ? E : 1];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    float v[V];
    const int c = (t + i * G) * V;
    load_vec<V>(c < C ? vec.w : nullptr, vec.fp32, c, 1.f, v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i * V + j] = v[j];
      aw[i * V + j] = 0.f;
      if (LAYER) ab[i * V + j] = 0.f;
    }
  }
  const float inv_c = 1.f / C;
  float2 next[R];
  auto stats_of = [&](uint32_t r0) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const uint32_t r = r0 + q * GROUPS + group;
      next[q] = r >= r0 && r < rows ? *reinterpret_cast<const float2*>(stats + 2 * (size_t)r) : make_float2(0.f, 0.f);
    }
  };
  stats_of(first);
  int stage = 0, flip = 0;
  for (uint64_t r64 = first; r64 < rows; r64 += step) {
    const uint32_t r0 = (uint32_t)r64;
    float2 st[R];
#pragma unroll
    for (int q = 0; q < R; ++q) st[q] = next[q];
    const int ahead = stage == 0 ? DEPTH - 1 : stage - 1;  // the stage consumed in the last turn
    const uint64_t r_ahead = r64 + (uint64_t)(DEPTH - 1) * step;
    fetch(r_ahead < rows ? (uint32_t)r_ahead : rows, ahead);
    copy_commit();
    stats_of(r64 + step < rows ? r0 + step : rows);
    copy_wait<DEPTH - 1>();
    float s[N * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
#pragma unroll
      for (int n = 0; n < N; ++n) s[q * N + n] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        float g[V], v[V];
        dy_of(stage, q * UPT + i, g);
        x_of(stage, q * UPT + i, (t + i * G) * V, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = LAYER ? v[j] - st[q].x : v[j];
          const float gw = g[j] * w[i * V + j];
          s[q * N] += gw * d;
          aw[i * V + j] += g[j] * (d * st[q].y);
          if (LAYER) {
            s[q * N + N - 1] += gw;
            ab[i * V + j] += g[j];
          }
        }
      }
    }
    if (dx != nullptr) {
      group_sum<G, N * R>(s, ws[flip]);
      flip ^= 1;
      asm volatile("" ::: "memory");  // the fragments are read from the ring again, not held in registers
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const uint32_t r = r0 + q * GROUPS + group;
        if (r >= rows) continue;
        const float rstd = st[q].y;
        const float a = LAYER ? s[q * N + N - 1] * inv_c * rstd : 0.f;
        const float b = s[q * N] * inv_c * rstd * rstd * rstd;  // s holds sum gw (x - mean)
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
          const int c = (t + i * G) * V;
          if (c >= C) continue;
          float g[V], v[V];
          dy_of(stage, q * UPT + i, g);
          x_of(stage, q * UPT + i, c, v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float d = LAYER ? v[j] - st[q].x : v[j];
            v[j] = (g[j] * w[i * V + j]) * rstd - a - d * b;
          }
          store_v<T, V>(dx + (long long)r * C + c, v);
        }
      }
    }
    stage = stage == DEPTH - 1 ? 0 : stage + 1;
  }
  copy_wait<0>();
  if (part == nullptr) return;
  join_groups<V, G, GROUPS, UPT, LAYER>(aw, ab, t, group);
  if (group == 0) store_partial<V, G, UPT, LAYER>(aw, ab, t, C, vec.fp32, part, dw, db);
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
  __shared__ float ws[kThreads / 32];
  __syncthreads();
  float s[1] = {v};
  group_sum<kThreads, 1>(s, ws);
  return s[0];
}

__device__ __forceinline__ float vec_at(const void* p, bool fp32, int c, float missing) {
  float v[1];
  load_vec<1>(p, fp32, c, missing, v);
  return v[0];
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
    if (threadIdx.x == 0) *reinterpret_cast<float2*>(stats + 2 * (size_t)r) = make_float2(mean, rstd);
    T* yr = y + (long long)r * C;
    for (int c = threadIdx.x; c < (k.codes != nullptr ? k.Cp : C); c += kThreads) {
      float v[1] = {c < C ? to_f32(xr[c]) : 0.f};
      if (k.codes != nullptr) {  // Cp % 32 == 0: warps stay whole
        const uint32_t sb = kept8_byte(kept8_amax<1>(v));
        kept8_store_codes<1>(k.codes + (long long)r * k.Cp + c, v, sb);
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

int sm_count() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

uint32_t wide_grid(long long rows) { return (uint32_t)(rows < 148 * 64 ? rows : 148 * 64); }

template <typename T, int V, int G, int UPT>
void fwd_rows(const NormArgs& a, const RowsArg& x, void* y, float* stats, const Kept8Buf& k, cudaStream_t s) {
  constexpr int NT = G > kThreads ? G : kThreads, GROUPS = NT / G;
  norm_fwd_kernel<T, V, G, UPT><<<(uint32_t)((a.rows + GROUPS - 1) / GROUPS), NT, 0, s>>>(
      view_of(x), a.rows, a.C, Vectors{a.w, a.b, a.w_fp32}, a.eps, a.layer, (T*)y, stats, kept_of(k));
}

template <typename T>
void fwd(const NormArgs& a, const RowsArg& x, void* y, float* stats, const Kept8Buf& k, cudaStream_t s) {
  const int C = a.C;
#define ROWS(V, G, UPT) return fwd_rows<T, V, G, UPT>(a, x, y, stats, k, s)
  if (C % 8 == 0 && rows_aligned16(x, a.fp32) && aligned16(a.w) && aligned16(a.b)) {
    // the smallest group whose threads hold the row in at most 4 fragments up to a warp; then up to
    // 16 bf16 / 8 fp32 fragments (64 registers), then more warps
    if (C <= 128) ROWS(8, 4, 4);
    if (C <= 256) ROWS(8, 8, 4);
    if (C <= 512) ROWS(8, 16, 4);
    if (C <= 1024) ROWS(8, 32, 4);
    if (C <= 2048) ROWS(8, 32, 8);
    if constexpr (sizeof(T) == 2) {
      if (C <= 4096) ROWS(8, 32, 16);
    }
    if (C <= 8192) ROWS(8, 128, 8);
    if (C <= 16384) ROWS(8, 256, 8);
    if (C <= 32768) ROWS(8, 512, 8);
  } else {
    if (C <= 256) ROWS(1, 32, 8);
    if (C <= 1024) ROWS(1, 32, 32);
    if (C <= 4096) ROWS(1, 128, 32);
    if (C <= 16384) ROWS(1, 512, 32);
  }
#undef ROWS
  norm_fwd_wide_kernel<T><<<wide_grid(a.rows), kThreads, 0, s>>>(
      view_of(x), a.rows, C, Vectors{a.w, a.b, a.w_fp32}, a.eps, a.layer, (T*)y, stats, kept_of(k));
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
  int* parts;  // asked for the number of partial rows instead of a launch when not null
};

template <typename T, int V, int G, int UPT, int R, bool KEPT>
void bwd_rows(const BwdCall& b) {
  constexpr int NT = G > kThreads ? G : kThreads, GROUPS = NT / G;
  static int resident = 0;
  if (resident == 0) {
    int n = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_bwd_kernel<T, V, G, UPT, R, KEPT>, NT, 0);
    resident = n < 1 ? 1 : n;
  }
  const long long want = (b.a.rows + GROUPS * R - 1) / (GROUPS * R), most = (long long)sm_count() * resident;
  const int grid = (int)(want < 1 ? 1 : want < most ? want : most);
  if (b.parts != nullptr) {
    *b.parts = grid;
    return;
  }
  norm_bwd_kernel<T, V, G, UPT, R, KEPT><<<grid, NT, 0, b.s>>>(
      view_of(b.dy), view_of(b.x), kept_of(b.k), b.a.rows, b.a.C, Vectors{b.a.w, nullptr, b.a.w_fp32}, b.a.layer,
      b.stats, (T*)b.dx, b.part, b.dw, b.db);
  if (b.part != nullptr && grid > 1)
    norm_bwd_final_kernel<<<dim3((b.a.C + 31) / 32, 2), 32 * kFinalChains, 0, b.s>>>(b.part, grid, b.a.C, b.a.w_fp32,
                                                                                     b.dw, b.db);
}

template <typename T, int G, int UPT, int R, int DEPTH, int CTAS, bool LAYER, bool KEPT>
void bwd_staged(const BwdCall& b) {
  using S = Staged<T, G, UPT, R, DEPTH, KEPT>;
  static_assert(S::BYTES * CTAS <= 220 * 1024, "the rings of an SM's CTAs do not fit its shared memory");
  const auto kernel = norm_bwd_staged_kernel<T, G, UPT, R, DEPTH, CTAS, LAYER, KEPT>;
  static bool ready = false;
  if (!ready) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
    ready = true;
  }
  const long long want = (b.a.rows + S::GROUPS * R - 1) / (S::GROUPS * R), most = (long long)sm_count() * CTAS;
  const int grid = (int)(want < 1 ? 1 : want < most ? want : most);
  if (b.parts != nullptr) {
    *b.parts = grid;
    return;
  }
  kernel<<<grid, S::NT, S::BYTES, b.s>>>(view_of(b.dy), view_of(b.x), kept_of(b.k), b.a.rows, b.a.C,
                                         Vectors{b.a.w, nullptr, b.a.w_fp32}, b.stats, (T*)b.dx, b.part, b.dw, b.db);
  if (b.part != nullptr && grid > 1)
    norm_bwd_final_kernel<<<dim3((b.a.C + 31) / 32, 2), 32 * kFinalChains, 0, b.s>>>(b.part, grid, b.a.C, b.a.w_fp32,
                                                                                     b.dw, b.db);
}

template <typename T, bool KEPT>
void bwd_wide(const BwdCall& b) {
  const NormArgs& a = b.a;
  const int parts = (int)(a.rows < 128 ? 1 : a.rows > 1024 * 128 ? 1024 : (a.rows + 127) / 128);
  if (b.parts != nullptr) {
    *b.parts = parts;
    return;
  }
  const Vectors vec{a.w, nullptr, a.w_fp32};
  if (b.dx != nullptr && a.rows > 0)
    norm_bwd_wide_dx_kernel<T><<<wide_grid(a.rows), kThreads, 0, b.s>>>(view_of(b.dy), view_of(b.x), kept_of(b.k),
                                                                        a.rows, a.C, vec, a.layer, b.stats, (T*)b.dx);
  if (b.part == nullptr) return;
  norm_bwd_wide_partial_kernel<T><<<dim3((a.C + kThreads - 1) / kThreads, parts), kThreads, 0, b.s>>>(
      view_of(b.dy), view_of(b.x), kept_of(b.k), a.rows, a.C, b.stats, (uint32_t)((a.rows + parts - 1) / parts),
      b.part);
  norm_bwd_final_kernel<<<dim3((a.C + 31) / 32, 2), 32 * kFinalChains, 0, b.s>>>(b.part, parts, a.C, a.w_fp32, b.dw,
                                                                                 b.db);
}

// 16 columns a thread, so 16 accumulators for each of dw and db; 2 CTAs an SM with rings of about 100 KB
template <typename T, bool LAYER, bool KEPT>
void bwd_staged_any(const BwdCall& b) {
  const int C = b.a.C;
  constexpr int R = sizeof(T) == 2 ? 2 : 1;
#define STAGED(G) return bwd_staged<T, G, 2, R, 3, 2, LAYER, KEPT>(b)
  if (C <= 64) STAGED(4);
  if (C <= 128) STAGED(8);
  if (C <= 256) STAGED(16);
  if (C <= 512) STAGED(32);
  if (C <= 1024) STAGED(64);
  if (C <= 2048) STAGED(128);
  if (C <= 4096) STAGED(256);
#undef STAGED
  if (C <= 8192) return bwd_staged<T, 512, 2, R, 3, 1, LAYER, KEPT>(b);
  bwd_staged<T, 512, 4, 1, 6 / (int)sizeof(T), 1, LAYER, KEPT>(b);
}

template <typename T, bool KEPT>
void bwd(const BwdCall& b) {
  const int C = b.a.C;
  const bool fp32 = sizeof(T) == 4;
  if (C % 8 == 0 && C <= 16384 && rows_aligned16(b.dy, fp32) && (KEPT || rows_aligned16(b.x, fp32)) && aligned16(b.a.w))
    return b.a.layer ? bwd_staged_any<T, true, KEPT>(b) : bwd_staged_any<T, false, KEPT>(b);
#define ROWS(G, UPT, R) return bwd_rows<T, 1, G, UPT, R, KEPT>(b)
  if (C <= 256) ROWS(32, 8, 4);
  if (C <= 512) ROWS(32, 16, 2);
  if (C <= 2048) ROWS(128, 16, 2);
  if (C <= 4096) ROWS(256, 16, 2);
  if (C <= 8192) ROWS(512, 16, 1);
#undef ROWS
  bwd_wide<T, KEPT>(b);
}

void bwd_any(const BwdCall& b) {
  if (b.a.fp32) b.k.codes != nullptr ? bwd<float, true>(b) : bwd<float, false>(b);
  else b.k.codes != nullptr ? bwd<__nv_bfloat16, true>(b) : bwd<__nv_bfloat16, false>(b);
}

}  // namespace

void launch_norm_fwd(const NormArgs& a, const RowsArg& x, void* y, float* stats, const Kept8Buf& k, cudaStream_t s) {
  if (a.rows <= 0) return;
  a.fp32 ? fwd<float>(a, x, y, stats, k, s) : fwd<__nv_bfloat16>(a, x, y, stats, k, s);
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
