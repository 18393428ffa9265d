// Layer norm and RMS norm with learned weight and bias, forward and backward (sm_100a).
//
//   n = (x - mean) * rstd,  y = n * w + b                (RMS norm: mean = 0, no b)
//   g = dy * w,  dx = rstd * (g - mean_c(g) - n * mean_c(g n))      (RMS norm without mean_c(g))
//   dw = sum_rows dy * n,  db = sum_rows dy
//
// Statistics are fp32 and two-pass (mean first, then the centred squares), so a large common offset
// does not cancel the variance away.  The backward reads x either as it was or from its 8-bit codes
// (kept8.cuh); mean and rstd are always those of the exact x.
#include "kept8.cuh"
#include "launchers.h"

namespace pan {
namespace {

constexpr int kThreads = 256;

// Sum over the CTA of one value per thread; every thread gets it.
__device__ __forceinline__ float cta_sum(float v) {
  __shared__ float ws[kThreads / 32];
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += ws[i];
  return t;
}

__device__ __forceinline__ float vec_at(const void* p, bool fp32, int c, float missing) {
  if (p == nullptr) return missing;
  return fp32 ? reinterpret_cast<const float*>(p)[c] : to_f32(reinterpret_cast<const __nv_bfloat16*>(p)[c]);
}

struct Kept {
  int8_t* codes;
  uint8_t* scales;
  int Cp, nb, nbp;
};

// One CTA per row, three sweeps over it (mean, variance, output).
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_fwd_kernel(RowView x, uint32_t rows, int C, const void* w,
                                                            const void* b, bool w_fp32, float eps, bool layer,
                                                            T* __restrict__ y, float* __restrict__ stats, Kept k) {
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
    if (stats != nullptr && threadIdx.x == 0) *reinterpret_cast<float2*>(stats + 2 * (size_t)r) = make_float2(mean, rstd);
    T* yr = y + (long long)r * C;
    for (int c = threadIdx.x; c < (k.codes != nullptr ? k.Cp : C); c += kThreads) {
      float v[1] = {c < C ? to_f32(xr[c]) : 0.f};
      if (k.codes != nullptr) {  // Cp % 32 == 0: warps stay whole
        const uint32_t sb = kept8_byte(kept8_amax<1>(v));
        kept8_store_codes<1>(k.codes + (long long)r * k.Cp + c, v, sb);
        if (c % kKeptBlock == 0) kept8_store_byte(k.scales + (long long)r * k.nbp, c / kKeptBlock, k.nb, k.nbp, sb);
      }
      if (c < C) yr[c] = from_f32<T>((v[0] - mean) * rstd * vec_at(w, w_fp32, c, 1.f) + vec_at(b, w_fp32, c, 0.f));
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
__global__ void __launch_bounds__(kThreads) norm_bwd_dx_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C,
                                                               const void* w, bool w_fp32, bool layer,
                                                               const float* __restrict__ stats, T* __restrict__ dx) {
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* gr = row_ptr<T>(dy, r);
    const T* xr = k.codes == nullptr ? row_ptr<T>(x, r) : nullptr;
    const float2 st = *reinterpret_cast<const float2*>(stats + 2 * (size_t)r);
    float a = 0.f, b = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float g = to_f32(gr[c]) * vec_at(w, w_fp32, c, 1.f);
      a += g;
      b += g * (x_at(xr, k, r, c) - st.x) * st.y;
    }
    a = layer ? cta_sum(a) / C : 0.f;
    b = cta_sum(b) / C;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float g = to_f32(gr[c]) * vec_at(w, w_fp32, c, 1.f);
      const float n = (x_at(xr, k, r, c) - st.x) * st.y;
      dx[(long long)r * C + c] = from_f32<T>(st.y * (g - a - n * b));
    }
  }
}

// part[chunk, 0, c] = sum of dy * n, part[chunk, 1, c] = sum of dy over a chunk of rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_bwd_partial_kernel(RowView dy, RowView x, Kept k, uint32_t rows, int C,
                                                                    const float* __restrict__ stats, uint32_t chunk,
                                                                    float* __restrict__ part) {
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

// dw[c], db[c]: the partial sums added in chunk order.
template <typename W>
__global__ void __launch_bounds__(kThreads) norm_bwd_final_kernel(const float* __restrict__ part, int parts, int C,
                                                                  W* __restrict__ dw, W* __restrict__ db) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  W* out = blockIdx.y == 0 ? dw : db;
  if (c >= C || out == nullptr) return;
  float acc = 0.f;
  for (int p = 0; p < parts; ++p) acc += part[((long long)p * 2 + blockIdx.y) * C + c];
  out[c] = from_f32<W>(acc);
}

RowView view_of(const RowsArg& a) { return RowView{a.p, a.outer_stride, a.inner_stride, FastDiv((uint32_t)a.inner)}; }

Kept kept_of(const Kept8Buf& b) {
  Kept k;
  k.codes = (int8_t*)b.codes;
  k.scales = (uint8_t*)b.scales;
  k.Cp = (b.C + kKeptBlock - 1) / kKeptBlock * kKeptBlock;
  k.nb = k.Cp / kKeptBlock;
  k.nbp = (k.nb + 3) / 4 * 4;
  return k;
}

uint32_t row_grid(long long rows) { return (uint32_t)(rows < 148 * 64 ? rows : 148 * 64); }

}  // namespace

void launch_norm_fwd(const NormArgs& a, const RowsArg& x, void* y, float* stats, const Kept8Buf& k, cudaStream_t s) {
  if (a.rows <= 0) return;
  const uint32_t grid = row_grid(a.rows);
  if (a.fp32)
    norm_fwd_kernel<float><<<grid, kThreads, 0, s>>>(view_of(x), a.rows, a.C, a.w, a.b, a.w_fp32, a.eps, a.layer,
                                                     (float*)y, stats, kept_of(k));
  else
    norm_fwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(view_of(x), a.rows, a.C, a.w, a.b, a.w_fp32, a.eps,
                                                             a.layer, (__nv_bfloat16*)y, stats, kept_of(k));
}

int norm_bwd_parts(const NormArgs& a) {
  const long long p = (a.rows + 127) / 128;
  return p < 1 ? 1 : (p > 1024 ? 1024 : (int)p);
}

void launch_norm_bwd(const NormArgs& a, const RowsArg& dy, const RowsArg& x, const Kept8Buf& k, const float* stats,
                     void* dx, float* part, int parts, void* dw, void* db, cudaStream_t s) {
  if (dx != nullptr && a.rows > 0) {
    if (a.fp32)
      norm_bwd_dx_kernel<float><<<row_grid(a.rows), kThreads, 0, s>>>(view_of(dy), view_of(x), kept_of(k), a.rows, a.C,
                                                                      a.w, a.w_fp32, a.layer, stats, (float*)dx);
    else
      norm_bwd_dx_kernel<__nv_bfloat16><<<row_grid(a.rows), kThreads, 0, s>>>(
          view_of(dy), view_of(x), kept_of(k), a.rows, a.C, a.w, a.w_fp32, a.layer, stats, (__nv_bfloat16*)dx);
  }
  if (dw == nullptr && db == nullptr) return;
  const uint32_t chunk = (uint32_t)((a.rows + parts - 1) / parts);
  const dim3 grid((a.C + kThreads - 1) / kThreads, parts);
  if (a.fp32)
    norm_bwd_partial_kernel<float><<<grid, kThreads, 0, s>>>(view_of(dy), view_of(x), kept_of(k), a.rows, a.C, stats,
                                                             chunk, part);
  else
    norm_bwd_partial_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(view_of(dy), view_of(x), kept_of(k), a.rows, a.C,
                                                                     stats, chunk, part);
  const dim3 fin(grid.x, 2);
  if (a.w_fp32) norm_bwd_final_kernel<float><<<fin, kThreads, 0, s>>>(part, parts, a.C, (float*)dw, (float*)db);
  else norm_bwd_final_kernel<__nv_bfloat16><<<fin, kThreads, 0, s>>>(part, parts, a.C, (__nv_bfloat16*)dw,
                                                                      (__nv_bfloat16*)db);
}

}  // namespace pan
