// 8-bit kept activations (sm_100a): store, reload, the SwiGLU whose gate and value are kept in 8 bits,
// and the column sums that its neighbours' bias gradients need.  The format is in kept8.cuh.
//
// All kernels here are element streams bounded by DRAM.  Work is cut into fragments of V elements
// (V = 8 when every row is 16-byte aligned and C % 8 == 0, V = 1 otherwise); the 32 / V lanes that
// hold one block of 32 agree on its scale by shuffles, so every input is read once.
#include "kept8.cuh"
#include "launchers.h"

namespace pan {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxUnits = 1u << 30;  // fragments per launch; larger tensors run as several launches

struct Kept8Out {
  int8_t* codes;
  uint8_t* scales;
  int C, Cp, nb, nbp;
};

// The row chunk of one launch: fragments of V elements over rows [row0, row0 + rows).
struct Units {
  uint32_t row0, total;
  FastDiv per_row;
};

template <int V>
__device__ __forceinline__ void unit_at(const Units& un, uint32_t u, uint32_t& row, int& c) {
  const uint32_t r = un.per_row.div(u);
  row = un.row0 + r;
  c = (int)(u - r * un.per_row.d) * V;
}

// Block maximum, scale byte and codes of one fragment of (row, c); `act` lanes store.
template <int V>
__device__ __forceinline__ void keep_fragment(const Kept8Out& o, uint32_t row, int c, bool act, const float (&v)[V]) {
  const uint32_t b = kept8_byte(kept8_amax<V>(v));
  if (!act) return;
  kept8_store_codes<V>(o.codes + (long long)row * o.Cp + c, v, b);
  if (c % kKeptBlock == 0) kept8_store_byte(o.scales + (long long)row * o.nbp, c / kKeptBlock, o.nb, o.nbp, b);
}

template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) keep8_kernel(RowView x, Units un, Kept8Out o) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
  float v[U][V];
  uint32_t row[U];
  int c[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    unit_at<V>(un, u, row[k], c[k]);
    if (u < un.total && c[k] < o.C) {
      load_v<T, V>(row_ptr<T>(x, row[k]) + c[k], v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) keep_fragment<V>(o, row[k], c[k], u0 + k * kThreads < un.total, v[k]);
}

template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) restore8_kernel(const int8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, Units un, int C, int Cp,
                                                            int nbp, T* __restrict__ out, long long ld) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    uint32_t row;
    int c;
    unit_at<V>(un, u, row, c);
    if (u >= un.total || c >= C) continue;
    float v[V];
    kept8_load<V>(codes + (long long)row * Cp + c, scales[(long long)row * nbp + c / kKeptBlock], v);
    store_v<T, V>(out + (long long)row * ld + c, v);
  }
}

// ---------------------------------------------------------------- SwiGLU
// h = silu(g) * u; both inputs' codes are written beside it.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) swiglu_fwd_kernel(RowView gate, RowView value, Units un, Kept8Out og,
                                                              Kept8Out ov, T* __restrict__ h) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    uint32_t row;
    int c;
    unit_at<V>(un, u, row, c);
    float g[V], w[V];
    const bool in = u < un.total && c < og.C;
    if (in) {
      load_v<T, V>(row_ptr<T>(gate, row) + c, g);
      load_v<T, V>(row_ptr<T>(value, row) + c, w);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = w[i] = 0.f;
    }
    if (og.codes != nullptr) {
      keep_fragment<V>(og, row, c, u < un.total, g);
      keep_fragment<V>(ov, row, c, u < un.total, w);
    }
    if (in) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = g[i] / (1.f + expf(-g[i])) * w[i];
      store_v<T, V>(h + (long long)row * og.C + c, o);
    }
  }
}

// dg = dh u s (1 + g (1 - s)),  du = dh g s  with s = sigmoid(g) and g, u read from their codes;
// h, when asked for, is silu(g) u of the same values (the input of the projection that follows).
template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) swiglu_bwd_kernel(RowView dh, Kept8Out kg, Kept8Out kv, Units un,
                                                              T* __restrict__ dgate, T* __restrict__ dvalue,
                                                              T* __restrict__ h) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    uint32_t row;
    int c;
    unit_at<V>(un, u, row, c);
    if (u >= un.total || c >= kg.C) continue;
    float d[V], g[V], w[V], dg[V], dv[V];
    load_v<T, V>(row_ptr<T>(dh, row) + c, d);
    kept8_load<V>(kg.codes + (long long)row * kg.Cp + c, kg.scales[(long long)row * kg.nbp + c / kKeptBlock], g);
    kept8_load<V>(kv.codes + (long long)row * kv.Cp + c, kv.scales[(long long)row * kv.nbp + c / kKeptBlock], w);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = 1.f / (1.f + expf(-g[i]));
      dg[i] = d[i] * w[i] * s * (1.f + g[i] * (1.f - s));
      dv[i] = d[i] * g[i] * s;
      w[i] *= g[i] * s;
    }
    const long long at = (long long)row * kg.C + c;
    store_v<T, V>(dgate + at, dg);
    store_v<T, V>(dvalue + at, dv);
    if (h != nullptr) store_v<T, V>(h + at, w);
  }
}

// ---------------------------------------------------------------- column sums
// part[chunk, c] = sum of a chunk of rows, then out[c] = sum over chunks: a fixed order, no atomics.
template <typename T>
__global__ void __launch_bounds__(kThreads) column_partial_kernel(RowView x, uint32_t rows, int C, uint32_t chunk,
                                                                  float* __restrict__ part) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= C) return;
  const uint32_t r1 = min(rows, (blockIdx.y + 1) * chunk);
  float acc = 0.f;
  for (uint32_t r = blockIdx.y * chunk; r < r1; ++r) acc += to_f32(row_ptr<T>(x, r)[c]);
  part[(long long)blockIdx.y * C + c] = acc;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) column_final_kernel(const float* __restrict__ part, int parts, int C,
                                                                T* __restrict__ out) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= C) return;
  float acc = 0.f;
  for (int p = 0; p < parts; ++p) acc += part[(long long)p * C + c];
  out[c] = from_f32<T>(acc);
}

// Runs `launch(units, grid)` over row chunks of at most kMaxUnits fragments.
template <int V, int U, typename F>
void over_rows(long long rows, int cols, F&& launch) {
  const uint32_t per_row = (uint32_t)((cols + V - 1) / V);
  const long long chunk = kMaxUnits / per_row;
  for (long long r0 = 0; r0 < rows; r0 += chunk) {
    Units un;
    un.row0 = (uint32_t)r0;
    un.per_row = FastDiv(per_row);
    un.total = (uint32_t)((rows - r0 < chunk ? rows - r0 : chunk) * per_row);
    launch(un, (un.total + kThreads * U - 1) / (kThreads * U));
  }
}

Kept8Out out_of(const Kept8Buf& k) {
  Kept8Out o;
  o.codes = (int8_t*)k.codes;
  o.scales = (uint8_t*)k.scales;
  o.C = k.C;
  o.Cp = (k.C + kKeptBlock - 1) / kKeptBlock * kKeptBlock;
  o.nb = o.Cp / kKeptBlock;
  o.nbp = (o.nb + 3) / 4 * 4;
  return o;
}

RowView view_of(const RowsArg& a) { return RowView{a.p, a.outer_stride, a.inner_stride, FastDiv((uint32_t)a.inner)}; }

template <typename T, int V>
void keep8_t(const RowsArg& x, long long rows, const Kept8Buf& k, cudaStream_t s) {
  constexpr int U = V == 1 ? 8 : 4;
  const Kept8Out o = out_of(k);
  over_rows<V, U>(rows, o.Cp, [&](const Units& un, uint32_t grid) {
    keep8_kernel<T, V, U><<<grid, kThreads, 0, s>>>(view_of(x), un, o);
  });
}

template <typename T, int V>
void restore8_t(const Kept8Buf& k, long long row0, long long rows, void* out, long long ld, cudaStream_t s) {
  constexpr int U = V == 1 ? 8 : 4;
  const Kept8Out o = out_of(k);
  const int8_t* codes = o.codes + row0 * o.Cp;
  const uint8_t* scales = o.scales + row0 * o.nbp;
  over_rows<V, U>(rows, o.Cp, [&](const Units& un, uint32_t grid) {
    restore8_kernel<T, V, U><<<grid, kThreads, 0, s>>>(codes, scales, un, o.C, o.Cp, o.nbp, (T*)out, ld);
  });
}

template <typename T, int V>
void swiglu_fwd_t(const RowsArg& g, const RowsArg& v, long long rows, const Kept8Buf& kg, const Kept8Buf& kv, void* h,
                  cudaStream_t s) {
  constexpr int U = V == 1 ? 4 : 1;
  const Kept8Out a = out_of(kg), b = out_of(kv);
  over_rows<V, U>(rows, a.Cp, [&](const Units& un, uint32_t grid) {
    swiglu_fwd_kernel<T, V, U><<<grid, kThreads, 0, s>>>(view_of(g), view_of(v), un, a, b, (T*)h);
  });
}

template <typename T, int V>
void swiglu_bwd_t(const RowsArg& dh, long long rows, const Kept8Buf& kg, const Kept8Buf& kv, void* dg, void* dv, void* h,
                  cudaStream_t s) {
  constexpr int U = V == 1 ? 4 : 1;
  const Kept8Out a = out_of(kg), b = out_of(kv);
  over_rows<V, U>(rows, a.Cp, [&](const Units& un, uint32_t grid) {
    swiglu_bwd_kernel<T, V, U><<<grid, kThreads, 0, s>>>(view_of(dh), a, b, un, (T*)dg, (T*)dv, (T*)h);
  });
}

// 16-byte fragments: C in whole fragments and every row start aligned.
bool fragments_of_8(const RowsArg& a, int C, bool fp32) {
  const int e = fp32 ? 4 : 2;
  return C % 8 == 0 && reinterpret_cast<uintptr_t>(a.p) % 16 == 0 && a.outer_stride * e % 16 == 0 &&
         a.inner_stride * e % 16 == 0;
}

}  // namespace

#define PAN_BY_TYPE(fp32, vec, CALL)                       \
  do {                                                     \
    if (fp32) {                                            \
      if (vec) CALL(float, 8); else CALL(float, 1);        \
    } else {                                               \
      if (vec) CALL(__nv_bfloat16, 8);                     \
      else CALL(__nv_bfloat16, 1);                         \
    }                                                      \
  } while (0)

void launch_keep8(const RowsArg& x, long long rows, bool fp32, const Kept8Buf& k, cudaStream_t s) {
  if (rows <= 0) return;
#define CALL(T, V) keep8_t<T, V>(x, rows, k, s)
  PAN_BY_TYPE(fp32, fragments_of_8(x, k.C, fp32), CALL);
#undef CALL
}

void launch_restore8(const Kept8Buf& k, long long row0, long long rows, bool fp32, void* out, long long ld,
                     cudaStream_t s) {
  if (rows <= 0) return;
  const RowsArg o{out, ld, 0, 1};
#define CALL(T, V) restore8_t<T, V>(k, row0, rows, out, ld, s)
  PAN_BY_TYPE(fp32, fragments_of_8(o, k.C, fp32), CALL);
#undef CALL
}

void launch_swiglu_fwd(const RowsArg& g, const RowsArg& v, long long rows, bool fp32, const Kept8Buf& kg,
                       const Kept8Buf& kv, void* h, cudaStream_t s) {
  if (rows <= 0) return;
  const bool vec = fragments_of_8(g, kg.C, fp32) && fragments_of_8(v, kg.C, fp32);
#define CALL(T, V) swiglu_fwd_t<T, V>(g, v, rows, kg, kv, h, s)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
}

void launch_swiglu_bwd(const RowsArg& dh, long long rows, bool fp32, const Kept8Buf& kg, const Kept8Buf& kv, void* dg,
                       void* dv, void* h, cudaStream_t s) {
  if (rows <= 0) return;
#define CALL(T, V) swiglu_bwd_t<T, V>(dh, rows, kg, kv, dg, dv, h, s)
  PAN_BY_TYPE(fp32, fragments_of_8(dh, kg.C, fp32), CALL);
#undef CALL
}

int column_sum_parts(long long rows) {
  const long long p = (rows + 127) / 128;
  return p < 1 ? 1 : (p > 1024 ? 1024 : (int)p);
}

void launch_column_sum(const RowsArg& x, long long rows, int C, bool fp32, float* part, int parts, void* out,
                       bool out_fp32, cudaStream_t s) {
  const uint32_t chunk = (uint32_t)((rows + parts - 1) / parts);
  const uint32_t gx = (C + kThreads - 1) / kThreads;
  if (fp32) column_partial_kernel<float><<<dim3(gx, parts), kThreads, 0, s>>>(view_of(x), rows, C, chunk, part);
  else column_partial_kernel<__nv_bfloat16><<<dim3(gx, parts), kThreads, 0, s>>>(view_of(x), rows, C, chunk, part);
  if (out_fp32) column_final_kernel<float><<<gx, kThreads, 0, s>>>(part, parts, C, (float*)out);
  else column_final_kernel<__nv_bfloat16><<<gx, kThreads, 0, s>>>(part, parts, C, (__nv_bfloat16*)out);
}

}  // namespace pan
