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

// A fragment in registers: V = 8 as it lies in memory, V = 1 as one fp32.
template <typename T, int V>
struct Piece {
  Frag<T> f;
  __device__ __forceinline__ void load(const T* p) { f.load(p); }
  __device__ __forceinline__ void zero() { f.zero(); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const { f.get(v); }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = f.raw;
    } else {
      reinterpret_cast<float4*>(p)[0] = f.raw[0];
      reinterpret_cast<float4*>(p)[1] = f.raw[1];
    }
  }
};
template <typename T>
struct Piece<T, 1> {
  float f;
  __device__ __forceinline__ void load(const T* p) { f = to_f32(*p); }
  __device__ __forceinline__ void zero() { f = 0.f; }
  __device__ __forceinline__ void get(float2 (&v)[1]) const { v[0] = make_float2(f, 0.f); }
  __device__ __forceinline__ void store(T* p) const { *p = from_f32<T>(f); }
};
constexpr int pairs_of(int V) { return V == 8 ? 4 : 1; }

// V results; V = 1 has one in the pair's first half.
template <typename T, int V>
__device__ __forceinline__ void store_values(T* p, const float2 (&v)[pairs_of(V)]) {
  if constexpr (V == 8) store_pairs(p, v);
  else *p = from_f32<T>(v[0].x);
}

// Block maximum, scale byte and codes of one fragment of (row, c); `act` lanes store.
template <typename T, int V>
__device__ __forceinline__ void keep_fragment(const Kept8Out& o, uint32_t row, int c, bool act, const Piece<T, V>& x) {
  uint32_t b;
  int8_t* at = o.codes + (long long)row * o.Cp + c;
  if constexpr (V == 8) {
    uint2 codes;
    kept8_encode(x.f, b, codes);
    if (act) *reinterpret_cast<uint2*>(at) = codes;
  } else {
    const float v[1] = {x.f};
    b = kept8_byte(kept8_amax<1>(v));
    if (act) kept8_store_codes<1>(at, v, b);
  }
  if (act && c % kKeptBlock == 0) kept8_store_byte(o.scales + (long long)row * o.nbp, c / kKeptBlock, o.nb, o.nbp, b);
}

template <int V>
__device__ __forceinline__ void kept_pairs(const Kept8Out& k, uint32_t row, int c, float2 (&v)[pairs_of(V)]) {
  const int8_t* p = k.codes + (long long)row * k.Cp + c;
  const float step = kept8_step(k.scales[(long long)row * k.nbp + c / kKeptBlock]);
  if constexpr (V == 8) kept8_values(*reinterpret_cast<const uint2*>(p), step, v);
  else v[0] = make_float2(kept8_number(*p) * step, 0.f);
}

// `copy`, when given, also gets x itself with rows of `ld` elements and zeros past C: the operand that a
// GEMM can read of rows that are not 16-byte aligned.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) keep8_kernel(RowView x, Units un, Kept8Out o, T* __restrict__ copy,
                                                         long long ld) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
  Piece<T, V> v[U];
  uint32_t row[U];
  int c[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    unit_at<V>(un, u, row[k], c[k]);
    if (u < un.total && c[k] < o.C) v[k].load(row_ptr<T>(x, row[k]) + c[k]);
    else v[k].zero();
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool act = u0 + k * kThreads < un.total;
    keep_fragment<T, V>(o, row[k], c[k], act, v[k]);
    if (copy != nullptr && act && c[k] < ld) v[k].store(copy + (long long)row[k] * ld + c[k]);
  }
}

// out [rows, ld] = x [rows, C] with zeros past C, eight elements a thread (ld % 8 == 0).
__global__ void __launch_bounds__(kThreads) pad_rows_kernel(RowView x, Units un, int C,
                                                            __nv_bfloat16* __restrict__ out, long long ld) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= un.total) return;
  uint32_t row;
  int c;
  unit_at<8>(un, u, row, c);
  const __nv_bfloat16* p = row_ptr<__nv_bfloat16>(x, row);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < C ? to_f32(p[c + i]) : 0.f;
  store8(out + (long long)row * ld + c, v);
}

template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) restore8_kernel(Units un, Kept8Out k8, T* __restrict__ out, long long ld) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    uint32_t row;
    int c;
    unit_at<V>(un, u, row, c);
    if (u >= un.total || c >= k8.C) continue;
    float2 v[pairs_of(V)];
    kept_pairs<V>(k8, row, c, v);
    store_values<T, V>(out + (long long)row * ld + c, v);
  }
}

// ---------------------------------------------------------------- SwiGLU
// 1 / (1 + exp(-g)) by the hardware's base-2 exponential and reciprocal: their errors, and |g| 2^-24 from the
// product with log2(e), reach the result times s (1 - s), below 2^-22 everywhere.  exp(-g) = inf gives 0.
__device__ __forceinline__ float sigmoid_fast(float g) {
  float e, s;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}

// h = silu(g) * u; both inputs' codes are written beside it.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kThreads) swiglu_fwd_kernel(RowView gate, RowView value, Units un, Kept8Out og,
                                                              Kept8Out ov, T* __restrict__ h) {
  const uint32_t u0 = blockIdx.x * (kThreads * U) + threadIdx.x;
  Piece<T, V> g[U], w[U];
  uint32_t row[U];
  int c[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const uint32_t u = u0 + k * kThreads;
    unit_at<V>(un, u, row[k], c[k]);
    if (u < un.total && c[k] < og.C) {
      g[k].load(row_ptr<T>(gate, row[k]) + c[k]);
      w[k].load(row_ptr<T>(value, row[k]) + c[k]);
    } else {
      g[k].zero();
      w[k].zero();
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool act = u0 + k * kThreads < un.total;
    if (og.codes != nullptr) {
      keep_fragment<T, V>(og, row[k], c[k], act, g[k]);
      keep_fragment<T, V>(ov, row[k], c[k], act, w[k]);
    }
    if (!act || c[k] >= og.C) continue;
    float2 a[pairs_of(V)], b[pairs_of(V)];
    g[k].get(a);
    w[k].get(b);
#pragma unroll
    for (int i = 0; i < pairs_of(V); ++i)
      a[i] = mul2(mul2(a[i], make_float2(sigmoid_fast(a[i].x), sigmoid_fast(a[i].y))), b[i]);
    store_values<T, V>(h + (long long)row[k] * og.C + c[k], a);
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
    Piece<T, V> piece;
    piece.load(row_ptr<T>(dh, row) + c);
    float2 d[pairs_of(V)], g[pairs_of(V)], w[pairs_of(V)];
    kept_pairs<V>(kg, row, c, g);
    kept_pairs<V>(kv, row, c, w);
    piece.get(d);
    const long long at = (long long)row * kg.C + c;
    float2 o[pairs_of(V)];
#pragma unroll
    for (int i = 0; i < pairs_of(V); ++i) {
      const float2 s = make_float2(sigmoid_fast(g[i].x), sigmoid_fast(g[i].y));
      const float2 ds = mul2(d[i], s);
      const float2 gs = mul2(g[i], s);
      const float2 slope = fma2(g[i], fma2(s, twice(-1.f), twice(1.f)), twice(1.f));
      d[i] = mul2(ds, g[i]);
      o[i] = mul2(mul2(ds, w[i]), slope);
      w[i] = mul2(gs, w[i]);
    }
    store_values<T, V>(dgate + at, o);
    store_values<T, V>(dvalue + at, d);
    if (h != nullptr) store_values<T, V>(h + at, w);
  }
}

// ---------------------------------------------------------------- column sums
// A CTA sums a chunk of rows of 256 / TR column fragments, TR rows at a time; part[chunk, c] then goes to a second
// kernel unless there is one chunk.  A fixed order, no atomics.
template <typename T>
__device__ __forceinline__ void put(void* out, int c, float v) { reinterpret_cast<T*>(out)[c] = from_f32<T>(v); }

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) column_partial_kernel(RowView x, uint32_t rows, int C, uint32_t chunk,
                                                                  float* __restrict__ part, void* out, bool out_fp32) {
  constexpr int TC = V == 8 ? 8 : 32, TR = kThreads / TC;
  __shared__ float sum[TR][TC * V + 1];
  const int tc = threadIdx.x % TC, tr = threadIdx.x / TC, c = (blockIdx.x * TC + tc) * V;
  const uint32_t r1 = min(rows, (blockIdx.y + 1) * chunk);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (c < C) {
#pragma unroll 4
    for (uint32_t r = blockIdx.y * chunk + tr; r < r1; r += TR) {
      float v[V];
      load_v<T, V>(row_ptr<T>(x, r) + c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum[tr][tc * V + i] = acc[i];
  __syncthreads();
  const int col = blockIdx.x * TC * V + threadIdx.x;
  if (threadIdx.x >= TC * V || col >= C) return;
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < TR; ++i) total += sum[i][threadIdx.x];
  if (gridDim.y > 1) part[(long long)blockIdx.y * C + col] = total;
  else if (out_fp32) put<float>(out, col, total);
  else put<__nv_bfloat16>(out, col, total);
}

__global__ void __launch_bounds__(kThreads) column_final_kernel(const float* __restrict__ part, int parts, int C,
                                                                void* out, bool out_fp32) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= C) return;
  float acc = 0.f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) acc += part[(long long)p * C + c];
  if (out_fp32) put<float>(out, c, acc);
  else put<__nv_bfloat16>(out, c, acc);
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
void keep8_t(const RowsArg& x, long long rows, const Kept8Buf& k, void* copy, long long ld, cudaStream_t s) {
  constexpr int U = V == 1 ? 8 : 4;
  const Kept8Out o = out_of(k);
  over_rows<V, U>(rows, o.Cp, [&](const Units& un, uint32_t grid) {
    keep8_kernel<T, V, U><<<grid, kThreads, 0, s>>>(view_of(x), un, o, (T*)copy, ld);
  });
}

template <typename T, int V>
void restore8_t(const Kept8Buf& k, long long row0, long long rows, void* out, long long ld, cudaStream_t s) {
  constexpr int U = V == 1 ? 8 : 4;
  Kept8Out o = out_of(k);
  o.codes += row0 * o.Cp;
  o.scales += row0 * o.nbp;
  over_rows<V, U>(rows, o.Cp, [&](const Units& un, uint32_t grid) {
    restore8_kernel<T, V, U><<<grid, kThreads, 0, s>>>(un, o, (T*)out, ld);
  });
}

template <typename T, int V>
void swiglu_fwd_t(const RowsArg& g, const RowsArg& v, long long rows, const Kept8Buf& kg, const Kept8Buf& kv, void* h,
                  cudaStream_t s) {
  constexpr int U = V == 1 ? 4 : 2;
  const Kept8Out a = out_of(kg), b = out_of(kv);
  over_rows<V, U>(rows, a.Cp, [&](const Units& un, uint32_t grid) {
    swiglu_fwd_kernel<T, V, U><<<grid, kThreads, 0, s>>>(view_of(g), view_of(v), un, a, b, (T*)h);
  });
}

template <typename T, int V>
void swiglu_bwd_t(const RowsArg& dh, long long rows, const Kept8Buf& kg, const Kept8Buf& kv, void* dg, void* dv, void* h,
                  cudaStream_t s) {
  constexpr int U = V == 1 ? 4 : 2;
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

void launch_keep8(const RowsArg& x, long long rows, bool fp32, const Kept8Buf& k, void* copy, long long ld,
                  cudaStream_t s) {
  if (rows <= 0) return;
#define CALL(T, V) keep8_t<T, V>(x, rows, k, copy, ld, s)
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

void launch_pad_rows(const RowsArg& x, long long rows, int C, void* out, long long ld, cudaStream_t s) {
  const uint32_t per_row = (uint32_t)(ld / 8);
  const long long chunk = kMaxUnits / per_row;
  for (long long r0 = 0; r0 < rows; r0 += chunk) {
    Units un;
    un.row0 = (uint32_t)r0;
    un.per_row = FastDiv(per_row);
    un.total = (uint32_t)((rows - r0 < chunk ? rows - r0 : chunk) * per_row);
    pad_rows_kernel<<<(un.total + kThreads - 1) / kThreads, kThreads, 0, s>>>(view_of(x), un, C, (__nv_bfloat16*)out, ld);
  }
}

// One chunk (and one launch) up to 1024 rows; beyond, as many as fill the GPU about four times with chunks of at
// least 256 rows.
int column_sum_parts(long long rows, int C) {
  if (rows <= 1024) return 1;
  const long long ctas = (C + 63) / 64, want = (4 * 148 + ctas - 1) / ctas, most = (rows + 255) / 256;
  return (int)(want < most ? want : most);
}

void launch_column_sum(const RowsArg& x, long long rows, int C, bool fp32, float* part, int parts, void* out,
                       bool out_fp32, cudaStream_t s) {
  const uint32_t chunk = (uint32_t)((rows + parts - 1) / parts);
  const bool vec = fragments_of_8(x, C, fp32);
  const dim3 grid((uint32_t)(vec ? (C + 63) / 64 : (C + 31) / 32), (uint32_t)parts);
#define CALL(T, V) \
  column_partial_kernel<T, V><<<grid, kThreads, 0, s>>>(view_of(x), (uint32_t)rows, C, chunk, part, out, out_fp32)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
  if (parts > 1)
    column_final_kernel<<<(C + kThreads - 1) / kThreads, kThreads, 0, s>>>(part, parts, C, out, out_fp32);
}

}  // namespace pan
