// 8-bit kept activations (sm_100a): store, reload, the SwiGLU whose gate and value are kept in 8 bits,
// and the column sums that its neighbours' bias gradients need.  The format is in kept8.cuh.
//
// All kernels here are element streams bounded by DRAM.  Work is cut into fragments of V elements; the 32 / V lanes
// that hold one block of 32 agree on its scale by shuffles, so every input is read once.  Three forms:
//   V = 8   C % 8 == 0 and every row 16-byte aligned: 16-byte accesses
//   flat    contiguous tensors of any other width: tiles through shared memory (flat.cuh), fragments of 4 or 8
//   V = 1   what is left (odd views): one element a lane
#include "flat.cuh"
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
    if (act) kept8_store_code(at, x.f, b);
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

// A block's scale is the exponent of its largest |x|: four lanes agree on it by two exchanges, so x is read once.  Bound by
// DRAM (3.03 B an element in bf16, twice as many reads as writes): 110576 x 4096 240 us (5.7 TB/s), fp32 330 us
// (6.9 TB/s); odd widths through tiles 200001 x 1001 bf16 144 us (4.2 TB/s).  U = 4 fragments in flight a thread hide the latency.
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

// out [out_rows, ld] = x [rows, C] with zeros past C and past the rows, eight elements a thread (ld % 8 == 0).
__global__ void __launch_bounds__(kThreads) pad_rows_kernel(RowView x, Units un, uint32_t rows, int C,
                                                            __nv_bfloat16* __restrict__ out, long long ld) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= un.total) return;
  uint32_t row;
  int c;
  unit_at<8>(un, u, row, c);
  const __nv_bfloat16* p = row_ptr<__nv_bfloat16>(x, row < rows ? row : 0);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = row < rows && c + i < C ? to_f32(p[c + i]) : 0.f;
  store8(out + (long long)row * ld + c, v);
}

// code * step, exact in bf16, so one rounding-free store.  Bound by DRAM: 110576 x 4096 to bf16 232 us (5.9 TB/s), to fp32 430
// us (5.3 TB/s, where stores are four fifths of the bytes).
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
// s = 1 / (1 + exp(-g)) and 1 - s, to the type of the tensors.
//
// bf16: by the hardware's base-2 exponential and reciprocal.  Their errors and the rounding of g log2(e) reach s as a relative
// error of up to |g| 2^-24 (4e-6 at g = -80), far below the 2^-9 of the results' rounding.  What would be subnormal is 0: below g =
// -87.3 the results, under 1.1e-36 of the factors beside them, vanish (the forms that keep them take several instructions more).
//
// fp32: e = exp(-|g|) never overflows, and s or 1 - s = e / (1 + e) is formed without a difference: a few roundings of
// each, to the smallest numbers.  Forward / backward with the bf16 form and with this one: 8192 x 16384 279 / 285 and 283 / 285
// us, 30000 x 1001 90 / 98 and 98 / 98.
template <typename T>
__device__ __forceinline__ void sigmoid(float g, float& s, float& rest) {
  if constexpr (sizeof(T) == 2) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    rest = 1.f - s;
  } else {
    const float e = expf(-fabsf(g)), inv = 1.f / (1.f + e), low = e * inv;
    s = g >= 0.f ? inv : low;
    rest = g >= 0.f ? low : inv;
  }
}
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  float s, rest;
  sigmoid<T>(g, s, rest);
  return s;
}

// h = silu(g) * u; both inputs' codes are written beside it.  Bound by DRAM: 16384 x 16384 bf16 361 us (6.0 TB/s), the codes in
// packed pairs and the sigmoid in two hardware instructions to keep issue below it; 60000 x 1001 129 us (3.8 TB/s, tiles).
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
      a[i] = mul2(mul2(a[i], make_float2(sigmoid<T>(a[i].x), sigmoid<T>(a[i].y))), b[i]);
    store_values<T, V>(h + (long long)row[k] * og.C + c[k], a);
  }
}

// dg = dh u s (1 + g (1 - s)),  du = dh g s  with s = sigmoid(g) and g, u read from their codes;
// h, when asked for, is silu(g) u of the same values (the input of the projection that follows).  Bound by DRAM: 16384 x
// 16384 bf16 322 us without h (6.7 TB/s); 60000 x 1001 128 us (3.8 TB/s, tiles).
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
      float2 s, rest;
      sigmoid<T>(g[i].x, s.x, rest.x);
      sigmoid<T>(g[i].y, s.y, rest.y);
      const float2 ds = mul2(d[i], s);
      const float2 gs = mul2(g[i], s);
      const float2 slope = fma2(g[i], rest, twice(1.f));
      d[i] = mul2(ds, g[i]);
      o[i] = mul2(mul2(ds, w[i]), slope);
      w[i] = mul2(gs, w[i]);
    }
    store_values<T, V>(dgate + at, o);
    store_values<T, V>(dvalue + at, d);
    if (h != nullptr) store_values<T, V>(h + at, w);
  }
}

// ---------------------------------------------------------------- flat form
// A tile is 16 KB of whole rows, or of one row when that is longer.  Its fragments are (row, V columns) over rows padded
// to whole blocks, 32 / V lanes to a block.  V = 8 for bf16, where the kernels are bound by instructions: keep8 of 200001 x
// 1001 took 242 us with 4 columns and 8 KB tiles, 190 with 8, 172 with the packed encoding, 144 with 16 KB tiles whose ends are copied in parallel (4.2 TB/s).
// V = 4 for fp32, where 8 would read shared memory at half the rate.
constexpr int flat_v(bool fp32) { return fp32 ? 4 : 8; }
constexpr int flat_size(bool fp32) { return fp32 ? 4096 : 8192; }  // 16 KB
template <typename T>
constexpr bool is_fp32() { return sizeof(T) == 4; }

struct FlatTiles {
  FastDiv per_row, frag_row;  // tiles a row (1 unless rows are long), fragments a padded row of a tile
  int rows, C;                // rows a tile
  uint32_t total_rows;
};

struct FlatTile {
  uint32_t row0, rows;
  int c0, cols;      // columns c0 .. c0 + cols of every row
  uint32_t frags;    // fragments of the tile
};

template <typename T>
__device__ __forceinline__ FlatTile flat_tile(const FlatTiles& t) {
  constexpr int V = flat_v(is_fp32<T>()), SIZE = flat_size(is_fp32<T>());
  FlatTile f;
  if (t.rows > 1 || t.per_row.d == 1) {
    f.row0 = blockIdx.x * t.rows;
    f.rows = min((uint32_t)t.rows, t.total_rows - f.row0);
    f.c0 = 0;
    f.cols = t.C;
  } else {
    f.row0 = t.per_row.div(blockIdx.x);
    f.rows = 1;
    f.c0 = (int)(blockIdx.x - f.row0 * t.per_row.d) * SIZE;
    f.cols = min(SIZE, t.C - f.c0);
  }
  f.frags = f.rows * ((f.cols + kKeptBlock - 1) / kKeptBlock * (kKeptBlock / V));
  return f;
}

// Fragment u of the tile: its row (in the tile) and first column (in the tile).
template <int V>
__device__ __forceinline__ void flat_frag(const FlatTiles& t, const FlatTile& f, uint32_t u, uint32_t& r, int& c) {
  r = f.rows == 1 ? 0 : t.frag_row.div(u);
  c = (int)(u - r * t.frag_row.d) * V;
}

template <typename T, int V>
__device__ __forceinline__ void flat_read(const uint8_t* smem, const FlatTile& f, uint32_t r, int c, float (&v)[V]) {
  const T* p = reinterpret_cast<const T*>(smem) + r * f.cols + c;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = c + i < f.cols ? to_f32(p[i]) : 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void flat_write(uint8_t* smem, const FlatTile& f, uint32_t r, int c, const float (&v)[V]) {
  T* p = reinterpret_cast<T*>(smem) + r * f.cols + c;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (c + i < f.cols) p[i] = from_f32<T>(v[i]);
}

// Eight bf16 as they would lie in an aligned row.
__device__ __forceinline__ Frag<__nv_bfloat16> flat_frag8(const uint8_t* smem, const FlatTile& f, uint32_t r, int c) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(smem) + r * f.cols + c;
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = c + i < f.cols ? p[i] : 0u;
  Frag<__nv_bfloat16> x;
  x.raw = make_uint4(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410), __byte_perm(e[4], e[5], 0x5410),
                     __byte_perm(e[6], e[7], 0x5410));
  return x;
}

// Scale and codes of four columns; all lanes of the warp take part, `act` lanes store.
__device__ __forceinline__ void flat_keep(const Kept8Out& o, uint32_t row, int c, bool act, const float (&v)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < kKeptBlock / 4; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  const uint32_t b = kept8_byte(m);
  if (!act) return;
  const float inv = kept8_inv_step(b);
  *reinterpret_cast<uint32_t*>(o.codes + (long long)row * o.Cp + c) =
      pack4_low_bytes(kept8_code(v[0], inv), kept8_code(v[1], inv), kept8_code(v[2], inv), kept8_code(v[3], inv));
  if (c % kKeptBlock == 0) kept8_store_byte(o.scales + (long long)row * o.nbp, c / kKeptBlock, o.nb, o.nbp, b);
}

template <int V>
__device__ __forceinline__ void flat_values(const Kept8Out& k, uint32_t row, int c, float (&v)[V]) {
  const int8_t* at = k.codes + (long long)row * k.Cp + c;
  const float step = kept8_step(k.scales[(long long)row * k.nbp + c / kKeptBlock]);
  if constexpr (V == 8) {
    kept8_values(*reinterpret_cast<const uint2*>(at), step, v);
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(at) ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)) - 8388736.f) * step;
  }
}

template <typename T>
constexpr uint32_t flat_room() { return FlatRun<T>::room(flat_size(is_fp32<T>())); }
__device__ __forceinline__ void flat_wait() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
}
template <typename T>
__device__ __forceinline__ FlatRun<T> flat_run(const void* p, const FlatTiles& t, const FlatTile& f) {
  return FlatRun<T>(p, (long long)f.row0 * t.C + f.c0, f.rows * (uint32_t)f.cols);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) keep8_flat_kernel(const T* x, FlatTiles t, Kept8Out o, T* __restrict__ copy,
                                                              long long ld) {
  constexpr int V = flat_v(is_fp32<T>());
  __shared__ __align__(16) uint8_t sx[flat_room<T>()];
  const FlatTile f = flat_tile<T>(t);
  const FlatRun<T> run = flat_run<T>(x, t, f);
  run.fetch(sx);
  flat_wait();
  for (uint32_t u0 = 0; u0 < f.frags; u0 += kThreads) {  // whole warps: a block's lanes are in or out together
    const uint32_t u = u0 + threadIdx.x;
    const bool act = u < f.frags;
    uint32_t r;
    int c;
    flat_frag<V>(t, f, act ? u : 0, r, c);
    const uint32_t row = f.row0 + r;
    if constexpr (sizeof(T) == 2) {
      Piece<T, 8> piece;
      piece.f = flat_frag8(sx + run.head, f, r, c);
      keep_fragment<T, 8>(o, row, f.c0 + c, act, piece);
      if (copy != nullptr && act && f.c0 + c < ld) piece.store(copy + (long long)row * ld + f.c0 + c);  // ld % 8 == 0
    } else {
      float v[V];
      flat_read<T, V>(sx + run.head, f, r, c, v);
      flat_keep(o, row, f.c0 + c, act, v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) restore8_flat_kernel(FlatTiles t, Kept8Out k, T* __restrict__ out) {
  constexpr int V = flat_v(is_fp32<T>());
  __shared__ __align__(16) uint8_t so[flat_room<T>()];
  const FlatTile f = flat_tile<T>(t);
  const FlatRun<T> run = flat_run<T>(out, t, f);
#pragma unroll 2
  for (uint32_t u = threadIdx.x; u < f.frags; u += kThreads) {
    uint32_t r;
    int c;
    flat_frag<V>(t, f, u, r, c);
    float v[V];
    flat_values(k, f.row0 + r, f.c0 + c, v);
    flat_write<T, V>(so + run.head, f, r, c, v);
  }
  __syncthreads();
  run.store(so);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) swiglu_fwd_flat_kernel(const T* gate, const T* value, FlatTiles t,
                                                                   Kept8Out og, Kept8Out ov, T* __restrict__ h) {
  constexpr int V = flat_v(is_fp32<T>());
  __shared__ __align__(16) uint8_t sg[flat_room<T>()], sv[flat_room<T>()];
  const FlatTile f = flat_tile<T>(t);
  const FlatRun<T> rg = flat_run<T>(gate, t, f), rv = flat_run<T>(value, t, f), rh = flat_run<T>(h, t, f);
  rg.fetch(sg);
  rv.fetch(sv);
  flat_wait();
  for (uint32_t u0 = 0; u0 < f.frags; u0 += kThreads) {
    const uint32_t u = u0 + threadIdx.x;
    const bool act = u < f.frags;
    uint32_t r;
    int c;
    flat_frag<V>(t, f, act ? u : 0, r, c);
    if (!act) c = f.cols;  // reads nothing: the first fragment's thread writes h over its values meanwhile
    float g[V], v[V];
    if constexpr (sizeof(T) == 2) {
      Piece<T, 8> pg, pv;
      pg.f = flat_frag8(sg + rg.head, f, r, c);
      pv.f = flat_frag8(sv + rv.head, f, r, c);
      if (og.codes != nullptr) {
        keep_fragment<T, 8>(og, f.row0 + r, f.c0 + c, act, pg);
        keep_fragment<T, 8>(ov, f.row0 + r, f.c0 + c, act, pv);
      }
      float2 a[4], b[4];
      pg.get(a);
      pv.get(b);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[2 * i] = a[i].x, g[2 * i + 1] = a[i].y, v[2 * i] = b[i].x, v[2 * i + 1] = b[i].y;
    } else {
      flat_read<T, V>(sg + rg.head, f, r, c, g);
      flat_read<T, V>(sv + rv.head, f, r, c, v);
      if (og.codes != nullptr) {
        flat_keep(og, f.row0 + r, f.c0 + c, act, g);
        flat_keep(ov, f.row0 + r, f.c0 + c, act, v);
      }
    }
    if (!act) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= g[i] * sigmoid<T>(g[i]);
    flat_write<T, V>(sv + rv.head, f, r, c, v);  // h takes the place of value: same offsets, own elements
  }
  __syncthreads();
  rh.store(sv);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) swiglu_bwd_flat_kernel(const T* dh, Kept8Out kg, Kept8Out kv, FlatTiles t,
                                                                   T* __restrict__ dgate, T* __restrict__ dvalue,
                                                                   T* __restrict__ h) {
  constexpr int V = flat_v(is_fp32<T>());
  __shared__ __align__(16) uint8_t sd[flat_room<T>()], sv[flat_room<T>()];
  const FlatTile f = flat_tile<T>(t);
  const FlatRun<T> rd = flat_run<T>(dh, t, f);
  rd.fetch(sd);
  flat_wait();
  for (int pass = 0; pass < (h != nullptr ? 2 : 1); ++pass) {  // dgate over dh and dvalue; then h by itself
    for (uint32_t u = threadIdx.x; u < f.frags; u += kThreads) {
      uint32_t r;
      int c;
      flat_frag<V>(t, f, u, r, c);
      float g[V], w[V];
      flat_values(kg, f.row0 + r, f.c0 + c, g);
      flat_values(kv, f.row0 + r, f.c0 + c, w);
      if (pass == 0) {
        float d[V], o[V];
        flat_read<T, V>(sd + rd.head, f, r, c, d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float s, rest;
          sigmoid<T>(g[i], s, rest);
          const float ds = d[i] * s;
          o[i] = ds * w[i] * fmaf(g[i], rest, 1.f);
          d[i] = ds * g[i];
        }
        flat_write<T, V>(sd + rd.head, f, r, c, o);
        flat_write<T, V>(sv + rd.head, f, r, c, d);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] *= g[i] * sigmoid<T>(g[i]);
        flat_write<T, V>(sd + rd.head, f, r, c, w);
      }
    }
    __syncthreads();
    if (pass == 0) {
      flat_run<T>(dgate, t, f).store(sd);
      flat_run<T>(dvalue, t, f).store(sv);
      __syncthreads();
    } else {
      flat_run<T>(h, t, f).store(sd);
    }
  }
}

// ---------------------------------------------------------------- column sums
// A CTA sums a chunk of rows of 256 / TR column fragments, TR rows at a time; part[chunk, c] then goes to a second
// kernel unless there is one chunk.  A fixed order, no atomics.  Bias gradients of 4096 x 12288 bf16 41 us (2.5 TB/s),
// 32768 x 4096 89 us (3.0 TB/s), 777 x 1032 8.5 us: 0.4 to 0.5 of the copy rate, beside products that take several times as long.
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
void restore8_t(const Kept8Buf& k, long long row0, long long rows, void* out, long long ld, int cols, cudaStream_t s) {
  constexpr int U = V == 1 ? 8 : 4;
  Kept8Out o = out_of(k);
  o.C = cols;
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

// Whether `a` is a contiguous, 16-byte aligned tensor of rows of C.
bool contiguous_rows(const RowsArg& a, int C) {
  return a.inner == 1 && a.outer_stride == C && reinterpret_cast<uintptr_t>(a.p) % 16 == 0;
}

FlatTiles flat_tiles(long long rows, int C, bool fp32, uint32_t* grid) {
  FlatTiles t;
  const int size = flat_size(fp32), tiles = (C + size - 1) / size;
  t.per_row = FastDiv((uint32_t)tiles);
  t.rows = tiles > 1 ? 1 : size / C;
  t.C = C;
  t.frag_row = FastDiv((uint32_t)((tiles > 1 ? size : (C + kKeptBlock - 1) / kKeptBlock * kKeptBlock) / flat_v(fp32)));
  t.total_rows = (uint32_t)rows;
  *grid = tiles > 1 ? (uint32_t)rows * (uint32_t)tiles : (uint32_t)((rows + t.rows - 1) / t.rows);
  return t;
}
// Tiles are counted in 31 bits.
bool flat_fits(long long rows, int C) { return rows * ((C + 4095) / 4096) < (1ll << 31); }

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
  const bool vec = fragments_of_8(x, k.C, fp32);
  if (!vec && contiguous_rows(x, k.C) && flat_fits(rows, k.C)) {
    uint32_t grid;
    const FlatTiles t = flat_tiles(rows, k.C, fp32, &grid);
    if (fp32) keep8_flat_kernel<float><<<grid, kThreads, 0, s>>>((const float*)x.p, t, out_of(k), (float*)copy, ld);
    else keep8_flat_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>((const __nv_bfloat16*)x.p, t, out_of(k), (__nv_bfloat16*)copy, ld);
    return;
  }
#define CALL(T, V) keep8_t<T, V>(x, rows, k, copy, ld, s)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
}

void launch_restore8(const Kept8Buf& k, long long row0, long long rows, bool fp32, void* out, long long ld, int cols,
                     cudaStream_t s) {
  if (rows <= 0) return;
  const RowsArg o{out, ld, 0, 1};
  const bool vec = fragments_of_8(o, cols, fp32);
  if (!vec && cols == k.C && contiguous_rows(o, k.C) && flat_fits(rows, k.C)) {
    uint32_t grid;
    const FlatTiles t = flat_tiles(rows, k.C, fp32, &grid);
    Kept8Out from = out_of(k);
    from.codes += row0 * from.Cp;
    from.scales += row0 * from.nbp;
    if (fp32) restore8_flat_kernel<float><<<grid, kThreads, 0, s>>>(t, from, (float*)out);
    else restore8_flat_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(t, from, (__nv_bfloat16*)out);
    return;
  }
#define CALL(T, V) restore8_t<T, V>(k, row0, rows, out, ld, cols, s)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
}

void launch_swiglu_fwd(const RowsArg& g, const RowsArg& v, long long rows, bool fp32, const Kept8Buf& kg,
                       const Kept8Buf& kv, void* h, cudaStream_t s) {
  if (rows <= 0) return;
  const bool vec = fragments_of_8(g, kg.C, fp32) && fragments_of_8(v, kg.C, fp32);
  if (!vec && contiguous_rows(g, kg.C) && contiguous_rows(v, kg.C) && flat_fits(rows, kg.C)) {
    uint32_t grid;
    const FlatTiles t = flat_tiles(rows, kg.C, fp32, &grid);
    if (fp32)
      swiglu_fwd_flat_kernel<float><<<grid, kThreads, 0, s>>>((const float*)g.p, (const float*)v.p, t, out_of(kg),
                                                              out_of(kv), (float*)h);
    else
      swiglu_fwd_flat_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(
          (const __nv_bfloat16*)g.p, (const __nv_bfloat16*)v.p, t, out_of(kg), out_of(kv), (__nv_bfloat16*)h);
    return;
  }
#define CALL(T, V) swiglu_fwd_t<T, V>(g, v, rows, kg, kv, h, s)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
}

void launch_swiglu_bwd(const RowsArg& dh, long long rows, bool fp32, const Kept8Buf& kg, const Kept8Buf& kv, void* dg,
                       void* dv, void* h, cudaStream_t s) {
  if (rows <= 0) return;
  const bool vec = fragments_of_8(dh, kg.C, fp32);
  if (!vec && contiguous_rows(dh, kg.C) && flat_fits(rows, kg.C)) {
    uint32_t grid;
    const FlatTiles t = flat_tiles(rows, kg.C, fp32, &grid);
    if (fp32)
      swiglu_bwd_flat_kernel<float><<<grid, kThreads, 0, s>>>((const float*)dh.p, out_of(kg), out_of(kv), t, (float*)dg,
                                                              (float*)dv, (float*)h);
    else
      swiglu_bwd_flat_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>((const __nv_bfloat16*)dh.p, out_of(kg), out_of(kv),
                                                                      t, (__nv_bfloat16*)dg, (__nv_bfloat16*)dv,
                                                                      (__nv_bfloat16*)h);
    return;
  }
#define CALL(T, V) swiglu_bwd_t<T, V>(dh, rows, kg, kv, dg, dv, h, s)
  PAN_BY_TYPE(fp32, vec, CALL);
#undef CALL
}

void launch_pad_rows(const RowsArg& x, long long rows, int C, void* out, long long out_rows, long long ld,
                     cudaStream_t s) {
  over_rows<8, 1>(out_rows, (int)ld, [&](const Units& un, uint32_t grid) {
    pad_rows_kernel<<<grid, kThreads, 0, s>>>(view_of(x), un, (uint32_t)rows, C, (__nv_bfloat16*)out, ld);
  });
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
