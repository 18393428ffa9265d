// Contiguous rows whose width is no multiple of 16 bytes: the rows of a tile are one run of bytes, which
// moves between global and shared memory in aligned 16-byte pieces; single elements are touched only in shared
// memory, where their alignment costs nothing.  The run keeps its offset to a 16-byte boundary, so a
// piece is aligned on both sides; the pieces at the two ends, which share their 16 bytes with other tiles, go
// element by element.
#pragma once

#include "kept8.cuh"

namespace pan {

// The run of `count` elements of T from element `first` of a 16-byte aligned tensor.
template <typename T>
struct FlatRun {
  const uint8_t* base;   // aligned address at or below the first element
  uint32_t head, bytes;  // offset of the first element, and of the end, from base
  __device__ __forceinline__ FlatRun(const void* tensor, long long first, uint32_t count) {
    const long long at = first * (long long)sizeof(T);
    head = (uint32_t)(at & 15);
    base = reinterpret_cast<const uint8_t*>(tensor) + (at - head);
    bytes = head + count * (uint32_t)sizeof(T);
  }
  static constexpr uint32_t room(uint32_t count) { return (count * (uint32_t)sizeof(T) + 15 + 15) / 16 * 16; }

  // global -> shared, asynchronously: wait, then a barrier, before use.  The first piece brings its neighbour's bytes along (they
  // are the same tensor's); the last reads none past the run.  Taken element by element instead, the two end pieces
  // made every barrier wait for a chain of loads: layer norm backward of 141393 x 631 bf16 382 us, now 237.
  __device__ __forceinline__ void fetch(uint8_t* smem) const {
    const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
    const uint32_t whole = bytes & ~15u;
    for (uint32_t i = threadIdx.x * 16; i < whole; i += blockDim.x * 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s0 + i), "l"(base + i) : "memory");
    if (threadIdx.x == 0 && whole != bytes)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s0 + whole), "l"(base + whole),
                   "r"(bytes - whole) : "memory");
  }
  // shared -> global, after a barrier: the elements of the two end pieces one a lane of the last warp, the pieces between whole
  __device__ __forceinline__ void store(const uint8_t* smem) const {
    uint8_t* out = const_cast<uint8_t*>(base);
    if (threadIdx.x >= blockDim.x - 32) {
      const uint32_t lane = threadIdx.x & 31, j = (lane & 15) * (uint32_t)sizeof(T), tail = bytes & ~15u;
      const uint32_t i = lane < 16 ? j : tail + j;
      const bool mine = lane < 16 ? head != 0 && i >= head && i < bytes : (tail != 0 || head == 0) && i < bytes;
      if (j < 16 && mine) *reinterpret_cast<T*>(out + i) = *reinterpret_cast<const T*>(smem + i);
    }
    for (uint32_t i = threadIdx.x * 16; i + 16 <= bytes; i += blockDim.x * 16)
      if (i >= head) *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(smem + i);
  }
};

}  // namespace pan
