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

  // global -> shared (asynchronous except for the end pieces); wait, then a barrier, before use
  __device__ __forceinline__ void fetch(uint8_t* smem) const {
    const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) {
      if (i >= head && i + 16 <= bytes) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s0 + i), "l"(base + i) : "memory");
      } else {
        const uint32_t b = i + 16 < bytes ? i + 16 : bytes;
        for (uint32_t j = i < head ? head : i; j < b; j += sizeof(T))
          *reinterpret_cast<T*>(smem + j) = *reinterpret_cast<const T*>(base + j);
      }
    }
  }
  // shared -> global, after a barrier
  __device__ __forceinline__ void store(const uint8_t* smem) const {
    uint8_t* out = const_cast<uint8_t*>(base);
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) {
      if (i >= head && i + 16 <= bytes) {
        *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(smem + i);
      } else {
        const uint32_t b = i + 16 < bytes ? i + 16 : bytes;
        for (uint32_t j = i < head ? head : i; j < b; j += sizeof(T))
          *reinterpret_cast<T*>(out + j) = *reinterpret_cast<const T*>(smem + j);
      }
    }
  }
};

}  // namespace pan
