// warp_mma.cuh -- warp-level matrix instructions (m16n8k16), their operand loads,
// and the shared-memory layouts of K and V tiles they read.
#pragma once

#include "device_utils.cuh"

namespace sm120n {

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Mma<__half> {
  __device__ __forceinline__ static void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}

// 16 bytes from global to shared memory, zeros where `real` is false.
__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem),
               "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Where 16-byte chunk c of a row lies. 16-bit tiles: the 8 rows of a matrix
// hit 8 different chunks. fp8 tiles: two neighbouring rows read 64 bytes each
// (K) and rows 0, 2, 4, 6 read 32 bytes each (V) at once.
template <int kChunks, bool kFp8>
__device__ __forceinline__ int chunk_at(int row, int c) {
  if constexpr (!kFp8) return row * kChunks + (c ^ (row & 7));
  if constexpr (kChunks == 4) return row * kChunks + (c ^ (((row >> 1) & 1) << 1));
  return row * kChunks + (c ^ ((((row ^ (row >> 1)) & 1) << 2) | (((row >> 2) & 1) << 1)));
}

}  // namespace sm120n
