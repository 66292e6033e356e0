// What the kernels behind the encoder stem share (layernorm.hip, linear.hip, attention.hip):
// element types, 16-byte loads and stores at any element alignment, and one matrix step on
// 16-byte operand fragments.
#pragma once
#include "mia_internal.h"

namespace mia {
namespace nn {

typedef __bf16 bf16;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

// Rows of a view may start at any element, so 16-byte pieces are read and written through a type
// with the element's alignment: the same global_load_dwordx4 / global_store_dwordx4 (the memory
// system takes any 2- or 4-byte alignment), only never assumed aligned.
struct __attribute__((packed, aligned(2))) Raw16 {
  u4 v;
};

template <class T>
constexpr int kPer16 = 16 / (int)sizeof(T);

// Elements [0, n) of the 16-byte piece at p, zeros behind; n may be <= 0.  `room`: elements from p on that
// belong to the same array (its later rows): where that is a whole piece, a row's end costs one load and
// three masks; element by element (each a load of its own) only at the array's very end.
template <class T>
__device__ __forceinline__ u4 load_piece(const T* p, int n, long long room = 0) {
  constexpr int V = kPer16<T>;
  if (n >= V) return reinterpret_cast<const Raw16*>(p)->v;
  u4 x = u4{0, 0, 0, 0};
  if (n <= 0) return x;
  if (room >= V) {
    x = reinterpret_cast<const Raw16*>(p)->v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int bytes = n * (int)sizeof(T) - 4 * j;  // of this word inside
      x[j] = bytes >= 4 ? x[j] : bytes == 2 ? x[j] & 0xffffu : 0u;
    }
    return x;
  }
  union {
    u4 u;
    T e[V];
  } y;
  y.u = x;
#pragma unroll
  for (int j = 0; j < V - 1; ++j)
    if (j < n) y.e[j] = p[j];
  return y.u;
}
// PAST: the result goes past the caches (a nontemporal store).
template <class T, bool PAST = false>
__device__ __forceinline__ void store_piece(T* p, u4 v, int n) {
  constexpr int V = kPer16<T>;
  if (n >= V) {
    typedef u4 __attribute__((aligned(2))) u4a;
    if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<u4a*>(p));
    else reinterpret_cast<Raw16*>(p)->v = v;
    return;
  }
  union {
    u4 u;
    T e[V];
  } x;
  x.u = v;
#pragma unroll
  for (int j = 0; j < V - 1; ++j)
    if (j < n) p[j] = x.e[j];
}
template <class T>
__device__ __forceinline__ void unpack(u4 v, float* out) {
  union {
    u4 u;
    T e[kPer16<T>];
  } x;
  x.u = v;
#pragma unroll
  for (int j = 0; j < kPer16<T>; ++j) out[j] = (float)x.e[j];
}
// rounds to nearest, ties to even, like every conversion from float here
template <class T>
__device__ __forceinline__ u4 pack(const float* in) {
  union {
    u4 u;
    T e[kPer16<T>];
  } x;
#pragma unroll
  for (int j = 0; j < kPer16<T>; ++j) x.e[j] = (T)in[j];
  return x.u;
}

// One step of a 16 x 16 product over 64 bytes of each operand row (32 elements of 2 bytes, 16
// floats).  Lane l holds 16 bytes of row l & 15 of either operand: elements k = V (l >> 4) + j.  The
// result: column l & 15 (the second operand's row), rows 4 (l >> 4) + i (the first operand's).
// float runs four instructions of four k each: instruction j takes element j of both operands, so
// it sums k = j, 4 + j, 8 + j, 12 + j - the same k for both.
template <class T>
struct Mma;
template <>
struct Mma<_Float16> {
  static __device__ __forceinline__ f4 step(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16> {
  static __device__ __forceinline__ f4 step(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static __device__ __forceinline__ f4 step(u4 a, u4 b, f4 c) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[0], y[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[1], y[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[2], y[2], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x[3], y[3], c, 0, 0, 0);
  }
};

// Four 2-byte elements down a column of LDS: of the 16 lanes l & 15 of a group, lane j reads the 8
// bytes at `addr` (four columns of row j >> 2, quad j & 3) and receives column l & 15 of rows 0..3.
__device__ __forceinline__ s4 lds_read_column4(unsigned addr) {
  typedef __attribute__((address_space(3))) s4* lds_s4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(unsigned long long)addr);
}

// One wave-wide load into LDS: lane L's 16 bytes at gptr land at lds_byte_addr + 16 L.  No register
// receives data; the compiler does not count the load, so the kernel waits for it itself.
__device__ __forceinline__ void dma16(const void* gptr, unsigned lds_byte_addr) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(gptr), "s"(lds_byte_addr)
      : "memory");
}
// the same from a uniform base and a lane's unsigned byte offset: no address arithmetic per lane
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the compiler keeps nothing in it
__device__ __forceinline__ void dma16(const void* base, unsigned offset, unsigned lds_byte_addr) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %0"
      :
      : "s"(base), "v"(offset), "s"(lds_byte_addr)
      : "memory", "m0");
}
// either, of the lanes in `lanes` only; the others' places stay as they are
__device__ __forceinline__ void dma16(const void* base, unsigned offset, unsigned lds_byte_addr,
                                      unsigned long long lanes) {
  unsigned long long active;
  asm volatile(
      "s_mov_b32 m0, %3\n\t"
      "s_and_saveexec_b64 %0, %4\n\t"
      "global_load_lds_dwordx4 %2, %1\n\t"
      "s_mov_b64 exec, %0"
      : "=&s"(active)
      : "s"(base), "v"(offset), "s"(lds_byte_addr), "s"(lanes)
      : "memory", "m0", "scc");
}
__device__ __forceinline__ void dma16(const void* gptr, unsigned lds_byte_addr, unsigned long long lanes) {
  unsigned long long active;
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_and_saveexec_b64 %0, %3\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_mov_b64 exec, %0"
      : "=&s"(active)
      : "v"(gptr), "s"(lds_byte_addr), "s"(lanes)
      : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
// the same with 4 bytes a lane, at lds_byte_addr + 4 L
__device__ __forceinline__ void dma4(const void* gptr, unsigned lds_byte_addr) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(gptr), "s"(lds_byte_addr)
      : "memory");
}
// all but the newest N of this wave's vector loads have arrived, all its LDS operations are done
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
}
// A barrier that leaves loads into LDS in flight (__syncthreads would drain them).
__device__ __forceinline__ void barrier_keep_loads() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

static inline bool dtype_ok(int d) { return d == MIA_F32 || d == MIA_F16 || d == MIA_BF16; }
static inline size_t dtype_size(int d) { return d == MIA_F32 ? 4 : 2; }
static inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Calls f(T()) with the element type that `dtype` names.
template <class F>
static inline int with_dtype(int dtype, F f) {
  if (dtype == MIA_F32) return f(float());
  if (dtype == MIA_F16) return f((_Float16)0);
  return f((bf16)0.0f);
}

}  // namespace nn
}  // namespace mia
