// m3g_serve.cuh -- what the serving operators share: activation types, the
// planes of the quantised KV cache, and the checked view of a batch.
#pragma once
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/m3gemv.h"
#include "m3g_internal.h"

namespace m3g {
int host_fail(int code, const char* fmt, ...);

// ---------------------------------------------------------------- activations
template <class T> struct Act;
template <> struct Act<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Act<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct Act<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// A vector's values as f32 and back, two 16-bit values to a conversion.
template <class T, int N>
__device__ __forceinline__ void unpack_act(const T (&t)[N], float (&v)[N]) {
  if constexpr (std::is_same<T, __half>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 f = __half22float2(__halves2half2(t[i], t[i + 1]));
      v[i] = f.x;
      v[i + 1] = f.y;
    }
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 f = __bfloat1622float2(__halves2bfloat162(t[i], t[i + 1]));
      v[i] = f.x;
      v[i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<T>::to(t[i]);
  }
}
template <class T, int N>
__device__ __forceinline__ void pack_act(T (&t)[N], const float (&v)[N]) {
  if constexpr (std::is_same<T, __half>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
      t[i] = __low2half(h);
      t[i + 1] = __high2half(h);
    }
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
      t[i] = __low2bfloat16(h);
      t[i + 1] = __high2bfloat16(h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = Act<T>::from(v[i]);
  }
}

// N consecutive values; VEC: their address is a multiple of 16 bytes (of N * sizeof(T) where that is less).
template <class T, int N, bool VEC>
__device__ __forceinline__ void load_act(const T* p, float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16, E = B / sizeof(T);
    union { uint4 q; uint2 d; T t[E]; } u;
#pragma unroll
    for (int i = 0; i < N; i += E) {
      if constexpr (B == 16) u.q = *reinterpret_cast<const uint4*>(p + i);
      else u.d = *reinterpret_cast<const uint2*>(p + i);
#pragma unroll
      for (int j = 0; j < E; ++j) v[i + j] = Act<T>::to(u.t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<T>::to(p[i]);
  }
}
template <class T, int N, bool VEC>
__device__ __forceinline__ void store_act(T* p, const float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int B = N * sizeof(T) < 16 ? N * sizeof(T) : 16, E = B / sizeof(T);
    union U { uint4 q; uint2 d; T t[E]; __device__ U() {} } u;
#pragma unroll
    for (int i = 0; i < N; i += E) {
#pragma unroll
      for (int j = 0; j < E; ++j) u.t[j] = Act<T>::from(v[i + j]);
      if constexpr (B == 16) *reinterpret_cast<uint4*>(p + i) = u.q;
      else *reinterpret_cast<uint2*>(p + i) = u.d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = Act<T>::from(v[i]);
  }
}

// 16 bytes from global to shared memory without registers, the last 16 - bytes of them zeros.
__device__ __forceinline__ void cp16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

inline int act_size(uint32_t dtype) {
  return dtype == M3G_DTYPE_F32 ? 4 : (dtype == M3G_DTYPE_F16 || dtype == M3G_DTYPE_BF16) ? 2 : 0;
}

// Whether rows of `size`-byte values at p, `strides` apart, all start on 16-byte boundaries.
inline bool rows_aligned(const void* p, int64_t token_stride, int64_t head_stride, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token_stride * size % 16 == 0 && head_stride * size % 16 == 0;
}

// A pointer that is not a multiple of its elements' size (an access would fault).
inline bool misaligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// The current device and its status word for these operators.
inline int serve_device(int* dev, uint32_t** status) {
  if (cudaGetDevice(dev) != cudaSuccess) return host_fail(M3G_ECUDA, "no CUDA device");
  return serve_status_word(*dev, status);
}
inline cudaStream_t serve_stream(void* stream) {
  return stream ? static_cast<cudaStream_t>(stream) : cudaStreamLegacy;
}

// ---------------------------------------------------------------- the batch
struct SeqView {
  int q0, n, ctx;  // first token, new tokens, cached positions; n == 0: nothing to do
};

// Sequence s of the batch, empty where it passes the call's limits (bad set then).
__device__ __forceinline__ SeqView seq_view(const m3g_kv_batch& b, long long cap, int s, bool* bad) {
  const long long q0 = b.q_start[s], q1 = b.q_start[s + 1], ctx = b.ctx_len[s];
  SeqView v{static_cast<int>(q0), static_cast<int>(q1 - q0), static_cast<int>(ctx)};
  if (q0 < 0 || q1 < q0 || q1 > b.n_tokens || q1 - q0 > b.max_tokens || ctx < 0 || ctx + (q1 - q0) > cap) {
    if (!(q0 == q1 && ctx >= 0)) *bad = true;  // no new tokens: nothing is read, whatever the context
    v.n = 0;
  }
  return v;
}

// Positions a sequence may have: the call's limit and its row of the page table.
inline __host__ __device__ long long seq_cap(const m3g_kv_batch& b, uint32_t page_size) {
  const long long rows = static_cast<long long>(b.max_pages) * page_size;
  return rows < static_cast<long long>(b.max_len) ? rows : static_cast<long long>(b.max_len);
}

// ---------------------------------------------------------------- the cache
struct KvPlanes {
  uint8_t *kc, *ks, *vc, *vs;  // this layer's planes
  uint32_t* status;
  int kvh, hd, cb, sb;         // KV heads, head size, code and scale bytes per row
  int page_shift, page_size;
  int n_pages;
};

int kv_check(const m3g_kv_layout* l);
int kv_batch_check(const m3g_kv_layout* l, const m3g_kv_batch* b);
// The planes of one layer (checks layout, pool and layer); status: of the current device.
int kv_planes(const m3g_kv_layout* l, const void* pool, uint32_t layer, KvPlanes* out);

// Row number of (page, head, place) in a plane; a row is cb code or sb scale bytes.
__device__ __forceinline__ long long kv_row(const KvPlanes& p, int page, int head, int at) {
  return (static_cast<long long>(page) * p.kvh + head) * p.page_size + at;
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return static_cast<uint64_t>(__float_as_uint(lo)) | static_cast<uint64_t>(__float_as_uint(hi)) << 32;
}
__device__ __forceinline__ float low(uint64_t x) { return __uint_as_float(static_cast<uint32_t>(x)); }
__device__ __forceinline__ float high(uint64_t x) { return __uint_as_float(static_cast<uint32_t>(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <class Kern, class... Args>
cudaError_t serve_launch(Kern kern, dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace m3g
