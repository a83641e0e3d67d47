// Common CDNA4 (gfx950) kernel utilities for the LuminaAI-AMD framework.
// Hand-written HIP, MI355X-first: 64-wide wavefronts, bf16x8 vector loads,
// fp32 internal math. No CUDA compatibility paths.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#define WAVE 64
#define DEV_INLINE __device__ __forceinline__

// ---- vector types for 16-byte loads -------------------------------------
typedef __attribute__((ext_vector_type(4))) float    floatx4;
typedef __attribute__((ext_vector_type(4))) uint32_t uintx4;
typedef __attribute__((ext_vector_type(8))) uint16_t ushortx8;

// ---- dtype conversion helpers -------------------------------------------
DEV_INLINE float bf16_to_f32(uint16_t u) {
  union { uint32_t i; float f; } v;
  v.i = ((uint32_t)u) << 16;
  return v.f;
}

DEV_INLINE uint16_t f32_to_bf16(float f) {
  union { float f; uint32_t i; } v;
  v.f = f;
  // round-to-nearest-even
  uint32_t lsb = (v.i >> 16) & 1;
  v.i += 0x7fff + lsb;
  return (uint16_t)(v.i >> 16);
}

// ---- rows of 16-bit channels at any address -------------------------------
// 16 bytes at any element: one load, gfx950 takes any alignment there
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t uintx4_any;

// Channels 8 c .. 8 c + 7 of a row of D, zero past its end. Nothing outside the
// row is read: its last, partial piece is read as its last 8 channels and moved
// down, without a branch that lanes could take apart (a piece of one in twenty
// lanes, loaded channel by channel, made a copy of rows of 159 three times as
// long).
DEV_INLINE uintx4 load8_ragged(const uint16_t* row, int c, int D) {
  if (D >= 8) {                               // uniform, and below
    const int o = 8 * c < D - 8 ? 8 * c : D - 8;
    uintx4 v = *reinterpret_cast<const uintx4_any*>(row + o);
    const int e = (8 - (D & 7)) & 7;
    const bool part = 8 * c > D - 8;
    if (e & 1) {
      const uint32_t by = part ? 16 : 0;
      #pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = __builtin_amdgcn_alignbit(j < 3 ? v[j + 1] : (part ? 0 : v[3]),
                                         v[j], by);
    }
    if (e & 2) v = part ? uintx4{v[1], v[2], v[3], 0} : v;
    if (e & 4) v = part ? uintx4{v[2], v[3], 0, 0} : v;
    return 8 * c < D ? v : uintx4{0, 0, 0, 0};
  }
  uintx4 v = {0, 0, 0, 0};
  #pragma unroll
  for (int j = 0; j < 7; ++j)
    if (8 * c + j < D) v[j >> 1] |= (uint32_t)row[8 * c + j] << (16 * (j & 1));
  return v;
}

// inclusive sum over the wave's lanes up to this one
DEV_INLINE int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);  // row_bcast
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);
  return x;
}

// sum over the wave, the same in every lane
DEV_INLINE int wave_sum(int x) {
  return __builtin_amdgcn_readlane(wave_scan(x), 63);
}

// inclusive sum over a workgroup's threads; ws: an int for each wave
DEV_INLINE int block_scan(int x, int* ws) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  #pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();                           // the last call's reads are done
  if (lane == 63) ws[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += ws[i];
  return x;
}

// generic element accessors so kernels template over T in {float, bf16-as-u16}
struct F32Elem {
  using storage = float;
  static DEV_INLINE float load(const float* p) { return *p; }
  static DEV_INLINE void store(float* p, float v) { *p = v; }
};
struct BF16Elem {
  using storage = uint16_t;
  static DEV_INLINE float load(const uint16_t* p) { return bf16_to_f32(*p); }
  static DEV_INLINE void store(uint16_t* p, float v) { *p = f32_to_bf16(v); }
};

// ---- wave + block reductions --------------------------------------------
DEV_INLINE float wave_reduce_sum(float v) {
  #pragma unroll
  for (int off = WAVE / 2; off > 0; off >>= 1)
    v += __shfl_down(v, off, WAVE);
  return v;  // valid in lane 0
}

DEV_INLINE float wave_reduce_max(float v) {
  #pragma unroll
  for (int off = WAVE / 2; off > 0; off >>= 1)
    v = fmaxf(v, __shfl_down(v, off, WAVE));
  return v;
}

// Block reduction over up to 16 waves; smem must hold >= 16 floats.
// Returns the result broadcast to all threads.
DEV_INLINE float block_reduce_sum(float v, float* smem) {
  const int lane = threadIdx.x & (WAVE - 1);
  const int wid  = threadIdx.x / WAVE;
  const int nw   = (blockDim.x + WAVE - 1) / WAVE;
  v = wave_reduce_sum(v);
  if (lane == 0) smem[wid] = v;
  __syncthreads();
  float r = (threadIdx.x < nw) ? smem[threadIdx.x] : 0.0f;
  if (wid == 0) {
    r = wave_reduce_sum(r);
    if (lane == 0) smem[0] = r;
  }
  __syncthreads();
  r = smem[0];
  __syncthreads();
  return r;
}

DEV_INLINE float block_reduce_max(float v, float* smem) {
  const int lane = threadIdx.x & (WAVE - 1);
  const int wid  = threadIdx.x / WAVE;
  const int nw   = (blockDim.x + WAVE - 1) / WAVE;
  v = wave_reduce_max(v);
  if (lane == 0) smem[wid] = v;
  __syncthreads();
  float r = (threadIdx.x < nw) ? smem[threadIdx.x] : -INFINITY;
  if (wid == 0) {
    r = wave_reduce_max(r);
    if (lane == 0) smem[0] = r;
  }
  __syncthreads();
  r = smem[0];
  __syncthreads();
  return r;
}

// ---- grid sizing ---------------------------------------------------------
// memory-bound ops: cap the grid and grid-stride the rest (guide G11)
DEV_INLINE int64_t gstride() { return (int64_t)gridDim.x * blockDim.x; }

static inline int elementwise_grid(int64_t n, int block, int per_thread = 8) {
  int64_t want = (n + (int64_t)block * per_thread - 1) / ((int64_t)block * per_thread);
  int64_t cap = 2048;
  return (int)(want < cap ? (want < 1 ? 1 : want) : cap);
}

#define HIP_CHECK_LAST()                                                   \
  do {                                                                     \
    hipError_t e_ = hipGetLastError();                                     \
    if (e_ != hipSuccess) return e_;                                       \
  } while (0)
