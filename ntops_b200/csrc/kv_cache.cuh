// Shared parts of the paged 8-bit KV cache kernels (kv_store.cu, kv_pages.cu, kv_attention*.cu).
//
// A cache layer holds key and value codes [P, H, T, D] (P pages of T tokens, H kv heads), one
// byte each: e4m3 or int8, and one fp32 scale for each (page, head): value = code * scale.  A
// block table int32 [B, M] names, for row b, the page that holds tokens [m * T, (m + 1) * T);
// an entry outside [0, P) is a hole: nothing is stored there and attention skips its tokens.
#pragma once

#include <cuda_fp8.h>

#include "elementwise.cuh"
#include "ntb_common.cuh"

namespace ntb {
namespace kv {

// One layer as the store and attention kernels see it.  Strides in elements (codes: bytes).
struct Layer {
  uint8_t *key, *value;
  float *key_scale, *value_scale;
  int64_t k_p, k_h, k_t, v_p, v_h, v_t;  // code strides: page, head, token (unit inner stride)
  int64_t ks_p, ks_h, vs_p, vs_h;        // scale strides: page, head
  int P, H, T, D;
  int code;                              // NTB_F8E4M3 or NTB_I8
};

struct Table {
  const int* ids;
  int64_t s_b, s_m;
  int B, M;
};

// Checks a cache (codes `layers ? 5 : 4`-D, scales one less than two) and fills *l with layer 0.
int check_cache(const NtbKvCache* c, bool layers, Layer* l);
// Checks an int32 tensor of the given rank; its name appears in the error.
int check_i32(const NtbTensor* t, int ndim, const char* name);

// Blocks of a kernel that the current device keeps resident at once (cached occupancy query).
int resident_blocks(const void* kernel, int threads, size_t smem);

__device__ __forceinline__ int page_of(const Table& t, int P, int b, int m) {
  if (m >= t.M) return -1;
  const int id = t.ids[(int64_t)b * t.s_b + (int64_t)m * t.s_m];
  return (unsigned)id < (unsigned)P ? id : -1;
}

// ------------------------------------------------------------------------------ codes -----
template <int CODE> struct CodeMax;
template <> struct CodeMax<NTB_F8E4M3> { static constexpr float value = 448.f; };
template <> struct CodeMax<NTB_I8> { static constexpr float value = 127.f; };

// Exponent e of the smallest power of two 2^e with amax <= qmax * 2^e, within [-100, 120].  With
// qmax = M * 2^k, M in [1, 2) (448 = 1.75 * 2^8, 127 = 1.984375 * 2^6) and amax = m * 2^x, it is
// x - k, plus one where m > M: integer operations on amax's bits, exact, so every implementation
// finds the same scale.  Powers of two make x / scale exact, the only rounding is the code's own,
// and re-coding a page under a larger scale changes e4m3 codes in their subnormal range only.
template <int CODE>
__device__ __forceinline__ int scale_exp(float amax) {
  constexpr uint32_t kTop = CODE == NTB_F8E4M3 ? 0x600000u : 0x7E0000u;  // mantissa bits of M
  constexpr int kExp = CODE == NTB_F8E4M3 ? 8 : 6;
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - kExp + ((u & 0x7FFFFFu) > kTop ? 1 : 0);  // subnormal amax: clamped below
  return min(max(e, -100), 120);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four values (already divided by the scale) -> four codes, first in the low byte.  e4m3: round
// to nearest even, saturating to +-448 (infinities too), NaN stays NaN.  int8: round to nearest
// even, saturating to +-127, NaN becomes 0.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (CODE == NTB_F8E4M3) {
    uint32_t r;  // (the conversion's first source is the upper byte)
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  } else {
    auto q = [](float x) -> uint32_t {
      // a NaN loses both comparisons of fminf / fmaxf, so it is set to 0 first
      return (uint32_t)(__float2int_rn(fminf(fmaxf(x == x ? x : 0.f, -127.f), 127.f)) & 0xFF);
    };
    return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
  }
}
template <int CODE>
__device__ __forceinline__ uint8_t encode1(float a) {
  return (uint8_t)(encode4<CODE>(a, 0.f, 0.f, 0.f) & 0xFFu);
}
template <int CODE>
__device__ __forceinline__ float decode1(uint8_t c) {
  if constexpr (CODE == NTB_F8E4M3) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
  } else {
    return (float)(int8_t)c;
  }
}

// ------------------------------------------------------------- programmatic launch --------
// A kernel launched with programmatic stream serialisation may start before its predecessor
// ends; this waits until the predecessor has finished and its writes are visible.  Every block of
// such a kernel calls it, before it returns or touches memory that the stream's earlier work
// touches.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches `kernel` so that it may be scheduled before the preceding kernel of the stream ends;
// the kernel calls grid_dependency_wait() before it touches anything that one wrote.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace kv
}  // namespace ntb
