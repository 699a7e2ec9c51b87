// 16-bit element types of the mixed-precision training operators (gemm_half.hip, embedding.hip, adamw.hip): loads that
// need no more than the element's alignment, conversions to and from fp32 (round to nearest even, the hardware's).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hd {

typedef __bf16 bf16;
typedef _Float16 f16;

// N elements from an address that is aligned to the element only: the compiler emits wide loads (the unaligned access mode
// is on), which cost nothing extra where the address happens to be 16-byte aligned
template <typename T, int N> struct Pack { T v[N]; };
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    Pack<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) { __builtin_memcpy(p, &r, sizeof(r)); }

// host side: element type codes of the C ABI (HD_DT_F32 / HD_DT_BF16 / HD_DT_F16)
inline int dt_size(int dt) { return dt == 0 ? 4 : 2; }

}  // namespace hd
