// gdr_rows.hpp -- row access shared by the Local block's prologue, norms and
// their backward passes.
#pragma once

#include <type_traits>

#include "gdr_device.hpp"

namespace rhz {

// N consecutive elements as floats: one 16-byte access when VEC (N = 4 fp32
// or 8 bf16, 16-byte aligned), else N = 1.
template <typename T, bool VEC>
struct Vec {
    static constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
    // the loaded bits, unpacked later (4 registers for 16 bytes)
    using Raw = typename std::conditional<VEC, uint4, T>::type;
    static __device__ __forceinline__ Raw load_raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&x)[N]) {
        if constexpr (!VEC) {
            x[0] = Elem<T>::load(&r, 0);
        } else if constexpr (sizeof(T) == 4) {
            x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y);
            x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
        } else {
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ void load(const T* p, float (&x)[N]) { unpack(load_raw(p), x); }
    // NT: a non-temporal store (streaming output that this kernel does not
    // read back).
    template <bool NT = false>
    static __device__ __forceinline__ void store(T* p, const float (&x)[N]) {
        if constexpr (!VEC) {
            Elem<T>::store(p, 0, x[0]);
        } else if constexpr (sizeof(T) == 4) {
            const f32x4 v = {x[0], x[1], x[2], x[3]};
            if constexpr (NT)
                __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
            else
                *reinterpret_cast<f32x4*>(p) = v;
        } else {
            typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
            const u32x4 u = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                             pack_bf16x2(x[6], x[7])};
            if constexpr (NT)
                __builtin_nontemporal_store(u, reinterpret_cast<u32x4*>(p));
            else
                *reinterpret_cast<u32x4*>(p) = u;
        }
    }
};

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Sum over aligned groups of G lanes, G a power of two up to 64.
template <int G>
__device__ __forceinline__ float row_sum(float x) {
    if constexpr (G >= 32) {
        x = lane_group_sum<16>(x);
        x += __shfl_xor(x, 16, kWave);
        if constexpr (G == 64) x += __shfl_xor(x, 32, kWave);
        return x;
    } else if constexpr (G > 1) {
        return lane_group_sum<G>(x);
    } else {
        return x;
    }
}

}  // namespace rhz
