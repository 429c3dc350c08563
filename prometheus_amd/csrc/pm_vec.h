// pm_vec.h — rows of V elements between memory and registers, for the elementwise kernels.
//
// A row is loaded and stored whole (16 bytes or more in one or two instructions) at any alignment
// of its elements: gfx950 takes global accesses at any byte address, so views at odd offsets and
// rows of odd widths run the same code, and only a tensor's last, partial row goes element by
// element.
#pragma once

#include "pm_common.h"

namespace pm {

// V elements of type E (uint16_t: bf16 bit patterns) as they are in memory
template <typename E, int V>
struct Row {
    uint32_t raw[V * sizeof(E) / 4];

    // elements [0, n) of p, zeros beyond
    __device__ __forceinline__ void load(const E* p, int n) {
        if (n >= V) {
            __builtin_memcpy(raw, p, sizeof raw);
            return;
        }
#pragma unroll
        for (int i = 0; i < static_cast<int>(V * sizeof(E) / 4); ++i) raw[i] = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                if constexpr (sizeof(E) == 2) raw[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i % 2));
                else raw[i] = __float_as_uint(p[i]);
            }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(E) == 2) return __uint_as_float(i % 2 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
        else return __uint_as_float(raw[i]);
    }
};

typedef __bf16 bf16_pair __attribute__((ext_vector_type(2)));
typedef float f32_pair __attribute__((ext_vector_type(2)));

// the first n of V floats to p, rounded to nearest even where E is bf16
template <typename E, int V>
__device__ __forceinline__ void store_row(E* p, const float (&v)[V], int n) {
    uint32_t raw[V * sizeof(E) / 4];
    if constexpr (sizeof(E) == 2) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const f32_pair two = {v[2 * i], v[2 * i + 1]};
            raw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16_pair));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) raw[i] = __float_as_uint(v[i]);
    }
    if (n >= V) {
        __builtin_memcpy(p, raw, sizeof raw);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) {
            if constexpr (sizeof(E) == 2) p[i] = static_cast<uint16_t>(raw[i / 2] >> (16 * (i % 2)));
            else p[i] = v[i];
        }
}

}  // namespace pm
