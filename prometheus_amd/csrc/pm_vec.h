// pm_vec.h — rows of V elements between memory and registers, for the elementwise kernels.
//
// A row is loaded and stored whole (16 bytes or more in one or two instructions) at any alignment
// of its elements: gfx950 takes global accesses at any byte address, so views at odd offsets and
// rows of odd widths run the same code, and only a tensor's last, partial row goes element by
// element.
#pragma once

#include "pm_common.h"

namespace pm {

typedef __bf16 bf16_pair __attribute__((ext_vector_type(2)));
typedef float f32_pair __attribute__((ext_vector_type(2)));

// V elements of type E (uint16_t: bf16 bit patterns) as they are in memory
template <typename E, int V>
struct Row {
    uint32_t raw[V * sizeof(E) / 4];

    __device__ __forceinline__ void load(const E* p) { __builtin_memcpy(raw, p, sizeof raw); }
    // elements [0, n) of p, zeros beyond
    __device__ __forceinline__ void load(const E* p, int n) {
        if (n >= V) {
            load(p);
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
    // element i, rounded to nearest even where E is bf16; elements are set in order
    __device__ __forceinline__ void set(int i, float v) {
        if constexpr (sizeof(E) == 4) {
            raw[i] = __float_as_uint(v);
        } else if (i % 2 == 0) {
            raw[i / 2] = __float_as_uint(v);  // (kept whole until its neighbour comes: one conversion for both)
        } else {
            const f32_pair two = {__uint_as_float(raw[i / 2]), v};
            raw[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16_pair));
        }
    }
    __device__ __forceinline__ void store(E* p) const {
        // (outputs are not read again here: they go past the caches)
        typedef uint32_t vec __attribute__((ext_vector_type(V * sizeof(E) / 4), aligned(sizeof(E))));
        vec v;
        __builtin_memcpy(&v, raw, sizeof raw);
        __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
    }
    // the first n elements to p
    __device__ __forceinline__ void store(E* p, int n) const {
        if (n >= V) {
            store(p);
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                if constexpr (sizeof(E) == 2) p[i] = static_cast<uint16_t>(raw[i / 2] >> (16 * (i % 2)));
                else p[i] = __uint_as_float(raw[i]);
            }
    }
};

// the first n of V floats to p, rounded to nearest even where E is bf16
template <typename E, int V>
__device__ __forceinline__ void store_row(E* p, const float (&v)[V], int n) {
    Row<E, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.set(i, v[i]);
    r.store(p, n);
}

}  // namespace pm
