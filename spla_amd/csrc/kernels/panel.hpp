// panel.hpp — element types and wide accesses of the panel operators (route.hip, expert_product.hip, global_norm.hip): a panel is a dense row-major
// matrix [rows, width] of fp32, fp16 or bf16 elements.  Sums are kept in fp32 or wider and rounded to the panel's type once, by the hardware's
// round-to-nearest-even conversion.
#pragma once

#include "common.hpp"

namespace splahip {

    using bf16_t = __bf16;
    using fp16_t = _Float16;

    inline bool panel_type_valid(int type) { return type == SPLAHIP_PANEL_FLOAT || type == SPLAHIP_PANEL_HALF || type == SPLAHIP_PANEL_BFLOAT16; }

    // elements of a 16-byte unit
    template<typename T>
    constexpr int kUnit = 16 / (int) sizeof(T);

    // a unit in memory: a row of odd width starts at any element, so the access claims the element's alignment only (gfx950 serves wide global accesses at
    // any address; an aligned address costs no more for it)
    template<typename T>
    struct UnitOf {
        typedef T mem __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    };

    // the unit at p as floats; `left` elements of the row from p on: the last unit of a row is read element by element, zeros behind it
    template<typename T>
    __device__ __forceinline__ void load_unit(const T* __restrict__ p, uint32_t left, float (&x)[kUnit<T>]) {
        if (left >= (uint32_t) kUnit<T>) {
            const typename UnitOf<T>::mem v = *reinterpret_cast<const typename UnitOf<T>::mem*>(p);
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i) x[i] = (float) v[i];
        } else {
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i) x[i] = (uint32_t) i < left ? (float) p[i] : 0.0f;
        }
    }

    template<typename T>
    __device__ __forceinline__ void store_unit(T* __restrict__ p, uint32_t left, const float (&x)[kUnit<T>]) {
        if (left >= (uint32_t) kUnit<T>) {
            typename UnitOf<T>::mem v;
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i) v[i] = (T) x[i];
            *reinterpret_cast<typename UnitOf<T>::mem*>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i)
                if ((uint32_t) i < left) p[i] = (T) x[i];
        }
    }

    // runs f(T{}) for the element type of `type`
    template<typename F>
    inline void panel_dispatch(int type, F&& f) {
        switch (type) {
            case SPLAHIP_PANEL_HALF: f(fp16_t{}); break;
            case SPLAHIP_PANEL_BFLOAT16: f(bf16_t{}); break;
            default: f(float{}); break;
        }
    }

}// namespace splahip
