// global_norm.hip — the 2-norm over many arrays as if they were one, and the arrays scaled down to a largest norm: the reduction of splahip_reduce over a list
// of panels of mixed element types, whose result stays on the device.
//
//   norm = sqrt(sum over all arrays of x^2),  out = x * min(1, limit / norm)
//
// The norm is used in 64 bits, where only a NaN or infinity among the values makes it one: that scales nothing.  Rounded to 32 bits it is infinity beyond FLT_MAX, while
// the values are scaled all the same.  A norm that the caller gives has 32 bits: NaN and infinity scale nothing.
//
// Squares are taken and summed in 64 bits: the square of an fp32 value is exact there and no sum of them leaves the range, so neither a large gradient
// overflows nor do many small ones get lost.  Every partial sum has its own word and a fixed order: the norm is the same from run to run.
// The arrays' addresses travel as kernel arguments (kBatch of them per launch): no table in device memory to fill, keep alive or race with.
#include "panel.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <new>
#include <vector>

namespace splahip {

    constexpr uint32_t kBatch = 128, kSmallBatch = 16;// arrays per launch: 3.7 KB of arguments, or 0.5 where they do (each launch copies them)

    template<uint32_t N>
    struct NormBatch {
        const void* src[N];
        void*       dst[N];
        uint64_t    n[N];
        uint32_t    first[N + 1];// first chunk of array i, ascending; [count] = chunks of the launch
        uint8_t     type[N];
        uint32_t    count;
    };

    // which array chunk b belongs to
    template<uint32_t N>
    __device__ __forceinline__ uint32_t array_of(const NormBatch<N>& a, uint32_t b) {
        uint32_t lo = 0, hi = a.count;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (a.first[mid] <= b) lo = mid;
            else
                hi = mid;
        }
        return lo;
    }

    __device__ __forceinline__ double block_sum(double x) {
        __shared__ double part[16];
#pragma unroll
        for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
        if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        double s = 0.0;
        for (uint32_t w = 0; w < (blockDim.x >> 6); ++w) s += part[w];
        return s;
    }

    // A workgroup's chunk: kAhead units per thread under way, then what is left unit by unit.  Both passes are bound by HBM.  Streaming accesses, eight of them and chunks of 2^14
    // elements: 400 M elements of 300 arrays (1.0 GB) are read in 154 us = 6.4 TB/s, read twice and written in 501 us = 5.9 TB/s (cached accesses, four, 2^16: 191 and 627 us).
    constexpr uint32_t kAhead = 8;

    template<typename T>
    __device__ __forceinline__ double chunk_squares(const T* __restrict__ x, uint64_t n) {
        constexpr uint32_t U = kUnit<T>, BLOCK = 256 * U * kAhead;
        double             s0 = 0.0, s1 = 0.0;
        uint64_t           at = 0;
        for (; at + BLOCK <= n; at += BLOCK) {
            typename UnitOf<T>::mem v[kAhead];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) v[k] = __builtin_nontemporal_load(reinterpret_cast<const typename UnitOf<T>::mem*>(x + at + (k * 256 + threadIdx.x) * U));
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k)
#pragma unroll
                for (uint32_t q = 0; q < U; q += 2) {
                    s0 = fma((double) (float) v[k][q], (double) (float) v[k][q], s0);
                    s1 = fma((double) (float) v[k][q + 1], (double) (float) v[k][q + 1], s1);
                }
        }
        for (uint64_t c = at + (uint64_t) threadIdx.x * U; c < n; c += 256 * U) {
            float v[U];
            load_unit<T>(x + c, (uint32_t) min(n - c, (uint64_t) U), v);
#pragma unroll
            for (uint32_t q = 0; q < U; ++q) s0 = fma((double) v[q], (double) v[q], s0);
        }
        return s0 + s1;
    }

    template<uint32_t N>
    __global__ __launch_bounds__(256) void norm_partials_kernel(const NormBatch<N> a, uint32_t chunk, double* __restrict__ partials) {
        const uint32_t i   = array_of(a, blockIdx.x);
        const uint64_t at  = (uint64_t) (blockIdx.x - a.first[i]) * chunk;
        const uint64_t len = min(a.n[i] - at, (uint64_t) chunk);
        double         s;
        if (a.type[i] == SPLAHIP_PANEL_FLOAT) s = chunk_squares(static_cast<const float*>(a.src[i]) + at, len);
        else if (a.type[i] == SPLAHIP_PANEL_HALF)
            s = chunk_squares(static_cast<const fp16_t*>(a.src[i]) + at, len);
        else
            s = chunk_squares(static_cast<const bf16_t*>(a.src[i]) + at, len);
        s = block_sum(s);
        if (threadIdx.x == 0) partials[blockIdx.x] = s;
    }

    __global__ __launch_bounds__(1024) void norm_finish_kernel(uint32_t n, const double* __restrict__ partials, float* __restrict__ norm, double* __restrict__ norm64) {
        double s = 0.0;
#pragma unroll 8
        for (uint32_t i = threadIdx.x; i < n; i += 1024) s += partials[i];
        s = sqrt(block_sum(s));
        if (threadIdx.x == 0) {
            *norm   = (float) s;
            *norm64 = s;
        }
    }

    // how the arrays are scaled: by a factor of 32 bits, by one of 64 where 32 cannot hold it to full precision (a norm near or beyond fp32's largest value: the
    // factor is subnormal there), or not at all
    enum Scaling { kCopy, kFactor32, kFactor64 };

    template<typename T, Scaling HOW>
    __device__ __forceinline__ void chunk_scale(const T* x, T* y, uint64_t n, double factor) {
        constexpr uint32_t U = kUnit<T>;
        constexpr uint32_t BLOCK = 256 * U * kAhead;
        const float        f     = (float) factor;
        auto               scale = [&](float v) { return HOW == kFactor32 ? v * f : HOW == kFactor64 ? (float) ((double) v * factor) : v; };
        uint64_t           at    = 0;
        for (; at + BLOCK <= n; at += BLOCK) {
            typename UnitOf<T>::mem v[kAhead];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) v[k] = __builtin_nontemporal_load(reinterpret_cast<const typename UnitOf<T>::mem*>(x + at + (k * 256 + threadIdx.x) * U));
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) {
#pragma unroll
                for (uint32_t q = 0; q < U; ++q) v[k][q] = (T) scale((float) v[k][q]);
                __builtin_nontemporal_store(v[k], reinterpret_cast<typename UnitOf<T>::mem*>(y + at + (k * 256 + threadIdx.x) * U));
            }
        }
        for (uint64_t c = at + (uint64_t) threadIdx.x * U; c < n; c += 256 * U) {
            const uint32_t left = (uint32_t) min(n - c, (uint64_t) U);
            float          v[U];
            load_unit<T>(x + c, left, v);
#pragma unroll
            for (uint32_t q = 0; q < U; ++q) v[q] = scale(v[q]);
            store_unit<T>(y + c, left, v);
        }
    }
    template<Scaling HOW, uint32_t N>
    __device__ __forceinline__ void chunk_scale_any(const NormBatch<N>& a, uint32_t i, uint64_t at, uint64_t len, double factor) {
        if (a.type[i] == SPLAHIP_PANEL_FLOAT) chunk_scale<float, HOW>(static_cast<const float*>(a.src[i]) + at, static_cast<float*>(a.dst[i]) + at, len, factor);
        else if (a.type[i] == SPLAHIP_PANEL_HALF)
            chunk_scale<fp16_t, HOW>(static_cast<const fp16_t*>(a.src[i]) + at, static_cast<fp16_t*>(a.dst[i]) + at, len, factor);
        else
            chunk_scale<bf16_t, HOW>(static_cast<const bf16_t*>(a.src[i]) + at, static_cast<bf16_t*>(a.dst[i]) + at, len, factor);
    }

    // the factor is rounded to 32 bits once, each product to 32 bits and to the array's type
    template<uint32_t N>
    __global__ __launch_bounds__(256) void norm_scale_kernel(const NormBatch<N> a, uint32_t chunk, float limit, const float* __restrict__ norm32,
                                                             const double* __restrict__ norm64) {
        const double   norm   = norm64 ? *norm64 : (double) *norm32;
        const bool     same   = !(norm > (double) limit) || norm == INFINITY;// (a NaN compares false)
        const double   factor = same ? 1.0 : (double) limit / norm;
        const uint32_t i      = array_of(a, blockIdx.x);
        const uint64_t at     = (uint64_t) (blockIdx.x - a.first[i]) * chunk;
        const uint64_t len    = min(a.n[i] - at, (uint64_t) chunk);
        if (same && a.src[i] == a.dst[i]) return;
        if (same) chunk_scale_any<kCopy>(a, i, at, len, factor);
        else if (factor >= (double) FLT_MIN || factor == 0.0)
            chunk_scale_any<kFactor32>(a, i, at, len, factor);
        else
            chunk_scale_any<kFactor64>(a, i, at, len, factor);
    }

    // elements of a workgroup's chunk: about 4096 chunks in all, so that the card is full, between 2048 (a workgroup's one step of 16-bit units) and 2^14
    static uint32_t chunk_elements(uint64_t total) {
        uint32_t c = 2048;
        while (c < 16384 && (uint64_t) c * 4096 < total) c <<= 1;
        return c;
    }

    static uint64_t total_elements(uint32_t n_arrays, const uint64_t* lengths) {
        uint64_t t = 0;
        for (uint32_t i = 0; i < n_arrays; ++i) t += lengths[i];
        return t;
    }

    // launches f(batch, chunks, chunks before it) for the arrays in batches
    template<uint32_t N, typename F>
    static void for_batches_of(uint32_t n_arrays, const void* const* src, void* const* dst, const uint64_t* lengths, const int* types, uint32_t chunk, F&& f) {
        NormBatch<N> a;
        a.count        = 0;
        uint64_t done  = 0;
        uint32_t first = 0;
        for (uint32_t i = 0; i < n_arrays; ++i) {
            if (lengths[i]) {
                a.src[a.count]   = src[i];
                a.dst[a.count]   = dst ? dst[i] : nullptr;
                a.n[a.count]     = lengths[i];
                a.type[a.count]  = (uint8_t) types[i];
                a.first[a.count] = first;
                first += (uint32_t) ((lengths[i] + chunk - 1) / chunk);
                ++a.count;
            }
            if (a.count && (a.count == N || i + 1 == n_arrays)) {
                a.first[a.count] = first;
                f(a, first, done);
                done += first;
                a.count = 0;
                first   = 0;
            }
        }
    }

    template<typename F>
    static void for_batches(uint32_t n_arrays, const void* const* src, void* const* dst, const uint64_t* lengths, const int* types, uint32_t chunk, F&& f) {
        if (n_arrays <= kSmallBatch) for_batches_of<kSmallBatch>(n_arrays, src, dst, lengths, types, chunk, f);
        else
            for_batches_of<kBatch>(n_arrays, src, dst, lengths, types, chunk, f);
    }

    static uint64_t bytes_of(uint64_t length, int type) { return length * (type == SPLAHIP_PANEL_FLOAT ? 4u : 2u); }
    static bool     overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
        return (uintptr_t) a < (uintptr_t) b + b_bytes && (uintptr_t) b < (uintptr_t) a + a_bytes;
    }

    static int check_arrays(uint32_t n_arrays, const void* const* ptrs, const uint64_t* lengths, const int* types) {
        SPLAHIP_REQUIRE(n_arrays == 0 || (ptrs && lengths && types), "null list");
        uint64_t total = 0;
        for (uint32_t i = 0; i < n_arrays; ++i) {
            SPLAHIP_REQUIRE(panel_type_valid(types[i]), "element type");
            SPLAHIP_REQUIRE(lengths[i] == 0 || ptrs[i], "null array");
            SPLAHIP_REQUIRE(lengths[i] < (1ull << 40), "array length: below 2^40");
            total += lengths[i];
        }
        SPLAHIP_REQUIRE(total < (1ull << 44), "elements in all: below 2^44");
        return SPLAHIP_OK;
    }

    // the partial sums are written while the arrays are read, the norm behind them
    static int check_workspace(uint32_t n_arrays, const void* const* ptrs, const uint64_t* lengths, const int* types, const void* work, uint64_t work_bytes, const float* norm) {
        SPLAHIP_REQUIRE(!overlap(norm, sizeof(float), work, work_bytes), "the norm lies inside the workspace");
        for (uint32_t i = 0; i < n_arrays; ++i) SPLAHIP_REQUIRE(!lengths[i] || !overlap(ptrs[i], bytes_of(lengths[i], types[i]), work, work_bytes), "an array overlaps the workspace");
        return SPLAHIP_OK;
    }

    // no two results may share memory, and a result may share it with its own source only, element for element: anything else would be scaled twice or read
    // after it was scaled.  A norm that is computed (`written`) may not lie inside a source either, which is read again after it was written.
    static int check_overlap(uint32_t n_arrays, const void* const* src, void* const* dst, const uint64_t* lengths, const int* types, const float* norm,
                             bool written) {
        struct Span {
            uintptr_t a, b;
            uint32_t  i;
        };
        std::vector<Span> out;
        out.reserve(n_arrays);
        auto span = [&](const void* p, uint32_t i) { return Span{(uintptr_t) p, (uintptr_t) p + bytes_of(lengths[i], types[i]), i}; };
        for (uint32_t i = 0; i < n_arrays; ++i)
            if (lengths[i]) out.push_back(span(dst[i], i));
        std::sort(out.begin(), out.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
        for (size_t k = 1; k < out.size(); ++k) SPLAHIP_REQUIRE(out[k - 1].b <= out[k].a, "results overlap (the same array twice?)");
        auto free_of_results = [&](uintptr_t a, uintptr_t b) {
            auto it = std::upper_bound(out.begin(), out.end(), a, [](uintptr_t p, const Span& y) { return p < y.b; });
            return it == out.end() || it->a >= b;
        };
        SPLAHIP_REQUIRE(free_of_results((uintptr_t) norm, (uintptr_t) norm + sizeof(float)), "the norm lies inside a result");
        for (uint32_t i = 0; i < n_arrays; ++i) {
            if (lengths[i] == 0 || src[i] == dst[i]) continue;// (its own result: the check above covers the others)
            const Span x = span(src[i], i);
            SPLAHIP_REQUIRE(!written || !overlap(norm, sizeof(float), src[i], x.b - x.a), "the norm lies inside an array");
            SPLAHIP_REQUIRE(free_of_results(x.a, x.b), "an array overlaps a result other than itself");
        }
        return SPLAHIP_OK;
    }

}// namespace splahip

using namespace splahip;

extern "C" size_t splahip_global_norm_workspace(uint32_t n_arrays, const uint64_t* h_lengths) {
    const uint32_t chunk  = chunk_elements(total_elements(n_arrays, h_lengths));
    uint64_t       chunks = 0;
    for (uint32_t i = 0; i < n_arrays; ++i) chunks += (h_lengths[i] + chunk - 1) / chunk;
    return (size_t) (chunks + 1) * sizeof(double);
}

extern "C" int splahip_global_norm(uint32_t n_arrays, const void* const* h_arrays, const uint64_t* h_lengths, const int* h_types, void* d_workspace,
                                   size_t workspace_bytes, float* d_norm, void* stream) {
    if (int st = check_arrays(n_arrays, h_arrays, h_lengths, h_types)) return st;
    SPLAHIP_REQUIRE(d_norm, "null result");
    SPLAHIP_REQUIRE(d_workspace && ((uintptr_t) d_workspace & 7u) == 0 && workspace_bytes >= splahip_global_norm_workspace(n_arrays, h_lengths), "workspace too small");
    if (int st = check_workspace(n_arrays, h_arrays, h_lengths, h_types, d_workspace, splahip_global_norm_workspace(n_arrays, h_lengths), d_norm)) return st;
    if (int st = ensure_device()) return st;
    hipStream_t    s        = as_stream(stream);
    double*        norm64   = static_cast<double*>(d_workspace);
    double*        partials = norm64 + 1;
    const uint32_t chunk    = chunk_elements(total_elements(n_arrays, h_lengths));
    uint64_t       n        = 0;
    for_batches(n_arrays, h_arrays, nullptr, h_lengths, h_types, chunk, [&](const auto& a, uint32_t chunks, uint64_t before) {
        norm_partials_kernel<<<chunks, 256, 0, s>>>(a, chunk, partials + before);
        n = before + chunks;
    });
    norm_finish_kernel<<<1, 1024, 0, s>>>((uint32_t) n, partials, d_norm, norm64);
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}

extern "C" int splahip_clip_global_norm(uint32_t n_arrays, const void* const* h_arrays, void* const* h_out, const uint64_t* h_lengths, const int* h_types, float limit,
                                        int norm_given, void* d_workspace, size_t workspace_bytes, float* d_norm, void* stream) {
    if (int st = check_arrays(n_arrays, h_arrays, h_lengths, h_types)) return st;
    SPLAHIP_REQUIRE(limit >= 0.0f && std::isfinite(limit), "largest norm: finite, not negative");
    SPLAHIP_REQUIRE(d_norm, "null norm");
    SPLAHIP_REQUIRE(n_arrays == 0 || h_out, "null list");
    for (uint32_t i = 0; i < n_arrays; ++i) SPLAHIP_REQUIRE(h_lengths[i] == 0 || h_out[i], "null array");
    try {
        if (int st = check_overlap(n_arrays, h_arrays, h_out, h_lengths, h_types, d_norm, !norm_given)) return st;
    } catch (const std::bad_alloc&) { return fail(SPLAHIP_ERROR, "out of host memory"); }
    if (!norm_given && h_out != h_arrays && d_workspace)// (the 64-bit norm is read from there while the results are written)
        if (int st = check_workspace(n_arrays, h_out, h_lengths, h_types, d_workspace, splahip_global_norm_workspace(n_arrays, h_lengths), d_norm)) return st;
    if (!norm_given)
        if (int st = splahip_global_norm(n_arrays, h_arrays, h_lengths, h_types, d_workspace, workspace_bytes, d_norm, stream)) return st;
    if (int st = ensure_device()) return st;
    hipStream_t    s     = as_stream(stream);
    const uint32_t chunk = chunk_elements(total_elements(n_arrays, h_lengths));
    for_batches(n_arrays, h_arrays, h_out, h_lengths, h_types, chunk, [&](const auto& a, uint32_t chunks, uint64_t) {
        norm_scale_kernel<<<chunks, 256, 0, s>>>(a, chunk, limit, d_norm, norm_given ? nullptr : static_cast<const double*>(d_workspace));
    });
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}
