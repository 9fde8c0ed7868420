// route.hip — products with a routing matrix: rows (tokens) x columns (experts), per_row entries in every row, as a router of a layer of experts hands
// them over.  Sorting the entries by expert is the transpose of that matrix; bringing rows of a panel into that order and back, with weights, is a
// product of it with a dense operand of many columns.
//
//   splahip_route_sort       offsets[e] = number of entries with an expert below e; order = the entries (row * per_row + choice) by (expert, entry);
//                            place = order's inverse.  An expert outside [0, n_experts) is no entry: its place is -1, order is -1 behind the last entry.
//   splahip_route_rows       out[p, :] = w_i x[row(i), :], i = order[p]; rows behind the last entry become 0
//   splahip_route_back       out[r, :] = sum over the row's entries of w_i y[place_i, :]
//   splahip_route_back_grad  dy[p, :] = w_i dout[row(i), :], dw_i = <dout[row(i), :], y[place_i, :]>
//
// Every sum has a fixed order: results are the same from run to run.
#include "panel.hpp"

#include <algorithm>
#include <type_traits>

namespace splahip {

    constexpr uint32_t kMaxExperts = 2048;

    // ---- the sort: a stable counting sort ------------------------------------------------------------------------------------------------------------
    // A workgroup owns kSortTile consecutive entries, each of its wavefronts a part of them.  Entry i's position is
    //   offsets[e] + (entries of e in earlier tiles) + (in earlier wavefronts of the tile) + (in earlier steps of the wavefront) + (in lower lanes of the step),
    // the last by a ballot per bit of the expert's number.  Three launches (count, scan over the tiles, place); a tile's entries are brought into order in LDS first, so
    // that `order` is written in runs.  Floor: 12 bytes per entry; what is left is the launches and the latency of each: 1 M entries over 128 experts 17 us (3 us of
    // bytes).  Up to 8192 entries one workgroup sorts them in one launch: 3 us, behind 7 of the host's.
    constexpr uint32_t kSortThreads = 512, kSortTile = 4096, kSortSteps = kSortTile / kSortThreads;

    __device__ __forceinline__ uint64_t lanes_alike(uint32_t key, bool valid, uint32_t bits) {
        uint64_t m = __ballot(valid);
        for (uint32_t b = 0; b < bits; ++b) {
            const uint64_t with = __ballot((key >> b) & 1u);
            m &= ((key >> b) & 1u) ? with : ~with;
        }
        return m;
    }

    // counts[tile, e]
    __global__ __launch_bounds__(512) void route_count_kernel(uint32_t n_entries, uint32_t n_experts, const int32_t* __restrict__ experts, uint32_t* __restrict__ counts) {
        __shared__ uint32_t hist[kMaxExperts];
        for (uint32_t e = threadIdx.x; e < n_experts; e += kSortThreads) hist[e] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t s = 0; s < kSortSteps; ++s) {
            const uint32_t i = blockIdx.x * kSortTile + s * kSortThreads + threadIdx.x;
            if (i < n_entries) {
                const uint32_t e = (uint32_t) experts[i];
                if (e < n_experts) atomicAdd(&hist[e], 1u);
            }
        }
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < n_experts; e += kSortThreads) counts[(size_t) blockIdx.x * n_experts + e] = hist[e];
    }

    // exclusive scan of one value per thread over the workgroup; total returned through `sum`
    template<uint32_t THREADS>
    __device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t* sum) {
        __shared__ uint32_t wave_sum[THREADS / 64];
        const uint32_t      lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint32_t            inc = x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(inc, d);
            if (lane >= (uint32_t) d) inc += up;
        }
        if (lane == 63) wave_sum[wave] = inc;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            if (w < wave) before += wave_sum[w];
            all += wave_sum[w];
        }
        __syncthreads();
        *sum = all;
        return before + inc - x;
    }

    // 16 experts a workgroup, the tiles in 64 contiguous parts: the counts become exclusive prefixes over the tiles, their sums the totals.  (64 experts and 16 parts: 4.7 instead of
    // 3.5 us at 256 tiles x 128 experts, the loads of a part coming one after another.)
    __global__ __launch_bounds__(1024) void route_scan_kernel(uint32_t n_tiles, uint32_t n_experts, uint32_t* __restrict__ counts, uint32_t* __restrict__ totals) {
        __shared__ uint32_t part[16][65];
        const uint32_t      lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = threadIdx.x & 15u, g = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
        const uint32_t      per = (n_tiles + 63) / 64, t0 = min(g * per, n_tiles), t1 = min(t0 + per, n_tiles);
        uint32_t            sum = 0, kept[8];// a part of up to 8 tiles stays in registers
        const bool          few = per <= 8;
        if (e < n_experts) {
            if (few)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) kept[i] = t0 + i < t1 ? counts[(size_t) (t0 + i) * n_experts + e] : 0u, sum += kept[i];
            else
#pragma unroll 8
                for (uint32_t t = t0; t < t1; ++t) sum += counts[(size_t) t * n_experts + e];
        }
        part[col][g] = sum;
        __syncthreads();
        const uint32_t own = part[wave][lane];// a wavefront scans an expert's parts
        uint32_t       inc = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(inc, d);
            if (lane >= (uint32_t) d) inc += up;
        }
        part[wave][lane] = inc - own;
        if (lane == 63 && blockIdx.x * 16 + wave < n_experts) totals[blockIdx.x * 16 + wave] = inc;
        __syncthreads();
        if (e >= n_experts) return;
        uint32_t at = part[col][g];
        if (few) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (t0 + i < t1) counts[(size_t) (t0 + i) * n_experts + e] = at;
                at += kept[i];
            }
            return;
        }
#pragma unroll 8
        for (uint32_t t = t0; t < t1; ++t) {
            const uint32_t c                       = counts[(size_t) t * n_experts + e];
            counts[(size_t) t * n_experts + e] = at;
            at += c;
        }
    }

    // EXPERTS >= n_experts: the size of the tables in LDS, one per wavefront (more wavefronts, fewer steps one after another: 10.1 -> 9.6 us at 256 tiles x 128 experts)
    template<uint32_t EXPERTS, uint32_t THREADS>
    __global__ __launch_bounds__(THREADS) void route_place_kernel(uint32_t n_entries, uint32_t n_experts, uint32_t bits, const int32_t* __restrict__ experts,
                                                              const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals, uint32_t* __restrict__ offsets,
                                                              int32_t* __restrict__ order, int32_t* __restrict__ place) {
        constexpr uint32_t  WAVES = THREADS / 64, STEPS = kSortTile / THREADS;
        __shared__ uint32_t wave_count[WAVES][EXPERTS];
        __shared__ uint32_t shift[EXPERTS];// place of an entry of e - its place in the tile's order
        __shared__ uint32_t entry[kSortTile], place_of[kSortTile];
        const uint32_t      lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, first = blockIdx.x * kSortTile + wave * STEPS * 64;
        uint32_t            mine[STEPS];
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) {
            const uint32_t i = first + s * 64 + lane;
            mine[s]          = i < n_entries ? (uint32_t) experts[i] : ~0u;
        }
        for (uint32_t e = lane; e < n_experts; e += 64) wave_count[wave][e] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s)
            if (mine[s] < n_experts) atomicAdd(&wave_count[wave][mine[s]], 1u);
        __syncthreads();
        uint32_t run = 0, here = 0;
        for (uint32_t e0 = 0; e0 < n_experts; e0 += THREADS) {
            const uint32_t e = e0 + threadIdx.x;
            uint32_t       all, in_tile = 0, count = 0;
            const uint32_t at = run + block_exclusive<THREADS>(e < n_experts ? totals[e] : 0u, &all);
            run += all;
            if (e < n_experts)
#pragma unroll
                for (uint32_t w = 0; w < WAVES; ++w) count += wave_count[w][e];
            in_tile = here + block_exclusive<THREADS>(count, &all);
            here += all;
            if (e < n_experts) {
                if (blockIdx.x == 0) offsets[e] = at;
                shift[e] = at + (n_entries ? counts[(size_t) blockIdx.x * n_experts + e] : 0u) - in_tile;
                for (uint32_t w = 0; w < WAVES; ++w) {
                    const uint32_t c = wave_count[w][e];
                    wave_count[w][e] = in_tile;
                    in_tile += c;
                }
            }
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) offsets[n_experts] = run;
        __syncthreads();
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) {// (a wavefront's own counts only: its LDS accesses stay in program order)
            const uint32_t i = first + s * 64 + lane, e = mine[s];
            const bool     valid = e < n_experts;
            const uint64_t alike = lanes_alike(e, valid, bits);
            const uint32_t below = __popcll(alike & ((1ull << lane) - 1ull));
            uint32_t       p     = ~0u;
            if (valid) {
                const uint32_t at = *(volatile uint32_t*) &wave_count[wave][e] + below;
                p                 = at + shift[e];
                entry[at]         = i;
                place_of[at]      = p;
                if (below == 0) *(volatile uint32_t*) &wave_count[wave][e] = at + (uint32_t) __popcll(alike);
            }
            if (i < n_entries) place[i] = (int32_t) p;
        }
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < here; at += THREADS) order[place_of[at]] = (int32_t) entry[at];
        // order behind the last entry: this tile's share of those places
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) {
            const uint32_t i = first + s * 64 + lane;
            if (i < n_entries && i >= run) order[i] = -1;
        }
    }

    // a wavefront's entries, 64 at a time from `first`: mine[e] (LDS) = where its next entry of e goes
    __device__ __forceinline__ void place_wave(uint32_t first, uint32_t steps, uint32_t n_entries, uint32_t n_experts, uint32_t bits, const int32_t* __restrict__ experts,
                                               int32_t* __restrict__ order, int32_t* __restrict__ place, uint32_t* mine) {
        const uint32_t lane = threadIdx.x & 63u;
        for (uint32_t s = 0; s < steps; ++s) {// (the wavefront's own words only: its LDS accesses stay in program order)
            const uint32_t i     = first + s * 64 + lane;
            const uint32_t e     = i < n_entries ? (uint32_t) experts[i] : ~0u;
            const bool     valid = e < n_experts;
            const uint64_t alike = lanes_alike(e, valid, bits);
            const uint32_t below = __popcll(alike & ((1ull << lane) - 1ull));
            uint32_t       p     = 0;
            if (valid) p = *(volatile uint32_t*) &mine[e] + below;
            if (i < n_entries) place[i] = valid ? (int32_t) p : -1;
            if (valid) {
                order[p] = (int32_t) i;
                if (below == 0) *(volatile uint32_t*) &mine[e] = p + (uint32_t) __popcll(alike);
            }
        }
    }

    // The whole sort in one workgroup of 16 wavefronts: a wavefront counts and places a contiguous part of the entries.
    constexpr uint32_t kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64, kSmallEntries = 8192, kSmallExperts = 512;

    __global__ __launch_bounds__(1024) void route_sort_small_kernel(uint32_t n_entries, uint32_t n_experts, uint32_t bits, const int32_t* __restrict__ experts,
                                                                    uint32_t* __restrict__ offsets, int32_t* __restrict__ order, int32_t* __restrict__ place) {
        extern __shared__ uint32_t wave_count[];// kSmallWaves x n_experts
        const uint32_t             lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const uint32_t             steps = (n_entries + kSmallThreads - 1) / kSmallThreads, first = wave * steps * 64;
        for (uint32_t i = threadIdx.x; i < kSmallWaves * n_experts; i += kSmallThreads) wave_count[i] = 0;
        __syncthreads();
        for (uint32_t s = 0; s < steps; ++s) {
            const uint32_t i = first + s * 64 + lane;
            const uint32_t e = i < n_entries ? (uint32_t) experts[i] : ~0u;
            if (e < n_experts) atomicAdd(&wave_count[wave * n_experts + e], 1u);
        }
        __syncthreads();
        uint32_t mine = 0;// (n_experts <= kSmallThreads: a thread each)
        if (threadIdx.x < n_experts)
            for (uint32_t w = 0; w < kSmallWaves; ++w) mine += wave_count[w * n_experts + threadIdx.x];
        uint32_t       all;
        const uint32_t base = block_exclusive<kSmallThreads>(mine, &all);
        if (threadIdx.x < n_experts) {
            offsets[threadIdx.x] = base;
            uint32_t at          = base;
            for (uint32_t w = 0; w < kSmallWaves; ++w) {
                const uint32_t c                              = wave_count[w * n_experts + threadIdx.x];
                wave_count[w * n_experts + threadIdx.x] = at;
                at += c;
            }
        }
        if (threadIdx.x == 0) offsets[n_experts] = all;
        for (uint32_t p = all + threadIdx.x; p < n_entries; p += kSmallThreads) order[p] = -1;
        __syncthreads();
        place_wave(first, steps, n_entries, n_experts, bits, experts, order, place, wave_count + wave * n_experts);
    }

    // ---- panels ----------------------------------------------------------------------------------------------------------------------------------------
    // A row is served by `lanes` neighbouring threads (a power of two, 16 bytes each per step).  All of it is streaming, bound by HBM: 16384 rows to 65536 places of 2048 bf16 62 us =
    // 5.4 TB/s, 30021 rows of 1001 fp32 back to 10007 32 us = 5.0 TB/s, the gradient of 65536 rows of 2048 bf16 118 us = 5.1 TB/s.
    struct RowShape {
        uint32_t lanes;// threads per row
        uint32_t shift;// log2
    };
    static RowShape row_shape(uint32_t units) {
        RowShape r{1, 0};
        while (r.lanes < 256 && r.lanes < units) r.lanes <<= 1, ++r.shift;
        return r;
    }

    // one unit of a row whose end may cut it; LARGE panels are streamed past the caches
    template<typename T, bool LARGE>
    __device__ __forceinline__ typename UnitOf<T>::mem unit_at(const T* __restrict__ p, uint32_t left) {
        typename UnitOf<T>::mem v;
        if (left >= (uint32_t) kUnit<T>) {
            auto* from = reinterpret_cast<const typename UnitOf<T>::mem*>(p);
            v          = LARGE ? __builtin_nontemporal_load(from) : *from;
        } else {
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i) v[i] = (uint32_t) i < left ? p[i] : (T) 0.0f;
        }
        return v;
    }
    template<typename T, bool LARGE>
    __device__ __forceinline__ void put_unit(T* __restrict__ p, uint32_t left, typename UnitOf<T>::mem v) {
        if (left >= (uint32_t) kUnit<T>) {
            auto* to = reinterpret_cast<typename UnitOf<T>::mem*>(p);
            if (LARGE) __builtin_nontemporal_store(v, to);
            else
                *to = v;
        } else {
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i)
                if ((uint32_t) i < left) p[i] = v[i];
        }
    }
    template<typename T>
    __device__ __forceinline__ typename UnitOf<T>::mem scaled(typename UnitOf<T>::mem v, float w) {
#pragma unroll
        for (int i = 0; i < kUnit<T>; ++i) v[i] = (T) (w * (float) v[i]);
        return v;
    }
    // rows [first, n_places) of a panel become 0; `rows` rows at a time, `lanes` threads each, `workers` workgroups
    template<typename T>
    __device__ __forceinline__ void clear_rows(T* __restrict__ out, uint32_t first, uint32_t n_places, uint32_t width, uint32_t worker, uint32_t workers, uint32_t shift) {
        constexpr uint32_t U = kUnit<T>;
        const uint32_t     lanes = 1u << shift, sub = threadIdx.x & (lanes - 1u), rows = 256u >> shift;
        for (uint64_t p = (uint64_t) first + worker * rows + (threadIdx.x >> shift); p < n_places; p += (uint64_t) workers * rows)
            for (uint32_t c = sub * U; c < width; c += lanes * U) put_unit<T, false>(out + p * width + c, width - c, typename UnitOf<T>::mem{});
    }

    // x is read once and written to each of the row's places (gathered instead, a row would be fetched once per entry from places far apart in time).
    template<typename T, bool WEIGHTED, bool LARGE>
    __global__ __launch_bounds__(256) void route_rows_kernel(uint32_t n_rows, uint32_t per_row, uint32_t width, uint32_t n_experts, uint32_t row_blocks, uint32_t shift,
                                                             const uint32_t* __restrict__ offsets, const int32_t* __restrict__ place, const float* __restrict__ weights,
                                                             const T* __restrict__ x, T* __restrict__ out) {
        constexpr uint32_t U        = kUnit<T>;
        const uint32_t     lanes    = 1u << shift, sub = threadIdx.x & (lanes - 1u);
        const uint32_t     n_places = n_rows * per_row;
        if (blockIdx.x >= row_blocks) {
            clear_rows(out, min(offsets[n_experts], n_places), n_places, width, blockIdx.x - row_blocks, gridDim.x - row_blocks, shift);
            return;
        }
        for (uint32_t r = blockIdx.x * (256u >> shift) + (threadIdx.x >> shift); r < n_rows; r += row_blocks * (256u >> shift))
            for (uint32_t c = sub * U; c < width; c += lanes * U) {
                const auto v = unit_at<T, LARGE>(x + (size_t) r * width + c, width - c);
                for (uint32_t j = 0; j < per_row; ++j) {
                    const uint32_t i = r * per_row + j;
                    const uint32_t p = (uint32_t) place[i];
                    if (p >= n_places) continue;
                    put_unit<T, LARGE>(out + (size_t) p * width + c, width - c, WEIGHTED ? scaled<T>(v, weights[i]) : v);
                }
            }
    }

    // four entries' units under way
    template<typename T, bool WEIGHTED, bool LARGE>
    __global__ __launch_bounds__(256) void route_back_kernel(uint32_t n_rows, uint32_t per_row, uint32_t width, uint32_t shift, const int32_t* __restrict__ place,
                                                             const float* __restrict__ weights, const T* __restrict__ y, T* __restrict__ out) {
        constexpr uint32_t U        = kUnit<T>, AHEAD = 4;
        const uint32_t     lanes    = 1u << shift, sub = threadIdx.x & (lanes - 1u);
        const uint32_t     n_places = n_rows * per_row;
        for (uint32_t r = blockIdx.x * (256u >> shift) + (threadIdx.x >> shift); r < n_rows; r += gridDim.x * (256u >> shift))
            for (uint32_t c = sub * U; c < width; c += lanes * U) {
                float s[U] = {};
                for (uint32_t j0 = 0; j0 < per_row; j0 += AHEAD) {
                    typename UnitOf<T>::mem v[AHEAD];
                    bool                    here[AHEAD];// (no entry: its weight does not count either)
#pragma unroll
                    for (uint32_t j = 0; j < AHEAD; ++j) {
                        const uint32_t p = j0 + j < per_row ? (uint32_t) place[r * per_row + j0 + j] : ~0u;
                        here[j]          = p < n_places;
                        if (here[j]) v[j] = unit_at<T, LARGE>(y + (size_t) p * width + c, width - c);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < AHEAD; ++j)
                        if (here[j]) {
                            const float w = WEIGHTED ? weights[r * per_row + j0 + j] : 1.0f;
#pragma unroll
                            for (uint32_t q = 0; q < U; ++q) s[q] = WEIGHTED ? fmaf(w, (float) v[j][q], s[q]) : s[q] + (float) v[j][q];
                        }
                }
                typename UnitOf<T>::mem o;
#pragma unroll
                for (uint32_t q = 0; q < U; ++q) o[q] = (T) s[q];
                put_unit<T, false>(out + (size_t) r * width + c, width - c, o);
            }
    }

    // One wavefront per row: an entry's weight gradient is reduced inside it.  UNITS units of dout's row stay in its registers (0: a row longer than eight per lane is read
    // again for every entry).
    template<typename T, uint32_t UNITS, bool LARGE>
    __global__ __launch_bounds__(256) void route_back_grad_kernel(uint32_t n_rows, uint32_t per_row, uint32_t width, uint32_t n_experts, uint32_t row_blocks,
                                                                  const uint32_t* __restrict__ offsets, const int32_t* __restrict__ place,
                                                                  const float* __restrict__ weights, const T* __restrict__ y, const T* __restrict__ dout,
                                                                  T* __restrict__ dy, float* __restrict__ dweights) {
        constexpr uint32_t U        = kUnit<T>, KEPT = UNITS ? UNITS : 1;
        const uint32_t     lane     = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const uint32_t     n_places = n_rows * per_row;
        if (blockIdx.x >= row_blocks) {
            clear_rows(dy, min(offsets[n_experts], n_places), n_places, width, blockIdx.x - row_blocks, gridDim.x - row_blocks, 6);
            return;
        }
        for (uint32_t r = blockIdx.x * 4 + wave; r < n_rows; r += row_blocks * 4) {
            const T*                grow = dout + (size_t) r * width;
            typename UnitOf<T>::mem kept[KEPT];
            if (UNITS)
#pragma unroll
                for (uint32_t u = 0; u < KEPT; ++u) {
                    const uint32_t c = (u * 64 + lane) * U;
                    if (c < width) kept[u] = unit_at<T, LARGE>(grow + c, width - c);
                }
            for (uint32_t j = 0; j < per_row; ++j) {
                const uint32_t i   = r * per_row + j;
                const uint32_t p   = (uint32_t) place[i];
                float          dot = 0.0f;
                if (p < n_places) {
                    const float w    = weights[i];
                    const T*    yrow = y + (size_t) p * width;
                    T*          drow = dy + (size_t) p * width;
                    auto        part = [&](uint32_t c, typename UnitOf<T>::mem g, typename UnitOf<T>::mem v) {
#pragma unroll
                        for (uint32_t q = 0; q < U; ++q) dot = fmaf((float) g[q], (float) v[q], dot);
                        put_unit<T, LARGE>(drow + c, width - c, scaled<T>(g, w));
                    };
                    if (UNITS) {
                        typename UnitOf<T>::mem v[KEPT];
#pragma unroll
                        for (uint32_t u = 0; u < KEPT; ++u) {
                            const uint32_t c = (u * 64 + lane) * U;
                            if (c < width) v[u] = unit_at<T, LARGE>(yrow + c, width - c);
                        }
#pragma unroll
                        for (uint32_t u = 0; u < KEPT; ++u) {
                            const uint32_t c = (u * 64 + lane) * U;
                            if (c < width) part(c, kept[u], v[u]);
                        }
                    } else {
                        for (uint32_t c = lane * U; c < width; c += 64 * U) part(c, unit_at<T, false>(grow + c, width - c), unit_at<T, LARGE>(yrow + c, width - c));
                    }
#pragma unroll
                    for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
                }
                if (lane == 0) dweights[i] = dot;
            }
        }
    }

    static int check_route(uint32_t n_rows, uint32_t per_row, uint32_t n_experts) {
        SPLAHIP_REQUIRE(per_row >= 1, "entries per row: at least one");
        SPLAHIP_REQUIRE(n_experts >= 1 && n_experts <= kMaxExperts, "experts: 1 .. 2048");
        SPLAHIP_REQUIRE((uint64_t) n_rows * per_row < (1ull << 31), "rows x entries per row: below 2^31");
        return SPLAHIP_OK;
    }
    static int check_width(uint32_t width) {
        SPLAHIP_REQUIRE(width < (1u << 30), "width: below 2^30");
        return SPLAHIP_OK;
    }
    constexpr uint32_t kRowBlocks  = 1u << 20;// at most: a launch holds fewer than 2^32 threads
    constexpr uint32_t kTailBlocks = 128;// workgroups that clear the rows behind the last entry (none of them: they return at once)
    // A panel that the caches (256 MB behind the L2s) do not hold along with what else is read: streamed past the L2 (the gradient of 65536 x 2048 bf16 rows 125 -> 119 us).
    static bool large_panel(uint32_t n_places, uint32_t width, size_t element) { return (uint64_t) n_places * width * element > (128ull << 20); }

}// namespace splahip

using namespace splahip;

static bool sorts_small(uint64_t n_entries, uint32_t n_experts) { return n_entries <= kSmallEntries && n_experts <= kSmallExperts; }

extern "C" size_t splahip_route_sort_workspace(uint32_t n_rows, uint32_t per_row, uint32_t n_experts) {
    if (sorts_small((uint64_t) n_rows * per_row, n_experts)) return 0;
    const size_t tiles = ((size_t) n_rows * per_row + kSortTile - 1) / kSortTile;
    return ((size_t) n_experts * tiles + n_experts) * 4;
}

extern "C" int splahip_route_sort(uint32_t n_rows, uint32_t per_row, uint32_t n_experts, const int32_t* d_experts, uint32_t* d_offsets, int32_t* d_order,
                                  int32_t* d_place, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (int st = check_route(n_rows, per_row, n_experts)) return st;
    const uint32_t n     = n_rows * per_row;
    const uint32_t tiles = (n + kSortTile - 1) / kSortTile;
    SPLAHIP_REQUIRE(d_offsets && (n == 0 || (d_experts && d_order && d_place)), "null array");
    const size_t need = splahip_route_sort_workspace(n_rows, per_row, n_experts);
    SPLAHIP_REQUIRE(workspace_bytes >= need && (need == 0 || d_workspace), "workspace too small");
    if (int st = ensure_device()) return st;
    hipStream_t s    = as_stream(stream);
    uint32_t    bits = 0;
    while ((1u << bits) < n_experts) ++bits;
    if (sorts_small(n, n_experts)) {
        route_sort_small_kernel<<<1, kSmallThreads, n_experts * 4 * kSmallWaves, s>>>(n, n_experts, bits, d_experts, d_offsets, d_order, d_place);
        SPLAHIP_TRY(hipGetLastError());
        return SPLAHIP_OK;
    }
    uint32_t* counts = static_cast<uint32_t*>(d_workspace);
    uint32_t* totals = counts + (size_t) n_experts * tiles;
    if (tiles) route_count_kernel<<<tiles, kSortThreads, 0, s>>>(n, n_experts, d_experts, counts);
    route_scan_kernel<<<(n_experts + 15) / 16, 1024, 0, s>>>(tiles, n_experts, counts, totals);
    const bool few = n_experts <= 512;
    auto*      place_kernel = few ? route_place_kernel<512, 1024> : route_place_kernel<kMaxExperts, 512>;
    place_kernel<<<tiles ? tiles : 1, few ? 1024 : 512, 0, s>>>(n, n_experts, bits, d_experts, counts, totals, d_offsets, d_order, d_place);
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}

extern "C" int splahip_route_rows(int panel_type, uint32_t n_rows, uint32_t per_row, uint32_t n_experts, uint32_t width, const uint32_t* d_offsets,
                                  const int32_t* d_place, const float* d_weights, const void* d_x, void* d_out, void* stream) {
    if (int st = check_route(n_rows, per_row, n_experts)) return st;
    if (int st = check_width(width)) return st;
    SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
    if (n_rows == 0 || width == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_place && d_x && d_out, "null array");
    if (int st = ensure_device()) return st;
    hipStream_t s = as_stream(stream);
    panel_dispatch(panel_type, [&](auto zero) {
        using T              = decltype(zero);
        const RowShape sh    = row_shape((width + kUnit<T> - 1) / kUnit<T>);
        const uint32_t rows  = 256u >> sh.shift, blocks = std::min((n_rows + rows - 1) / rows, kRowBlocks);
        auto*          x     = static_cast<const T*>(d_x);
        auto*          out   = static_cast<T*>(d_out);
        const bool     large = large_panel(n_rows * per_row, width, sizeof(T));
        auto*          kernel = d_weights ? (large ? route_rows_kernel<T, true, true> : route_rows_kernel<T, true, false>) : (large ? route_rows_kernel<T, false, true> : route_rows_kernel<T, false, false>);
        kernel<<<blocks + kTailBlocks, 256, 0, s>>>(n_rows, per_row, width, n_experts, blocks, sh.shift, d_offsets, d_place, d_weights, x, out);
    });
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}

extern "C" int splahip_route_back(int panel_type, uint32_t n_rows, uint32_t per_row, uint32_t width, const int32_t* d_place, const float* d_weights, const void* d_y,
                                  void* d_out, void* stream) {
    if (int st = check_route(n_rows, per_row, 1)) return st;
    if (int st = check_width(width)) return st;
    SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
    if (n_rows == 0 || width == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_place && d_y && d_out, "null array");
    if (int st = ensure_device()) return st;
    hipStream_t s = as_stream(stream);
    panel_dispatch(panel_type, [&](auto zero) {
        using T             = decltype(zero);
        const RowShape sh   = row_shape((width + kUnit<T> - 1) / kUnit<T>);
        const uint32_t rows = 256u >> sh.shift, blocks = std::min((n_rows + rows - 1) / rows, kRowBlocks);
        auto*          y    = static_cast<const T*>(d_y);
        auto*          out  = static_cast<T*>(d_out);
        const bool     large = large_panel(n_rows * per_row, width, sizeof(T));
        auto*          kernel = d_weights ? (large ? route_back_kernel<T, true, true> : route_back_kernel<T, true, false>) : (large ? route_back_kernel<T, false, true> : route_back_kernel<T, false, false>);
        kernel<<<blocks, 256, 0, s>>>(n_rows, per_row, width, sh.shift, d_place, d_weights, y, out);
    });
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}

extern "C" int splahip_route_back_grad(int panel_type, uint32_t n_rows, uint32_t per_row, uint32_t n_experts, uint32_t width, const uint32_t* d_offsets,
                                       const int32_t* d_place, const float* d_weights, const void* d_y, const void* d_dout, void* d_dy, float* d_dweights, void* stream) {
    if (int st = check_route(n_rows, per_row, n_experts)) return st;
    if (int st = check_width(width)) return st;
    SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
    if (n_rows == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_place && d_weights && d_dweights && (width == 0 || (d_y && d_dout && d_dy)), "null array");
    if (int st = ensure_device()) return st;
    hipStream_t    s      = as_stream(stream);
    const uint32_t blocks = std::min((n_rows + 3) / 4, kRowBlocks);
    panel_dispatch(panel_type, [&](auto zero) {
        using T = decltype(zero);
        const uint32_t per_lane = (width + 64 * kUnit<T> - 1) / (64 * kUnit<T>);
        const bool     large = large_panel(n_rows * per_row, width, sizeof(T));
        auto           pick = [&](auto units) {
            constexpr uint32_t N = decltype(units)::value;
            return large ? route_back_grad_kernel<T, N, true> : route_back_grad_kernel<T, N, false>;
        };
        auto* kernel = per_lane <= 1 ? pick(std::integral_constant<uint32_t, 1>{}) : per_lane <= 2 ? pick(std::integral_constant<uint32_t, 2>{})
                     : per_lane <= 4 ? pick(std::integral_constant<uint32_t, 4>{}) : per_lane <= 8 ? pick(std::integral_constant<uint32_t, 8>{}) : pick(std::integral_constant<uint32_t, 0>{});
        kernel<<<blocks + kTailBlocks, 256, 0, s>>>(n_rows, per_row, width, n_experts, blocks, d_offsets, d_place, d_weights, static_cast<const T*>(d_y),
                                                    static_cast<const T*>(d_dout), static_cast<T*>(d_dy), d_dweights);
    });
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}
