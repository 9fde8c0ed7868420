// expert_product.hip — a block-diagonal product: the rows of a panel sorted by expert (route.hip), every expert's range times that expert's dense matrix, and
// the gradients of that product for the rows and for the matrices, on the matrix cores.
//
//   splahip_expert_product     y[p, :]  = w[e(p)] x[p, :]            w [n_experts, n_out, n_in]
//   splahip_expert_product_dx  dx[p, :] = w[e(p)]^T dy[p, :]
//   splahip_expert_product_dw  dw[e]    = sum over the expert's rows of dy[p, :] x[p, :]^T
//
// Rows behind the last entry (offsets[n_experts] ..) become 0; an expert without rows has dw = 0.  fp32 sums in a fixed order, one rounding to the panel's
// type.  fp32 panels are multiplied in full fp32 (v_mfma_f32_16x16x4_f32).
#include "panel.hpp"

namespace splahip {

    typedef float    f32x4 __attribute__((ext_vector_type(4)));
    typedef bf16_t   bf16x8 __attribute__((ext_vector_type(8)));
    typedef fp16_t   fp16x8 __attribute__((ext_vector_type(8)));

    // ---- which rows a row tile covers ------------------------------------------------------------------------------------------------------------------
    // Row tiles are numbered expert by expert, ceil(rows / BM) each, the rows behind the last entry last (as expert number n_experts).
    struct RowTile {
        uint32_t expert;// n_experts: rows behind the last entry; > n_experts: no such tile
        uint32_t row0, rows;
    };
    __device__ __forceinline__ uint32_t bounded(const uint32_t* __restrict__ offsets, uint32_t e, uint32_t n_experts, uint32_t n_places) {
        return e > n_experts ? n_places : min(offsets[e], n_places);
    }
    // every wavefront finds it for itself: 64 experts per step, a scan over the lanes
    __device__ __forceinline__ RowTile find_row_tile(uint32_t tile, uint32_t bm, uint32_t n_experts, uint32_t n_places, const uint32_t* __restrict__ offsets) {
        const uint32_t lane = threadIdx.x & 63u;
        uint32_t       done = 0;
        for (uint32_t e0 = 0; e0 <= n_experts; e0 += 64) {
            const uint32_t e     = e0 + lane;
            const uint32_t begin = e <= n_experts ? bounded(offsets, e, n_experts, n_places) : n_places;
            const uint32_t end   = e <= n_experts ? bounded(offsets, e + 1, n_experts, n_places) : n_places;
            const uint32_t rows  = end > begin ? end - begin : 0u;
            const uint32_t tiles = (rows + bm - 1) / bm;
            uint32_t       inc   = tiles;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(inc, d);
                if (lane >= (uint32_t) d) inc += up;
            }
            const uint32_t ex   = done + inc - tiles;
            const uint64_t mine = __ballot(tile >= ex && tile < ex + tiles);
            if (mine) {
                const int      src = __ffsll((unsigned long long) mine) - 1;
                const uint32_t k   = tile - __shfl(ex, src), r = __shfl(rows, src);
                return RowTile{(uint32_t) __builtin_amdgcn_readfirstlane(e0 + src), (uint32_t) __builtin_amdgcn_readfirstlane(__shfl(begin, src) + k * bm),
                               (uint32_t) __builtin_amdgcn_readfirstlane(min(bm, r - k * bm))};
            }
            done += __builtin_amdgcn_readfirstlane(__shfl(inc, 63));
        }
        return RowTile{n_experts + 1, 0, 0};
    }
    // upper bound of the number of row tiles (the host does not know the ranges)
    static uint64_t row_tiles_bound(uint32_t n_places, uint32_t n_experts, uint32_t bm) {
        return n_places / bm + (uint64_t) min(n_experts + 1, n_places);
    }

    // ---- the general kernel ----------------------------------------------------------------------------------------------------------------------------
    // C[m, n] = sum over k of A(m, k) B(n, k) for any sizes, strides and alignment: 64 x 64 tiles, 32 of k per step through LDS, element loads with bounds.
    enum Form { kForward, kRowGrad, kMatrixGrad };

    struct GeneralArgs {
        const void *a, *b;
        void*       c;
        uint32_t    n_places, n_experts, m, n, k;// kForward: n = n_out, k = n_in; kRowGrad: n = n_in, k = n_out; kMatrixGrad: m = n_out, n = n_in
        const uint32_t* offsets;
    };

    template<typename T>
    struct Step;// one 16 x 16 result tile, 32 of k, operands of lane l: row l % 16, k = 8 (l / 16) ..
    template<>
    struct Step<bf16_t> {
        static __device__ __forceinline__ f32x4 mul(const bf16_t* a, const bf16_t* b, f32x4 c) {
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(a), *reinterpret_cast<const bf16x8*>(b), c, 0, 0, 0);
        }
    };
    template<>
    struct Step<fp16_t> {
        static __device__ __forceinline__ f32x4 mul(const fp16_t* a, const fp16_t* b, f32x4 c) {
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const fp16x8*>(a), *reinterpret_cast<const fp16x8*>(b), c, 0, 0, 0);
        }
    };
    template<>
    struct Step<float> {// (the order of k inside a step is free as long as both operands share it)
        static __device__ __forceinline__ f32x4 mul(const float* a, const float* b, f32x4 c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
            return c;
        }
    };

    template<typename T, Form FORM>
    __global__ __launch_bounds__(256) void product_general_kernel(const GeneralArgs g, uint32_t col_tiles) {
        constexpr uint32_t BM = 64, BN = 64, BK = 32, LD = BK + kUnit<T>;// (row stride of the LDS tiles: a unit more than BK against bank conflicts)
        __shared__ __align__(16) T As[BM * LD];
        __shared__ __align__(16) T Bs[BN * LD];
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const T*       A    = static_cast<const T*>(g.a);
        const T*       B    = static_cast<const T*>(g.b);
        T*             C    = static_cast<T*>(g.c);
        uint32_t       m0, n0, rows, cols, depth, expert;
        size_t         sam, sak, sbn, sbk, ldc;// element strides of A(m, k), B(n, k) and C's rows
        const uint32_t tile = blockIdx.x / col_tiles, col = blockIdx.x % col_tiles;
        n0 = col * BN;
        if (FORM == kMatrixGrad) {
            const uint32_t row_tiles = (g.m + BM - 1) / BM;
            expert                   = tile / row_tiles;
            m0                       = tile % row_tiles * BM;
            rows                     = min(BM, g.m - m0);
            cols                     = min(BN, g.n - n0);
            const uint32_t begin = bounded(g.offsets, expert, g.n_experts, g.n_places), end = bounded(g.offsets, expert + 1, g.n_experts, g.n_places);
            depth = end > begin ? end - begin : 0u;
            A += (size_t) begin * g.m + m0;
            B += (size_t) begin * g.n + n0;
            sam = 1, sak = g.m, sbn = 1, sbk = g.n;
            C += ((size_t) expert * g.m + m0) * g.n + n0;
        } else {
            const RowTile t = find_row_tile(tile, BM, g.n_experts, g.n_places, g.offsets);
            if (t.expert > g.n_experts) return;
            m0 = t.row0, rows = t.rows, expert = t.expert;
            cols  = min(BN, g.n - n0);
            depth = expert < g.n_experts ? g.k : 0u;
            A += (size_t) m0 * g.k;
            sam = g.k, sak = 1;
            if (FORM == kForward) B += ((size_t) expert * g.n + n0) * g.k, sbn = g.k, sbk = 1;
            else
                B += (size_t) expert * g.n * g.k + n0, sbn = 1, sbk = g.n;
            C += (size_t) m0 * g.n + n0;
        }
        ldc = g.n;
        f32x4 acc[2][2] = {};
        const uint32_t wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
        for (uint32_t k0 = 0; k0 < depth; k0 += BK) {
            __syncthreads();
#pragma unroll
            for (uint32_t s = 0; s < BM * BK / 256; ++s) {
                const uint32_t i = s * 256 + threadIdx.x;
                // neighbouring threads along the axis that is contiguous in memory
                const uint32_t am = FORM == kMatrixGrad ? i % BM : i / BK, ak = FORM == kMatrixGrad ? i / BM : i % BK;
                const uint32_t bn = FORM == kForward ? i / BK : i % BN, bk = FORM == kForward ? i % BK : i / BN;
                As[am * LD + ak]  = am < rows && k0 + ak < depth ? A[am * sam + (k0 + ak) * sak] : (T) 0.0f;
                Bs[bn * LD + bk]  = bn < cols && k0 + bk < depth ? B[bn * sbn + (k0 + bk) * sbk] : (T) 0.0f;
            }
            __syncthreads();
            const uint32_t r = lane & 15u, q = (lane >> 4) * 8;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = Step<T>::mul(As + (wm + i * 16 + r) * LD + q, Bs + (wn + j * 16 + r) * LD + q, acc[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const uint32_t m = wm + i * 16 + (lane >> 4) * 4 + v, n = wn + j * 16 + (lane & 15u);
                    if (m < rows && n < cols) C[m * ldc + n] = (T) acc[i][j][v];
                }
    }

    static int check_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out) {
        SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
        SPLAHIP_REQUIRE(n_experts >= 1 && n_experts <= 2048, "experts: 1 .. 2048");
        SPLAHIP_REQUIRE(n_places < (1u << 31), "rows: below 2^31");
        SPLAHIP_REQUIRE(n_in >= 1 && n_out >= 1 && n_in < (1u << 24) && n_out < (1u << 24), "matrix sizes: 1 .. 2^24 - 1");
        return SPLAHIP_OK;
    }

    template<Form FORM>
    static int launch_product(int panel_type, const GeneralArgs& g, hipStream_t s) {
        const uint64_t col_tiles = (g.n + 63) / 64;
        const uint64_t row_tiles = FORM == kMatrixGrad ? (uint64_t) g.n_experts * ((g.m + 63) / 64) : row_tiles_bound(g.n_places, g.n_experts, 64);
        SPLAHIP_REQUIRE(col_tiles * row_tiles < (1ull << 31), "too many tiles for one launch");
        panel_dispatch(panel_type, [&](auto zero) {
            product_general_kernel<decltype(zero), FORM><<<(uint32_t) (col_tiles * row_tiles), 256, 0, s>>>(g, (uint32_t) col_tiles);
        });
        SPLAHIP_TRY(hipGetLastError());
        return SPLAHIP_OK;
    }

}// namespace splahip

using namespace splahip;

extern "C" int splahip_expert_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets, const void* d_x,
                                      const void* d_w, void* d_y, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    if (n_places == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_x && d_w && d_y, "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kForward>(panel_type, GeneralArgs{d_x, d_w, d_y, n_places, n_experts, n_places, n_out, n_in, d_offsets}, as_stream(stream));
}

extern "C" int splahip_expert_product_dx(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_w, void* d_dx, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    if (n_places == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_dy && d_w && d_dx, "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kRowGrad>(panel_type, GeneralArgs{d_dy, d_w, d_dx, n_places, n_experts, n_places, n_in, n_out, d_offsets}, as_stream(stream));
}

extern "C" int splahip_expert_product_dw(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_x, void* d_dw, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    SPLAHIP_REQUIRE(d_offsets && d_dw && (n_places == 0 || (d_dy && d_x)), "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kMatrixGrad>(panel_type, GeneralArgs{d_dy, d_x, d_dw, n_places, n_experts, n_out, n_in, 0, d_offsets}, as_stream(stream));
}
