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

    // ---- 16-bit panels: large tiles -------------------------------------------------------------------------------------------------------------------
    // A workgroup computes BM x BN of the result, BK = 64 of k per step: both operands' slabs go from global memory straight into LDS (16 bytes per lane, no
    // registers between), double buffered, and feed v_mfma_f32_16x16x32.  The product is taken transposed (the instruction's rows are the result's columns), so that
    // a lane holds four neighbouring columns of a result row and stores 8 bytes.
    //
    // An operand whose k axis is contiguous in memory lies in LDS as [rows][64 of k], one whose row axis is contiguous as [64 of k][rows] and is read
    // with the transposing LDS read.  The units (16 bytes) of an LDS row are permuted by an exclusive-or with bits of the row's number so that the lanes of
    // one read meet different banks; the direct loads write LDS in lane order, so the permutation is in the lanes' global addresses.
    // Units outside the operand (k beyond the depth, rows beyond the tile) come from a page of zeros.
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));

    __device__ const uint4 zero_page[4] = {};

    constexpr uint32_t kDepthStep = 64;

    __device__ __forceinline__ uint32_t swz_rows(uint32_t row) { return row & 7u; }                          // [rows][64 of k]: unit ^= this
    __device__ __forceinline__ uint32_t swz_depth(uint32_t k) { return (k & 3u) | ((k >> 1) & 4u); }          // [64 of k][rows]: pair of units ^= this

    // 16 bytes per lane from global memory to LDS at dst + 16 lane (dst the same for the whole wavefront).  Written as assembly because the compiler waits for every
    // such load before the next LDS read of any address; the kernel waits itself, by loads_arrived().  It has no result register: nothing the compiler could reuse early.
    __device__ __forceinline__ void load_to_lds(const void* src, void* dst) {
        const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (__attribute__((address_space(3))) void*) dst);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src) : "memory", "m0");
    }
    template<uint32_t LEFT>
    __device__ __forceinline__ void loads_arrived() {// all but the last LEFT of this wavefront's loads
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
    }

    // one operand's slab of ROWS x 64: THREADS threads, base = its element (row 0, k 0), stride = elements between rows (k contiguous) or between k (rows contiguous)
    template<typename T, uint32_t ROWS, uint32_t THREADS, bool DEPTH_CONTIGUOUS>
    __device__ __forceinline__ void stage(const T* __restrict__ base, uint32_t stride, uint32_t rows, uint32_t depth, uint32_t k0, T* lds) {
        constexpr uint32_t kUnits = ROWS * kDepthStep / 8;
        static_assert(kUnits % THREADS == 0, "whole steps");
        const uint32_t wave_base = threadIdx.x & ~63u;
#pragma unroll
        for (uint32_t i = 0; i < kUnits / THREADS; ++i) {
            const uint32_t u = i * THREADS + threadIdx.x;// the unit's place in LDS
            const void*    src;
            if (DEPTH_CONTIGUOUS) {
                const uint32_t row = u >> 3, k = k0 + (((u & 7u) ^ swz_rows(row)) << 3);
                src = row < rows && k < depth ? (const void*) (base + (size_t) row * stride + k) : (const void*) zero_page;
            } else {
                constexpr uint32_t per = ROWS / 8;
                const uint32_t     kk = u / per, at = u % per, row = (at ^ (swz_depth(kk) << 1)) << 3, k = k0 + kk;
                src = row < rows && k < depth ? (const void*) (base + (size_t) k * stride + row) : (const void*) zero_page;
            }
            load_to_lds(src, lds + (size_t) (i * THREADS + wave_base) * 8);
        }
    }

    // the operand of one v_mfma_f32_16x16x32: lane l holds row r0 + l % 16, k = 8 (l / 16) .. + 7 of the 32 at k0
    template<typename T, uint32_t ROWS, bool DEPTH_CONTIGUOUS>
    __device__ __forceinline__ s16x8 operand(const T* lds, uint32_t r0, uint32_t k0) {
        const uint32_t lane = threadIdx.x & 63u;
        if (DEPTH_CONTIGUOUS) {
            const uint32_t row = r0 + (lane & 15u), unit = (k0 >> 3) + (lane >> 4);
            return *reinterpret_cast<const s16x8*>(lds + (size_t) row * kDepthStep + ((unit ^ swz_rows(row)) << 3));
        } else {
            // 16 lanes read 4 of k x 16 rows (8 bytes each) and get them transposed: 4 of k of one row
            s16x4 part[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t k = k0 + (lane >> 4) * 8 + h * 4 + ((lane & 15u) >> 2);
                const uint32_t at = ((r0 >> 4) ^ swz_depth(k)) * 16 + (lane & 3u) * 4;
                part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (lds + (size_t) k * ROWS + at));
            }
            return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    __device__ __forceinline__ f32x4 matrix_step(s16x8 a, s16x8 b, f32x4 c, bf16_t) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x4 matrix_step(s16x8 a, s16x8 b, f32x4 c, fp16_t) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0, 0);
    }

    // Workgroup number -> tile: workgroups go round the 8 XCDs, each of which has an L2 of its own; an XCD gets a contiguous run of tiles, and a run
    // walks the columns of kGroup row tiles side by side, so that the workgroups at work in an XCD share both operands' slabs.
    struct TileAt {
        uint32_t row, col;
    };
    __device__ __forceinline__ TileAt tile_at(uint32_t block, uint32_t row_tiles, uint32_t col_tiles) {
        constexpr uint32_t kGroup = 4;
        const uint32_t     total = row_tiles * col_tiles, per = total / 8, extra = total % 8;
        const uint32_t     xcd = block % 8, local = block / 8;
        const uint32_t     id    = xcd * per + min(xcd, extra) + local;
        const uint32_t     group = id / (kGroup * col_tiles), in = id % (kGroup * col_tiles);
        const uint32_t     height = min(kGroup, row_tiles - group * kGroup);
        return TileAt{group * kGroup + in % height, in / height};
    }

    template<typename T, Form FORM, uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN>
    __global__ __launch_bounds__(WM* WN * 64) void product_tile_kernel(const GeneralArgs g, uint32_t row_tiles, uint32_t col_tiles) {
        constexpr uint32_t THREADS = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16;
        constexpr bool     A_DEPTH = FORM != kMatrixGrad, B_DEPTH = FORM == kForward;
        __shared__ __align__(1024) T As[2][BM * kDepthStep];
        __shared__ __align__(1024) T Bs[2][BN * kDepthStep];
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const T*       A    = static_cast<const T*>(g.a);
        const T*       B    = static_cast<const T*>(g.b);
        T*             C    = static_cast<T*>(g.c);
        const TileAt   at   = tile_at(blockIdx.x, row_tiles, col_tiles);
        uint32_t       rows, depth, stride_a, stride_b;
        const uint32_t n0 = at.col * BN, cols = min(BN, g.n - n0);
        if (FORM == kMatrixGrad) {
            const uint32_t per = (g.m + BM - 1) / BM, expert = at.row / per, m0 = at.row % per * BM;
            const uint32_t begin = bounded(g.offsets, expert, g.n_experts, g.n_places), end = bounded(g.offsets, expert + 1, g.n_experts, g.n_places);
            rows                 = min(BM, g.m - m0);
            depth                = end > begin ? end - begin : 0u;
            A += (size_t) begin * g.m + m0;
            B += (size_t) begin * g.n + n0;
            C += ((size_t) expert * g.m + m0) * g.n + n0;
            stride_a = g.m, stride_b = g.n;
        } else {
            const RowTile t = find_row_tile(at.row, BM, g.n_experts, g.n_places, g.offsets);
            if (t.expert > g.n_experts) return;
            rows  = t.rows;
            depth = t.expert < g.n_experts ? g.k : 0u;
            A += (size_t) t.row0 * g.k;
            if (t.expert < g.n_experts) B += FORM == kForward ? ((size_t) t.expert * g.n + n0) * g.k : (size_t) t.expert * g.n * g.k + n0;
            C += (size_t) t.row0 * g.n + n0;
            stride_a = g.k, stride_b = FORM == kForward ? g.k : g.n;
        }
        const uint32_t wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
        f32x4          acc[TM][TN] = {};
        const uint32_t steps       = (depth + kDepthStep - 1) / kDepthStep;
        if (steps) {
            stage<T, BM, THREADS, A_DEPTH>(A, stride_a, rows, depth, 0, As[0]);
            stage<T, BN, THREADS, B_DEPTH>(B, stride_b, cols, depth, 0, Bs[0]);
        }
        for (uint32_t s = 0; s < steps; ++s) {
            loads_arrived<0>();
            __syncthreads();// every wavefront's part of this step's slabs has arrived, the other buffers have been read
            if (s + 1 < steps) {
                stage<T, BM, THREADS, A_DEPTH>(A, stride_a, rows, depth, (s + 1) * kDepthStep, As[(s + 1) & 1]);
                stage<T, BN, THREADS, B_DEPTH>(B, stride_b, cols, depth, (s + 1) * kDepthStep, Bs[(s + 1) & 1]);
            }
            const T *as = As[s & 1], *bs = Bs[s & 1];
#pragma unroll
            for (uint32_t kk = 0; kk < kDepthStep; kk += 32) {
                s16x8 a[TM], b[TN];
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i) a[i] = operand<T, BM, A_DEPTH>(as, wm + i * 16, kk);
#pragma unroll
                for (uint32_t j = 0; j < TN; ++j) b[j] = operand<T, BN, B_DEPTH>(bs, wn + j * 16, kk);
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < TN; ++j) acc[i][j] = matrix_step(b[j], a[i], acc[i][j], T{});
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < TM; ++i) {
            const uint32_t m = wm + i * 16 + (lane & 15u);
            if (m >= rows) continue;
#pragma unroll
            for (uint32_t j = 0; j < TN; ++j) {
                const uint32_t n = wn + j * 16 + (lane >> 4) * 4;
                if (n >= cols) continue;// (columns come in eights)
                typedef T four __attribute__((ext_vector_type(4)));
                four      v;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = (T) acc[i][j][q];
                *reinterpret_cast<four*>(C + (size_t) m * g.n + n) = v;
            }
        }
    }

    static int check_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out) {
        SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
        SPLAHIP_REQUIRE(n_experts >= 1 && n_experts <= 2048, "experts: 1 .. 2048");
        SPLAHIP_REQUIRE(n_places < (1u << 31), "rows: below 2^31");
        SPLAHIP_REQUIRE(n_in >= 1 && n_out >= 1 && n_in < (1u << 24) && n_out < (1u << 24), "matrix sizes: 1 .. 2^24 - 1");
        return SPLAHIP_OK;
    }

    template<typename T, Form FORM, uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN>
    static int launch_tiles(const GeneralArgs& g, hipStream_t s) {
        const uint64_t col_tiles = (g.n + BN - 1) / BN;
        const uint64_t row_tiles = FORM == kMatrixGrad ? (uint64_t) g.n_experts * ((g.m + BM - 1) / BM) : row_tiles_bound(g.n_places, g.n_experts, BM);
        SPLAHIP_REQUIRE(col_tiles * row_tiles < (1ull << 31), "too many tiles for one launch");
        product_tile_kernel<T, FORM, BM, BN, WM, WN><<<(uint32_t) (col_tiles * row_tiles), WM * WN * 64, 0, s>>>(g, (uint32_t) row_tiles, (uint32_t) col_tiles);
        return SPLAHIP_OK;
    }

    template<Form FORM>
    static int launch_product(int panel_type, const GeneralArgs& g, hipStream_t s) {
        const bool units = ((uintptr_t) g.a % 16 == 0) && ((uintptr_t) g.b % 16 == 0) && ((uintptr_t) g.c % 16 == 0) && g.n % 8 == 0 && g.k % 8 == 0 && g.m % 8 == 0;
        int        st    = SPLAHIP_OK;
        if (panel_type != SPLAHIP_PANEL_FLOAT && units) {
            if (panel_type == SPLAHIP_PANEL_HALF) st = launch_tiles<fp16_t, FORM, 256, 256, 2, 4>(g, s);
            else
                st = launch_tiles<bf16_t, FORM, 256, 256, 2, 4>(g, s);
            if (st) return st;
            SPLAHIP_TRY(hipGetLastError());
            return SPLAHIP_OK;
        }
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
    return launch_product<kForward>(panel_type, GeneralArgs{d_x, d_w, d_y, n_places, n_experts, 0, n_out, n_in, d_offsets}, as_stream(stream));
}

extern "C" int splahip_expert_product_dx(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_w, void* d_dx, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    if (n_places == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_dy && d_w && d_dx, "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kRowGrad>(panel_type, GeneralArgs{d_dy, d_w, d_dx, n_places, n_experts, 0, n_in, n_out, d_offsets}, as_stream(stream));
}

extern "C" int splahip_expert_product_dw(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_x, void* d_dw, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    SPLAHIP_REQUIRE(d_offsets && d_dw && (n_places == 0 || (d_dy && d_x)), "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kMatrixGrad>(panel_type, GeneralArgs{d_dy, d_x, d_dw, n_places, n_experts, n_out, n_in, 0, d_offsets}, as_stream(stream));
}
