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
#include <type_traits>


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

    __device__ __forceinline__ uint32_t swz_rows(uint32_t row) { return (row >> 1) & 7u; }                          // [rows][64 of k]: unit ^= this
    __device__ __forceinline__ uint32_t swz_depth(uint32_t k) { return (k & 3u) << 1; }          // [64 of k][rows]: pair of units ^= this

    // 16 bytes per lane from global memory to LDS at dst + 16 lane (dst the same for the whole wavefront).  Written as assembly because the compiler waits for every
    // such load before the next LDS read of any address; the kernel waits itself, by loads_arrived().  It has no result register: nothing the compiler could reuse early.
    __device__ __forceinline__ void load_to_lds(const void* src, uint32_t dst) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
    }
    template<uint32_t LEFT>
    __device__ __forceinline__ void loads_arrived() {// all but the last LEFT of this wavefront's loads
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
    }

    // the operand of one v_mfma_f32_32x32x16: lane l holds row r0 + l % 32, k = k0 + 8 (l / 32) .. + 7
    template<typename T, uint32_t ROWS, bool DEPTH_CONTIGUOUS>
    __device__ __forceinline__ s16x8 operand(const T* lds, uint32_t r0, uint32_t k0) {
        const uint32_t lane = threadIdx.x & 63u;
        if (DEPTH_CONTIGUOUS) {
            const uint32_t row = r0 + (lane & 31u), unit = (k0 >> 3) + (lane >> 5);
            return *reinterpret_cast<const s16x8*>(lds + (size_t) row * kDepthStep + ((unit ^ swz_rows(row)) << 3));
        } else {
            // 16 lanes read 4 of k x 16 rows (8 bytes each) and get them transposed: 4 of k of one row
            s16x4 part[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t k  = k0 + (lane >> 5) * 8 + h * 4 + ((lane & 15u) >> 2);
                const uint32_t at = (((r0 >> 4) + ((lane >> 4) & 1u)) ^ swz_depth(k)) * 16 + (lane & 3u) * 4;
                part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (lds + (size_t) k * ROWS + at));
            }
            return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    typedef float f32x16 __attribute__((ext_vector_type(16)));
    __device__ __forceinline__ f32x16 matrix_step(s16x8 a, s16x8 b, f32x16 c, bf16_t) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x16 matrix_step(s16x8 a, s16x8 b, f32x16 c, fp16_t) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0, 0);
    }

    // The row tiles of the first 64 experts stay in a wavefront's registers (lane = expert), so that finding a tile's rows costs no memory access; further ones are found by
    // find_row_tile.
    struct RowTiles {
        uint32_t begin, rows, first;// of the lane's expert
        uint32_t known, total;      // row tiles of the first 64, of all
    };
    __device__ __forceinline__ RowTiles row_tiles_of(uint32_t bm, uint32_t n_experts, uint32_t n_places, const uint32_t* __restrict__ offsets) {
        const uint32_t lane = threadIdx.x & 63u;
        RowTiles       t{};
        for (uint32_t e0 = 0; e0 <= n_experts; e0 += 64) {
            const uint32_t e     = e0 + lane;
            const uint32_t begin = e <= n_experts ? bounded(offsets, e, n_experts, n_places) : n_places;
            const uint32_t end   = e <= n_experts ? bounded(offsets, e + 1, n_experts, n_places) : n_places;
            const uint32_t rows  = end > begin ? end - begin : 0u;
            uint32_t       inc   = (rows + bm - 1) / bm;
            const uint32_t own   = inc;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(inc, d);
                if (lane >= (uint32_t) d) inc += up;
            }
            const uint32_t sum = __builtin_amdgcn_readfirstlane(__shfl(inc, 63));
            if (e0 == 0) t.begin = begin, t.rows = rows, t.first = inc - own, t.known = sum;
            t.total += sum;
        }
        return t;
    }
    __device__ __forceinline__ RowTile row_tile(const RowTiles& t, uint32_t tile, uint32_t bm, uint32_t n_experts, uint32_t n_places, const uint32_t* __restrict__ offsets) {
        if (tile >= t.known) return find_row_tile(tile, bm, n_experts, n_places, offsets);
        // the last lane whose first tile is not behind it, among those that have one
        const uint64_t at = __ballot(t.first <= tile && t.rows);
        const int      e  = 63 - __clzll((long long) at);
        const uint32_t begin = __builtin_amdgcn_readlane(t.begin, e), rows = __builtin_amdgcn_readlane(t.rows, e), skip = (tile - __builtin_amdgcn_readlane(t.first, e)) * bm;
        return RowTile{(uint32_t) e, begin + skip, min(bm, rows - skip)};
    }

    // The tiles go to the workgroups in patches of about 32 neighbouring ones (up to 8 columns wide): a patch to the 32 CUs of one XCD, whose L2 then holds what they share, the
    // patches to the XCDs in turn.  Workgroup b runs in XCD b % 8 and takes one tile of each of the XCD's patches.
    template<typename P>
    __device__ __forceinline__ P* uniform(P* p) {// the same in every lane, as the compiler may not see
        const uint64_t v = (uint64_t) p;
        return (P*) (((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((uint32_t) (v >> 32)) << 32) | (uint32_t) __builtin_amdgcn_readfirstlane((uint32_t) v));
    }

    struct Patches {
        uint32_t row_tiles, col_tiles, wide, width, height, count;
    };
    __device__ __forceinline__ Patches patches_of(uint32_t row_tiles, uint32_t col_tiles) {
        Patches p{row_tiles, col_tiles, (col_tiles + 7) / 8, 0, 0, 0};
        p.width  = (col_tiles + p.wide - 1) / p.wide;
        p.height = 32 / p.width;
        p.count  = p.wide * ((row_tiles + p.height - 1) / p.height);
        return p;
    }

    // One operand's slab of ROWS x 64 of k, THREADS threads, 16 bytes each per load.  stride = elements between rows (k contiguous) or between k (rows contiguous).  The lane's byte offsets
    // from the slab's first element are made once per tile; the slab's address moves in scalar registers.  Rows outside the tile read the tile's first row instead (their
    // results are not stored).
    template<typename T, uint32_t ROWS, uint32_t THREADS, bool DEPTH_CONTIGUOUS>
    struct Slab {
        static constexpr uint32_t kLoads = ROWS * 8 / THREADS, kPerDepth = ROWS / 8;
        static __device__ __forceinline__ void offsets(uint32_t stride, uint32_t rows, uint32_t (&off)[kLoads]) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t u = i * THREADS + threadIdx.x;
                if (DEPTH_CONTIGUOUS) {
                    const uint32_t row = u >> 3;
                    off[i]             = ((row < rows ? row * stride : 0u) + depth_of(i)) * sizeof(T);
                } else {
                    const uint32_t kk = depth_of(i), row = ((u % kPerDepth) ^ (swz_depth(kk) << 1)) << 3;
                    off[i] = (kk * stride + (row < rows ? row : 0u)) * sizeof(T);
                }
            }
        }
        // the lane's first k inside the slab
        static __device__ __forceinline__ uint32_t depth_of(uint32_t i) {
            const uint32_t u = i * THREADS + threadIdx.x;
            return DEPTH_CONTIGUOUS ? ((u & 7u) ^ swz_rows(u >> 3)) << 3 : u / kPerDepth;
        }
    };
    __device__ __forceinline__ void load_to_lds_at(const void* base, uint32_t offset, uint32_t dst) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "memory");
    }

    // the slab that the depth ends in: units behind it come from the page of zeros
    template<typename S, typename T>
    __device__ __forceinline__ void last_slab(const T* base, const uint32_t (&off)[S::kLoads], uint32_t left, uint32_t dst, uint32_t step) {
#pragma unroll
        for (uint32_t i = 0; i < S::kLoads; ++i)
            load_to_lds(S::depth_of(i) < left ? reinterpret_cast<const char*>(base) + off[i] : reinterpret_cast<const char*>(zero_page), dst + i * step);
    }

    // A workgroup stays and computes one tile after another.  A step of k (64) is four quarters of 16: while a quarter's matrix instructions run from registers, the operands of the
    // next are read from LDS.  LDS holds five slabs, A0 B0 A1 B1 A2 ..: one barrier per step, before its last quarter: behind it every wavefront has read this step's two slabs, so the
    // next two loads may overwrite them, and the next step's slabs have arrived (issued one step ago, A's two steps ago).  The loads of the next tile's first slabs are
    // under way while a tile's result is stored.
    template<typename T, Form FORM, uint32_t BM, uint32_t WM, uint32_t WN, uint32_t OCC>
    __global__ __launch_bounds__(WM* WN * 64, OCC) void product_tile_kernel(const GeneralArgs g, uint32_t col_tiles) {
        constexpr uint32_t BN = BM, THREADS = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
        constexpr uint32_t LOADS = BM * 8 / THREADS;// per thread and slab
        constexpr bool     A_DEPTH = FORM != kMatrixGrad, B_DEPTH = FORM == kForward;
        using SlabA = Slab<T, BM, THREADS, A_DEPTH>;
        using SlabB = Slab<T, BN, THREADS, B_DEPTH>;
        constexpr uint32_t kSlots = 5, kSlab = BM * kDepthStep;
        constexpr uint32_t kMul = TM * TN, kReads = TM + TN;
        constexpr uint32_t kCols = BN / WN, kRowUnits = kCols / 8, kStores = TM * 32 * kRowUnits / 64;
        __shared__ __align__(1024) T slabs[kSlots][kSlab];
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
        const uint32_t stride_a = FORM == kMatrixGrad ? g.m : g.k, stride_b = FORM == kForward ? g.k : g.n;
        const size_t   move_a = A_DEPTH ? kDepthStep : (size_t) kDepthStep * stride_a, move_b = B_DEPTH ? kDepthStep : (size_t) kDepthStep * stride_b;
        const uint32_t lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void*) slabs + wave * 1024;

        RowTiles       tiles{};
        const uint32_t m_tiles = (g.m + BM - 1) / BM;// kMatrixGrad: row tiles of an expert
        if (FORM != kMatrixGrad) tiles = row_tiles_of(BM, g.n_experts, g.n_places, g.offsets);
        const Patches  patches = patches_of(FORM == kMatrixGrad ? g.n_experts * m_tiles : tiles.total, col_tiles);
        const uint32_t team = gridDim.x / 8, member = blockIdx.x / 8;// (the grid is a multiple of 8)

        // the tile at hand
        const T *      A, *B;
        T*             C;
        uint32_t       rows, cols, depth, steps, whole;
        uint32_t       off_a[LOADS], off_b[LOADS];
        // the XCD's tiles are numbered patch by patch; at >= its count: done
        const uint32_t area = patches.width * patches.height;
        uint32_t       at   = member;
        auto           next = [&]() -> bool {
            for (;; at += team) {
                const uint32_t p = at / area * 8 + blockIdx.x % 8, in = at % area;
                if (p >= patches.count) return false;
                const uint32_t row = p / patches.wide * patches.height + in / patches.width, col = p % patches.wide * patches.width + in % patches.width;
                if (row >= patches.row_tiles || col >= patches.col_tiles) continue;
                const uint32_t n0 = col * BN;
                cols              = min(BN, g.n - n0);
                if (FORM == kMatrixGrad) {
                    const uint32_t expert = row / m_tiles, m0 = row % m_tiles * BM;
                    const uint32_t begin = bounded(g.offsets, expert, g.n_experts, g.n_places), end = bounded(g.offsets, expert + 1, g.n_experts, g.n_places);
                    rows                 = min(BM, g.m - m0);
                    depth                = end > begin ? end - begin : 0u;
                    A = static_cast<const T*>(g.a) + (size_t) begin * g.m + m0;
                    B = static_cast<const T*>(g.b) + (size_t) begin * g.n + n0;
                    C = static_cast<T*>(g.c) + ((size_t) expert * g.m + m0) * g.n + n0;
                } else {
                    const RowTile t = row_tile(tiles, row, BM, g.n_experts, g.n_places, g.offsets);
                    const uint32_t e = min(t.expert, g.n_experts - 1);
                    rows            = t.rows;
                    depth           = t.expert < g.n_experts ? g.k : 0u;
                    A = static_cast<const T*>(g.a) + (size_t) t.row0 * g.k;
                    B = static_cast<const T*>(g.b) + (FORM == kForward ? ((size_t) e * g.n + n0) * g.k : (size_t) e * g.n * g.k + n0);
                    C = static_cast<T*>(g.c) + (size_t) t.row0 * g.n + n0;
                }
                A = uniform(A), B = uniform(B), C = uniform(C);
                rows = __builtin_amdgcn_readfirstlane(rows), depth = __builtin_amdgcn_readfirstlane(depth);
                steps = (depth + kDepthStep - 1) / kDepthStep, whole = depth / kDepthStep;
                uint32_t sa = stride_a, sb = stride_b;// (opaque: what depends on them is made anew for each tile, not kept in registers)
                asm volatile("" : "+s"(sa), "+s"(sb));
                SlabA::offsets(sa, rows, off_a);
                SlabB::offsets(sb, cols, off_b);
                at += team;
                return true;
            }
        };
        auto slot_after = [](uint32_t slot, uint32_t n) { return slot + n >= kSlots ? slot + n - kSlots : slot + n; };
        auto load_a = [&](uint32_t s, uint32_t slot, uint32_t i) { load_to_lds_at(A + s * move_a, off_a[i], lds0 + slot * (kSlab * 2) + i * (THREADS * 16)); };
        auto load_b = [&](uint32_t s, uint32_t slot, uint32_t i) { load_to_lds_at(B + s * move_b, off_b[i], lds0 + slot * (kSlab * 2) + i * (THREADS * 16)); };
        auto slab_a = [&](uint32_t s, uint32_t slot) {
            if (s < whole) {
#pragma unroll
                for (uint32_t i = 0; i < LOADS; ++i) load_a(s, slot, i);
            } else if (s < steps)
                last_slab<SlabA>(A + s * move_a, off_a, depth - s * kDepthStep, lds0 + slot * (kSlab * 2), THREADS * 16);
        };
        auto slab_b = [&](uint32_t s, uint32_t slot) {
            if (s < whole) {
#pragma unroll
                for (uint32_t i = 0; i < LOADS; ++i) load_b(s, slot, i);
            } else if (s < steps)
                last_slab<SlabB>(B + s * move_b, off_b, depth - s * kDepthStep, lds0 + slot * (kSlab * 2), THREADS * 16);
        };

        if (!next()) return;
        slab_a(0, 0), slab_b(0, 1), slab_a(1, 2), slab_b(1, 3);
        bool stored = false;// a whole tile's stores are among the loads under way
        for (bool more = true; more;) {
            f32x16 acc[TM][TN] = {};
            slab_a(2, 4);
            if (steps) {
                // the first two slabs: behind them three more, and a whole tile's stores
                if (whole < 3) loads_arrived<0>();
                else if (stored)
                    loads_arrived<3 * LOADS + kStores>();
                else
                    loads_arrived<3 * LOADS>();
                __syncthreads();
                s16x8 fa[2][TM], fb[2][TN];
#pragma unroll
                for (uint32_t j = 0; j < TN; ++j) fb[0][j] = operand<T, BN, B_DEPTH>(slabs[1], wn + j * 32, 0);
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i) fa[0][i] = operand<T, BM, A_DEPTH>(slabs[0], wm + i * 32, 0);
                // quarter q's matrix instructions; the next quarter's operands are read meanwhile, and with `load` the loads of B's slab ls and A's next one issued
                auto quarter = [&](auto q_, auto load_, const T* as, const T* bs, uint32_t ls, uint32_t slot) {
                    constexpr uint32_t q = decltype(q_)::value, cur = q & 1u, k0 = (q + 1) % 4 * 16;
                    constexpr bool     load = decltype(load_)::value;
#pragma unroll
                    for (uint32_t x = 0; x < kMul; ++x) {
                        if (x < TN) fb[cur ^ 1][x] = operand<T, BN, B_DEPTH>(bs, wn + x * 32, k0);
                        else if (x < kReads)
                            fa[cur ^ 1][x - TN] = operand<T, BM, A_DEPTH>(as, wm + (x - TN) * 32, k0);
                        if (load)
#pragma unroll
                            for (uint32_t l = x * 2 * LOADS / kMul; l < (x + 1) * 2 * LOADS / kMul; ++l) {
                                if (l < LOADS) load_b(ls, slot, l);
                                else
                                    load_a(ls + 1, slot_after(slot, 1), l - LOADS);
                            }
                        acc[x / TN][x % TN] = matrix_step(fb[cur][x % TN], fa[cur][x / TN], acc[x / TN][x % TN], T{});
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                using std::integral_constant;
                constexpr integral_constant<bool, true>  yes{};
                constexpr integral_constant<bool, false> no{};
                uint32_t                                 slot = 0;// of A's slab
                auto                                     step = [&](auto load_, uint32_t s) {
                    const T *as = slabs[slot], *bs = slabs[slot_after(slot, 1)];
                    quarter(integral_constant<uint32_t, 0>{}, no, as, bs, 0, 0);
                    quarter(integral_constant<uint32_t, 1>{}, no, as, bs, 0, 0);
                    quarter(integral_constant<uint32_t, 2>{}, no, as, bs, 0, 0);
                    if (decltype(load_)::value) loads_arrived<LOADS>();
                    else
                        loads_arrived<0>();
                    __syncthreads();
                    // B's slab s + 2 goes where A's s was, A's s + 3 where B's s was
                    if (!decltype(load_)::value) slab_b(s + 2, slot), slab_a(s + 3, slot_after(slot, 1));
                    quarter(integral_constant<uint32_t, 3>{}, load_, slabs[slot_after(slot, 2)], slabs[slot_after(slot, 3)], s + 2, slot);
                    slot = slot_after(slot, 2);
                };
                uint32_t s = 0;
                for (; s + 3 < whole; ++s) step(yes, s);
                for (; s < steps; ++s) step(no, s);
                __syncthreads();// nothing reads a slab any more
            }
            T* const       out = C;
            uint32_t       ldc = g.n;
            asm volatile("" : "+s"(ldc));
            const uint32_t out_rows = rows, out_cols = cols;
            more = next();
            if (more) slab_a(0, 0), slab_b(0, 1), slab_a(1, 2), slab_b(1, 3);
            stored = out_rows == BM && out_cols == BN;
            // A lane holds four neighbouring columns (8 bytes) of a row, its neighbours hold other rows.  Every wavefront turns its part in the fifth slab, 32 rows at a time, and stores
            // rows of BN / WN columns.
            T*   turn = slabs[4] + wave * (32 * kCols);
            auto swz  = [](uint32_t m) { return (m / (16 / kRowUnits)) % kRowUnits; };
#pragma unroll
            for (uint32_t i = 0; i < TM; ++i) {
                const uint32_t m = lane & 31u;
#pragma unroll
                for (uint32_t j = 0; j < TN; ++j)
#pragma unroll
                    for (uint32_t v = 0; v < 16; v += 4) {
                        typedef T four __attribute__((ext_vector_type(4)));
                        four      c;
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) c[q] = (T) acc[i][j][v + q];
                        const uint32_t unit = j * 4 + v / 4;
                        *reinterpret_cast<four*>(turn + m * kCols + ((unit ^ swz(m)) * 8 + (lane >> 5) * 4)) = c;
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (uint32_t x = 0; x < 32 * kRowUnits / 64; ++x) {
                    const uint32_t u = x * 64 + lane, row = u / kRowUnits, unit = u % kRowUnits;
                    const s16x8    c = *reinterpret_cast<const s16x8*>(turn + row * kCols + ((unit ^ swz(row)) * 8));
                    const uint32_t gm = wm + i * 32 + row, gn = wn + unit * 8;
                    if (gm < out_rows && gn < out_cols) *reinterpret_cast<s16x8*>(out + (size_t) gm * ldc + gn) = c;// (columns come in eights)
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            if (more) __syncthreads();// the fifth slab is free again
        }
    }

    static int check_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out) {
        SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
        SPLAHIP_REQUIRE(n_experts >= 1 && n_experts <= 2048, "experts: 1 .. 2048");
        SPLAHIP_REQUIRE(n_places < (1u << 31), "rows: below 2^31");
        SPLAHIP_REQUIRE(n_in >= 1 && n_out >= 1 && n_in < (1u << 24) && n_out < (1u << 24), "matrix sizes: 1 .. 2^24 - 1");
        return SPLAHIP_OK;
    }

    template<typename T, Form FORM, uint32_t BM, uint32_t WM, uint32_t WN, uint32_t OCC>
    static int launch_tiles(const GeneralArgs& g, hipStream_t s) {
        const uint64_t col_tiles = (g.n + BM - 1) / BM;
        const uint64_t row_tiles = FORM == kMatrixGrad ? (uint64_t) g.n_experts * ((g.m + BM - 1) / BM) : row_tiles_bound(g.n_places, g.n_experts, BM);
        SPLAHIP_REQUIRE(col_tiles * row_tiles < (1ull << 31), "too many tiles for one launch");
        constexpr uint32_t kResident = 256 * (OCC * 4 / (WM * WN));// workgroups the card holds at once
        product_tile_kernel<T, FORM, BM, WM, WN, OCC><<<kResident, WM * WN * 64, 0, s>>>(g, (uint32_t) col_tiles);
        return SPLAHIP_OK;
    }

    template<Form FORM>
    static int launch_product(int panel_type, const GeneralArgs& g, hipStream_t s) {
        const bool units = g.n < (1u << 22) && g.k < (1u << 22) && g.m < (1u << 22) && ((uintptr_t) g.a % 16 == 0) && ((uintptr_t) g.b % 16 == 0) && ((uintptr_t) g.c % 16 == 0) && g.n % 8 == 0 && g.k % 8 == 0 && g.m % 8 == 0;
        int        st    = SPLAHIP_OK;
        if (panel_type != SPLAHIP_PANEL_FLOAT && units) {
            const uint64_t tiles = FORM == kMatrixGrad ? (uint64_t) g.n_experts * ((g.m + 255) / 256) * ((g.n + 255) / 256) : (uint64_t) (g.n_places / 256 + 1) * ((g.n + 255) / 256);
            const bool     large = tiles >= 200;
            if (panel_type == SPLAHIP_PANEL_HALF) st = large ? launch_tiles<fp16_t, FORM, 256, 2, 4, 2>(g, s) : launch_tiles<fp16_t, FORM, 128, 2, 2, 2>(g, s);
            else
                st = large ? launch_tiles<bf16_t, FORM, 256, 2, 4, 2>(g, s) : launch_tiles<bf16_t, FORM, 128, 2, 2, 2>(g, s);
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
