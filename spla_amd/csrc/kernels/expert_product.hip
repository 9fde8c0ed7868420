// expert_product.hip — a block-diagonal product: the rows of a panel sorted by expert (route.hip), every expert's range times that expert's dense matrix, and
// the gradients of that product for the rows and for the matrices, on the matrix cores.
//
//   splahip_expert_product     y[p, :]  = w[e(p)] x[p, :]            w [n_experts, n_out, n_in]
//   splahip_expert_product_dx  dx[p, :] = w[e(p)]^T dy[p, :]
//   splahip_expert_product_dw  dw[e]    = sum over the expert's rows of dy[p, :] x[p, :]^T
//
// Rows behind the last entry (offsets[n_experts] ..) become 0, and what operands hold there does not count; an expert without rows has dw = 0.  fp32 sums in a fixed order, one rounding to the panel's
// type.  fp32 panels are multiplied in full fp32 (v_mfma_f32_32x32x2_f32).
#include "panel.hpp"

#include <algorithm>
#include <type_traits>

namespace splahip {

    typedef float    f32x4 __attribute__((ext_vector_type(4)));
    typedef float    f32x16 __attribute__((ext_vector_type(16)));
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

    template<typename P>
    __device__ __forceinline__ P* uniform(P* p) {// the same in every lane, as the compiler may not see
        const uint64_t v = (uint64_t) p;
        const uint64_t u = ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((uint32_t) (v >> 32)) << 32) | (uint32_t) __builtin_amdgcn_readfirstlane((uint32_t) v);
        return (P*) (__attribute__((address_space(1))) P*) u;// (global memory: not the flat accesses that a number turned pointer would get)
    }

    // Tile number t of a grid of row_tiles x col_tiles: H row tiles side by side, column by column, so that neighbouring tiles share both operands' slabs.
    struct TileAt {
        uint32_t row, col;
    };
    template<uint32_t H>
    __device__ __forceinline__ TileAt tile_at(uint32_t t, uint32_t row_tiles, uint32_t col_tiles) {
        const uint32_t group = t / (H * col_tiles), in = t % (H * col_tiles), height = min(H, row_tiles - group * H);
        return TileAt{group * H + in % height, in / height};
    }

    // rank -> expert with the most rows first, for up to 64 experts (the order is free); lane = expert
    __device__ __forceinline__ uint32_t rank_by_rows(uint32_t rows, uint32_t n_experts) {
        const uint32_t lane = threadIdx.x & 63u;
        uint32_t       rank = 0;
        for (uint32_t e = 0; e < n_experts; ++e) {
            const uint32_t r = __builtin_amdgcn_readlane(rows, e);
            rank += r > rows || (r == rows && e < lane);
        }
        return rank;
    }

    // C[m, n] = sum over k of A(m, k) B(n, k).  A result tile is a workgroup's; rows of A and B are the result's rows and columns.
    enum Form { kForward, kRowGrad, kMatrixGrad };

    struct ProductArgs {
        const void *a, *b;
        void*       c;
        uint32_t    n_places, n_experts, m, n, k;// kForward: n = n_out, k = n_in; kRowGrad: n = n_in, k = n_out; kMatrixGrad: m = n_out, n = n_in
        const uint32_t* offsets;
        uint32_t        splits = 1;// kMatrixGrad: parts that an expert's rows are taken in, c then = fp32 [splits, n_experts, m, n]
    };

    // ---- LDS ---------------------------------------------------------------------------------------------------------------------------------------------
    // A step of k takes kStep elements (128 bytes).  An operand's slab of a step lies in LDS as [rows][128 bytes of k] if its k axis is contiguous in memory, as
    // [k][rows] if its rows are.  16-byte units are permuted by an exclusive-or with bits of the LDS row's number: the lanes that LDS serves in one clock (16 of them
    // at 16 bytes, 256 bytes in all) then meet different banks (no conflict counted in either layout).
    template<typename T>
    constexpr uint32_t kStep = 128 / sizeof(T);

    __device__ __forceinline__ uint32_t swz_rows(uint32_t row) { return (row >> 1) & 7u; }
    template<typename T>
    __device__ __forceinline__ uint32_t swz_depth(uint32_t k) {
        return sizeof(T) == 2 ? (k & 3u) << 2 : ((k >> 2) & 1u) << 3;
    }

    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));// 16 bytes of any element type

    // What a matrix instruction takes: lane l holds row r0 + l % 32, 16 bytes of k from k0 + (l / 32) * kUnit
    template<typename T, uint32_t ROWS, bool DEPTH_CONTIGUOUS>
    __device__ __forceinline__ s16x8 operand(const T* lds, uint32_t r0, uint32_t k0) {
        const uint32_t lane = threadIdx.x & 63u;
        if constexpr (DEPTH_CONTIGUOUS) {
            const uint32_t row = r0 + (lane & 31u), unit = k0 / kUnit<T> + (lane >> 5);
            return *reinterpret_cast<const s16x8*>(lds + row * kStep<T> + ((unit ^ swz_rows(row)) * kUnit<T>));
        } else if constexpr (sizeof(T) == 2) {
            // the transposing read: 16 lanes take 4 of k x 16 rows (8 bytes each) and get 4 of k of one row each
            static_assert(ROWS >= 128, "the permutation needs 16 units per row");
            s16x4 part[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t k = k0 + (lane >> 5) * 8 + h * 4 + ((lane & 15u) >> 2), row = r0 + (lane & 16u) + (lane & 3u) * 4;
                const uint32_t at = ((row >> 3) ^ swz_depth<T>(k)) * 8 + (row & 7u);
                part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (lds + k * ROWS + at));
            }
            return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            const uint32_t row = r0 + (lane & 31u);
            f32x4          v;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t k = k0 + (lane >> 5) * 4 + i;
                v[i]             = lds[k * ROWS + (((row >> 2) ^ swz_depth<T>(k)) * 4 + (row & 3u))];
            }
            return __builtin_bit_cast(s16x8, v);
        }
    }

    // 32 x 32 of the result, two units of k.  fp32: the order of k inside the step is free as long as both operands share it.
    __device__ __forceinline__ f32x16 matrix_step(s16x8 a, s16x8 b, f32x16 c, bf16_t) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x16 matrix_step(s16x8 a, s16x8 b, f32x16 c, fp16_t) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x16 matrix_step(s16x8 a, s16x8 b, f32x16 c, float) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }

    // ---- from memory to LDS ------------------------------------------------------------------------------------------------------------------------------
    // kUnits: 16 bytes per lane straight into LDS; operands, rows and the result begin at multiples of 16 bytes.
    // kWords: 4 bytes per lane straight into LDS; fp32 of any sizes.  4800 rows x 250 x 333 over 5, forward, dx, dw: 15, 18, 19 us, and 13, 16, 18 as kUnits at 252 x 336; as
    // kElements 1.3, 1.2 and 1.1 times as long, and 1.6, 1.4 and 1.1 times at 8000 rows x 1001 x 1003 over 8 (155, 155, 132 us, random loads).  The lane's addresses cost: the
    // compiler spills 31 to 144 scalar registers in these kernels.
    // kElements: through registers, 16 bytes per lane from any address, the ends of rows element by element; 16-bit elements of odd sizes or alignment.
    enum Load { kUnits, kWords, kElements };

    __device__ const uint4 zero_page[4] = {};

    // One load per lane into LDS at dst + (16 or 4) lane, dst the same for the whole wavefront.  Assembly, because the compiler waits for every such load before the next LDS
    // read of any address; the kernel waits itself, by loads_arrived().  There is no result register that the compiler could reuse early.  M0 holds dst
    // and is named as changed, so that the compiler keeps nothing there across it (it warns that M0 is reserved, which is meant).  Five wait states lie between
    // whatever may have made `base` - a read of a lane is vector work - and the load, which the compiler sees to for its own instructions only.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    template<Load LOAD>
    __device__ __forceinline__ void load_to_lds(const void* src, uint32_t dst) {
        if constexpr (LOAD == kUnits) asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
        else
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
    }
    template<Load LOAD>
    __device__ __forceinline__ void load_to_lds_at(const void* base, uint32_t offset, uint32_t dst) {
        if constexpr (LOAD == kUnits) asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "memory", "m0");
        else
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "memory", "m0");
    }
#pragma clang diagnostic pop
    template<uint32_t LEFT>
    __device__ __forceinline__ void loads_arrived() {// all but the last LEFT of this wavefront's loads (and stores) into memory order
        static_assert(LEFT < 64, "a six-bit counter");
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
    }

    // One operand's slab: ROWS rows, THREADS threads, kLoads loads each.  stride = elements between rows (k contiguous) or between k (rows contiguous).  The lane's byte
    // offsets from the slab's first element are made once per tile; the slab's address moves in scalar registers.  Rows outside the tile read the tile's first row
    // instead: their results are not stored.
    template<typename T, uint32_t ROWS, uint32_t THREADS, bool DEPTH_CONTIGUOUS, Load LOAD>
    struct Slab {
        static constexpr uint32_t kPiece = LOAD == kWords ? 4 : 16, kLoads = ROWS * 128 / (THREADS * kPiece), kPerDepth = ROWS / kUnit<T>;
        static __device__ __forceinline__ uint32_t unit(uint32_t i) { return (i * THREADS + threadIdx.x) * kPiece / 16; }
        static __device__ __forceinline__ uint32_t sub(uint32_t i) { return (i * THREADS + threadIdx.x) * kPiece % 16 / sizeof(T); }
        // the lane's first k and row inside the slab
        static __device__ __forceinline__ uint32_t depth_of(uint32_t i) {
            return DEPTH_CONTIGUOUS ? ((unit(i) & 7u) ^ swz_rows(unit(i) >> 3)) * kUnit<T> + sub(i) : unit(i) / kPerDepth;
        }
        static __device__ __forceinline__ uint32_t row_of(uint32_t i) {
            return DEPTH_CONTIGUOUS ? unit(i) >> 3 : ((unit(i) % kPerDepth) ^ swz_depth<T>(depth_of(i))) * kUnit<T> + sub(i);
        }
        static __device__ __forceinline__ void offsets(uint32_t stride, uint32_t rows, uint32_t (&off)[kLoads]) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t row = row_of(i) < rows ? row_of(i) : 0u;
                off[i]             = (DEPTH_CONTIGUOUS ? row * stride + depth_of(i) : depth_of(i) * stride + row) * (uint32_t) sizeof(T);
            }
        }
        static __device__ __forceinline__ void load(const T* base, const uint32_t (&off)[kLoads], uint32_t i, uint32_t dst) {
            load_to_lds_at<LOAD>(base, off[i], dst + i * (THREADS * kPiece));
        }
        // the slab that the depth ends in (left < kStep of it): what lies behind comes from a page of zeros
        static __device__ __forceinline__ void load_last(const T* base, const uint32_t (&off)[kLoads], uint32_t left, uint32_t dst) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i)
                load_to_lds<LOAD>(depth_of(i) < left ? reinterpret_cast<const char*>(base) + off[i] : reinterpret_cast<const char*>(zero_page), dst + i * (THREADS * kPiece));
        }
        // kElements: into registers ..  A unit may reach beyond its row into the next one: elements behind `rows` belong to results that are not stored, elements of k behind `left` are
        // cleared.  At the array's end it is read element by element.
        static __device__ __forceinline__ void fetch(const T* base, const T* end, const uint32_t (&off)[kLoads], uint32_t left, s16x8 (&r)[kLoads]) {
            constexpr uint32_t U = kUnit<T>;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const T*       p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off[i]);
                const uint32_t k = depth_of(i);
                r[i]             = s16x8{};
                if (k >= left) continue;
                if (p + U <= end) r[i] = __builtin_bit_cast(s16x8, *reinterpret_cast<const typename UnitOf<T>::mem*>(p));
                else
#pragma unroll
                    for (uint32_t q = 0; q < U; ++q)
                        if (p + q < end) r[i][q] = __builtin_bit_cast(short, p[q]);
            }
            if (DEPTH_CONTIGUOUS && left < kStep<T>)
#pragma unroll
                for (uint32_t i = 0; i < kLoads; ++i)
#pragma unroll
                    for (uint32_t q = 0; q < U; ++q)
                        if (depth_of(i) + q >= left) r[i][q] = 0;
        }
        // .. and on into LDS
        static __device__ __forceinline__ void put(const s16x8 (&r)[kLoads], T* slab) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) *reinterpret_cast<s16x8*>(slab + unit(i) * kUnit<T>) = r[i];
        }
    };

    // ---- the kernel --------------------------------------------------------------------------------------------------------------------------------------
    // 16 bytes of a result row, or as many of their elements as the row has left.  A large result passes the L2 by: it would push out the slabs that the workgroups share
    // (all of them store at about the same time).
    template<bool LARGE, typename T>
    __device__ __forceinline__ void store_part(T* p, uint32_t left, s16x8 c) {
        if (left >= (uint32_t) kUnit<T>) {
            auto* to = reinterpret_cast<typename UnitOf<T>::mem*>(p);
            if (LARGE) __builtin_nontemporal_store(__builtin_bit_cast(typename UnitOf<T>::mem, c), to);
            else
                *to = __builtin_bit_cast(typename UnitOf<T>::mem, c);
        } else {
            const auto v = __builtin_bit_cast(typename UnitOf<T>::mem, c);
#pragma unroll
            for (uint32_t q = 0; q < (uint32_t) kUnit<T>; ++q)
                if (q < left) p[q] = v[q];
        }
    }

    template<typename T, typename O>
    struct Tile {
        const T *a, *b;
        O*       c;
        uint32_t rows, cols, depth;
    };

    // A workgroup stays and computes one BM x BM tile after another, WM x WN wavefronts side by side.  A step of k is four quarters of two units: while a quarter's matrix
    // instructions run from registers, the operands of the next are read from LDS.  LDS holds five slabs, A0 B0 A1 B1 A2 ..: one barrier per step, before its last
    // quarter: behind it every wavefront has read this step's two slabs, so the next two loads may overwrite them, and the next step's slabs have arrived (issued one
    // step ago, A's two steps ago).  The loads of the next tile's first slabs are under way while a tile's result is stored.
    // Bound: in 16 bits the card's power.  32768 rows x 2048 x 4096 over 8 even experts, 256 x 256 tiles: 472 us = 1.17 PFLOP/s forward, 442 and 453 for the gradients, at 1.7 GHz
    // (on zeros, which cost no power, 353 us = 1.56); 128 x 128 tiles 1.3 times as long: an operand's byte is used half as often.  256 x 256 tiles of the forward product and the
    // row gradient take all 256 vector registers and spill three (16 bytes a lane of scratch).  fp32: the matrix cores, 8192 x 1024 x 1024 over 8 even experts 127 us =
    // 135 TFLOP/s.  kElements at 16384 x 1001 x 1003 over 8: 560, 590 and 600 TFLOP/s (forward, dx, dw) at even loads, 450, 470 and 590 at random ones, where 1000 x 1008
    // has 785, 850, 800 and 650, 690, 780: its slabs go through registers, with misaligned 16-byte accesses; which of the two costs was not measured apart.
    // Small problems (4096 x 1024 x 1024 over 16 experts: 14 us at even loads, 20 at random ones) wait for the CUs that have two tiles.
    //
    // take(tile): the workgroup's next tile, false behind the last.  O: the result's type, T or (partial sums) float
    template<typename T, typename O, Form FORM, Load LOAD, uint32_t BM, uint32_t WM, uint32_t WN, typename TAKE>
    __device__ __forceinline__ void run_tiles(const ProductArgs& g, T* lds, TAKE&& take) {
        constexpr uint32_t BN = BM, THREADS = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
        constexpr bool     A_DEPTH = FORM != kMatrixGrad, B_DEPTH = FORM == kForward;
        using SlabA                   = Slab<T, BM, THREADS, A_DEPTH, LOAD>;
        using SlabB                   = Slab<T, BN, THREADS, B_DEPTH, LOAD>;
        constexpr uint32_t LOADS      = SlabA::kLoads;// per thread and slab
        constexpr uint32_t kSlots     = 5, kSlab = BM * kStep<T>;
        constexpr uint32_t kMul       = TM * TN, kReads = TM + TN, kReadsPer = (kReads + kMul - 1) / kMul, kQuarter = 2 * kUnit<T>;
        // the result is turned in the fifth slab, 32 rows x kTurn tiles of 32 columns at a time and wavefront
        constexpr uint32_t kTurn = sizeof(T) == 2 ? TN : 1, kTurnCols = kTurn * 32, kRowUnits = kTurnCols / kUnit<T>;
        constexpr bool     kTurns = std::is_same_v<T, O> && WM * WN * 32 * kTurnCols <= kSlab;
        constexpr uint32_t kStores = kTurns ? TM * (TN / kTurn) * 32 * kRowUnits / 64 : TM * TN * 4;
        auto slabs = [&](uint32_t slot) { return lds + slot * kSlab; };
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
        const uint32_t stride_a = FORM == kMatrixGrad ? g.m : g.k, stride_b = FORM == kForward ? g.k : g.n;
        const size_t   move_a = A_DEPTH ? kStep<T> : (size_t) kStep<T> * stride_a, move_b = B_DEPTH ? kStep<T> : (size_t) kStep<T> * stride_b;
        const uint32_t lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void*) lds + wave * (64 * SlabA::kPiece);
        constexpr uint32_t kSlabBytes = kSlab * sizeof(T);

        // the tile at hand
        const T *A, *B;
        O*       C;
        uint32_t rows, cols, depth, steps, whole;
        uint32_t off_a[LOADS], off_b[LOADS];
        auto     next = [&]() -> bool {
            Tile<T, O> t;
            if (!take(t)) return false;
            A = uniform(t.a), B = uniform(t.b), C = uniform(t.c);
            rows = __builtin_amdgcn_readfirstlane(t.rows), cols = __builtin_amdgcn_readfirstlane(t.cols), depth = __builtin_amdgcn_readfirstlane(t.depth);
            steps = (depth + kStep<T> - 1) / kStep<T>, whole = depth / kStep<T>;
            uint32_t sa = stride_a, sb = stride_b;// (opaque: what depends on them is made anew for each tile, not kept in registers)
            asm volatile("" : "+s"(sa), "+s"(sb));
            SlabA::offsets(sa, rows, off_a);
            SlabB::offsets(sb, cols, off_b);
            return true;
        };
        auto slot_after = [](uint32_t slot, uint32_t n) { return slot + n >= kSlots ? slot + n - kSlots : slot + n; };
        auto dst_of     = [&](uint32_t slot) { return lds0 + slot * kSlabBytes; };
        auto slab_a     = [&](uint32_t s, uint32_t slot) {
            if constexpr (LOAD != kElements) {
                if (s < whole) {
#pragma unroll
                    for (uint32_t i = 0; i < LOADS; ++i) SlabA::load(A + s * move_a, off_a, i, dst_of(slot));
                } else if (s < steps)
                    SlabA::load_last(A + s * move_a, off_a, depth - s * kStep<T>, dst_of(slot));
            }
        };
        auto slab_b = [&](uint32_t s, uint32_t slot) {
            if constexpr (LOAD != kElements) {
                if (s < whole) {
#pragma unroll
                    for (uint32_t i = 0; i < LOADS; ++i) SlabB::load(B + s * move_b, off_b, i, dst_of(slot));
                } else if (s < steps)
                    SlabB::load_last(B + s * move_b, off_b, depth - s * kStep<T>, dst_of(slot));
            }
        };
        // kElements: a slab of each operand on its way, the operands' ends
        const T* const end_a = static_cast<const T*>(g.a) + (size_t) g.n_places * (FORM == kMatrixGrad ? g.m : g.k);
        const T* const end_b = static_cast<const T*>(g.b) + (FORM == kMatrixGrad ? (size_t) g.n_places * g.n : (size_t) g.n_experts * g.n * g.k);
        s16x8 ra[LOADS], rb[LOADS];
        auto  fetch_a = [&](uint32_t s) { if constexpr (LOAD == kElements) if (s < steps) SlabA::fetch(A + s * move_a, end_a, off_a, min(kStep<T>, depth - s * kStep<T>), ra); };
        auto  fetch_b = [&](uint32_t s) { if constexpr (LOAD == kElements) if (s < steps) SlabB::fetch(B + s * move_b, end_b, off_b, min(kStep<T>, depth - s * kStep<T>), rb); };

        if (!next()) return;
        slab_a(0, 0), slab_b(0, 1), slab_a(1, 2), slab_b(1, 3);
        bool stored = false;// a whole tile's stores are among what is under way
        for (bool more = true; more;) {
            f32x16 acc[TM][TN] = {};
            slab_a(2, 4);
            if (steps) {
                if constexpr (LOAD == kElements) {
                    fetch_a(0), fetch_b(0);
                    SlabA::put(ra, slabs(0)), SlabB::put(rb, slabs(1));
                    fetch_a(1);
                    SlabA::put(ra, slabs(2));
                    fetch_b(1), fetch_a(2);
                } else {
                    // the first two slabs: behind them three more, and a whole tile's stores
                    constexpr uint32_t kBehind = 3 * LOADS + kStores < 64 ? 3 * LOADS + kStores : 3 * LOADS;
                    if (whole < 3) loads_arrived<0>();
                    else if (stored)
                        loads_arrived<kBehind>();
                    else
                        loads_arrived<3 * LOADS>();
                }
                __syncthreads();
                s16x8 fa[2][TM], fb[2][TN];
#pragma unroll
                for (uint32_t j = 0; j < TN; ++j) fb[0][j] = operand<T, BN, B_DEPTH>(slabs(1), wn + j * 32, 0);
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i) fa[0][i] = operand<T, BM, A_DEPTH>(slabs(0), wm + i * 32, 0);
                // quarter q's matrix instructions; the next quarter's operands are read meanwhile, and with `load` the loads of B's slab ls and A's next one issued
                auto quarter = [&](auto q_, auto load_, const T* as, const T* bs, uint32_t ls, uint32_t slot) {
                    constexpr uint32_t q = decltype(q_)::value, cur = q & 1u, k0 = (q + 1) % 4 * kQuarter;
                    constexpr bool     load = decltype(load_)::value && LOAD != kElements;
#pragma unroll
                    for (uint32_t x = 0; x < kMul; ++x) {
#pragma unroll
                        for (uint32_t r = x * kReadsPer; r < (x + 1) * kReadsPer && r < kReads; ++r) {
                            if (r < TN) fb[cur ^ 1][r] = operand<T, BN, B_DEPTH>(bs, wn + r * 32, k0);
                            else
                                fa[cur ^ 1][r - TN] = operand<T, BM, A_DEPTH>(as, wm + (r - TN) * 32, k0);
                        }
                        if constexpr (load)
#pragma unroll
                            for (uint32_t l = x * 2 * LOADS / kMul; l < (x + 1) * 2 * LOADS / kMul; ++l) {
                                if (l < LOADS) SlabB::load(B + ls * move_b, off_b, l, dst_of(slot));
                                else
                                    SlabA::load(A + (ls + 1) * move_a, off_a, l - LOADS, dst_of(slot_after(slot, 1)));
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
                    const T *as = slabs(slot), *bs = slabs(slot_after(slot, 1));
                    quarter(integral_constant<uint32_t, 0>{}, no, as, bs, 0, 0);
                    quarter(integral_constant<uint32_t, 1>{}, no, as, bs, 0, 0);
                    quarter(integral_constant<uint32_t, 2>{}, no, as, bs, 0, 0);
                    if constexpr (LOAD == kElements) SlabB::put(rb, slabs(slot_after(slot, 3))), SlabA::put(ra, slabs(slot_after(slot, 4)));
                    else if (decltype(load_)::value)
                        loads_arrived<LOADS>();
                    else
                        loads_arrived<0>();
                    __syncthreads();
                    // B's slab s + 2 goes where A's s was, A's s + 3 where B's s was
                    if constexpr (LOAD == kElements) fetch_b(s + 2), fetch_a(s + 3);
                    else if (!decltype(load_)::value)
                        slab_b(s + 2, slot), slab_a(s + 3, slot_after(slot, 1));
                    quarter(integral_constant<uint32_t, 3>{}, load_, slabs(slot_after(slot, 2)), slabs(slot_after(slot, 3)), s + 2, slot);
                    slot = slot_after(slot, 2);
                };
                uint32_t s = 0;
                if constexpr (LOAD != kElements)
                    for (; s + 3 < whole; ++s) step(yes, s);
                for (; s < steps; ++s) step(no, s);
                __syncthreads();// nothing reads a slab any more
            }
            O* const       out = C;
            uint32_t       ldc = g.n;
            asm volatile("" : "+s"(ldc));
            const uint32_t out_rows = rows, out_cols = cols;
            more = next();
            if (more) slab_a(0, 0), slab_b(0, 1), slab_a(1, 2), slab_b(1, 3);
            stored = out_rows == BM && out_cols == BN;
            // A lane holds four neighbouring columns of a row, its neighbours hold other rows.
            auto quad = [&](uint32_t i, uint32_t j, uint32_t v) {
                typedef O four __attribute__((ext_vector_type(4)));
                four      c;
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) c[q] = (O) acc[i][j][v + q];
                return c;
            };
            if constexpr (kTurns) {
                // every wavefront turns its part in LDS and stores lines
                T*   turn = slabs(4) + wave * (32 * kTurnCols);
                auto swz  = [](uint32_t m) { return (m / (16 / kRowUnits)) % kRowUnits; };
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i)
#pragma unroll
                    for (uint32_t j0 = 0; j0 < TN; j0 += kTurn) {
                        const uint32_t m = lane & 31u;
#pragma unroll
                        for (uint32_t j = 0; j < kTurn; ++j)
#pragma unroll
                            for (uint32_t v = 0; v < 16; v += 4) {
                                const auto     c = quad(i, j0 + j, v);
                                const uint32_t n = j * 32 + v * 2 + (lane >> 5) * 4;
                                __builtin_memcpy(__builtin_assume_aligned(turn + m * kTurnCols + (((n / kUnit<T>) ^ swz(m)) * kUnit<T> + n % kUnit<T>), 4 * sizeof(T)), &c, sizeof c);
                            }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
#pragma unroll
                        for (uint32_t x = 0; x < 32 * kRowUnits / 64; ++x) {
                            const uint32_t u = x * 64 + lane, row = u / kRowUnits, unit = u % kRowUnits;
                            s16x8          c;
                            __builtin_memcpy(&c, __builtin_assume_aligned(turn + row * kTurnCols + (unit ^ swz(row)) * kUnit<T>, 16), 16);
                            const uint32_t gm = wm + i * 32 + row, gn = wn + j0 * 32 + unit * kUnit<T>;
                            if (gm < out_rows && gn < out_cols) store_part<(BM > 128)>(out + (size_t) gm * ldc + gn, out_cols - gn, c);
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                    }
                if (more) __syncthreads();// the fifth slab is free again
            } else {
#pragma unroll
                for (uint32_t i = 0; i < TM; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < TN; ++j)
#pragma unroll
                        for (uint32_t v = 0; v < 16; v += 4) {
                            const uint32_t gm = wm + i * 32 + (lane & 31u), gn = wn + j * 32 + v * 2 + (lane >> 5) * 4;
                            if (gm < out_rows && gn < out_cols) store_part<(BM > 128)>(out + (size_t) gm * ldc + gn, out_cols - gn, __builtin_bit_cast(s16x8, quad(i, j, v)));
                        }
            }
        }
    }

    // SPLIT: the tiles left over when every workgroup has had the same number are cut in four, if there are few of them: most CUs would wait for a whole tile's time
    // otherwise (132 row tiles x 16 columns on 256 CUs: nine tiles' time for 8.25 tiles' work; both gradients of 32768 x 2048 x 1024 over 32
    // experts 307 -> 301 us, 8192 x 1024 x 1024 over 8 in fp32 192 -> 152).
    template<typename T, Form FORM, Load LOAD, uint32_t BM, uint32_t WM, uint32_t WN, uint32_t OCC, bool SPLIT, bool PARTIAL>
    __global__ __launch_bounds__(WM* WN * 64, OCC) void product_kernel(const ProductArgs g, uint32_t col_tiles) {
        __shared__ __align__(1024) T lds[5 * BM * kStep<T>];
        const uint32_t lane = threadIdx.x & 63u;
        RowTiles       tiles{};
        const uint32_t m_tiles = (g.m + BM - 1) / BM;// kMatrixGrad: row tiles of an expert
        if (FORM != kMatrixGrad) tiles = row_tiles_of(BM, g.n_experts, g.n_places, g.offsets);
        using O                = std::conditional_t<PARTIAL, float, T>;
        const uint32_t n_tiles = (FORM == kMatrixGrad ? g.n_experts * m_tiles * (PARTIAL ? g.splits : 1u) : tiles.total) * col_tiles;
        const bool     ranked = FORM == kMatrixGrad && g.n_experts <= 64;
        uint32_t       rank = 0;
        if (ranked && lane < g.n_experts) {
            const uint32_t begin = bounded(g.offsets, lane, g.n_experts, g.n_places), end = bounded(g.offsets, lane + 1, g.n_experts, g.n_places);
            rank                 = end > begin ? end - begin : 0u;
        }
        if (ranked) rank = rank_by_rows(rank, g.n_experts);

        // The tiles go out in runs of RUN neighbours, a run to RUN workgroups of one XCD (workgroup b runs in XCD b % 8), whose L2 then holds what they share; the runs go to
        // such groups in turn.  kForward, kRowGrad: every tile costs the same and a run fills an XCD.  kMatrixGrad: a tile's cost is its expert's number of rows;
        // the experts go out by falling number, there and back over the groups, in shorter runs (one expert's tiles on one XCD made it the last by a third).
        constexpr uint32_t RUN = FORM == kMatrixGrad ? 8 : 32, HIGH = FORM == kMatrixGrad ? 2 : 4;
        auto               tile = [&](uint32_t t, Tile<T, O>& out) {
            const uint32_t each = m_tiles * col_tiles, part = PARTIAL ? t / each % g.splits : 0u;// tiles of an expert and part, the part
            const TileAt   at = FORM == kMatrixGrad ? tile_at<HIGH>(t % each, m_tiles, col_tiles) : tile_at<HIGH>(t, tiles.total, col_tiles);
            const uint32_t n0 = at.col * BM;
            out.cols          = min(BM, g.n - n0);
            if (FORM == kMatrixGrad) {
                uint32_t expert = t / (each * (PARTIAL ? g.splits : 1u));
                if (ranked) expert = __ffsll((unsigned long long) __ballot(lane < g.n_experts && rank == expert)) - 1;
                const uint32_t m0 = at.row * BM;
                uint32_t       begin = bounded(g.offsets, expert, g.n_experts, g.n_places);
                const uint32_t end = max(begin, bounded(g.offsets, expert + 1, g.n_experts, g.n_places));
                out.rows           = min(BM, g.m - m0);
                out.depth          = end - begin;
                if (PARTIAL) {// whole steps to each part
                    const uint32_t chunk = ((out.depth + kStep<T> - 1) / kStep<T> + g.splits - 1) / g.splits * kStep<T>;
                    begin                = min(begin + part * chunk, end);
                    out.depth            = min(chunk, end - begin);
                }
                out.a = static_cast<const T*>(g.a) + (size_t) begin * g.m + m0;
                out.b = static_cast<const T*>(g.b) + (size_t) begin * g.n + n0;
                out.c = static_cast<O*>(g.c) + (((size_t) part * g.n_experts + expert) * g.m + m0) * g.n + n0;
            } else {
                const RowTile  r = row_tile(tiles, at.row, BM, g.n_experts, g.n_places, g.offsets);
                const uint32_t e = min(r.expert, g.n_experts - 1);
                out.rows         = r.rows;
                out.depth        = r.expert < g.n_experts ? g.k : 0u;
                out.a = static_cast<const T*>(g.a) + (size_t) r.row0 * g.k;
                out.b = static_cast<const T*>(g.b) + (FORM == kForward ? ((size_t) e * g.n + n0) * g.k : (size_t) e * g.n * g.k + n0);
                out.c = static_cast<O*>(g.c) + (size_t) r.row0 * g.n + n0;
            }
        };
        const uint32_t groups = gridDim.x / RUN, group = blockIdx.x / 8 / RUN * 8 + blockIdx.x % 8, in = blockIdx.x / 8 % RUN;// (the grid is a multiple of 8 RUN)
        uint32_t       left = n_tiles % gridDim.x;
        if (!SPLIT || left * 2 > gridDim.x) left = 0;
        const uint32_t n_whole = n_tiles - left;
        uint32_t       round = 0;
        run_tiles<T, O, FORM, LOAD, BM, WM, WN>(g, lds, [&](Tile<T, O>& out) {
            for (;; ++round) {
                const uint64_t run = (uint64_t) round * groups + (FORM == kMatrixGrad && (round & 1u) ? groups - 1 - group : group);
                if ((uint64_t) round * groups * RUN >= n_whole) return false;
                if (run * RUN + in >= n_whole) continue;
                tile((uint32_t) run * RUN + in, out);
                ++round;
                return true;
            }
        });
        if constexpr (SPLIT) {
            if (left == 0) return;
            __syncthreads();// the slabs' memory changes hands
            constexpr uint32_t HALF = BM / 2, WAVES = WM * WN;
            // four neighbouring parts per tile, a contiguous stretch of them per XCD
            const uint32_t parts = left * 4, per = (parts + 7) / 8, end = min(parts, (blockIdx.x % 8 + 1) * per);
            uint32_t       part = blockIdx.x % 8 * per + blockIdx.x / 8;
            run_tiles<T, O, FORM, LOAD, HALF, 2, WAVES / 2>(g, lds, [&](Tile<T, O>& out) {
                for (; part < end; part += gridDim.x / 8) {
                    tile(n_whole + part / 4, out);
                    const uint32_t r = part % 4 / 2 * HALF, c = part % 2 * HALF;
                    if (r >= out.rows || c >= out.cols) continue;
                    out.rows = min(HALF, out.rows - r), out.cols = min(HALF, out.cols - c);
                    out.a += FORM == kMatrixGrad ? r : (size_t) r * g.k;
                    out.b += FORM == kForward ? (size_t) c * g.k : c;
                    out.c += (size_t) r * g.n + c;
                    part += gridDim.x / 8;
                    return true;
                }
                return false;
            });
        }
    }

    // ---- few rows per expert -----------------------------------------------------------------------------------------------------------------------------
    // Serving: every matrix is read for a few rows, the time is that of reading them.  A workgroup computes all rows of an expert x 16 NF columns, 32 at a time (for more, its
    // part of the matrix is read again, from the cache); its WAVES wavefronts take the depth in turns of 128 bytes, so that a matrix row is read in runs of
    // 512 and more, and go from memory to the matrix instruction without LDS: lane l holds row l % 16, 16 bytes of k from unit l / 16.  The wavefronts' sums are joined in LDS in
    // a fixed order.  Many small workgroups instead of a few that stay: what counts is bytes under way.
    // 256 rows over 32 matrices of 2048 x 2048 bf16, none of it cached: 51 us = 5.3 TB/s (the tile kernel: 64); 2 rows through two of eight 2048 x 4096: 9 us with the matrices
    // in the cache behind the L2s, 11 without (18).  One row block of
    // 16 and 32 columns instead of 64: 61 us (the rows are read too often); through LDS in whole rows: 65.  Where that leaves CUs without work, 16 columns and eight
    // wavefronts (8 rows through 8 of 13 matrices of 4032 x 192: 14.0 -> 7.7 us).
    // The choice goes by the average of the rows per expert, all that the host knows: up to 24.  Even loads meet there (2048 x 2048 bf16, 768 rows over 32 experts 59 us, the tile
    // kernel 55 over 31; 1536 over 64: 106, and 124 over 63).  It does not bound uneven ones: an expert's blocks of 32 rows come one after another in one column of
    // workgroups, so that all rows at one expert take 96 us for 256 rows, 284 for 768 and 565 for 1536, where the tile kernel takes 22.
    __device__ __forceinline__ f32x4 matrix_step16(s16x8 a, s16x8 b, f32x4 c, bf16_t) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x4 matrix_step16(s16x8 a, s16x8 b, f32x4 c, fp16_t) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ f32x4 matrix_step16(s16x8 a, s16x8 b, f32x4 c, float) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }

    constexpr uint32_t kZeroBlocks = 64;// workgroups for the rows behind the last entry

    template<typename T, uint32_t NF, uint32_t WAVES>
    __global__ __launch_bounds__(WAVES * 64) void product_few_rows_kernel(const ProductArgs g, uint32_t col_tiles) {
        constexpr uint32_t MF = 2, U = kUnit<T>, CHUNK = 8 * U, AHEAD = 2;// chunks of a wavefront under way
        __shared__ f32x4   part[WAVES][NF * MF][64];
        const uint32_t     lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const uint32_t     expert = blockIdx.x / col_tiles;
        typedef T          four __attribute__((ext_vector_type(4)));
        if (expert >= g.n_experts) {
            const uint64_t end = (uint64_t) g.n_places * (g.n / 4), step = (uint64_t) (gridDim.x - g.n_experts * col_tiles) * (WAVES * 64);
            for (uint64_t i = (uint64_t) bounded(g.offsets, g.n_experts, g.n_experts, g.n_places) * (g.n / 4) + (blockIdx.x - g.n_experts * col_tiles) * (WAVES * 64) + threadIdx.x; i < end; i += step)
                reinterpret_cast<four*>(g.c)[i] = four{};
            return;
        }
        const uint32_t begin = bounded(g.offsets, expert, g.n_experts, g.n_places), end = bounded(g.offsets, expert + 1, g.n_experts, g.n_places);
        const uint32_t n0 = blockIdx.x % col_tiles * (16 * NF), depth = g.k;
        const T*       w[NF];
#pragma unroll
        for (uint32_t j = 0; j < NF; ++j)
            w[j] = static_cast<const T*>(g.b) + ((size_t) expert * g.n + min(n0 + j * 16 + (lane & 15u), g.n - 1)) * g.k + (lane >> 4) * U;
        for (uint32_t row0 = begin; row0 < end; row0 += 16 * MF) {
            const uint32_t rows = end - row0;
            const T*       x[MF];
#pragma unroll
            for (uint32_t i = 0; i < MF; ++i) x[i] = static_cast<const T*>(g.a) + (size_t) (row0 + min(i * 16 + (lane & 15u), rows - 1)) * g.k + (lane >> 4) * U;
            f32x4 acc[MF][NF] = {};
            for (uint32_t k0 = wave * CHUNK; k0 < depth; k0 += WAVES * CHUNK * AHEAD) {
                s16x8 a[AHEAD][2][NF], b[AHEAD][2][MF];
#pragma unroll
                for (uint32_t c = 0; c < AHEAD; ++c) {
#pragma unroll
                    for (uint32_t j = 0; j < NF; ++j)
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const uint32_t k = k0 + c * WAVES * CHUNK + h * 4 * U;
                            a[c][h][j]       = k + (lane >> 4) * U < depth ? *reinterpret_cast<const s16x8*>(w[j] + k) : s16x8{};// (the depth comes in whole units)
                        }
#pragma unroll
                    for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const uint32_t k = k0 + c * WAVES * CHUNK + h * 4 * U;
                            b[c][h][i]       = k + (lane >> 4) * U < depth ? *reinterpret_cast<const s16x8*>(x[i] + k) : s16x8{};
                        }
                }
#pragma unroll
                for (uint32_t c = 0; c < AHEAD; ++c)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                        for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
                            for (uint32_t j = 0; j < NF; ++j) acc[i][j] = matrix_step16(a[c][h][j], b[c][h][i], acc[i][j], T{});
            }
            __syncthreads();// (the last rows' sums have been read)
#pragma unroll
            for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
                for (uint32_t j = 0; j < NF; ++j) part[wave][i * NF + j][lane] = acc[i][j];
            __syncthreads();
            for (uint32_t f = wave; f < MF * NF; f += WAVES) {
                f32x4 sum = part[0][f][lane];
#pragma unroll
                for (uint32_t w = 1; w < WAVES; ++w) sum += part[w][f][lane];
                const uint32_t m = f / NF * 16 + (lane & 15u), n = n0 + f % NF * 16 + (lane >> 4) * 4;
                if (m < rows && n < g.n) {// (columns come in fours)
                    four c;
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) c[q] = (T) sum[q];
                    *reinterpret_cast<four*>(static_cast<T*>(g.c) + (size_t) (row0 + m) * g.n + n) = c;
                }
            }
        }
    }

    template<typename T, uint32_t NF, uint32_t WAVES>
    static int launch_few_rows(const ProductArgs& g, hipStream_t s) {
        const uint64_t col_tiles = (g.n + 16 * NF - 1) / (16 * NF), blocks = g.n_experts * col_tiles + kZeroBlocks;
        SPLAHIP_REQUIRE(blocks < (1ull << 31), "too many tiles for one launch");
        product_few_rows_kernel<T, NF, WAVES><<<(uint32_t) blocks, WAVES * 64, 0, s>>>(g, (uint32_t) col_tiles);
        SPLAHIP_TRY(hipGetLastError());
        return SPLAHIP_OK;
    }

    static int check_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out) {
        SPLAHIP_REQUIRE(panel_type_valid(panel_type), "panel type");
        SPLAHIP_REQUIRE(n_experts >= 1 && n_experts <= 2048, "experts: 1 .. 2048");
        SPLAHIP_REQUIRE(n_places < (1u << 31), "rows: below 2^31");
        SPLAHIP_REQUIRE(n_in >= 1 && n_out >= 1 && n_in < (1u << 21) && n_out < (1u << 21), "matrix sizes: 1 .. 2^21 - 1");
        return SPLAHIP_OK;
    }

    // out = the sum of the parts, in their order
    template<typename T>
    __global__ __launch_bounds__(256) void join_parts_kernel(uint64_t n, uint32_t parts, const float* __restrict__ part, T* __restrict__ out) {
        for (uint64_t i = (uint64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t) gridDim.x * 256) {
            float s = 0.0f;
#pragma unroll 8
            for (uint32_t p = 0; p < parts; ++p) s += part[p * n + i];
            out[i] = (T) s;
        }
    }

    template<typename T, Form FORM, Load LOAD, uint32_t BM, uint32_t WM, uint32_t WN, uint32_t OCC, bool SPLIT = false, bool PARTIAL = false>
    static int launch_tiles(const ProductArgs& g, hipStream_t s) {
        const uint64_t col_tiles = (g.n + BM - 1) / BM;
        const uint64_t row_tiles = FORM == kMatrixGrad ? (uint64_t) g.n_experts * g.splits * ((g.m + BM - 1) / BM) : row_tiles_bound(g.n_places, g.n_experts, BM);
        SPLAHIP_REQUIRE(col_tiles * row_tiles < (1ull << 31), "too many tiles for one launch");
        constexpr uint32_t kResident = 256 * (OCC * 4 / (WM * WN));// workgroups the card holds at once
        product_kernel<T, FORM, LOAD, BM, WM, WN, OCC, SPLIT, PARTIAL><<<kResident, WM * WN * 64, 0, s>>>(g, (uint32_t) col_tiles);
        SPLAHIP_TRY(hipGetLastError());
        return SPLAHIP_OK;
    }

    static uint64_t matrix_tiles(const ProductArgs& g, uint64_t bm) { return g.n_experts * ((g.m + bm - 1) / bm) * ((g.n + bm - 1) / bm); }
    // The size of tile that fills the card: 256 (128 in fp32) takes 0.76 of the time of the next smaller one if there are enough of them (200 here, 200 by the average of the rows in
    // launch_of_type; 400 in fp32, two to a CU), up to twice the time if most CUs get none.
    static uint32_t matrix_grad_tile(const ProductArgs& g, uint32_t element, bool aligned) {
        if (element == 4) return matrix_tiles(g, 128) >= 400 ? 128 : 64;
        return aligned && matrix_tiles(g, 256) >= 200 ? 256 : 128;
    }
    // kMatrixGrad: parts that the experts' rows are taken in where there are too few tiles to fill the card: up to about 512 tiles in all, six steps of k or more for each on
    // the average, and no more parts than pay: S parts save (1 - 1/S) of the steps (t = 0.9 us each in fp32, 0.4 in 16 bits) and write and read S N fp32 sums
    // (5 TB/s), least at S^2 = steps t 5 TB/s / 8 N.  (The gradient for 5 matrices of 250 x 333 over 4800 fp32 rows, 120 tiles of 30 steps: 27 us in one part, 20 in four.)
    static uint32_t matrix_grad_splits(const ProductArgs& g, uint32_t element, bool aligned) {
        const uint32_t bm = matrix_grad_tile(g, element, aligned);
        if (bm == 256) return 1;
        const uint64_t steps = g.n_places / g.n_experts / (128 / element), most = std::min<uint64_t>({512 / std::max<uint64_t>(matrix_tiles(g, bm), 1), steps / 6, 16});
        const uint64_t n     = (uint64_t) g.n_experts * g.m * g.n;
        uint32_t       parts = 1;
        while (parts < most && (uint64_t) (parts + 1) * (parts + 1) * n <= steps * (element == 4 ? 562500 : 250000)) ++parts;
        return parts;
    }

    static bool aligned_product(const ProductArgs& g, uint32_t unit) {
        return ((uintptr_t) g.a % 16 == 0) && ((uintptr_t) g.b % 16 == 0) && ((uintptr_t) g.c % 16 == 0) && g.n % unit == 0 && g.k % unit == 0 && g.m % unit == 0;
    }

    template<Form FORM, typename T>
    static int launch_of_type(const ProductArgs& g, hipStream_t s) {
        const bool aligned = aligned_product(g, kUnit<T>);
        if constexpr (FORM == kMatrixGrad) {
            const uint32_t bm = matrix_grad_tile(g, sizeof(T), aligned);
            if constexpr (sizeof(T) == 4) {
                if (g.splits > 1)// (more than 256 tiles of 128 are not split)
                    return aligned ? launch_tiles<T, FORM, kUnits, 64, 2, 2, 4, false, true>(g, s) : launch_tiles<T, FORM, kWords, 64, 2, 2, 4, false, true>(g, s);
                if (bm == 128) return aligned ? launch_tiles<T, FORM, kUnits, 128, 2, 2, 2, true>(g, s) : launch_tiles<T, FORM, kWords, 128, 2, 2, 2, true>(g, s);
                return aligned ? launch_tiles<T, FORM, kUnits, 64, 2, 2, 4>(g, s) : launch_tiles<T, FORM, kWords, 64, 2, 2, 4>(g, s);
            } else {
                if (g.splits > 1) return aligned ? launch_tiles<T, FORM, kUnits, 128, 2, 2, 2, false, true>(g, s) : launch_tiles<T, FORM, kElements, 128, 2, 2, 2, false, true>(g, s);
                if (!aligned) return launch_tiles<T, FORM, kElements, 128, 2, 2, 2>(g, s);
                return bm == 256 ? launch_tiles<T, FORM, kUnits, 256, 2, 4, 2, true>(g, s) : launch_tiles<T, FORM, kUnits, 128, 2, 2, 2>(g, s);
            }
        } else {
            auto tiles = [&](uint64_t bm) { return (g.n_places / bm + 1) * ((g.n + bm - 1) / bm); };
            if constexpr (FORM == kForward)
                if (aligned && g.n_places <= 24 * (uint64_t) g.n_experts && g.n_experts * (uint64_t) (g.n / 32 + 1) < (1u << 23)) {// (a launch holds fewer than 2^32 threads)
                    const uint64_t rows = std::min(g.n_places, g.n_experts);// experts that have some, at most
                    if (rows * (g.n / 64) >= 1024) return launch_few_rows<T, 4, 4>(g, s);
                    return rows * (g.n / 32) >= 192 ? launch_few_rows<T, 2, 4>(g, s) : launch_few_rows<T, 1, 8>(g, s);
                }
            if constexpr (sizeof(T) == 4) {
                const bool large = tiles(128) >= 400;
                if (aligned) return large ? launch_tiles<T, FORM, kUnits, 128, 2, 2, 2, true>(g, s) : launch_tiles<T, FORM, kUnits, 64, 2, 2, 4>(g, s);
                return large ? launch_tiles<T, FORM, kWords, 128, 2, 2, 2, true>(g, s) : launch_tiles<T, FORM, kWords, 64, 2, 2, 4>(g, s);
            } else {
                if (!aligned) return launch_tiles<T, FORM, kElements, 128, 2, 2, 2>(g, s);
                return tiles(256) >= 200 ? launch_tiles<T, FORM, kUnits, 256, 2, 4, 2, true>(g, s) : launch_tiles<T, FORM, kUnits, 128, 2, 2, 2>(g, s);
            }
        }
    }

    template<Form FORM>
    static int launch_product(int panel_type, const ProductArgs& g, hipStream_t s) {
        int st = SPLAHIP_OK;
        panel_dispatch(panel_type, [&](auto zero) { st = launch_of_type<FORM, decltype(zero)>(g, s); });
        return st;
    }

}// namespace splahip

using namespace splahip;

extern "C" int splahip_expert_product(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets, const void* d_x,
                                      const void* d_w, void* d_y, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    if (n_places == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_x && d_w && d_y, "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kForward>(panel_type, ProductArgs{d_x, d_w, d_y, n_places, n_experts, 0, n_out, n_in, d_offsets}, as_stream(stream));
}

extern "C" int splahip_expert_product_dx(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_w, void* d_dx, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    if (n_places == 0) return SPLAHIP_OK;
    SPLAHIP_REQUIRE(d_offsets && d_dy && d_w && d_dx, "null array");
    if (int st = ensure_device()) return st;
    return launch_product<kRowGrad>(panel_type, ProductArgs{d_dy, d_w, d_dx, n_places, n_experts, 0, n_in, n_out, d_offsets}, as_stream(stream));
}

// the parts' sums; 0: the call needs none
extern "C" size_t splahip_expert_product_dw_workspace(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out) {
    if (check_product(panel_type, n_places, n_experts, n_in, n_out)) return 0;
    const uint32_t    element = panel_type == SPLAHIP_PANEL_FLOAT ? 4 : 2;
    const ProductArgs g{nullptr, nullptr, nullptr, n_places, n_experts, n_out, n_in, 0, nullptr};
    // (enough for operands of any alignment)
    const uint32_t splits = std::max(matrix_grad_splits(g, element, true), matrix_grad_splits(g, element, false));
    return splits > 1 ? (size_t) splits * n_experts * n_in * n_out * sizeof(float) : 0;
}

extern "C" int splahip_expert_product_dw(int panel_type, uint32_t n_places, uint32_t n_experts, uint32_t n_in, uint32_t n_out, const uint32_t* d_offsets,
                                         const void* d_dy, const void* d_x, void* d_dw, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (int st = check_product(panel_type, n_places, n_experts, n_in, n_out)) return st;
    SPLAHIP_REQUIRE(d_offsets && d_dw && (n_places == 0 || (d_dy && d_x)), "null array");
    const size_t need = splahip_expert_product_dw_workspace(panel_type, n_places, n_experts, n_in, n_out);
    SPLAHIP_REQUIRE(workspace_bytes >= need && (need == 0 || (d_workspace && (uintptr_t) d_workspace % 16 == 0)), "workspace too small");
    if (int st = ensure_device()) return st;
    hipStream_t    s       = as_stream(stream);
    const uint32_t element = panel_type == SPLAHIP_PANEL_FLOAT ? 4 : 2;
    ProductArgs    g{d_dy, d_x, d_dw, n_places, n_experts, n_out, n_in, 0, d_offsets};
    g.splits = matrix_grad_splits(g, element, aligned_product(g, 16 / element));
    if (g.splits == 1) return launch_product<kMatrixGrad>(panel_type, g, s);
    g.c = d_workspace;// (aligned, so that operands in units take the kernel for units even if d_dw starts between two: both have tiles of the size that g.splits was chosen for)
    if (int st = launch_product<kMatrixGrad>(panel_type, g, s)) return st;
    const uint64_t n = (uint64_t) n_experts * n_in * n_out;
    panel_dispatch(panel_type, [&](auto zero) {
        using T = decltype(zero);
        join_parts_kernel<T><<<(uint32_t) std::min<uint64_t>((n + 255) / 256, 4096), 256, 0, s>>>(n, g.splits, static_cast<const float*>(d_workspace), static_cast<T*>(d_dw));
    });
    SPLAHIP_TRY(hipGetLastError());
    return SPLAHIP_OK;
}
