// Products of a layer on macro tiles for gfx950: forward with bias, activation, gate and residual in the epilogue, and both gradients, for one
// matrix of weights or for one per group of rows.  No counterpart in the reference.
//
// A macro tile of 32 WM x 32 WN results is four waves of 16 WM x 16 WN each, on v_mfma_f32_16x16x32 with the accumulators in place; a stage is 64 of the sum.  Operands go
// to LDS by direct loads in the images of operand_tile.hpp and come back whole or, where they are not contiguous along the sum, through transposing reads.  LDS
// holds two images of A and three of B, so that loads run two stages ahead (B of the small tiles three).  The buffers go round at run time: the loop is one stage long, and
// what that costs, an addition for each address of a read, hides behind matrix instructions (six stages unrolled, as the GEMM has them, would be 36 KB of code for each epilogue).
//
// Bound by the matrix cores under the power limit where the sum is long and the tiles are whole (bf16 8192^3 706 to 734 us, 1.50 to 1.56 PFLOP/s; 4000 x 8192 x 4096 with GELU and two results 207 us, matrix cores
// busy 67 % of the CU's cycles, 72 % in the gradients of 4096 x 4096); by the start and end of a tile, some 11 us of the large one, where it is short; by HBM and the loads' latency where
// a group has few rows of its own weights (16384 rows over 64 groups of 2048 x 2048 203 us, 37 %).
//
// Rows are ragged: a workgroup finds its group from the offsets in device memory (GroupTiles).  A tile that has fewer rows reads its last one again, what that gives is not
// stored; a sum that ends inside a stage is completed with zeros by loads past the end of their buffer.
//
// Compiled once per type.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "lds_dma.hpp"
#include "linear.hpp"
#include "operand_tile.hpp"

namespace
{
    using r355::f32x4;
    using r355::GroupTile;
    using r355::GroupTiles;
    using r355::ldsBarrier;
    using r355::LinearParams;
    using r355::loadToLds;
    using r355::OUTSIDE;
    using r355::u32x2;
    using r355::u32x4;
    using r355::vec;
    using r355::waitVmcnt;
    using r355::tile::CHUNK;
    using r355::tile::i32x4;
    using r355::tile::laneOffsets8;
    using r355::tile::readBlock8;
    using r355::tile::readOffsets8;
    using r355::tile::STAGE_KB;
    using r355::tile::swzK8;
    using r355::tile::THREADS;

#ifdef R355_LINEAR_BF16
    using T = __bf16;
#else
    using T = _Float16;
#endif
    constexpr uint32_t TK = STAGE_KB / 2u; // of the sum per stage

    // (inline assembly: of the builtin the compiler makes instructions whose result is not tied to their addend, and moves the accumulators about)
    __device__ __forceinline__ void multiply(f32x4& acc, i32x4 x, i32x4 y)
    {
        if constexpr(__is_same(T, __bf16))
            asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
        else
            asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
    }

    // What a workgroup multiplies: Y rows first .. first + rowsLeft, columns col0 .. col0 + colsLeft, of group `group`; the sum's share [kFirst, kFirst + k).
    struct Work
    {
        uint32_t group, first, rowsLeft, col0, colsLeft, k, kFirst, share;
        uint64_t sumRow; // weights' gradient: first row of the group
    };

    // of workgroup `id` of those that have share `share` of the sums (an XCD has those of the same id % 8)
    template <bool AK, uint32_t ROWS, uint32_t COLS>
    __device__ __forceinline__ bool workOf(const LinearParams& p, Work& w, uint32_t id, uint32_t share)
    {
        uint32_t tm, tn, k;
        if constexpr(AK)
        {
            GroupTiles<ROWS> tiles{p};
            const uint32_t   tilesM = tiles.total();
            if(!r355::tileCoordRange(id, tilesM, p.tilesN, 0u, tilesM * p.tilesN, false, tm, tn))
                return false;
            const GroupTile t = tiles.at(tm);
            w.group = t.group, w.first = t.first, w.rowsLeft = t.count, w.sumRow = 0u, k = p.k;
        }
        else
        {
            // Few groups: an eighth of each one's tiles for every XCD, as their sums are of uneven lengths (4 gradients of 4096 x 2048 over 8000 uneven rows 288 -> 254 us, 8 310 -> 289); of
            // more, whole groups, whose operands one XCD alone then reads (16 of 4096 x 1536 264 us, in eighths 315).
            if(p.groups > 1u && p.groups < 16u)
            {
                const uint32_t eighth = (p.tilesM * p.tilesN + 7u) / 8u, slot = id / 8u;
                w.group               = slot / eighth;
                const uint32_t tile   = (id + w.group) % 8u * eighth + slot % eighth;
                if(w.group >= p.groups || tile >= p.tilesM * p.tilesN)
                    return false;
                r355::tileOfId(tile, p.tilesM, p.tilesN, tm, tn);
            }
            else
            {
                if(!r355::tileCoordRange(id, p.groups * p.tilesM, p.tilesN, 0u, p.groups * p.tilesM * p.tilesN, false, tm, tn))
                    return false;
                w.group = tm / p.tilesM, tm %= p.tilesM;
            }
            w.first           = tm * ROWS;
            w.rowsLeft        = p.m - w.first < ROWS ? p.m - w.first : ROWS;
            const auto  rows  = r355::rowsOf(p, w.group);
            w.sumRow = rows.first, k = rows.count;
        }
        w.col0     = tn * COLS;
        w.colsLeft = p.n - w.col0 < COLS ? p.n - w.col0 : COLS;
        // (whole stages for every share but the last ones)
        const uint32_t stages = k / TK + (k % TK != 0u ? 1u : 0u), part = p.splits > 1u ? (stages + p.splits - 1u) / p.splits : stages;
        w.share  = share;
        w.kFirst = share * part * TK;
        w.kFirst = w.kFirst < k ? w.kFirst : k;
        w.k      = k - w.kFirst < part * TK ? k - w.kFirst : part * TK;
        // (uniform, which the compiler does not see through the lanes' part in finding it)
        w.group = __builtin_amdgcn_readfirstlane(w.group), w.first = __builtin_amdgcn_readfirstlane(w.first), w.rowsLeft = __builtin_amdgcn_readfirstlane(w.rowsLeft);
        w.col0 = __builtin_amdgcn_readfirstlane(w.col0), w.colsLeft = __builtin_amdgcn_readfirstlane(w.colsLeft);
        w.k = __builtin_amdgcn_readfirstlane(w.k), w.kFirst = __builtin_amdgcn_readfirstlane(w.kFirst);
        return true;
    }

    // Where a lane's eight columns of a row lie: RUN = 8 neighbours, or two runs of 4, half of the row's width apart.  A run that is there as a whole moves as a vector, whatever its alignment
    // (the memory pipeline takes that); one that is not lies outside the buffer, and with `some` (uniform: the last columns are not a whole run) its `left` elements move one by one.
    template <uint32_t RUN>
    struct Columns
    {
        uint32_t at[8 / RUN], left[8 / RUN];
        bool     some;
    };

    // A lane's eight elements of type E of a row.
    template <typename E, uint32_t RUN>
    struct Eight
    {
        static constexpr uint32_t PER = 16u / sizeof(E) < RUN ? 16u / sizeof(E) : RUN; // elements an access
        vec<E, PER>               w[8u / PER];
        __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, uint32_t row, const Columns<RUN>& c) // row: byte offset
        {
#pragma unroll
            for(uint32_t r = 0; r < 8u / RUN; ++r)
            {
                const uint32_t offset = row + c.at[r] * static_cast<uint32_t>(sizeof(E));
                const bool     whole  = c.left[r] >= RUN;
#pragma unroll
                for(uint32_t i = 0; i < RUN / PER; ++i)
                {
                    const uint32_t at = whole ? offset + i * 16u : OUTSIDE;
                    if constexpr(PER * sizeof(E) == 16u)
                        w[r * (RUN / PER) + i] = __builtin_bit_cast(vec<E, PER>, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0));
                    else
                        w[r * (RUN / PER) + i] = __builtin_bit_cast(vec<E, PER>, __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0));
                }
                if(c.some && !whole)
#pragma unroll
                    for(uint32_t e = 0; e + 1u < RUN; ++e)
                    {
                        const uint32_t at = e < c.left[r] ? offset + e * static_cast<uint32_t>(sizeof(E)) : OUTSIDE, of = r * RUN + e;
                        if constexpr(sizeof(E) == 2u)
                            w[of / PER][of % PER] = __builtin_bit_cast(E, static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0)));
                        else
                            w[of / PER][of % PER] = __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
                    }
            }
        }
        __device__ __forceinline__ float operator[](uint32_t e) const
        {
            return static_cast<float>(w[e / PER][e % PER]);
        }
    };
    template <typename E, int POLICY, uint32_t RUN>
    __device__ __forceinline__ void storeRow(__amdgpu_buffer_rsrc_t to, uint32_t row, const Columns<RUN>& c, const float (&v)[8])
    {
        constexpr uint32_t PER = Eight<E, RUN>::PER;
#pragma unroll
        for(uint32_t r = 0; r < 8u / RUN; ++r)
        {
            const uint32_t offset = row + c.at[r] * static_cast<uint32_t>(sizeof(E));
            const bool     whole  = c.left[r] >= RUN;
#pragma unroll
            for(uint32_t i = 0; i < RUN / PER; ++i)
            {
                vec<E, PER> w;
#pragma unroll
                for(uint32_t e = 0; e < PER; ++e)
                    w[e] = static_cast<E>(v[r * RUN + i * PER + e]);
                // (the offset in the lane's register: gemm_tiled.hip says why)
                const uint32_t at = whole ? offset + i * 16u : OUTSIDE;
                if constexpr(PER * sizeof(E) == 16u)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, w), to, at, 0, POLICY);
                else
                    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, w), to, at, 0, POLICY);
            }
            if(c.some && !whole)
#pragma unroll
                for(uint32_t e = 0; e + 1u < RUN; ++e)
                {
                    const uint32_t at = e < c.left[r] ? offset + e * static_cast<uint32_t>(sizeof(E)) : OUTSIDE;
                    if constexpr(sizeof(E) == 2u)
                        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<E>(v[r * RUN + e])), to, at, 0, 0);
                    else
                        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, static_cast<E>(v[r * RUN + e])), to, at, 0, 0);
                }
        }
    }

    // Nontemporally where rows begin with a cache line, as what is written once; otherwise the L2 puts the lines together that neighbouring tiles write parts of
    // (8 gradients of 8144 x 5544 in f32 569 -> 277 us; of 4096 x 1536 102 instead of 76).
    template <typename E, uint32_t BATCH, uint32_t RUN>
    __device__ __forceinline__ void storeRows(bool lines, __amdgpu_buffer_rsrc_t to, uint32_t first, uint32_t step, const Columns<RUN>& c, const float (&v)[BATCH][8])
    {
        if(lines) // (uniform)
        {
#pragma unroll
            for(uint32_t u = 0; u < BATCH; ++u)
                storeRow<E, 2>(to, first + u * step, c, v[u]);
        }
        else
        {
#pragma unroll
            for(uint32_t u = 0; u < BATCH; ++u)
                storeRow<E, 0>(to, first + u * step, c, v[u]);
        }
    }

    // The buffer of `rows` rows of `cols` elements from (row, col) on, `bytes` an element: it ends with the last one
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rowsBuffer(const char* base, uint64_t row, uint32_t col, uint32_t ld, uint32_t rows, uint32_t cols, uint32_t bytes)
    {
        const uint64_t addr    = r355::uniformAddress(base + (row * ld + col) * bytes);
        const uint32_t records = rows && cols ? ((rows - 1u) * ld + cols) * bytes : 0u;
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(addr), 0, static_cast<int>(__builtin_amdgcn_readfirstlane(records)), 0x00020000);
    }

    // Results of one wave's tile of 16 WM x 16 WN, rows row0 .. and columns col0 .. of Y, `rows` x `cols` of them there: staged in f32 through the wave's own LDS, so that an
    // access covers whole rows of the wave's tile and the epilogue is taken of sums that nothing has rounded.
    //   z = sum + bias;  y = act(z) gate + c     (FULL; otherwise y = sum + c)
    // each rounded once.  Rows and columns that are not there lie outside the buffers: no branch around an access.
    template <uint32_t WM, uint32_t WN, bool FULL, typename Out>
    __device__ __forceinline__ void storeWave(f32x4 (&acc)[WM][WN], const LinearParams& p, const Work& w, uint32_t rowIn, uint32_t colIn, uint32_t lane, char* scratch)
    {
        constexpr uint32_t WT = 16u * WN, ROW = WT * 4u, PASS = WM % 4u == 0u ? 64u : 32u; // LDS bytes of a row, rows at a time
        constexpr uint32_t SWZ = WN * 4u < 16u ? WN * 4u - 1u : 15u;
        constexpr uint32_t LANES = WT / 8u, RPI = 64u / LANES, ITERS = PASS / RPI; // lanes of a row, rows an access, accesses
        constexpr uint32_t RUN = sizeof(Out) == 4u ? 4u : 8u; // (f32 in runs of 8 would leave every other 16 bytes to the next store: 16 gradients of 4096 x 1536 225 us instead of 165)
        constexpr uint32_t OS = sizeof(Out), MOST = OS == 4u ? 2u : 4u, BATCH = ITERS / 2u < MOST ? ITERS / 2u : MOST; // (more would not fit the registers)
        if(rowIn >= w.rowsLeft || colIn >= w.colsLeft)
            return; // (uniform)
        const uint32_t rows = w.rowsLeft - rowIn < 16u * WM ? w.rowsLeft - rowIn : 16u * WM, cols = w.colsLeft - colIn < WT ? w.colsLeft - colIn : WT;
        const uint64_t row0 = (uint64_t)w.first + rowIn;
        const uint32_t col0 = w.col0 + colIn, r16 = lane & 15u, quad = lane >> 4, rowLane = lane / LANES;
        Columns<RUN>   at;
        at.some = cols % RUN != 0u;
#pragma unroll
        for(uint32_t r = 0; r < 8u / RUN; ++r)
            at.at[r] = lane % LANES * RUN + r * LANES * RUN, at.left[r] = at.at[r] < cols ? cols - at.at[r] : 0u;
        // a share of a split sum goes to the workspace: [split][group, row of Y][column]
        char* const y = p.y + (uint64_t)w.group * p.strideY + (p.splits > 1u ? (uint64_t)w.share * p.strideSplit : 0u);
        const char* c = p.c ? p.c + (uint64_t)w.group * p.strideC : nullptr;

        Eight<T, RUN> bias;
        if constexpr(FULL)
            bias.load(rowsBuffer(p.bias, w.group, col0, p.n, p.bias ? 1u : 0u, cols, 2u), 0u, at);
#pragma unroll
        for(uint32_t pass = 0; pass < 16u * WM / PASS; ++pass)
        {
            const uint32_t under = pass * PASS < rows ? rows - pass * PASS : 0u, here = under < PASS ? under : PASS;
            const uint64_t row   = row0 + pass * PASS;
            const auto toY = rowsBuffer(y, row, col0, p.ldy, here, cols, OS);
            const auto fromC = rowsBuffer(c, row, col0, p.ldc, c ? here : 0u, cols, OS);
            const auto toZ = rowsBuffer(p.z, row, col0, p.ldz, FULL && p.z ? here : 0u, cols, 2u), fromG = rowsBuffer(p.gate, row, col0, p.ldg, FULL && p.gate ? here : 0u, cols, 2u);
            // two batches of accesses in turn: what one reads is under way while the other is worked on
            Eight<T, RUN>   gate[2][BATCH];
            Eight<Out, RUN> add[2][BATCH];
            auto request = [&](auto which, uint32_t b) __attribute__((always_inline)) {
                constexpr uint32_t W = decltype(which)::value;
                if(FULL && p.gate)
#pragma unroll
                    for(uint32_t u = 0; u < BATCH; ++u)
                        gate[W][u].load(fromG, ((b + u) * RPI + rowLane) * p.ldg * 2u, at);
                if(c)
#pragma unroll
                    for(uint32_t u = 0; u < BATCH; ++u)
                        add[W][u].load(fromC, ((b + u) * RPI + rowLane) * p.ldc * OS, at);
            };
            auto finish = [&](auto which, uint32_t b) __attribute__((always_inline)) {
                constexpr uint32_t W = decltype(which)::value;
                float              sum[BATCH][8];
#pragma unroll
                for(uint32_t u = 0; u < BATCH; ++u)
                {
                    const uint32_t r = (b + u) * RPI + rowLane;
#pragma unroll
                    for(uint32_t part = 0; part < 2u; ++part)
                    {
                        const uint32_t chunk = RUN == 8u ? at.at[0] / 4u + part : at.at[part % (8u / RUN)] / 4u;
                        const f32x4    v     = *reinterpret_cast<const f32x4*>(scratch + r * ROW + ((chunk ^ (r & SWZ)) * CHUNK));
#pragma unroll
                        for(uint32_t e = 0; e < 4u; ++e)
                            sum[u][part * 4u + e] = v[e];
                    }
                }
                if constexpr(FULL)
                {
#pragma unroll
                    for(uint32_t u = 0; u < BATCH; ++u)
#pragma unroll
                        for(uint32_t e = 0; e < 8u; ++e)
                            sum[u][e] += bias[e];
                    if(p.z)
                        storeRows<T>(p.linesZ != 0u, toZ, (b * RPI + rowLane) * p.ldz * 2u, RPI * p.ldz * 2u, at, sum);
                    r355::withActivation(p.activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
                        for(uint32_t u = 0; u < BATCH; ++u)
#pragma unroll
                            for(uint32_t e = 0; e < 8u; ++e)
                                sum[u][e] = r355::activate<decltype(act)::value>(sum[u][e]);
                    });
                    if(p.gate)
#pragma unroll
                        for(uint32_t u = 0; u < BATCH; ++u)
#pragma unroll
                            for(uint32_t e = 0; e < 8u; ++e)
                                sum[u][e] *= gate[W][u][e];
                }
                if(c)
#pragma unroll
                    for(uint32_t u = 0; u < BATCH; ++u)
#pragma unroll
                        for(uint32_t e = 0; e < 8u; ++e)
                            sum[u][e] += add[W][u][e];
                storeRows<Out>(p.linesY != 0u, toY, (b * RPI + rowLane) * p.ldy * OS, RPI * p.ldy * OS, at, sum);
            };
            constexpr std::integral_constant<uint32_t, 0> even;
            constexpr std::integral_constant<uint32_t, 1> odd;
            request(even, 0u);
#pragma unroll
            for(uint32_t i = 0; i < PASS / 16u; ++i)
#pragma unroll
                for(uint32_t j = 0; j < WN; ++j)
                {
                    const uint32_t r = 16u * i + r16;
                    *reinterpret_cast<f32x4*>(scratch + r * ROW + (((4u * j + quad) ^ (r & SWZ)) * CHUNK)) = acc[pass * (PASS / 16u) + i][j];
                }
            __builtin_amdgcn_wave_barrier(); // the same wave reads back what it wrote (LDS is in order per wave)
#pragma unroll 1
            for(uint32_t b = 0; b < ITERS && b * RPI < here; b += 2u * BATCH) // (uniform)
            {
                request(odd, b + BATCH);
                finish(even, b);
                if(b + 2u * BATCH < ITERS)
                    request(even, b + 2u * BATCH);
                finish(odd, b + BATCH);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    template <uint32_t WM, uint32_t WN, bool FULL>
    __device__ __forceinline__ void storeTile(f32x4 (&acc)[WM][WN], const LinearParams& p, const Work& w, uint32_t rowIn, uint32_t colIn, uint32_t lane, char* scratch)
    {
        if(p.outF32)
            storeWave<WM, WN, FULL, float>(acc, p, w, rowIn, colIn, lane, scratch);
        else
            storeWave<WM, WN, FULL, T>(acc, p, w, rowIn, colIn, lane, scratch);
    }

    // A stage of an operand that has `valid` bytes of the sum left per row: past its end the loads write zeros (K-contiguous: by tailOffset, otherwise the buffer ends there)
    template <bool KCONTIG>
    __device__ __forceinline__ i32x4 stageBuffer(uint64_t addr, uint32_t valid, uint32_t ld)
    {
        return i32x4{static_cast<int>(static_cast<uint32_t>(addr)), static_cast<int>(static_cast<uint32_t>(addr >> 32) & 0xFFFFu), static_cast<int>(KCONTIG ? 0x7FFFFFFFu : valid * ld),
                     0x00020000};
    }

    // Blocks of 32 rows of A's image.  Of an operand that is not contiguous along the sum there are images of 2, 4 and 8 (a load brings whole rows of the sum, whose swizzle stays
    // inside them): 192 rows of one lie in an image of 256, whose last quarter no wave reads (dW of 4096 x 2880 x 2880 71 us, on tiles of 256 rows 87; 8840 rows over 4 groups of 536 x 3552
    // 40 and 75).
    constexpr uint32_t imageOf(bool aK, uint32_t wm)
    {
        return aK || wm != 6u ? wm : 8u;
    }
    // bytes of LDS of a tile
    constexpr uint32_t ldsOf(bool aK, uint32_t wm, uint32_t wn)
    {
        return (2u * imageOf(aK, wm) + 3u * wn) * 32u * STAGE_KB;
    }

    template <bool AK, bool BK, uint32_t WM, uint32_t WN>
    __device__ __forceinline__ void linearTile(const LinearParams& p, const Work& w, char* lds)
    {
        constexpr uint32_t IA = imageOf(AK, WM);
        constexpr uint32_t SIZE_A = 32u * IA * STAGE_KB, SIZE_B = 32u * WN * STAGE_KB; // bytes of the operands' stages
        constexpr uint32_t FIRST_B = 2u * SIZE_A, LAST_B = FIRST_B + 2u * SIZE_B; // two buffers of A, three of B
        constexpr uint32_t NS = WM * WN, XS = WM + WN, BOTH = 2u * (WM < WN ? WM : WN); // matrix instructions and operand blocks of half a stage
        // the large tile's loads are dealt out over the whole stage, B two stages ahead; the small tiles', whose stages are a quarter as long and less, come in the
        // second half, B three stages ahead (gemm_tiled.hip has both measured), where there is room for all of them
        constexpr bool     SPREAD  = IA == 8u || WN == 8u;
        constexpr uint32_t B_AHEAD = SPREAD ? 2u : 3u;
        constexpr uint32_t SCRATCH = 64u * WN * (WM % 4u == 0u ? 64u : 32u); // of a wave's part of the epilogue
        static_assert(ldsOf(AK, WM, WN) <= 160u * 1024u && 4u * SCRATCH <= ldsOf(AK, WM, WN), "what a CU has");
        static_assert(SPREAD ? IA <= XS && WN <= XS : IA == WM, "one load an operand block at most");
        const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1u;
        const uint32_t ldsBase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
        const uint32_t dma     = ldsBase + wave * 64u * CHUNK;

        uint32_t offA[IA], offB[WN], stepA, stepB, kByteA, kByteB;
        uint64_t stageA, stageB;
        laneOffsets8<AK, IA, 2>(tid, p.lda, w.rowsLeft, offA, stepA, stageA, kByteA);
        laneOffsets8<BK, WN, 2>(tid, p.ldb, w.colsLeft, offB, stepB, stageB, kByteB);
        uint64_t fromA, fromB;
        if constexpr(AK)
        {
            if(p.source) // rows by their numbers; one that is none of A's reads as zeros
            {
                const uint32_t r = tid >> 3, slot = tid & 7u;
#pragma unroll
                for(uint32_t j = 0; j < WM; ++j)
                {
                    const uint32_t row = r + 32u * j < w.rowsLeft ? r + 32u * j : w.rowsLeft - 1u, from = static_cast<uint32_t>(p.source[(uint64_t)w.first + row]);
                    offA[j]            = from < p.sourceRows ? from * p.lda * 2u + ((slot ^ swzK8(r)) * CHUNK) : OUTSIDE;
                }
            }
            fromA = r355::uniformAddress(p.a + ((p.source ? 0u : (uint64_t)w.first * p.lda) + w.kFirst) * 2u);
            fromB = r355::uniformAddress(p.b + (uint64_t)w.group * p.strideB + (BK ? (uint64_t)w.col0 * p.ldb + w.kFirst : (uint64_t)w.kFirst * p.ldb + w.col0) * 2u);
        }
        else
        {
            fromA = r355::uniformAddress(p.a + ((w.sumRow + w.kFirst) * p.lda + w.first) * 2u);
            fromB = r355::uniformAddress(p.b + ((w.sumRow + w.kFirst) * p.ldb + w.col0) * 2u);
        }
        // (an empty sum has one stage of zeros)
        const uint32_t stages = w.k > TK ? (w.k - 1u) / TK + 1u : 1u, lastBytes = (w.k - (stages - 1u) * TK) * 2u;
        auto validOf = [&](uint32_t s) { return s + 1u < stages ? STAGE_KB : s + 1u == stages ? lastBytes : 0u; };
        auto tailA = [&](uint32_t j, uint32_t valid) { return AK && kByteA >= valid ? OUTSIDE : offA[j]; };
        auto tailB = [&](uint32_t j, uint32_t valid) { return BK && kByteB >= valid ? OUTSIDE : offB[j]; };
        // By groups, the sum's whole stages begin elsewhere in every group, or, of short sums, on every XCD: workgroups that go through rows of a power of two of bytes side by side, all at the same
        // place of a row, keep some of the memory's channels busy and others not (64 groups of 64 rows, 2048 x 2048: 130 -> 99 us, 32 68 -> 51, their dx in 64 groups of 2048 x 4096 219 -> 184;
        // 2048 x 1024 by groups 58 -> 60, by XCDs 54; 32 groups of 4096 x 4096 by groups 184 -> 176, by XCDs 202).  Weights that many rows read come from the caches: no difference, or a loss (4 groups
        // of 4096 rows, 8192 x 2048 458 -> 478).
        uint32_t turn = 0u;
        const uint32_t turns = w.k / TK;
        if(AK && p.groups > 1u && turns != 0u && p.rows / p.groups <= 1024u)
            turn = turns >= 24u ? ((w.group * 0x9E3779B1u) >> 16) * turns >> 16 : blockIdx.x % 8u * turns / 8u;
        auto placeOf = [&](uint32_t s) {
            const uint32_t at = s < stages ? s : stages - 1u; // (of a stage that is not there no lane reads anything)
            return static_cast<uint64_t>(at >= turns ? at : at + turn < turns ? at + turn : at + turn - turns);
        };
        auto addrA = [&](uint32_t s) { return fromA + placeOf(s) * stageA; };
        auto addrB = [&](uint32_t s) { return fromB + placeOf(s) * stageB; };
        auto issueA = [&](uint32_t s, uint32_t at) {
            const uint32_t valid = validOf(s);
#pragma unroll
            for(uint32_t j = 0; j < IA; ++j)
                loadToLds(stageBuffer<AK>(addrA(s), valid, p.lda), tailA(j, valid), j * stepA, dma + at + j * THREADS * CHUNK);
        };
        auto issueB = [&](uint32_t s, uint32_t at) {
            const uint32_t valid = validOf(s);
#pragma unroll
            for(uint32_t j = 0; j < WN; ++j)
                loadToLds(stageBuffer<BK>(addrB(s), valid, p.ldb), tailB(j, valid), j * stepB, dma + at + j * THREADS * CHUNK);
        };

        uint32_t rdA[8], rdB[8];
        readOffsets8<AK, IA, 2, WM>(wm, lane, rdA);
        readOffsets8<BK, WN, 2>(wn, lane, rdB);
        f32x4 acc[WM][WN];
#pragma unroll
        for(uint32_t i = 0; i < WM; ++i)
#pragma unroll
            for(uint32_t j = 0; j < WN; ++j)
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        i32x4 fa[2][WM], fb[2][WN];
        // matrix instruction n of half a stage, in shells around block (0, 0) as the operand blocks come, A0 B0 A1 B1 ... and then the rest of the longer operand; the
        // operands swapped: a lane holds four neighbouring columns of a row
        auto multiplyAt = [&](uint32_t half, uint32_t n) {
            constexpr uint32_t LESS = BOTH / 2u;
            uint32_t           d    = 0;
            while(d < LESS && (d + 1u) * (d + 1u) <= n)
                ++d;
            const uint32_t r = n - d * d, past = n - LESS * LESS;
            const uint32_t i = n < LESS * LESS ? (r <= d ? d : r - d - 1u) : WM > WN ? LESS + past / LESS : past % LESS;
            const uint32_t j = n < LESS * LESS ? (r <= d ? r : d) : WM > WN ? past % LESS : LESS + past / LESS;
            multiply(acc[i][j], fb[half][j], fa[half][i]);
        };
        auto readAt = [&](uint32_t atA, uint32_t atB, uint32_t half, uint32_t x, uint32_t part) {
            const bool     ofB = x < BOTH ? (x & 1u) != 0u : WN > WM;
            const uint32_t i   = x < BOTH ? x >> 1 : x - BOTH / 2u;
            if(ofB)
                readBlock8<BK, WN, 2>(lds + atB, rdB, i, half, part, fb[half][i], 0u);
            else
                readBlock8<AK, IA, 2>(lds + atA, rdA, i, half, part, fa[half][i], 0u);
        };
        auto after = [](uint32_t at) { return at == LAST_B ? FIRST_B : at + SIZE_B; }; // B's buffers go round
        // matrix instructions firstOf(x) .. firstOf(x + 1) - 1 of half a stage go with operand block x, one at least: with the first two its reads, with the third, or the last, a load
        auto firstOf = [](uint32_t x) { return x * NS / XS; };
        auto readsAt = [&](uint32_t atA, uint32_t atB, uint32_t half, uint32_t x, uint32_t n) {
            if(n == firstOf(x))
                readAt(atA, atB, half, x, 0);
            if(n == firstOf(x) + 1u || firstOf(x + 1u) == firstOf(x) + 1u)
                readAt(atA, atB, half, x, 1);
        };
        auto loadsAt = [&](uint32_t x, uint32_t n) {
            const uint32_t q = n - firstOf(x), of = firstOf(x + 1u) - firstOf(x);
            return q == (of > 2u ? 2u : of - 1u);
        };

        // prologue: stages 0 and 1 (and B of stage 2) requested in the order that the loop keeps
        if constexpr(SPREAD)
        {
            issueB(0u, FIRST_B), issueA(0u, 0u), issueB(1u, FIRST_B + SIZE_B), issueA(1u, SIZE_A);
            waitVmcnt<IA + WN>();
        }
        else
        {
            issueA(0u, 0u), issueB(0u, FIRST_B), issueA(1u, SIZE_A), issueB(1u, FIRST_B + SIZE_B), issueB(2u, LAST_B);
            waitVmcnt<IA + 2u * WN>();
        }
        ldsBarrier();
#pragma unroll
        for(uint32_t x = 0; x < XS; ++x)
        {
            readAt(0u, FIRST_B, 0, x, 0);
            readAt(0u, FIRST_B, 0, x, 1);
        }
        uint32_t aCur = 0u, bCur = FIRST_B;
        // One stage, its first half in registers: the second half arrives under the first's matrix instructions, then the first half of the next stage under the second's.
        // FULL: all that this stage requests lies inside the sum.
        auto stage = [&](auto full, uint32_t kt) {
            constexpr bool FULL = decltype(full)::value;
            const uint32_t aNxt = SIZE_A - aCur, bNxt = after(bCur), bTo = SPREAD ? after(bNxt) : bCur;
            const uint32_t vB   = FULL ? STAGE_KB : validOf(kt + B_AHEAD);
            const i32x4    bufB = stageBuffer<BK>(addrB(kt + B_AHEAD), vB, p.ldb);
            auto loadA = [&](i32x4 buf, uint32_t valid, uint32_t j) { loadToLds(buf, FULL ? offA[j] : tailA(j, valid), j * stepA, dma + aCur + j * THREADS * CHUNK); };
            auto loadB = [&](uint32_t j) { loadToLds(bufB, FULL ? offB[j] : tailB(j, vB), j * stepB, dma + bTo + j * THREADS * CHUNK); };
#pragma unroll
            for(uint32_t x = 0; x < XS; ++x)
#pragma unroll
                for(uint32_t n = firstOf(x); n < firstOf(x + 1u); ++n)
                {
                    multiplyAt(0, n);
                    readsAt(aCur, bCur, 1, x, n);
                    if(SPREAD && loadsAt(x, n))
                        if(const uint32_t j = x * WN / XS; (x + 1u) * WN / XS > j)
                            loadB(j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            waitVmcnt<WN>(); // all but the youngest loads, B of stage kt + 2
            ldsBarrier();
            const uint32_t vA   = FULL ? STAGE_KB : validOf(kt + 2u);
            const i32x4    bufA = stageBuffer<AK>(addrA(kt + 2u), vA, p.lda);
#pragma unroll
            for(uint32_t x = 0; x < XS; ++x)
#pragma unroll
                for(uint32_t n = firstOf(x); n < firstOf(x + 1u); ++n)
                {
                    multiplyAt(1, n);
                    readsAt(aNxt, bNxt, 0, x, n);
                    if(loadsAt(x, n))
                    {
                        if constexpr(SPREAD)
                        {
                            if(const uint32_t j = x * IA / XS; (x + 1u) * IA / XS > j)
                                loadA(bufA, vA, j);
                        }
                        else if(x < WM)
                            loadA(bufA, vA, x);
                        else
                            loadB(x - WM);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            aCur = aNxt, bCur = bNxt;
        };
        const uint32_t whole = w.k / TK, main = whole > B_AHEAD ? whole - B_AHEAD : 0u;
        uint32_t       kt    = 0u;
        for(; kt < main; ++kt)
            stage(std::true_type{}, kt);
        for(; kt < stages; ++kt)
            stage(std::false_type{}, kt);

        // the last matrix instructions are still under way, which the compiler does not know, and loads past the last stage are writing zeros to buffers that the
        // epilogue uses
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
        waitVmcnt<0>();
        ldsBarrier();
        storeTile<WM, WN, AK && BK>(acc, p, w, wm * 16u * WM, wn * 16u * WN, lane, lds + wave * SCRATCH);
    }

    // (a kernel per tile: the attribute cannot depend on a template parameter)
    // Of ragged rows, the last tile of a group takes a form as high as its rows (64 groups of 64 rows, 2048 x 2048: 112 -> 47 us with the weights at hand, 130 with those of each group from memory).
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) linearTiles256(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 8, 8)];
        Work                                           w;
        if(!workOf<AK, 256, 256>(p, w, blockIdx.x, blockIdx.y))
            return;
        if(!AK || w.rowsLeft > 192u)
            linearTile<AK, BK, 8, 8>(p, w, lds);
        else if constexpr(AK)
        {
            if(w.rowsLeft > 128u)
                linearTile<AK, BK, 6, 8>(p, w, lds);
            else if(w.rowsLeft > 64u)
                linearTile<AK, BK, 4, 8>(p, w, lds);
            else
                linearTile<AK, BK, 2, 8>(p, w, lds);
        }
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) linearTiles192x256(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 6, 8)];
        Work                                           w;
        if(workOf<AK, 192, 256>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 6, 8>(p, w, lds);
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) linearTiles192x128(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 6, 4)];
        Work                                           w;
        if(workOf<AK, 192, 128>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 6, 4>(p, w, lds);
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) linearTiles256x128(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 8, 4)];
        Work                                           w;
        if(workOf<AK, 256, 128>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 8, 4>(p, w, lds);
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) linearTiles128x256(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 4, 8)];
        Work                                           w;
        if(workOf<AK, 128, 256>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 4, 8>(p, w, lds);
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS, 2) linearTiles128(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 4, 4)];
        Work                                           w;
        if(workOf<AK, 128, 128>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 4, 4>(p, w, lds);
    }
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS, 4) linearTiles64(LinearParams p)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(AK, 2, 2)];
        Work                                           w;
        if(workOf<AK, 64, 64>(p, w, blockIdx.x, blockIdx.y))
            linearTile<AK, BK, 2, 2>(p, w, lds);
    }

    // Both gradients of a small layer in one launch: the input's by the first workgroups, the weights' by the others, on small tiles, four workgroups a CU (992 x 1008 x 1232 24.1 -> 17.3 us,
    // 100 x 512 x 512 11.1 -> 8.4, 2048 x 1024 x 1024 26.1 -> 18.9; of larger layers separate launches of larger tiles take less, by planBoth()).
    __global__ void __launch_bounds__(THREADS, 4) linearBoth64(LinearParams px, LinearParams pw, uint32_t workgroupsX, uint32_t workgroupsW)
    {
        __shared__ __attribute__((aligned(1024))) char lds[ldsOf(false, 2, 2)];
        Work                                           w;
        const uint32_t                                 first = workgroupsX * px.splits;
        if(blockIdx.x < first)
        {
            if(workOf<true, 64, 64>(px, w, blockIdx.x % workgroupsX, blockIdx.x / workgroupsX))
                linearTile<true, false, 2, 2>(px, w, lds);
        }
        else if(workOf<false, 64, 64>(pw, w, (blockIdx.x - first) % workgroupsW, (blockIdx.x - first) / workgroupsW))
            linearTile<false, false, 2, 2>(pw, w, lds);
    }

    // Eight elements of any alignment, `left` of them there: at once, or at the ends one by one
    __device__ __forceinline__ vec<T, 8> piece(const T* at, uint32_t left)
    {
        typedef T Unaligned __attribute__((ext_vector_type(8), aligned(2)));
        vec<T, 8> v{};
        if(left >= 8u)
            v = *reinterpret_cast<const Unaligned*>(at);
        else
#pragma unroll
            for(uint32_t e = 0; e < 7u; ++e)
                if(e < left)
                    v[e] = at[e];
        return v;
    }

    // The same on tiles of 64 x 64 for operands of any alignment, lengths and leading dimensions: through registers, 32 of the sum at a time (1500 x 1500 x 4096 backward, both
    // products, 460 us with single elements; even rows take 60).
    template <bool AK, bool BK>
    __global__ void __launch_bounds__(THREADS) linearAny(LinearParams p)
    {
        constexpr uint32_t TILE = 64u, STEP = 32u, PITCH = STEP + 8u; // (elements; rows 80 bytes apart: 16-byte reads of 16 rows meet in a bank at most twice)
        __shared__ __attribute__((aligned(16))) T   image[2][TILE * PITCH];
        __shared__ __attribute__((aligned(16))) char scratch[4u * 2u * 4096u];
        Work w;
        if(!workOf<AK, TILE, TILE>(p, w, blockIdx.x, blockIdx.y))
            return;
        const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1u;
        // a thread's eight elements of a step: neighbours along the sum, or along the rows of Y (columns, for B)
        const uint32_t rowA = AK ? tid >> 2 : (tid & 7u) * 8u, kA = AK ? (tid & 3u) * 8u : tid >> 3;
        const uint32_t rowB = BK ? tid >> 2 : (tid & 7u) * 8u, kB = BK ? (tid & 3u) * 8u : tid >> 3;
        const T* a = reinterpret_cast<const T*>(p.a);
        const T* b = reinterpret_cast<const T*>(p.b) + w.group * (p.strideB / 2u);
        bool     there = rowA < w.rowsLeft;
        if constexpr(AK)
        {
            uint64_t row = (uint64_t)w.first + rowA;
            if(there && p.source)
            {
                const uint32_t from = static_cast<uint32_t>(p.source[row]);
                there = from < p.sourceRows, row = from;
            }
            a += row * p.lda + w.kFirst;
            b += BK ? (uint64_t)(w.col0 + rowB) * p.ldb + w.kFirst : (uint64_t)w.kFirst * p.ldb + w.col0 + rowB;
        }
        else
        {
            a += (w.sumRow + w.kFirst) * p.lda + w.first + rowA;
            b += (w.sumRow + w.kFirst) * p.ldb + w.col0 + rowB;
        }
        f32x4 acc[2][2];
#pragma unroll
        for(uint32_t i = 0; i < 2u; ++i)
#pragma unroll
            for(uint32_t j = 0; j < 2u; ++j)
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for(uint32_t k0 = 0; k0 < w.k; k0 += STEP)
        {
            const uint32_t  leftK = w.k - k0; // of the sum
            const vec<T, 8> va = piece(a + (AK ? (uint64_t)k0 + kA : (uint64_t)(k0 + kA) * p.lda), AK ? (there && kA < leftK ? leftK - kA : 0u) : (kA < leftK && rowA < w.rowsLeft ? w.rowsLeft - rowA : 0u));
            const vec<T, 8> vb = piece(b + (BK ? (uint64_t)k0 + kB : (uint64_t)(k0 + kB) * p.ldb),
                                       BK ? (rowB < w.colsLeft && kB < leftK ? leftK - kB : 0u) : (kB < leftK && rowB < w.colsLeft ? w.colsLeft - rowB : 0u));
            __syncthreads();
            if constexpr(AK)
                *reinterpret_cast<vec<T, 8>*>(&image[0][rowA * PITCH + kA]) = va;
            else
#pragma unroll
                for(uint32_t e = 0; e < 8u; ++e)
                    image[0][(rowA + e) * PITCH + kA] = va[e];
            if constexpr(BK)
                *reinterpret_cast<vec<T, 8>*>(&image[1][rowB * PITCH + kB]) = vb;
            else
#pragma unroll
                for(uint32_t e = 0; e < 8u; ++e)
                    image[1][(rowB + e) * PITCH + kB] = vb[e];
            __syncthreads();
            u32x4 fa[2], fb[2];
#pragma unroll
            for(uint32_t i = 0; i < 2u; ++i)
            {
                fa[i] = *reinterpret_cast<const u32x4*>(&image[0][(wm * 32u + i * 16u + (lane & 15u)) * PITCH + (lane >> 4) * 8u]);
                fb[i] = *reinterpret_cast<const u32x4*>(&image[1][(wn * 32u + i * 16u + (lane & 15u)) * PITCH + (lane >> 4) * 8u]);
            }
#pragma unroll
            for(uint32_t i = 0; i < 2u; ++i)
#pragma unroll
                for(uint32_t j = 0; j < 2u; ++j)
                    acc[i][j] = r355::mfma32<T>(fb[j], fa[i], acc[i][j]);
        }
        storeTile<2, 2, AK && BK>(acc, p, w, wm * 32u, wn * 32u, lane, scratch + wave * 8192u);
    }

    template <bool AK, bool BK>
    void launch(const LinearParams& p, r355::LinearTile tile, uint32_t workgroups, hipStream_t s)
    {
        const auto kernel = tile == r355::TILE_256       ? linearTiles256<AK, BK>
                            : tile == r355::TILE_192_256 ? linearTiles192x256<AK, BK>
                            : tile == r355::TILE_256_128 ? linearTiles256x128<AK, BK>
                            : tile == r355::TILE_192_128 ? linearTiles192x128<AK, BK>
                            : tile == r355::TILE_128_256 ? linearTiles128x256<AK, BK>
                            : tile == r355::TILE_128     ? linearTiles128<AK, BK>
                            : tile == r355::TILE_64      ? linearTiles64<AK, BK>
                                                         : linearAny<AK, BK>;
        hipLaunchKernelGGL(kernel, dim3(workgroups, p.splits), dim3(THREADS), 0, s, p);
    }
} // namespace

#ifdef R355_LINEAR_BF16
void r355::linearTilesBF16(const LinearParams& p, bool aK, bool bK, LinearTile tile, uint32_t workgroups, hipStream_t s)
#else
void r355::linearTilesF16(const LinearParams& p, bool aK, bool bK, LinearTile tile, uint32_t workgroups, hipStream_t s)
#endif
{
    if(aK && bK)
        launch<true, true>(p, tile, workgroups, s);
    else if(aK)
        launch<true, false>(p, tile, workgroups, s);
    else
        launch<false, false>(p, tile, workgroups, s);
}

#ifdef R355_LINEAR_BF16
void r355::linearBothBF16(const LinearParams& px, const LinearParams& pw, uint32_t workgroupsX, uint32_t workgroupsW, hipStream_t s)
#else
void r355::linearBothF16(const LinearParams& px, const LinearParams& pw, uint32_t workgroupsX, uint32_t workgroupsW, hipStream_t s)
#endif
{
    hipLaunchKernelGGL(linearBoth64, dim3(workgroupsX * px.splits + workgroupsW * pw.splits), dim3(THREADS), 0, s, px, pw, workgroupsX, workgroupsW);
}
