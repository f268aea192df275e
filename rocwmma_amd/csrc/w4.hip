// Products with 4-bit weights and group scales on gfx950 matrix cores.
//
//   y[t][r] = alpha * sum_k x[t][k] (q[r][k] - z[k / g][r]) s[k / g][r] + beta c[t][r]
//
// No counterpart in the reference.  The weights q are stored in blocks of 16 rows x 128 k (r355_w4_pack), 1 KiB each in the order in
// which a wave's lanes load them, 16 bytes a lane: the four dwords of a lane are its second operands of four v_mfma_f32_16x16x32, x is the
// first, and up to 16 tokens cost what one costs.
//
// A nibble becomes an operand without a conversion: with the nibble in the four leading bits of the mantissa of 16.0 the 16-bit number
// is 16 + q, so a shift and an and-or make two operands.  The matrix instruction sums x (16 + q) over a group exactly as it would sum x q,
// one more instruction with ones for weights leaves sum x in the same lanes, and
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x
// in f32: the sums are about five times as large as the difference (16 + 7.5 against the spread of q), so their rounding costs about
// two bits of 24.  The scale of the group is applied to the f32 sum, never to a 16-bit weight.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"
#include "half_types.hpp"
#include "lds_dma.hpp"

namespace
{
    using r355::each;
    using r355::f32x4;
    using r355::u32x2;
    using r355::u32x4;
    using r355::vec;

    struct W4Params
    {
        const char*    x;
        const char*    w;
        const char*    scales;
        const uint8_t* zeros;
        const char*    c;
        char*          y;
        uint32_t       tokens, n, k, group, groups;
        uint32_t       ldx, ldc, ldy;
        uint32_t       blocksN, blocksK; // of 16 rows, of 128 k
        uint32_t       perGroup, groupMagic; // blocks of 128 k per group of 128 and more, and 2^32 over it, rounded up (exact: both numbers of blocks are at most 2^15)
        uint32_t       tilesN, tilesT, perXcd; // workgroups along n and tokens, and of each XCD
        uint32_t       outF32, wideN; // wideN: 4-element accesses of c and y
        float          alpha, beta;
    };

    constexpr uint32_t OUTSIDE = 0x7FFFFFF0u; // a lane's offset past the end of any buffer: it loads zeros

    // Eight weights of a dword as 16 + q each, two (nibbles p and p + 4) a register.  The two constants are kept from the compiler, which otherwise makes
    // an and and an or with literals of what is one instruction with registers.
    template <typename T>
    struct Expand
    {
        uint32_t mask, sixteen;
        __device__ __forceinline__ Expand()
        {
            mask = std::is_same_v<T, __bf16> ? 0x00780078u : 0x03C003C0u, sixteen = std::is_same_v<T, __bf16> ? 0x41804180u : 0x4C004C00u;
            asm volatile("" : "+s"(mask), "+v"(sixteen));
        }
        __device__ __forceinline__ u32x4 operator()(uint32_t d) const
        {
            if constexpr(std::is_same_v<T, __bf16>)
                return u32x4{((d << 3) & mask) | sixteen, ((d >> 1) & mask) | sixteen, ((d >> 5) & mask) | sixteen, ((d >> 9) & mask) | sixteen};
            else
                return u32x4{((d << 6) & mask) | sixteen, ((d << 2) & mask) | sixteen, ((d >> 2) & mask) | sixteen, ((d >> 6) & mask) | sixteen};
        }
    };

    // all 1, or all -24
    template <typename T, bool EARLY>
    __device__ __forceinline__ u32x4 timesOf()
    {
        constexpr uint32_t V = std::is_same_v<T, __bf16> ? (EARLY ? 0xC1C0C1C0u : 0x3F803F80u) : (EARLY ? 0xCE00CE00u : 0x3C003C00u);
        return u32x4{V, V, V, V};
    }

    // a 16-bit scale in the low half of a dword
    template <typename T>
    __device__ __forceinline__ float scaleOf(uint32_t v)
    {
        if constexpr(std::is_same_v<T, __bf16>)
            return __uint_as_float(v << 16);
        else
            return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v)));
    }

    // scale of the lane's row, and 16 + z of its zero point
    struct Values
    {
        float scale, zero;
    };
    __device__ __forceinline__ float zeroOf(uint32_t z)
    {
        return __uint_as_float(0x41800000u | (z << 19)); // (z < 16)
    }

    // the first group of block kb of 128 k
    template <uint32_t STEPS>
    __device__ __forceinline__ uint32_t groupOf(const W4Params& p, uint32_t kb)
    {
        return STEPS < 4u ? kb * (4u / STEPS) : p.perGroup == 1u ? kb : __umulhi(kb, p.groupMagic);
    }

    // One group (STEPS matrix instructions of 32 k): acc += s (sum x (16 + q) - (16 + z) sum x).  x is the first operand: a lane holds four tokens of one
    // row, so that it needs one scale and one zero point.  Every column of the product with ones is sum x.
    // EARLY: with z = 8 everywhere the product of all rows starts from -24 sum x, a product with that, instead of zero; x(c, i) is held meanwhile.
    template <typename T, uint32_t RB, uint32_t CB, uint32_t STEPS, bool ZEROS, bool EARLY, typename X, typename W, typename V>
    __device__ __forceinline__ void accumulate(f32x4 (&acc)[RB][CB], const Expand<T>& expand, X&& x, W&& weights, V&& values)
    {
        static_assert(!(ZEROS && EARLY), "one start for all rows");
        const u32x4 times = timesOf<T, EARLY>();
        f32x4       sumX[CB], sum[RB][CB];
        u32x4       held[CB][EARLY ? STEPS : 1u];
#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
            sumX[c] = f32x4{0, 0, 0, 0};
        if constexpr(EARLY)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
                    held[c][i] = x(c, i);
                    sumX[c]    = r355::mfma32<T>(held[c][i], times, sumX[c]);
                }
#pragma unroll
        for(uint32_t i = 0; i < STEPS; ++i)
        {
            if constexpr(!EARLY)
#pragma unroll
                for(uint32_t c = 0; c < CB; ++c)
                {
                    held[c][0] = x(c, i);
                    sumX[c]    = r355::mfma32<T>(held[c][0], times, sumX[c]);
                }
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
            {
                const u32x4 b = expand(weights(r, i));
#pragma unroll
                for(uint32_t c = 0; c < CB; ++c)
                    sum[r][c] = r355::mfma32<T>(held[c][EARLY ? i : 0u], b, i != 0u ? sum[r][c] : EARLY ? sumX[c] : f32x4{0, 0, 0, 0});
            }
        }
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
        {
            if constexpr(ZEROS && RB * CB >= 16u)
                __builtin_amdgcn_sched_barrier(0); // (the values of several blocks of rows at once would not fit beside the sums)
            const Values v = values(r);
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                for(uint32_t j = 0; j < 4; ++j)
                    acc[r][c][j] = fmaf(v.scale, EARLY ? sum[r][c][j] : fmaf(ZEROS ? -v.zero : -24.0f, sumX[c][j], sum[r][c][j]), acc[r][c][j]);
        }
    }

    template <typename O>
    __device__ __forceinline__ void storeRows(const W4Params& p, uint32_t token, uint32_t row, f32x4 sum)
    {
        const O* c = reinterpret_cast<const O*>(p.c) + (uint64_t)token * p.ldc + row;
        O*       y = reinterpret_cast<O*>(p.y) + (uint64_t)token * p.ldy + row;
        if(p.wideN && row + 4u <= p.n)
        {
            f32x4 out{p.alpha * sum[0], p.alpha * sum[1], p.alpha * sum[2], p.alpha * sum[3]};
            if(p.beta != 0.0f)
            {
                const vec<O, 4> was = *reinterpret_cast<const vec<O, 4>*>(c);
#pragma unroll
                for(uint32_t e = 0; e < 4; ++e)
                    out[e] += p.beta * static_cast<float>(was[e]);
            }
            *reinterpret_cast<vec<O, 4>*>(y) = vec<O, 4>{static_cast<O>(out[0]), static_cast<O>(out[1]), static_cast<O>(out[2]), static_cast<O>(out[3])};
        }
        else
#pragma unroll
            for(uint32_t e = 0; e < 4u; ++e)
                if(row + e < p.n)
                    y[e] = static_cast<O>(p.beta != 0.0f ? p.alpha * sum[e] + p.beta * static_cast<float>(c[e]) : p.alpha * sum[e]);
    }
    template <typename T>
    __device__ __forceinline__ void store(const W4Params& p, uint32_t token, uint32_t row, f32x4 sum)
    {
        if(token >= p.tokens || row >= p.n)
            return;
        if(p.outF32)
            storeRows<float>(p, token, row, sum);
        else
            storeRows<T>(p, token, row, sum);
    }

    // The sums of `sets` sets of waves, [token][STRIDE] with ROWS rows each, added up in order and stored, four rows of a token to a thread.
    template <typename T, uint32_t ROWS, uint32_t TOKENS, uint32_t STRIDE>
    __device__ __forceinline__ void storeTile(const W4Params& p, const float* sums, uint32_t sets, uint32_t token0, uint32_t row0)
    {
        const uint32_t left = p.tokens - token0 < TOKENS ? p.tokens - token0 : TOKENS;
        for(uint32_t i = threadIdx.x; i < left * (ROWS / 4u); i += blockDim.x)
        {
            const uint32_t token = i / (ROWS / 4u), row = i % (ROWS / 4u) * 4u;
            f32x4          sum   = *reinterpret_cast<const f32x4*>(sums + token * STRIDE + row);
            for(uint32_t v = 1u; v < sets; ++v)
                sum += *reinterpret_cast<const f32x4*>(sums + (v * TOKENS + token) * STRIDE + row);
            store<T>(p, token0 + token, row0 + row, sum);
        }
    }

    // Tile of n and tile of tokens of a workgroup: workgroups id, id + 8, ... run on one XCD and take a contiguous stretch of the tiles, those of one tile of
    // n after another (the scales of neighbouring rows share cache lines, the weights a tile of n).
    __device__ __forceinline__ bool tileOf(const W4Params& p, uint32_t& tileN, uint32_t& tileT)
    {
        const uint32_t id = blockIdx.x % 8u * p.perXcd + blockIdx.x / 8u;
        tileN = id / p.tilesT, tileT = id % p.tilesT;
        return tileN < p.tilesN;
    }

    // ---- A few tokens, or rows of x off 16-byte boundaries (FAST false: element by element, one tile for any number of tokens; 8192 x 4096, groups of 64, with rows 4097 apart
    // 1 token 14.5 us instead of 5.4, 24 tokens 48 instead of 8.1, 1000 tokens 2040 instead of 81).  A workgroup's waves share 16 RB rows x 16 CB tokens and take the 128-k blocks in
    // turn, x and the weights straight from global memory; their sums meet in LDS in the order of the waves, so the result does not depend on
    // scheduling.  STEPS: matrix instructions (32 k) per scale.  DEPTH blocks in flight, each in registers of its own.
    // Bound by the bytes of the weights from one wide row of workgroups on (16384 x 8192, groups of 128 with zero points, one token: 14.4 us, 4.9 TB/s of
    // weights, scales and zero points), below that by one load's latency and the launch (1024 x 2048: 5.6 us); with more tokens by x out of the L2 and, with small groups,
    // the vector instructions that make operands and apply scales (10250 x 4168, groups of 32, 24 tokens: 13.1 us in one round of 214 workgroups).  No LDS: no other wave reads the same weights.
    template <typename T, uint32_t RB, uint32_t CB, uint32_t DEPTH, uint32_t STEPS, bool ZEROS, bool FAST>
    __global__ void __launch_bounds__(512, FAST ? 2 : 1) w4Kernel(W4Params p)
    {
        extern __shared__ __attribute__((aligned(16))) float sums[]; // [waves][16 CB tokens][16 RB rows]
        constexpr uint32_t PARTS = 4u / STEPS;
        uint32_t           tileN, tileT;
        if(!tileOf(p, tileN, tileT))
            return;
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
        const uint32_t col = lane & 15u, quad = lane >> 4;
        const uint32_t block0 = tileN * RB, token0 = tileT * 16u * CB, left = p.tokens - token0;
        const Expand<T> expand;
        f32x4           acc[RB][CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                acc[r][c] = f32x4{0, 0, 0, 0};

        // Where a block of 128 k has several groups, the lanes of one row read one each and exchange them: one load instead of four.
        struct Stage
        {
            u32x4    w[RB], x[CB][4];
            uint32_t scale[RB], zero[RB];
        };
        const uint32_t mine = quad % PARTS;
        // (a buffer over the rows of x from token0 on, which ends with the last element; lanes without a token lie past it)
        const auto bufX = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.x) + (uint64_t)token0 * p.ldx * 2u, 0,
                                                            FAST ? ((left < 16u * CB ? left : 16u * CB) - 1u) * p.ldx * 2u + p.k * 2u : 0u, 0x00020000);
        uint32_t offX[CB];
#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
            offX[c] = c * 16u + col < left ? (c * 16u + col) * p.ldx * 2u + quad * 16u : OUTSIDE;
        auto load = [&](uint32_t kb) __attribute__((always_inline)) {
            Stage          s;
            const uint32_t of = groupOf<STEPS>(p, kb) + mine;
            const uint64_t g  = of < p.groups ? of : p.groups - 1u; // (past k: x is zero there)
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
            {
                const uint32_t b = block0 + r < p.blocksN ? block0 + r : p.blocksN - 1u;
                s.w[r]           = *reinterpret_cast<const u32x4*>(p.w + ((uint64_t)b * p.blocksK + kb) * 1024u + lane * 16u);
                const uint32_t row = (block0 + r) * 16u + col;
                const uint64_t at  = g * p.n + (row < p.n ? row : p.n - 1u);
                s.scale[r]         = reinterpret_cast<const uint16_t*>(p.scales)[at];
                s.zero[r]          = ZEROS ? p.zeros[at] : 0u;
            }
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                for(uint32_t i = 0; i < 4u; ++i)
                {
                    if constexpr(FAST)
                        s.x[c][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bufX, offX[c] + i * 64u, kb * 256u, 0));
                    else
                    {
                        const uint32_t k = kb * 128u + i * 32u + quad * 8u;
                        vec<T, 8>      v;
#pragma unroll
                        for(uint32_t e = 0; e < 8; ++e)
                            v[e] = c * 16u + col < left && k + e < p.k ? reinterpret_cast<const T*>(p.x)[(uint64_t)(token0 + c * 16u + col) * p.ldx + k + e] : T(0.0f);
                        s.x[c][i] = __builtin_bit_cast(u32x4, v);
                    }
                }
            return s;
        };
        // (in the last block of k a lane's pieces past k are those of the next token or of what lies between the rows)
        auto trim = [&](Stage& s, uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
            for(uint32_t i = 0; i < 4u; ++i)
                if(kb * 128u + i * 32u + quad * 8u >= p.k)
#pragma unroll
                    for(uint32_t c = 0; c < CB; ++c)
                        s.x[c][i] = u32x4{0u, 0u, 0u, 0u};
        };
        auto multiply = [&](const Stage& s) __attribute__((always_inline)) {
            uint32_t of[RB][PARTS]; // of each group: the scale and, in the upper half, the zero point
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
            {
                const uint32_t v = ZEROS ? s.scale[r] | (s.zero[r] << 16) : s.scale[r];
                if constexpr(PARTS == 1u)
                    of[r][0] = v;
                else if constexpr(PARTS == 2u)
                {
                    const auto pair = __builtin_amdgcn_permlane16_swap(v, v, false, false);
                    of[r][0] = pair[0], of[r][1] = pair[1];
                }
                else
                {
                    const auto half = __builtin_amdgcn_permlane32_swap(v, v, false, false);
                    const auto low = __builtin_amdgcn_permlane16_swap(half[0], half[0], false, false), high = __builtin_amdgcn_permlane16_swap(half[1], half[1], false, false);
                    of[r][0] = low[0], of[r][1] = low[1], of[r][2] = high[0], of[r][3] = high[1];
                }
            }
            each<PARTS>([&](auto partAt) __attribute__((always_inline)) {
                constexpr uint32_t part = decltype(partAt)::value;
                accumulate<T, RB, CB, STEPS, ZEROS, !ZEROS>(
                    acc, expand, [&](uint32_t c, uint32_t i) __attribute__((always_inline)) { return s.x[c][part * STEPS + i]; },
                    [&](uint32_t r, uint32_t i) __attribute__((always_inline)) { return s.w[r][part * STEPS + i]; },
                    [&](uint32_t r) __attribute__((always_inline)) { return Values{scaleOf<T>(of[r][part]), zeroOf(of[r][part] >> 16)}; });
            });
        };
        Stage stage[DEPTH]; // (a copy from one stage to the next would wait for its loads)
        each<DEPTH>([&](auto at) __attribute__((always_inline)) {
            constexpr uint32_t d = decltype(at)::value;
            if(wave + d * waves < p.blocksK)
                stage[d] = load(wave + d * waves);
        });
        for(uint32_t first = wave; first < p.blocksK; first += DEPTH * waves)
            each<DEPTH>([&](auto at) __attribute__((always_inline)) {
                constexpr uint32_t d  = decltype(at)::value;
                const uint32_t     kb = first + d * waves;
                if(kb < p.blocksK)
                {
                    if(FAST && kb + 1u == p.blocksK && p.k % 128u != 0u)
                        trim(stage[d], kb);
                    multiply(stage[d]);
                    if(kb + DEPTH * waves < p.blocksK)
                        stage[d] = load(kb + DEPTH * waves);
                }
            });

#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
            for(uint32_t j = 0; j < 4; ++j)
                if(c * 16u + quad * 4u + j < left)
#pragma unroll
                    for(uint32_t r = 0; r < RB; ++r)
                        sums[((wave * CB + c) * 16u + quad * 4u + j) * (16u * RB) + r * 16u + col] = acc[r][c][j];
        __syncthreads();
        storeTile<T, 16u * RB, 16u * CB, 16u * RB>(p, sums, waves, token0, block0 * 16u);
    }

    // ---- More tokens: 16 RB WN rows x 16 CB WT tokens a workgroup, 16 RB x 16 CB a wave; WK sets of such waves take the blocks of 128 k in turn.
    // Everything comes by direct loads into a ring of LDS buffers, as many steps ahead as fit: x in rows of 256 bytes (16-byte pieces in slots that depend on the
    // row: a wave reads 16 rows at one place), the weights as they are packed, a wave's scales and zero points one to a dword.  (Loads into registers among the
    // direct ones would have the compiler wait for all of them.)
    // Bound by the vector instructions that make operands, once per tile of tokens, and by LDS reads beside the matrix instructions: 8192 x 4096, groups of 64,
    // 1000 tokens, residual added: 85 us, 785 TFLOP/s (a product of the same size with weights made 16 bits beforehand, not counted: 57 us, 1180, in the vendor's
    // library and, 992 tokens, in this one's GEMM).
    __device__ __forceinline__ void loadShortToLds(r355::dma_i32x4 rsrc, uint32_t laneOffset, uint32_t ldsAddr)
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_ushort %0, %1, 0 offen lds" : : "v"(laneOffset), "s"(rsrc), "s"(ldsAddr) : "memory");
    }
    __device__ __forceinline__ void loadByteToLds(r355::dma_i32x4 rsrc, uint32_t laneOffset, uint32_t ldsAddr)
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_ubyte %0, %1, 0 offen lds" : : "v"(laneOffset), "s"(rsrc), "s"(ldsAddr) : "memory");
    }

    template <uint32_t RB, uint32_t CB, uint32_t WN, uint32_t WT, uint32_t WK, uint32_t STEPS, bool ZEROS>
    struct Ring
    {
        static constexpr uint32_t WAVES = WN * WT * WK, TOKENS = 16u * CB * WT, PARTS = 4u / STEPS;
        static constexpr uint32_t X = WK * TOKENS * 256u, W = WK * WN * RB * 1024u; // bytes of a step
        static constexpr uint32_t SCALES = (RB * PARTS + 3u) / 4u; // loads of 64 scales
        static constexpr uint32_t STAGE = X + W + WAVES * SCALES * 256u * (ZEROS ? 2u : 1u);
        static constexpr uint32_t LOADS_X = WK * TOKENS / 4u / WAVES, LOADS_W = W / 1024u / WAVES; // of a wave
        static constexpr uint32_t LOADS = LOADS_X + LOADS_W + SCALES * (ZEROS ? 2u : 1u);
        static constexpr uint32_t STRIDE = 16u * RB * WN + 4u, MERGE = WK * TOKENS * STRIDE * 4u; // of the sums, at the end
        static constexpr uint32_t FIT = 160u * 1024u / STAGE, BUFS = FIT > 4u ? 4u : FIT;
        static constexpr uint32_t LDS = BUFS * STAGE > MERGE ? BUFS * STAGE : MERGE;
        static_assert(LOADS_X * WAVES * 4u == WK * TOKENS && LOADS_W * WAVES * 1024u == W, "whole loads for every wave");
        static_assert(BUFS >= 2u && LOADS * (BUFS - 2u) < 64u && LDS <= 160u * 1024u, "LDS and counters");
    };

    template <typename T, uint32_t RB, uint32_t CB, uint32_t WN, uint32_t WT, uint32_t WK, uint32_t STEPS, bool ZEROS>
    __global__ void __launch_bounds__(64 * WN * WT * WK, 1) w4RingKernel(W4Params p)
    {
        using R                  = Ring<RB, CB, WN, WT, WK, STEPS, ZEROS>;
        constexpr uint32_t WAVES = R::WAVES, TOKENS = R::TOKENS, PARTS = R::PARTS, BUFS = R::BUFS;
        __shared__ __attribute__((aligned(1024))) char lds[R::LDS];
        uint32_t tileN, tileT;
        if(!tileOf(p, tileN, tileT))
            return;
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t col = lane & 15u, quad = lane >> 4, waveN = wave % WN, waveT = wave / WN % WT, waveK = wave / (WN * WT);
        const uint32_t group0 = tileN * WN * RB, block0 = group0 + waveN * RB, token0 = tileT * TOKENS, left = p.tokens - token0 < TOKENS ? p.tokens - token0 : TOKENS;
        const uint32_t ldsBase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
        constexpr uint32_t RECORDS = 0x7FFF0000u;

        // x: a load brings four rows of one block of k; past the tokens and past k: outside the buffer
        r355::dma_i32x4 bufX = r355::rawBuffer(reinterpret_cast<uint64_t>(p.x) + (uint64_t)token0 * p.ldx * 2u);
        bufX[2]              = __builtin_amdgcn_readfirstlane((left - 1u) * p.ldx * 2u + p.k * 2u);
        uint32_t offX[R::LOADS_X];
#pragma unroll
        for(uint32_t j = 0; j < R::LOADS_X; ++j)
        {
            const uint32_t row = (wave * R::LOADS_X + j) * 4u % TOKENS + quad;
            offX[j] = row < left ? row * p.ldx * 2u + (col ^ (row & 15u)) * 16u : OUTSIDE;
        }
        // scales: element (row block r, group of the block, row), 64 to a load
        uint32_t offS[R::SCALES], partS[R::SCALES];
#pragma unroll
        for(uint32_t j = 0; j < R::SCALES; ++j)
        {
            const uint32_t e = j * 64u + lane, r = e / (16u * PARTS), row = (block0 + r) * 16u + e % 16u;
            partS[j] = e / 16u % PARTS;
            offS[j]  = r < RB && row < p.n ? partS[j] * p.n + row : OUTSIDE / 2u;
        }
        auto issue = [&](uint32_t step, uint32_t buf) __attribute__((always_inline)) {
            const uint32_t to = ldsBase + buf * R::STAGE;
#pragma unroll
            for(uint32_t j = 0; j < R::LOADS_X; ++j)
            {
                const uint32_t at = wave * R::LOADS_X + j, kb = step * WK + at * 4u / TOKENS;
                const uint32_t k  = kb * 128u + (col ^ ((at * 4u % TOKENS + quad) & 15u)) * 8u;
                // (A lane's offset is held against the length of the buffer less the uniform one: that must not be more than the length, which with one token is 2 k
                // bytes, or the difference wraps around and OUTSIDE is inside.)
                r355::loadToLds(bufX, k < p.k ? offX[j] : OUTSIDE, __builtin_amdgcn_readfirstlane(kb < p.blocksK ? kb * 256u : 0u), __builtin_amdgcn_readfirstlane(to + at * 1024u));
            }
#pragma unroll
            for(uint32_t j = 0; j < R::LOADS_W; ++j)
            {
                const uint32_t at = wave * R::LOADS_W + j, kb = step * WK + at / (WN * RB), block = group0 + at % (WN * RB);
                r355::dma_i32x4 bufW = r355::rawBuffer(reinterpret_cast<uint64_t>(p.w) + ((uint64_t)block * p.blocksK + kb) * 1024u);
                bufW[2]              = __builtin_amdgcn_readfirstlane(block < p.blocksN && kb < p.blocksK ? 1024u : 0u);
                r355::loadToLds(bufW, lane * 16u, 0u, __builtin_amdgcn_readfirstlane(to + R::X + at * 1024u));
            }
            const uint32_t  g    = groupOf<STEPS>(p, step * WK + waveK);
            r355::dma_i32x4 bufS = r355::rawBuffer(reinterpret_cast<uint64_t>(p.scales) + (uint64_t)g * p.n * 2u);
            bufS[2]              = RECORDS;
#pragma unroll
            for(uint32_t j = 0; j < R::SCALES; ++j)
                loadShortToLds(bufS, (g + partS[j] < p.groups ? offS[j] : OUTSIDE / 2u) * 2u, __builtin_amdgcn_readfirstlane(to + R::X + R::W + (wave * R::SCALES + j) * 256u));
            if constexpr(ZEROS)
            {
                r355::dma_i32x4 bufZ = r355::rawBuffer(reinterpret_cast<uint64_t>(p.zeros) + (uint64_t)g * p.n);
                bufZ[2]              = RECORDS;
#pragma unroll
                for(uint32_t j = 0; j < R::SCALES; ++j)
                    loadByteToLds(bufZ, g + partS[j] < p.groups && offS[j] != OUTSIDE / 2u ? offS[j] : OUTSIDE,
                                  __builtin_amdgcn_readfirstlane(to + R::X + R::W + ((WAVES + wave) * R::SCALES + j) * 256u));
            }
        };

        const Expand<T> expand;
        f32x4           acc[RB][CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                acc[r][c] = f32x4{0, 0, 0, 0};

        using lds4 = const __attribute__((address_space(3))) u32x4*;
        using lds1 = const __attribute__((address_space(3))) uint32_t*;
        const uint32_t steps = (p.blocksK + WK - 1u) / WK;
        each<BUFS - 1u>([&](auto at) __attribute__((always_inline)) {
            if(decltype(at)::value < steps)
                issue(decltype(at)::value, decltype(at)::value);
        });
        uint32_t buf = 0u;
        for(uint32_t step = 0; step < steps; ++step)
        {
            const uint32_t after = steps - 1u - step; // steps whose loads may be outstanding
            if(BUFS == 4u && after >= 2u)
                r355::waitVmcnt<BUFS == 4u ? 2u * R::LOADS : 0u>();
            else if(BUFS >= 3u && after >= 1u)
                r355::waitVmcnt<BUFS >= 3u ? R::LOADS : 0u>();
            else
                r355::waitVmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            r355::ldsBarrier(); // everyone's part of this step is there, and everyone is done with the step before
            // The next loads, into the buffer of the step before: with groups of 128 behind the products (4096 x 4096, 512 tokens 77.4 -> 74.6 us), with smaller ones
            // before them, for want of registers.
            auto next = [&]() __attribute__((always_inline)) {
                if(step + BUFS - 1u < steps)
                    issue(step + BUFS - 1u, buf == 0u ? BUFS - 1u : buf - 1u);
            };
            if constexpr(PARTS > 1u)
                next();
            const uint32_t stage = ldsBase + buf * R::STAGE;
            const uint32_t fromX = stage + waveK * TOKENS * 256u + (waveT * CB * 16u + col) * 256u + (quad ^ col) * 16u;
            const uint32_t fromW = stage + R::X + ((waveK * WN + waveN) * RB * 64u + lane) * 16u;
            const uint32_t fromS = stage + R::X + R::W + wave * R::SCALES * 256u + col * 4u;
            each<PARTS>([&](auto partAt) __attribute__((always_inline)) {
                constexpr uint32_t part = decltype(partAt)::value;
                accumulate<T, RB, CB, STEPS, ZEROS, !ZEROS && (STEPS * CB <= 8u)>(
                    acc, expand,
                    [&](uint32_t c, uint32_t i) __attribute__((always_inline)) { return *(lds4)(uintptr_t)((fromX ^ ((part * STEPS + i) * 64u)) + c * 4096u); },
                    [&](uint32_t r, uint32_t i) __attribute__((always_inline)) { return *(lds1)(uintptr_t)(fromW + r * 1024u + (part * STEPS + i) * 4u); },
                    [&](uint32_t r) __attribute__((always_inline)) {
                        const uint32_t at = fromS + (r * PARTS + part) * 64u;
                        return Values{scaleOf<T>(*(lds1)(uintptr_t)at), ZEROS ? zeroOf(*(lds1)(uintptr_t)(at + WAVES * R::SCALES * 256u)) : 24.0f};
                    });
            });
            if constexpr(PARTS == 1u)
                next();
            buf = buf + 1u == BUFS ? 0u : buf + 1u;
        }
        __syncthreads();
        float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
            for(uint32_t j = 0; j < 4; ++j)
#pragma unroll
                for(uint32_t r = 0; r < RB; ++r)
                    sums[(waveK * TOKENS + (waveT * CB + c) * 16u + quad * 4u + j) * R::STRIDE + (waveN * RB + r) * 16u + col] = acc[r][c][j];
        __syncthreads();
        storeTile<T, 16u * RB * WN, TOKENS, R::STRIDE>(p, sums, WK, token0, group0 * 16u);
    }

    // one dword of the packed storage per thread: block of 16 rows, block of 128 k, lane, 32-k step
    __global__ void __launch_bounds__(256) w4PackKernel(const uint8_t* q, uint32_t n, uint32_t k, uint64_t ldq, uint32_t blocksK, uint32_t* packed)
    {
        const uint32_t i = threadIdx.x & 3u, lane = threadIdx.x >> 2;
        const uint32_t row = blockIdx.x * 16u + (lane & 15u);
        for(uint32_t kb = blockIdx.y; kb < blocksK; kb += gridDim.y)
        {
            const uint32_t k0 = kb * 128u + i * 32u + (lane >> 4) * 8u;
            uint32_t       d  = 0;
            if(row < n)
#pragma unroll
                for(uint32_t e = 0; e < 8; ++e)
                    if(k0 + e < k)
                    {
                        const uint32_t nibble = (q[row * ldq + (k0 + e) / 2u] >> (e % 2u * 4u)) & 15u;
                        d |= nibble << (4u * (e / 2u + e % 2u * 4u));
                    }
            packed[((uint64_t)blockIdx.x * blocksK + kb) * 256u + lane * 4u + i] = d;
        }
    }

    constexpr uint32_t MOST_ROWS = 1u << 24, MOST_TOKENS = 1u << 19, MOST_K = 1u << 22;
    constexpr uint64_t MOST_RESULTS = 1ull << 34;

    // most workgroups of a launch, a multiple of the XCDs (they have up to 512 threads, and the threads of a launch are counted in 32 bits)
    constexpr uint32_t MOST_GROUPS = r355::MAX_GROUPS / 16u * 8u;

    // Calls launch(parameters, workgroups) for tiles of rows x tokens, every XCD a stretch of them; several times, each with some of the tokens, where a
    // launch does not hold them all.
    template <typename F>
    void inLaunches(const W4Params& whole, uint32_t rows, uint32_t tokens, F&& launch)
    {
        const uint64_t outBytes = whole.outF32 ? 4u : 2u;
        W4Params       p        = whole;
        p.tilesN                = (p.n + rows - 1u) / rows;
        const uint32_t most     = MOST_GROUPS / p.tilesN * tokens; // (tilesN: 2^20 at most)
        for(uint32_t first = 0; first < whole.tokens; first += p.tokens)
        {
            p.tokens = whole.tokens - first < most ? whole.tokens - first : most;
            p.x      = whole.x + (uint64_t)first * p.ldx * 2u;
            p.y      = whole.y + (uint64_t)first * p.ldy * outBytes;
            p.c      = whole.c ? whole.c + (uint64_t)first * p.ldc * outBytes : nullptr;
            p.tilesT = (p.tokens + tokens - 1u) / tokens;
            p.perXcd = (p.tilesN * p.tilesT + 7u) / 8u;
            launch(p, dim3(p.perXcd * 8u));
        }
    }

    template <typename T, uint32_t RB, uint32_t CB, uint32_t DEPTH, uint32_t STEPS, bool FAST>
    void launchFew(const W4Params& whole, hipStream_t s)
    {
        const uint32_t waves = whole.blocksK >= 8u ? 8u : whole.blocksK >= 4u ? 4u : 1u;
        inLaunches(whole, 16u * RB, 16u * CB, [&](const W4Params& p, dim3 grid) {
            if(p.zeros)
                hipLaunchKernelGGL((w4Kernel<T, RB, CB, DEPTH, STEPS, true, FAST>), grid, dim3(waves * 64u), waves * RB * CB * 1024u, s, p);
            else
                hipLaunchKernelGGL((w4Kernel<T, RB, CB, DEPTH, STEPS, false, FAST>), grid, dim3(waves * 64u), waves * RB * CB * 1024u, s, p);
        });
    }

    template <typename T, uint32_t RB, uint32_t CB, uint32_t WN, uint32_t WT, uint32_t WK, uint32_t STEPS>
    void launchRing(const W4Params& whole, hipStream_t s)
    {
        inLaunches(whole, 16u * RB * WN, 16u * CB * WT, [&](const W4Params& p, dim3 grid) {
            if(p.zeros)
                hipLaunchKernelGGL((w4RingKernel<T, RB, CB, WN, WT, WK, STEPS, true>), grid, dim3(64u * WN * WT * WK), 0, s, p);
            else
                hipLaunchKernelGGL((w4RingKernel<T, RB, CB, WN, WT, WK, STEPS, false>), grid, dim3(64u * WN * WT * WK), 0, s, p);
        });
    }

    // The kernels that are launched, with what a workgroup of each takes for a block of 128 k while it has its CU to itself (hundredths of
    // a microsecond; groups of 128, of 64 and of 32; bf16, with and without zero points, 240 workgroups, from k = 4096 to 8192).
    struct Variant
    {
        uint32_t rows, tokens, time[3];
    };
    constexpr Variant VARIANTS[] = {
        {16, 16, {13, 13, 13}}, {32, 16, {15, 14, 15}}, {48, 16, {16, 17, 19}}, {64, 16, {18, 19, 23}}, // few tokens, one to four blocks of 16 rows
        {16, 32, {24, 25, 24}}, {32, 32, {26, 25, 26}}, {48, 32, {27, 27, 28}},
        {64, 32, {27, 29, 34}}, // (groups of 32: the ring, the others' registers spill)
        {128, 32, {49, 56, 63}}, {64, 64, {52, 57, 65}}, {128, 64, {78, 84, 106}}, // the ring
        {128, 128, {147, 161, 199}}, {256, 128, {251, 262, 319}}};

    // The least time of all, counting a round of workgroups over the CUs as long as one.  (24 tokens: 16384 x 8192, groups of 128: one to four blocks of rows
    // 55, 31, 34, 20 us; 10250 x 4168, groups of 32: 21, 20, 13, 16 us.)
    uint32_t variantOf(const W4Params& p)
    {
        const uint32_t by = p.group == 32u ? 2u : p.group == 64u ? 1u : 0u, cus = r355::computeUnits();
        uint32_t       best = 0u;
        uint64_t       least = ~0ull;
        for(uint32_t v = 0; v < sizeof(VARIANTS) / sizeof(VARIANTS[0]); ++v)
        {
            // up to four tokens x costs next to nothing, and two workgroups of up to three blocks share a CU well (16384 x 8192, one token: two blocks 14.3, four 15.2 us)
            if(p.tokens <= 4u && v > 2u)
                break;
            const uint64_t groups = (uint64_t)((p.n + VARIANTS[v].rows - 1u) / VARIANTS[v].rows) * ((p.tokens + VARIANTS[v].tokens - 1u) / VARIANTS[v].tokens);
            const uint64_t time   = ((groups + 7u) / 8u * 8u + cus - 1u) / cus * VARIANTS[v].time[by];
            if(time < least)
                least = time, best = v;
        }
        return best;
    }

    template <typename T, uint32_t STEPS>
    void launchSteps(const W4Params& p, bool fast, hipStream_t s)
    {
        if(!fast)
            return launchFew<T, 1, 2, 1, STEPS, false>(p, s);
        switch(variantOf(p))
        {
        case 0: return launchFew<T, 1, 1, 2, STEPS, true>(p, s);
        case 1: return launchFew<T, 2, 1, 1, STEPS, true>(p, s);
        case 2: return launchFew<T, 3, 1, 1, STEPS, true>(p, s);
        case 3: return launchFew<T, 4, 1, 1, STEPS, true>(p, s);
        case 4: return launchFew<T, 1, 2, 1, STEPS, true>(p, s);
        case 5: return launchFew<T, 2, 2, 1, STEPS, true>(p, s);
        case 6: return launchFew<T, 3, 2, 1, STEPS, true>(p, s);
        case 7:
            if constexpr(STEPS == 1u)
                return launchRing<T, 2, 2, 2, 1, 4, STEPS>(p, s);
            else
                return launchFew<T, 4, 2, 1, STEPS, true>(p, s);
        case 8: return launchRing<T, 2, 2, 4, 1, 2, STEPS>(p, s);
        case 9: return launchRing<T, 1, 4, 4, 1, 2, STEPS>(p, s);
        case 10: return launchRing<T, 2, 4, 4, 1, 2, STEPS>(p, s);
        case 11: return launchRing<T, 2, 4, 4, 2, 1, STEPS>(p, s);
        default: return launchRing<T, 4, 4, 4, 2, 1, STEPS>(p, s);
        }
    }

    template <typename T>
    void launchType(const W4Params& p, bool fast, hipStream_t s)
    {
        if(p.group == 32u)
            launchSteps<T, 1>(p, fast, s);
        else if(p.group == 64u)
            launchSteps<T, 2>(p, fast, s);
        else
            launchSteps<T, 4>(p, fast, s);
    }
} // namespace

extern "C" size_t r355_w4_packed_bytes(uint32_t n, uint32_t k)
{
    return ((size_t)n + 15u) / 16u * (((size_t)k + 127u) / 128u) * 1024u;
}

extern "C" int r355_w4_pack(const uint8_t* q, uint32_t n, uint32_t k, uint32_t ldq, void* packed, void* stream)
{
    if(!q || !packed)
        return r355::fail(R355_ERR_BAD_ARG, "w4_pack: null pointer");
    if(n == 0 || k == 0)
        return r355::fail(R355_ERR_BAD_ARG, "w4_pack: n and k must be non-zero");
    if(n > MOST_ROWS || k > MOST_K)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_pack: at most %u rows and %u columns, got %u and %u", MOST_ROWS, MOST_K, n, k);
    if(ldq < (k + 1u) / 2u)
        return r355::fail(R355_ERR_BAD_ARG, "w4_pack: ldq=%u is less than the %u bytes of a row", ldq, (k + 1u) / 2u);
    if(!r355::aligned(packed, 16))
        return r355::fail(R355_ERR_MISALIGNED, "w4_pack: the packed weights need 16-byte alignment");
    r355::beginCall();
    const uint32_t blocksK = (k + 127u) / 128u;
    hipLaunchKernelGGL(w4PackKernel, dim3((n + 15u) / 16u, blocksK < 65535u ? blocksK : 65535u), dim3(256), 0, static_cast<hipStream_t>(stream), q, n, k, ldq, blocksK,
                       static_cast<uint32_t*>(packed));
    return r355::checkLaunch("w4_pack");
}

extern "C" int r355_w4_matmul(const r355_w4_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "w4_matmul: null arguments");
    const r355_w4_args& a = *args;
    if(a.in_type != R355_F16 && a.in_type != R355_BF16)
        return r355::fail(R355_ERR_UNSUPPORTED, "w4_matmul: x is f16 or bf16");
    if(a.out_type != a.in_type && a.out_type != R355_F32)
        return r355::fail(R355_ERR_UNSUPPORTED, "w4_matmul: the result has the type of x or is f32");
    if(a.n == 0 || a.k == 0)
        return r355::fail(R355_ERR_BAD_ARG, "w4_matmul: n and k must be non-zero");
    if(a.n > MOST_ROWS || a.tokens > MOST_TOKENS || a.k > MOST_K)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: at most %u rows, %u tokens and %u columns, got %u, %u and %u", MOST_ROWS, MOST_TOKENS, MOST_K, a.n, a.tokens, a.k);
    if(a.group != 32u && a.group != 64u && (a.group == 0u || a.group % 128u))
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: group=%u must be 32, 64 or a multiple of 128", a.group);
    if((uint64_t)a.n * a.tokens >= MOST_RESULTS)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: n=%u times tokens=%u are 2^34 results and more", a.n, a.tokens);
    if(a.tokens == 0)
        return R355_OK;
    if(!a.x || !a.w || !a.scales || !a.y || (a.beta != 0.0 && !a.c))
        return r355::fail(R355_ERR_BAD_ARG, "w4_matmul: null pointer");
    if(a.ldx < a.k || a.ldy < a.n || (a.beta != 0.0 && a.ldc < a.n))
        return r355::fail(R355_ERR_BAD_ARG, "w4_matmul: a leading dimension is less than its row");
    const uint32_t outBytes = r355::dtypeBytes(a.out_type);
    if(!r355::aligned(a.w, 16))
        return r355::fail(R355_ERR_MISALIGNED, "w4_matmul: the packed weights need 16-byte alignment");
    if(!r355::aligned(a.x, 2) || !r355::aligned(a.scales, 2) || !r355::aligned(a.y, outBytes) || (a.beta != 0.0 && !r355::aligned(a.c, outBytes)))
        return r355::fail(R355_ERR_MISALIGNED, "w4_matmul: x, scales, c and y need the alignment of their elements");
    W4Params p;
    p.x = static_cast<const char*>(a.x), p.w = static_cast<const char*>(a.w), p.scales = static_cast<const char*>(a.scales), p.zeros = a.zeros;
    p.c = static_cast<const char*>(a.c), p.y = static_cast<char*>(a.y);
    p.tokens = a.tokens, p.n = a.n, p.k = a.k, p.group = a.group, p.groups = static_cast<uint32_t>(((uint64_t)a.k + a.group - 1u) / a.group), p.ldx = a.ldx, p.ldc = a.ldc, p.ldy = a.ldy;
    p.blocksN = (a.n + 15u) / 16u, p.blocksK = (a.k + 127u) / 128u;
    p.perGroup = a.group / 128u < p.blocksK ? a.group / 128u : p.blocksK; // (a group longer than k)
    p.groupMagic = p.perGroup > 1u ? static_cast<uint32_t>(((1ull << 32) + p.perGroup - 1u) / p.perGroup) : 0u;
    p.outF32 = a.out_type == R355_F32;
    p.wideN  = a.ldy % 4u == 0u && r355::aligned(a.y, 4u * outBytes) && (a.beta == 0.0 || (a.ldc % 4u == 0u && r355::aligned(a.c, 4u * outBytes)));
    p.alpha = static_cast<float>(a.alpha), p.beta = static_cast<float>(a.beta);
    // (the rows of x that a workgroup takes, 128 at most, lie within 2^31 bytes)
    const bool        fast = a.k % 8u == 0u && a.ldx % 8u == 0u && r355::aligned(a.x, 16) && a.ldx <= (1u << 22);
    const hipStream_t s    = static_cast<hipStream_t>(stream);
    r355::beginCall();
    if(a.in_type == R355_F16)
        launchType<_Float16>(p, fast, s);
    else
        launchType<__bf16>(p, fast, s);
    return r355::checkLaunch("w4_matmul");
}
