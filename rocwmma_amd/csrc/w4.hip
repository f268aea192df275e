// Products with 4-bit weights and group scales on gfx950 matrix cores.
//
//   y[t][r] = alpha * sum_k x[t][k] (q[r][k] - z[k / g][r]) s[k / g][r] + beta c[t][r]
//
// No counterpart in the reference.  The weights q are stored in blocks of 16 rows x 128 k (r355_w4_pack), 1 KiB each in the order in
// which a wave's lanes load them, 16 bytes a lane: the four dwords of a lane are its A operands of four v_mfma_f32_16x16x32, x is the B
// operand, and up to 16 tokens cost what one costs.
//
// A nibble becomes an operand without a conversion: with the nibble in the four leading bits of the mantissa of 16.0 the 16-bit number
// is 16 + q, so a shift and an and-or make two operands.  The matrix instruction sums x (16 + q) over a group exactly as it would sum x q,
// one more instruction with ones for A leaves sum x in the same lanes, and
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
        uint32_t       tilesN, tilesT, perXcd; // workgroups along n and tokens; tiles of n for each XCD
        uint32_t       outF32, wideN; // wideN: 4-element accesses of c and y
        float          alpha, beta;
    };

    // two weights of a dword (nibbles p and p + 4) as 16 + q each
    template <typename T>
    __device__ __forceinline__ u32x4 expand(uint32_t d)
    {
        if constexpr(std::is_same_v<T, __bf16>)
            return u32x4{((d << 3) & 0x00780078u) | 0x41804180u, ((d >> 1) & 0x00780078u) | 0x41804180u, ((d >> 5) & 0x00780078u) | 0x41804180u,
                         ((d >> 9) & 0x00780078u) | 0x41804180u};
        else
            return u32x4{((d << 6) & 0x03C003C0u) | 0x4C004C00u, ((d << 2) & 0x03C003C0u) | 0x4C004C00u, ((d >> 2) & 0x03C003C0u) | 0x4C004C00u,
                         ((d >> 6) & 0x03C003C0u) | 0x4C004C00u};
    }

    template <typename T>
    constexpr uint32_t ONES = std::is_same_v<T, __bf16> ? 0x3F803F80u : 0x3C003C00u;

    template <typename T>
    __device__ __forceinline__ f32x4 floats(u32x2 v)
    {
        const vec<T, 4> t = __builtin_bit_cast(vec<T, 4>, v);
        return f32x4{static_cast<float>(t[0]), static_cast<float>(t[1]), static_cast<float>(t[2]), static_cast<float>(t[3])};
    }
    // 16 + z of four zero points
    __device__ __forceinline__ f32x4 offsets(uint32_t v)
    {
        return f32x4{16.0f + static_cast<float>(v & 255u), 16.0f + static_cast<float>((v >> 8) & 255u), 16.0f + static_cast<float>((v >> 16) & 255u), 16.0f + static_cast<float>(v >> 24)};
    }

    struct __attribute__((packed, aligned(2))) Four16
    {
        u32x2 v;
    };
    struct __attribute__((packed, aligned(1))) Four8
    {
        uint32_t v;
    };

    // The scales (zero points) of four rows of a group.  At the end of a row of them the last four are read and moved down.
    struct RowsOf4
    {
        uint32_t at, past; // the first row read, and by how much the rows wanted lie behind it
        __device__ __forceinline__ RowsOf4(uint32_t row, uint32_t n)
        {
            at   = row + 4u <= n ? row : n - 4u;
            past = row - at < 3u ? row - at : 3u;
        }
        __device__ __forceinline__ u32x2 scales(const W4Params& p, uint32_t g) const
        {
            return reinterpret_cast<const Four16*>(p.scales + 2u * ((uint64_t)g * p.n + at))->v;
        }
        __device__ __forceinline__ uint32_t zeros(const W4Params& p, uint32_t g) const
        {
            return reinterpret_cast<const Four8*>(p.zeros + (uint64_t)g * p.n + at)->v;
        }
        __device__ __forceinline__ u32x2 moved(u32x2 v) const
        {
            return __builtin_bit_cast(u32x2, __builtin_bit_cast(uint64_t, v) >> (16u * past));
        }
        __device__ __forceinline__ uint32_t moved(uint32_t v) const
        {
            return v >> (8u * past);
        }
    };

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

    // Tile of n and tile of tokens of a workgroup: workgroups id, id + 8, ... run on one XCD and take a contiguous stretch of n (the scales of
    // neighbouring rows share cache lines), all tiles of tokens of one tile of n after another.
    __device__ __forceinline__ bool tileOf(const W4Params& p, uint32_t& tileN, uint32_t& tileT)
    {
        const uint32_t id = blockIdx.x / 8u;
        tileN = blockIdx.x % 8u * p.perXcd + id / p.tilesT, tileT = id % p.tilesT;
        return id / p.tilesT < p.perXcd && tileN < p.tilesN;
    }

    // ---- few tokens.  A workgroup's waves share 16 RB rows x 16 CB tokens and take the 128-k blocks in turn; their sums meet in LDS in the order
    // of the waves, so the result does not depend on scheduling.  STEPS: matrix instructions (32 k) per scale.  FAST: rows of x on 16-byte
    // boundaries; everything that a block of k needs is requested, without branches, while the one before it is multiplied.
    template <typename T, uint32_t RB, uint32_t CB, uint32_t STEPS, bool ZEROS, bool FAST>
    __global__ void __launch_bounds__(512) w4Kernel(W4Params p)
    {
        extern __shared__ __attribute__((aligned(16))) float sums[]; // [waves][RB * CB][64][4]
        constexpr uint32_t PARTS = 4u / STEPS;
        uint32_t           tileN, tileT;
        if(!tileOf(p, tileN, tileT))
            return;
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
        const uint32_t col = lane & 15u, quad = lane >> 4;
        const uint32_t block0 = tileN * RB, token0 = tileT * 16u * CB;
        const u32x4    ones{ONES<T>, ONES<T>, ONES<T>, ONES<T>};
        const f32x4    none{0, 0, 0, 0};
        f32x4          acc[RB][CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                acc[r][c] = none;

        struct Stage
        {
            u32x4    w[RB], x[CB][4];
            u32x2    scale[RB][PARTS];
            uint32_t zero[RB][PARTS];
        };
        const uint32_t left = p.tokens - token0;
        // (a buffer over the rows of x from token0 on, which ends with the last element; lanes without a token lie past it)
        constexpr uint32_t OUTSIDE = 0x7FFFFFF0u;
        const auto bufX = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.x) + (uint64_t)token0 * p.ldx * 2u, 0,
                                                            FAST ? ((left < 16u * CB ? left : 16u * CB) - 1u) * p.ldx * 2u + p.k * 2u : 0u, 0x00020000);
        auto load = [&](uint32_t kb) __attribute__((always_inline)) {
            Stage s;
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
            {
                const uint32_t b = block0 + r < p.blocksN ? block0 + r : p.blocksN - 1u;
                s.w[r]           = *reinterpret_cast<const u32x4*>(p.w + ((uint64_t)b * p.blocksK + kb) * 1024u + lane * 16u);
            }
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                for(uint32_t i = 0; i < 4u; ++i)
                {
                    const uint32_t k = kb * 128u + i * 32u + quad * 8u;
                    if constexpr(FAST)
                        s.x[c][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bufX, c * 16u + col < left && k < p.k ? (c * 16u + col) * p.ldx * 2u + k * 2u : OUTSIDE, 0, 0));
                    else
                    {
                        vec<T, 8> v;
#pragma unroll
                        for(uint32_t e = 0; e < 8; ++e)
                            v[e] = c * 16u + col < left && k + e < p.k ? reinterpret_cast<const T*>(p.x)[(uint64_t)(token0 + c * 16u + col) * p.ldx + k + e] : T(0.0f);
                        s.x[c][i] = __builtin_bit_cast(u32x4, v);
                    }
                }
#pragma unroll
            for(uint32_t part = 0; part < PARTS; ++part)
            {
                const uint32_t of = (kb * 128u + part * STEPS * 32u) / p.group, g = of < p.groups ? of : p.groups - 1u;
#pragma unroll
                for(uint32_t r = 0; r < RB; ++r)
                {
                    const uint32_t row = (block0 + r) * 16u + quad * 4u;
                    if constexpr(FAST)
                    {
                        const RowsOf4 rows(row, p.n);
                        s.scale[r][part] = rows.scales(p, g);
                        s.zero[r][part]  = ZEROS ? rows.zeros(p, g) : 0u;
                    }
                    else
                    {
                        s.scale[r][part] = u32x2{0u, 0u}, s.zero[r][part] = 0u;
#pragma unroll
                        for(uint32_t e = 0; e < 4; ++e)
                            if(row + e < p.n)
                            {
                                s.scale[r][part][e / 2u] |= (uint32_t)reinterpret_cast<const uint16_t*>(p.scales)[(uint64_t)g * p.n + row + e] << (e % 2u * 16u);
                                if(ZEROS)
                                    s.zero[r][part] |= (uint32_t)p.zeros[(uint64_t)g * p.n + row + e] << (e * 8u);
                            }
                    }
                }
            }
            return s;
        };
        auto multiply = [&](const Stage& s) __attribute__((always_inline)) {
#pragma unroll
            for(uint32_t part = 0; part < PARTS; ++part)
            {
                f32x4 sum[RB][CB], sumX[CB];
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
#pragma unroll
                    for(uint32_t c = 0; c < CB; ++c)
                        sumX[c] = r355::mfma32<T>(ones, s.x[c][part * STEPS + i], i == 0u ? none : sumX[c]);
#pragma unroll
                    for(uint32_t r = 0; r < RB; ++r)
                    {
                        const u32x4 a = expand<T>(s.w[r][part * STEPS + i]);
#pragma unroll
                        for(uint32_t c = 0; c < CB; ++c)
                            sum[r][c] = r355::mfma32<T>(a, s.x[c][part * STEPS + i], i == 0u ? none : sum[r][c]);
                    }
                }
#pragma unroll
                for(uint32_t r = 0; r < RB; ++r)
                {
                    const RowsOf4 rows((block0 + r) * 16u + quad * 4u, p.n);
                    const f32x4   scale = floats<T>(FAST ? rows.moved(s.scale[r][part]) : s.scale[r][part]);
                    f32x4         zero{24.0f, 24.0f, 24.0f, 24.0f};
                    if constexpr(ZEROS)
                        zero = offsets(FAST ? rows.moved(s.zero[r][part]) : s.zero[r][part]);
#pragma unroll
                    for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                        for(uint32_t j = 0; j < 4; ++j)
                            acc[r][c][j] = fmaf(scale[j], fmaf(-zero[j], sumX[c][j], sum[r][c][j]), acc[r][c][j]);
                }
            }
        };
        if(wave < p.blocksK)
        {
            Stage now = load(wave);
            for(uint32_t kb = wave;;)
            {
                const uint32_t next = kb + waves;
                if(next >= p.blocksK)
                {
                    multiply(now);
                    break;
                }
                const Stage then = load(next);
                __builtin_amdgcn_sched_barrier(0);
                multiply(now);
                __builtin_amdgcn_sched_barrier(0);
                now = then, kb = next;
            }
        }

#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                *reinterpret_cast<f32x4*>(sums + ((wave * RB * CB + r * CB + c) * 64u + lane) * 4u) = acc[r][c];
        __syncthreads();
        for(uint32_t u = wave; u < RB * CB; u += waves)
        {
            f32x4 sum = none;
            for(uint32_t v = 0; v < waves; ++v)
                sum += *reinterpret_cast<const f32x4*>(sums + ((v * RB * CB + u) * 64u + lane) * 4u);
            store<T>(p, token0 + u % CB * 16u + col, (block0 + u / CB) * 16u + quad * 4u, sum);
        }
    }

    // ---- many tokens: 128 rows x 128 tokens a workgroup, 64 x 64 a wave.  x goes to LDS by direct loads a block of 128 k ahead (16-byte pieces of a
    // row in slots that depend on the row: a wave reads 16 rows at one place), the weights of a wave's own rows straight to its registers.
    // Bound by the vector ALU: of 64 k (group 64) a wave's 40 matrix instructions take 640 cycles, two operands for each of its 4096 weights 290
    // and scaling its 4096 sums 510.
    template <typename T, uint32_t STEPS, bool ZEROS>
    __global__ void __launch_bounds__(256, 2) w4TileKernel(W4Params p)
    {
        constexpr uint32_t PARTS = 4u / STEPS, TILE = 128u * 256u, LOADS = 8, OUTSIDE = 0x7FFFFFF0u;
        __shared__ __attribute__((aligned(1024))) char lds[2u * TILE];
        uint32_t tileN, tileT;
        if(!tileOf(p, tileN, tileT))
            return;
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t col = lane & 15u, quad = lane >> 4, waveN = wave & 1u, waveT = wave >> 1;
        const uint32_t block0 = tileN * 8u + waveN * 4u, token0 = tileT * 128u, left = p.tokens - token0 < 128u ? p.tokens - token0 : 128u;
        const uint32_t ldsBase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));

        // rows 4 j + lane / 16 of the wave's 32 tokens; past the tokens and past k: outside the buffer, which loads zeros
        r355::dma_i32x4 bufX = r355::rawBuffer(reinterpret_cast<uint64_t>(p.x) + (uint64_t)token0 * p.ldx * 2u);
        bufX[2]              = __builtin_amdgcn_readfirstlane((left - 1u) * p.ldx * 2u + p.k * 2u);
        uint32_t offX[LOADS], pieceK[LOADS];
#pragma unroll
        for(uint32_t j = 0; j < LOADS; ++j)
        {
            const uint32_t row = wave * 32u + j * 4u + (lane >> 4), piece = col ^ (row & 15u);
            offX[j] = row < left ? row * p.ldx * 2u + piece * 16u : OUTSIDE, pieceK[j] = piece * 8u;
        }
        auto issue = [&](uint32_t kb, uint32_t buf) __attribute__((always_inline)) {
            const uint32_t to = __builtin_amdgcn_readfirstlane(ldsBase + buf * TILE + wave * 8192u);
#pragma unroll
            for(uint32_t j = 0; j < LOADS; ++j)
                r355::loadToLds(bufX, kb * 128u + pieceK[j] < p.k ? offX[j] : OUTSIDE, kb * 256u, to + j * 1024u);
        };

        struct Stage
        {
            u32x4    w[4];
            u32x2    scale[4][PARTS];
            uint32_t zero[4][PARTS];
        };
        auto load = [&](uint32_t kb) __attribute__((always_inline)) {
            Stage s;
#pragma unroll
            for(uint32_t r = 0; r < 4u; ++r)
            {
                const uint32_t b = block0 + r < p.blocksN ? block0 + r : p.blocksN - 1u;
                s.w[r]           = *reinterpret_cast<const u32x4*>(p.w + ((uint64_t)b * p.blocksK + kb) * 1024u + lane * 16u);
                const RowsOf4 rows((block0 + r) * 16u + quad * 4u, p.n);
#pragma unroll
                for(uint32_t part = 0; part < PARTS; ++part)
                {
                    const uint32_t of = (kb * 128u + part * STEPS * 32u) / p.group, g = of < p.groups ? of : p.groups - 1u;
                    s.scale[r][part] = rows.scales(p, g);
                    s.zero[r][part]  = ZEROS ? rows.zeros(p, g) : 0u;
                }
            }
            return s;
        };
        const u32x4 ones{ONES<T>, ONES<T>, ONES<T>, ONES<T>};
        const f32x4 none{0, 0, 0, 0};
        f32x4       acc[4][4];
#pragma unroll
        for(uint32_t r = 0; r < 4; ++r)
#pragma unroll
            for(uint32_t c = 0; c < 4; ++c)
                acc[r][c] = none;

        issue(0u, 0u);
        Stage now = load(0u);
        for(uint32_t kb = 0; kb < p.blocksK; ++kb)
        {
            r355::waitVmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            r355::ldsBarrier(); // everyone's part of block kb is there, and everyone is done with the other buffer
            Stage then = now;
            if(kb + 1u < p.blocksK)
            {
                issue(kb + 1u, (kb + 1u) & 1u);
                then = load(kb + 1u);
            }
            const uint32_t from = ldsBase + (kb & 1u) * TILE + (waveT * 64u + col) * 256u + (quad ^ col) * 16u;
#pragma unroll
            for(uint32_t part = 0; part < PARTS; ++part)
            {
                f32x4 sum[4][4], sumX[4];
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
                    u32x4 x[4];
#pragma unroll
                    for(uint32_t c = 0; c < 4; ++c)
                    {
                        x[c]    = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)((from ^ ((part * STEPS + i) * 64u)) + c * 4096u);
                        sumX[c] = r355::mfma32<T>(ones, x[c], i == 0u ? none : sumX[c]);
                    }
#pragma unroll
                    for(uint32_t r = 0; r < 4; ++r)
                    {
                        const u32x4 a = expand<T>(now.w[r][part * STEPS + i]);
#pragma unroll
                        for(uint32_t c = 0; c < 4; ++c)
                            sum[r][c] = r355::mfma32<T>(a, x[c], i == 0u ? none : sum[r][c]);
                    }
                }
#pragma unroll
                for(uint32_t r = 0; r < 4; ++r)
                {
                    const RowsOf4 rows((block0 + r) * 16u + quad * 4u, p.n);
                    const f32x4   scale = floats<T>(rows.moved(now.scale[r][part]));
                    f32x4         zero{24.0f, 24.0f, 24.0f, 24.0f};
                    if constexpr(ZEROS)
                        zero = offsets(rows.moved(now.zero[r][part]));
#pragma unroll
                    for(uint32_t c = 0; c < 4; ++c)
#pragma unroll
                        for(uint32_t j = 0; j < 4; ++j)
                            acc[r][c][j] = fmaf(scale[j], fmaf(-zero[j], sumX[c][j], sum[r][c][j]), acc[r][c][j]);
                }
            }
            now = then;
        }
#pragma unroll
        for(uint32_t r = 0; r < 4; ++r)
#pragma unroll
            for(uint32_t c = 0; c < 4; ++c)
                store<T>(p, token0 + waveT * 64u + c * 16u + col, (block0 + r) * 16u + quad * 4u, acc[r][c]);
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

    constexpr uint32_t MOST_ROWS = 1u << 24, MOST_TOKENS = 1u << 19;

    // workgroups: a multiple of eight, every XCD a stretch of the tiles of n
    dim3 gridOf(W4Params& p, uint32_t rows, uint32_t tokens)
    {
        p.tilesN = (p.n + rows - 1u) / rows, p.tilesT = (p.tokens + tokens - 1u) / tokens;
        p.perXcd = (p.tilesN + 7u) / 8u;
        return dim3(p.perXcd * 8u * p.tilesT);
    }

    template <typename T, uint32_t RB, uint32_t CB, uint32_t STEPS, bool FAST>
    void launchFew(W4Params& p, uint32_t waves, hipStream_t s)
    {
        const dim3 grid = gridOf(p, 16u * RB, 16u * CB);
        if(p.zeros)
            hipLaunchKernelGGL((w4Kernel<T, RB, CB, STEPS, true, FAST>), grid, dim3(waves * 64u), waves * RB * CB * 1024u, s, p);
        else
            hipLaunchKernelGGL((w4Kernel<T, RB, CB, STEPS, false, FAST>), grid, dim3(waves * 64u), waves * RB * CB * 1024u, s, p);
    }

    template <typename T, uint32_t STEPS>
    void launchSteps(W4Params& p, bool fast, hipStream_t s)
    {
        const uint32_t waves = p.blocksK >= 8u ? 8u : p.blocksK >= 4u ? 4u : 1u;
        if(!fast)
            launchFew<T, 1, 2, STEPS, false>(p, waves, s);
        else if(p.tokens <= 16u)
            launchFew<T, 1, 1, STEPS, true>(p, waves, s);
        else if(p.tokens <= 32u)
            launchFew<T, 1, 2, STEPS, true>(p, waves, s);
        else if(p.tokens <= 64u)
            launchFew<T, 1, 4, STEPS, true>(p, waves, s);
        else
        {
            const dim3 grid = gridOf(p, 128u, 128u);
            if(p.zeros)
                hipLaunchKernelGGL((w4TileKernel<T, STEPS, true>), grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((w4TileKernel<T, STEPS, false>), grid, dim3(256), 0, s, p);
        }
    }

    template <typename T>
    void launchType(W4Params& p, bool fast, hipStream_t s)
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
    if(n > MOST_ROWS || k > 0xFFFFFF00u)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_pack: at most %u rows and 0xFFFFFF00 columns, got %u and %u", MOST_ROWS, n, k);
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
    if(a.n > MOST_ROWS || a.tokens > MOST_TOKENS || a.k > 0xFFFFFF00u)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: at most %u rows, %u tokens and 0xFFFFFF00 columns, got %u, %u and %u", MOST_ROWS, MOST_TOKENS, a.n, a.tokens, a.k);
    if(a.group != 32u && a.group != 64u && (a.group == 0u || a.group % 128u))
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: group=%u must be 32, 64 or a multiple of 128", a.group);
    if(((uint64_t)a.n + 15u) / 16u * (((uint64_t)a.tokens + 15u) / 16u) > r355::MAX_GROUPS / 4u)
        return r355::fail(R355_ERR_BAD_SIZE, "w4_matmul: too many blocks of 16 rows x 16 tokens for one launch");
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
    p.tokens = a.tokens, p.n = a.n, p.k = a.k, p.group = a.group, p.groups = (a.k + a.group - 1u) / a.group, p.ldx = a.ldx, p.ldc = a.ldc, p.ldy = a.ldy;
    p.blocksN = (a.n + 15u) / 16u, p.blocksK = (a.k + 127u) / 128u;
    p.outF32 = a.out_type == R355_F32;
    p.wideN  = a.ldy % 4u == 0u && r355::aligned(a.y, 4u * outBytes) && (a.beta == 0.0 || (a.ldc % 4u == 0u && r355::aligned(a.c, 4u * outBytes)));
    p.alpha = static_cast<float>(a.alpha), p.beta = static_cast<float>(a.beta);
    // (the rows of x that a workgroup takes, 128 at most, lie within 2^31 bytes)
    const bool        fast = a.k % 8u == 0u && a.ldx % 8u == 0u && r355::aligned(a.x, 16) && a.n >= 4u && a.ldx <= (1u << 22);
    const hipStream_t s    = static_cast<hipStream_t>(stream);
    r355::beginCall();
    if(a.in_type == R355_F16)
        launchType<_Float16>(p, fast, s);
    else
        launchType<__bf16>(p, fast, s);
    return r355::checkLaunch("w4_matmul");
}
