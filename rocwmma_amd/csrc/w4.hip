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

namespace
{
    using r355::f32x4;
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
        uint32_t       tokens, n, k, group;
        uint32_t       ldx, ldc, ldy;
        uint32_t       blocksN, blocksK; // of 16 rows, of 128 k
        uint32_t       wideX, wideN; // 16-byte loads of x; 4-element accesses along n (scales, zero points, c, y)
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

    // 8 elements of x from k on, of a token; zeros past the tokens and past k
    template <typename T>
    __device__ __forceinline__ u32x4 loadX(const W4Params& p, uint32_t token, uint32_t k)
    {
        if(token >= p.tokens || k >= p.k)
            return u32x4{0u, 0u, 0u, 0u};
        const T* at = reinterpret_cast<const T*>(p.x) + (uint64_t)token * p.ldx + k;
        if(p.wideX)
            return *reinterpret_cast<const u32x4*>(at);
        vec<T, 8> v;
#pragma unroll
        for(uint32_t e = 0; e < 8; ++e)
            v[e] = k + e < p.k ? at[e] : T(0.0f);
        return __builtin_bit_cast(u32x4, v);
    }

    // four consecutive values along n, those past n as zero
    template <typename E>
    __device__ __forceinline__ vec<float, 4> load4(const E* at, uint32_t row, uint32_t n, bool wide)
    {
        if(row >= n)
            return vec<float, 4>{0, 0, 0, 0};
        if(wide)
        {
            const vec<E, 4> v = *reinterpret_cast<const vec<E, 4>*>(at + row);
            return vec<float, 4>{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]), static_cast<float>(v[3])};
        }
        vec<float, 4> v;
#pragma unroll
        for(uint32_t e = 0; e < 4; ++e)
            v[e] = row + e < n ? static_cast<float>(at[row + e]) : 0.0f;
        return v;
    }

    // A workgroup's waves share 16 RB rows x 16 CB tokens and take the 128-k blocks in turn; their sums meet in LDS in the order of the
    // waves, so the result does not depend on scheduling.  STEPS: matrix instructions (32 k) per scale.
    template <typename T, typename O, uint32_t RB, uint32_t CB, uint32_t STEPS>
    __global__ void __launch_bounds__(1024) w4Kernel(W4Params p)
    {
        extern __shared__ __attribute__((aligned(16))) float sums[]; // [waves][RB * CB][64][4]
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
        const uint32_t col = lane & 15u, quad = lane >> 4;
        const uint32_t block0 = blockIdx.x * RB, token0 = blockIdx.y * 16u * CB;
        constexpr uint32_t ONE = std::is_same_v<T, __bf16> ? 0x3F803F80u : 0x3C003C00u;
        const u32x4        ones{ONE, ONE, ONE, ONE};
        const f32x4        none{0, 0, 0, 0};
        f32x4              acc[RB][CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                acc[r][c] = none;

        for(uint32_t kb = wave; kb < p.blocksK; kb += waves)
        {
            u32x4 w[RB];
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
            {
                const uint32_t b = block0 + r < p.blocksN ? block0 + r : p.blocksN - 1u;
                w[r]             = *reinterpret_cast<const u32x4*>(p.w + (((uint64_t)b * p.blocksK + kb) * 64u + lane) * 16u);
            }
#pragma unroll
            for(uint32_t part = 0; part < 4u / STEPS; ++part)
            {
                const uint32_t k0 = kb * 128u + part * STEPS * 32u;
                if(k0 >= p.k)
                    break;
                f32x4 sum[RB][CB], sumX[CB];
#pragma unroll
                for(uint32_t c = 0; c < CB; ++c)
                {
                    sumX[c] = none;
#pragma unroll
                    for(uint32_t r = 0; r < RB; ++r)
                        sum[r][c] = none;
                }
#pragma unroll
                for(uint32_t s = 0; s < STEPS; ++s)
                {
                    u32x4 x[CB];
#pragma unroll
                    for(uint32_t c = 0; c < CB; ++c)
                    {
                        x[c]    = loadX<T>(p, token0 + c * 16u + col, k0 + s * 32u + quad * 8u);
                        sumX[c] = r355::mfma32<T>(ones, x[c], sumX[c]);
                    }
#pragma unroll
                    for(uint32_t r = 0; r < RB; ++r)
                    {
                        const u32x4 a = expand<T>(w[r][part * STEPS + s]);
#pragma unroll
                        for(uint32_t c = 0; c < CB; ++c)
                            sum[r][c] = r355::mfma32<T>(a, x[c], sum[r][c]);
                    }
                }
                const uint32_t g = k0 / p.group;
#pragma unroll
                for(uint32_t r = 0; r < RB; ++r)
                {
                    const uint32_t row   = (block0 + r) * 16u + quad * 4u;
                    const auto     scale = load4(reinterpret_cast<const T*>(p.scales) + (uint64_t)g * p.n, row, p.n, p.wideN);
                    auto           zero  = vec<float, 4>{8, 8, 8, 8};
                    if(p.zeros)
                        zero = load4(p.zeros + (uint64_t)g * p.n, row, p.n, p.wideN);
#pragma unroll
                    for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
                        for(uint32_t j = 0; j < 4; ++j)
                            acc[r][c][j] += scale[j] * (sum[r][c][j] - (16.0f + zero[j]) * sumX[c][j]);
                }
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
            const uint32_t r = u / CB, c = u % CB;
            f32x4          sum = none;
            for(uint32_t v = 0; v < waves; ++v)
                sum += *reinterpret_cast<const f32x4*>(sums + ((v * RB * CB + u) * 64u + lane) * 4u);
            const uint32_t token = token0 + c * 16u + col, row = (block0 + r) * 16u + quad * 4u;
            if(token >= p.tokens || row >= p.n)
                continue;
            vec<float, 4> out{p.alpha * sum[0], p.alpha * sum[1], p.alpha * sum[2], p.alpha * sum[3]};
            if(p.beta != 0.0f)
                out += p.beta * load4(reinterpret_cast<const O*>(p.c) + (uint64_t)token * p.ldc, row, p.n, p.wideN);
            O* to = reinterpret_cast<O*>(p.y) + (uint64_t)token * p.ldy + row;
            if(p.wideN)
                *reinterpret_cast<vec<O, 4>*>(to) = vec<O, 4>{static_cast<O>(out[0]), static_cast<O>(out[1]), static_cast<O>(out[2]), static_cast<O>(out[3])};
            else
                for(uint32_t e = 0; e < 4u && row + e < p.n; ++e)
                    to[e] = static_cast<O>(out[e]);
        }
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

    template <typename T, typename O, uint32_t RB, uint32_t CB, uint32_t STEPS>
    void launch(const W4Params& p, uint32_t waves, hipStream_t s)
    {
        const dim3 grid((p.blocksN + RB - 1u) / RB, (p.tokens + 16u * CB - 1u) / (16u * CB));
        hipLaunchKernelGGL((w4Kernel<T, O, RB, CB, STEPS>), grid, dim3(waves * 64u), waves * RB * CB * 1024u, s, p);
    }

    template <typename T, typename O, uint32_t RB, uint32_t CB>
    void launchSteps(const W4Params& p, uint32_t waves, hipStream_t s)
    {
        if(p.group == 32u)
            launch<T, O, RB, CB, 1>(p, waves, s);
        else if(p.group == 64u)
            launch<T, O, RB, CB, 2>(p, waves, s);
        else
            launch<T, O, RB, CB, 4>(p, waves, s);
    }

    template <typename T, typename O>
    void launchShape(const W4Params& p, hipStream_t s)
    {
        const uint32_t waves = p.blocksK >= 8u ? 8u : p.blocksK >= 4u ? 4u : 1u;
        if(p.tokens <= 16u)
            launchSteps<T, O, 1, 1>(p, waves, s);
        else
            launchSteps<T, O, 2, 4>(p, waves > 4u ? 4u : waves, s);
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
    p.tokens = a.tokens, p.n = a.n, p.k = a.k, p.group = a.group, p.ldx = a.ldx, p.ldc = a.ldc, p.ldy = a.ldy;
    p.blocksN = (a.n + 15u) / 16u, p.blocksK = (a.k + 127u) / 128u;
    p.wideX = a.k % 8u == 0u && a.ldx % 8u == 0u && r355::aligned(a.x, 16);
    p.wideN = a.n % 4u == 0u && a.ldy % 4u == 0u && r355::aligned(a.y, 4u * outBytes) && r355::aligned(a.scales, 8) && (!a.zeros || r355::aligned(a.zeros, 4))
              && (a.beta == 0.0 || (a.ldc % 4u == 0u && r355::aligned(a.c, 4u * outBytes)));
    p.alpha = static_cast<float>(a.alpha), p.beta = static_cast<float>(a.beta);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    r355::beginCall();
    if(a.in_type == R355_F16 && a.out_type == R355_F16)
        launchShape<_Float16, _Float16>(p, s);
    else if(a.in_type == R355_F16)
        launchShape<_Float16, float>(p, s);
    else if(a.out_type == R355_BF16)
        launchShape<__bf16, __bf16>(p, s);
    else
        launchShape<__bf16, float>(p, s);
    return r355::checkLaunch("w4_matmul");
}
