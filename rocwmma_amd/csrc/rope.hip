// Rotary positions, and the append of rotated keys and of values to a cache.  No counterpart in the reference.
//
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = 2 pi * position * turns[i]
//
// over the pairs (i, i + r/2) or (2 i, 2 i + 1) of the first r elements of every head; the rest of a head is copied.  The gradient is the
// rotation by -t.
//
// The angle: turns[i] is what pair i turns per position, as a 64-bit fraction of a turn.  The product with the position, modulo 2^64,
// wraps around just as the angle does, so any position is as exact as the first ones (an f32 product of position and frequency
// is 0.03 rad off at a position of a million) and no table has a last position.  The upper 32 bits give the quadrant and the rest, at most an
// eighth of a turn to either side, on which the Taylor sums of sine (to t^9) and cosine (to t^8) are within 4e-8.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "half_types.hpp"

namespace
{
    using r355::vec;

    struct Part
    {
        const char* x;
        char*       y;
        uint32_t    heads, rotate, toSlots;
        int64_t     xToken, xHead, yToken, yHead; // strides in elements
    };

    struct RopeParams
    {
        Part            part[R355_ROPE_MAX_PARTS];
        const int32_t*  positions;
        const uint64_t* turns;
        const int32_t*  slots;
        uint32_t        tokens, headDim, half, slotCount; // half: pairs
        uint32_t        split; // threads along a token's heads
        uint32_t        inverse;
        float           scale;
    };

    // cosine and sine of `phase` / 2^32 turns
    __device__ __forceinline__ void waveOf(int32_t phase, float& c, float& s)
    {
        const uint32_t quadrant = (static_cast<uint32_t>(phase) + 0x20000000u) >> 30;
        const int32_t  rest     = static_cast<int32_t>(static_cast<uint32_t>(phase) - (quadrant << 30)); // within an eighth of a turn
        const float    t        = static_cast<float>(rest) * 1.46291807926715968e-9f; // 2 pi / 2^32
        const float    z        = t * t;
        const float    sine     = t + t * z * (-1.66666667e-1f + z * (8.33333333e-3f + z * (-1.98412698e-4f + z * 2.75573192e-6f)));
        const float    cosine   = 1.0f + z * (-0.5f + z * (4.16666667e-2f + z * (-1.38888889e-3f + z * 2.48015873e-5f)));
        const bool     swapped  = quadrant & 1u;
        c = swapped ? sine : cosine;
        s = swapped ? cosine : sine;
        if(quadrant == 1u || quadrant == 2u)
            c = -c;
        if(quadrant >= 2u)
            s = -s;
    }

    // A thread takes V pairs (or V elements of what is only copied) of one token, and every `split`-th head: the sines are computed once for
    // all of them.  blockIdx.y: the part.
    // Bound by the bytes, each read and written once (8192 tokens, 32 / 8 / 8 heads of 128, f16: 42.5 us, 4.74 TB/s, what a copy of 4 GiB
    // reaches), for a few tokens by the launch (8 tokens of the same: 3.3 us of kernel).  V = 1, where half of what is rotated, the rest or a stride is no multiple of four
    // elements, by the number of accesses (8192 tokens, 40 heads of 80, one after another on the same data: 80 rotated 19 us, 40 rotated with V = 4 30, 20 rotated 44).
    template <typename T, bool HALF, uint32_t V>
    __global__ void __launch_bounds__(256) ropeKernel(RopeParams p)
    {
        using VecT = vec<T, V>;
        const Part&    part   = p.part[blockIdx.y];
        const uint32_t turned = part.rotate ? p.half / V : 0u; // threads with pairs
        const uint32_t units  = turned + (part.rotate ? (p.headDim - 2u * p.half) / V : p.headDim / V);
        const uint32_t perToken = units * p.split;
        const uint64_t id       = (uint64_t)blockIdx.x * 256u + threadIdx.x;
        const uint64_t token64  = id / perToken;
        if(token64 >= p.tokens)
            return;
        const uint32_t token = static_cast<uint32_t>(token64), within = static_cast<uint32_t>(id - token64 * perToken);
        const uint32_t unit = within % units, first = within / units;
        int64_t        row = token;
        if(part.toSlots)
        {
            row = p.slots[token];
            if(row < 0 || row >= (int64_t)p.slotCount)
                return;
        }
        const T* x = reinterpret_cast<const T*>(part.x) + token * part.xToken;
        T*       y = reinterpret_cast<T*>(part.y) + row * part.yToken;
        if(unit >= turned)
        {
            const uint32_t at = (part.rotate ? 2u * p.half : 0u) + (unit - turned) * V;
            for(uint32_t h = first; h < part.heads; h += p.split)
                *reinterpret_cast<VecT*>(y + h * part.yHead + at) = *reinterpret_cast<const VecT*>(x + h * part.xHead + at);
            return;
        }
        const int64_t position = p.positions[token];
        float         c[V], s[V];
#pragma unroll
        for(uint32_t e = 0; e < V; ++e)
        {
            waveOf(static_cast<int32_t>((static_cast<uint64_t>(position) * p.turns[unit * V + e]) >> 32), c[e], s[e]);
            c[e] *= p.scale;
            s[e] *= p.inverse ? -p.scale : p.scale;
        }
        const uint32_t at0 = HALF ? unit * V : 2u * unit * V, at1 = HALF ? p.half + unit * V : at0 + V;
        for(uint32_t h = first; h < part.heads; h += p.split)
        {
            const VecT u = *reinterpret_cast<const VecT*>(x + h * part.xHead + at0), v = *reinterpret_cast<const VecT*>(x + h * part.xHead + at1);
            VecT       outU, outV;
#pragma unroll
            for(uint32_t e = 0; e < V; ++e)
            {
                // interleaved: pair e lies at 2 e and 2 e + 1 of the 2 V elements
                float a, b;
                if constexpr(HALF)
                    a = static_cast<float>(u[e]), b = static_cast<float>(v[e]);
                else
                    a = static_cast<float>(2u * e < V ? u[2u * e % V] : v[2u * e % V]), b = static_cast<float>(2u * e + 1u < V ? u[(2u * e + 1u) % V] : v[(2u * e + 1u) % V]);
                const T ra = static_cast<T>(a * c[e] - b * s[e]), rb = static_cast<T>(a * s[e] + b * c[e]);
                if constexpr(HALF)
                    outU[e] = ra, outV[e] = rb;
                else
                {
                    (2u * e < V ? outU : outV)[2u * e % V]               = ra;
                    (2u * e + 1u < V ? outU : outV)[(2u * e + 1u) % V] = rb;
                }
            }
            *reinterpret_cast<VecT*>(y + h * part.yHead + at0) = outU;
            *reinterpret_cast<VecT*>(y + h * part.yHead + at1) = outV;
        }
    }

    // whether every access of V elements is aligned
    bool fits(const r355_rope_args& a, uint32_t v, uint32_t bytes)
    {
        if(a.rotary_dim / 2u % v || (a.head_dim - a.rotary_dim) % v || a.head_dim % v)
            return false;
        for(uint32_t i = 0; i < a.parts; ++i)
        {
            const r355_rope_part& q = a.part[i];
            if(q.x_token_stride % v || q.x_head_stride % v || q.y_token_stride % v || q.y_head_stride % v || !r355::aligned(q.x, v * bytes) || !r355::aligned(q.y, v * bytes))
                return false;
        }
        return true;
    }

    template <typename T, uint32_t V>
    void launch(const r355_rope_args& a, RopeParams& p, hipStream_t s)
    {
        uint32_t units = 0, heads = 0;
        for(uint32_t i = 0; i < a.parts; ++i)
        {
            const uint32_t u = a.part[i].rotate ? (a.head_dim - p.half) / V : a.head_dim / V;
            units = u > units ? u : units;
            heads = a.part[i].heads > heads ? a.part[i].heads : heads;
        }
        // one head a thread while that leaves the chip short of threads, up to eight with many tokens
        const uint64_t threads = (uint64_t)a.tokens * units * heads;
        uint64_t       each    = threads / (256u * 1024u);
        each                   = each < 1u ? 1u : each > 8u ? 8u : each;
        p.split                = static_cast<uint32_t>((heads + each - 1u) / each);
        // (tokens are taken in several launches where one would count 2^32 threads)
        const uint64_t perToken = (uint64_t)units * p.split;
        const uint32_t most     = static_cast<uint32_t>((uint64_t)r355::MAX_GROUPS * 256u / perToken < 0xFFFFFFFFu ? (uint64_t)r355::MAX_GROUPS * 256u / perToken : 0xFFFFFFFFu);
        const int32_t* positions = p.positions;
        for(uint32_t first = 0; first < a.tokens; first += p.tokens)
        {
            p.tokens = a.tokens - first < most ? a.tokens - first : most;
            RopeParams q = p;
            for(uint32_t i = 0; i < a.parts; ++i)
            {
                q.part[i].x += (int64_t)first * q.part[i].xToken * (int64_t)sizeof(T);
                if(!q.part[i].toSlots)
                    q.part[i].y += (int64_t)first * q.part[i].yToken * (int64_t)sizeof(T);
            }
            q.positions = positions + first;
            q.slots     = p.slots ? p.slots + first : nullptr;
            const dim3 grid(static_cast<uint32_t>((p.tokens * perToken + 255u) / 256u), a.parts);
            if(a.layout == R355_ROPE_HALF)
                hipLaunchKernelGGL((ropeKernel<T, true, V>), grid, dim3(256), 0, s, q);
            else
                hipLaunchKernelGGL((ropeKernel<T, false, V>), grid, dim3(256), 0, s, q);
        }
    }

    template <typename T>
    void launchWidth(const r355_rope_args& a, RopeParams& p, hipStream_t s)
    {
        if constexpr(sizeof(T) == 2u)
            if(fits(a, 8, 2))
                return launch<T, 8>(a, p, s);
        if(fits(a, 4, sizeof(T)))
            return launch<T, 4>(a, p, s);
        launch<T, 1>(a, p, s);
    }
} // namespace

extern "C" int r355_rope_turns(uint32_t rotary_dim, double base, double factor, uint32_t original_length, double slow, double fast, uint64_t* turns)
{
    if(!turns)
        return r355::fail(R355_ERR_BAD_ARG, "rope_turns: null pointer");
    if(rotary_dim == 0 || rotary_dim % 2u)
        return r355::fail(R355_ERR_BAD_SIZE, "rope_turns: rotary_dim=%u must be even and not zero", rotary_dim);
    if(!(base > 0.0) || !std::isfinite(base) || !(factor > 0.0) || !std::isfinite(factor) || (original_length != 0 && !(slow < fast)))
        return r355::fail(R355_ERR_BAD_ARG, "rope_turns: base and factor must be positive, and slow less than fast");
    for(uint32_t i = 0; i < rotary_dim / 2u; ++i)
    {
        const double turn = std::pow(base, -2.0 * i / rotary_dim) / (2.0 * 3.14159265358979323846);
        double       keep = original_length ? (original_length * turn - slow) / (fast - slow) : 0.0;
        keep              = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        double scaled     = turn * (keep + (1.0 - keep) / factor);
        scaled -= std::floor(scaled); // (whole turns per position are none)
        turns[i] = static_cast<uint64_t>(std::ldexp(scaled, 64));
    }
    return R355_OK;
}

extern "C" int r355_rope(const r355_rope_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "rope: null arguments");
    const r355_rope_args& a = *args;
    if(a.type != R355_F16 && a.type != R355_BF16 && a.type != R355_F32)
        return r355::fail(R355_ERR_UNSUPPORTED, "rope: f16, bf16 and f32");
    if(a.layout != R355_ROPE_HALF && a.layout != R355_ROPE_INTERLEAVED)
        return r355::fail(R355_ERR_BAD_ARG, "rope: unknown layout");
    if(a.parts == 0 || a.parts > R355_ROPE_MAX_PARTS)
        return r355::fail(R355_ERR_BAD_ARG, "rope: 1 to %u parts, got %u", R355_ROPE_MAX_PARTS, a.parts);
    if(a.head_dim == 0 || a.rotary_dim == 0 || a.rotary_dim % 2u || a.rotary_dim > a.head_dim)
        return r355::fail(R355_ERR_BAD_SIZE, "rope: rotary_dim=%u must be even, not zero and at most head_dim=%u", a.rotary_dim, a.head_dim);
    if(a.head_dim > 4096u)
        return r355::fail(R355_ERR_BAD_SIZE, "rope: head_dim=%u is over 4096", a.head_dim);
    if(!a.turns)
        return r355::fail(R355_ERR_BAD_ARG, "rope: null turns");
    if(!r355::aligned(a.turns, 8))
        return r355::fail(R355_ERR_MISALIGNED, "rope: turns need 8-byte alignment");
    const uint32_t bytes = r355::dtypeBytes(a.type);
    RopeParams     p{};
    for(uint32_t i = 0; i < a.parts; ++i)
    {
        const r355_rope_part& q = a.part[i];
        if(q.heads == 0 || q.heads > 65536u)
            return r355::fail(R355_ERR_BAD_SIZE, "rope: part %u has %u heads: 1 to 65536", i, q.heads);
        if(a.tokens != 0 && (!q.x || !q.y || (q.to_slots && !a.slots)))
            return r355::fail(R355_ERR_BAD_ARG, "rope: null pointer in part %u", i);
        if(!r355::aligned(q.x, bytes) || !r355::aligned(q.y, bytes))
            return r355::fail(R355_ERR_MISALIGNED, "rope: x and y of part %u need the alignment of their elements", i);
        p.part[i] = Part{static_cast<const char*>(q.x), static_cast<char*>(q.y), q.heads, q.rotate != 0, q.to_slots != 0,
                         q.x_token_stride, q.x_head_stride, q.y_token_stride, q.y_head_stride};
    }
    if(a.tokens == 0)
        return R355_OK;
    if(!a.positions)
        return r355::fail(R355_ERR_BAD_ARG, "rope: null positions");
    if(!r355::aligned(a.positions, 4) || !r355::aligned(a.slots, 4))
        return r355::fail(R355_ERR_MISALIGNED, "rope: positions and slots need 4-byte alignment");
    p.positions = a.positions, p.turns = a.turns, p.slots = a.slots;
    p.tokens = a.tokens, p.headDim = a.head_dim, p.half = a.rotary_dim / 2u, p.slotCount = a.slot_count;
    p.inverse = a.inverse != 0, p.scale = static_cast<float>(a.scale);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    r355::beginCall();
    if(a.type == R355_F16)
        launchWidth<_Float16>(a, p, s);
    else if(a.type == R355_BF16)
        launchWidth<__bf16>(a, p, s);
    else
        launchWidth<float>(a, p, s);
    return r355::checkLaunch("rope");
}
