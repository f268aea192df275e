// The router of a layer with experts, and the rows' way to the experts and back, with the gradients of both.  No counterpart in the reference.
//
//   route      the `top` experts of each token by logit (plus bias) or by score plus bias, their weights, and the rows in order of experts: place[t][j], source[row], offsets[e]
//   combine    y_t = sum_j w_tj rows[place_tj] + c_t
//   dispatch   rows[place_tj] = w_tj x_t;  dw_tj = x_t . values[place_tj]      (the gradient of combine; without weights that of its own, and the way to the experts)
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "half_types.hpp"

namespace
{
    using r355::vec;

    // ---- reductions over a wave, by lanes of a row and then of rows (data-parallel operands); the result is in every lane
    template <int CTRL, int ROWS>
    __device__ __forceinline__ uint32_t moved(uint32_t identity, uint32_t v)
    {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(identity), static_cast<int>(v), CTRL, ROWS, 0xF, false));
    }
    template <typename F>
    __device__ __forceinline__ uint32_t reduce(uint32_t identity, uint32_t v, F&& f)
    {
        v = f(v, moved<0x111, 0xF>(identity, v)); // row_shr 1, 2, 4, 8
        v = f(v, moved<0x112, 0xF>(identity, v));
        v = f(v, moved<0x114, 0xF>(identity, v));
        v = f(v, moved<0x118, 0xF>(identity, v));
        v = f(v, moved<0x142, 0xA>(identity, v)); // row_bcast 15, 31
        v = f(v, moved<0x143, 0xC>(identity, v));
        return __builtin_amdgcn_readlane(v, 63);
    }
    __device__ __forceinline__ uint32_t largest(uint32_t v)
    {
        return reduce(0u, v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    }
    // numbers as integers in their order, infinities at their ends and NaN beyond them, and back
    __device__ __forceinline__ uint32_t orderOf(float v)
    {
        const uint32_t b = __float_as_uint(v);
        return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    }
    __device__ __forceinline__ float largest(float v) // (of integers a step is one instruction, of floats it is four; where one is NaN so is all that is made of the result)
    {
        const uint32_t k = largest(orderOf(v));
        return __uint_as_float(k ^ (~static_cast<uint32_t>(static_cast<int32_t>(k) >> 31) | 0x80000000u));
    }
    __device__ __forceinline__ float sum(float v)
    {
        return __uint_as_float(reduce(0u, __float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
    }

    struct RouteParams
    {
        const char*    logits;
        const float*   bias;
        float*         weights;
        int32_t*       chosen;
        int32_t*       place;
        int32_t*       source;
        int32_t*       offsets;
        uint32_t*      counts; // [experts][blocks]: of each block of tokens; then what the blocks before it have
        uint32_t*      totals; // [experts]
        const int32_t* given;  // gradient: the experts chosen
        const float*   dweights;
        char*          dlogits;
        uint32_t       tokens, experts, top, ldl, ldd, blocks, perBlock;
        int32_t        score, chosenOnly, even; // even: rows of logits on the boundaries of what a lane reads of them
        int32_t        scoreBias; // the bias is added to the score, otherwise to the logit
        float          scale;
    };

    constexpr uint32_t MOST_EXPERTS = 1024u, MOST_TOP = 32u;
    constexpr uint32_t THREADS = 256u, WAVES = 4u;

    // log of a score: the logit itself (softmax, up to what its sum takes off) or log sigma
    __device__ __forceinline__ float logScore(int32_t score, float x)
    {
        // (the logarithm's argument lies in [1, 2]: nothing to scale)
        return score == R355_ROUTE_SIGMOID ? fminf(x, 0.0f) - 0.69314718056f * __builtin_amdgcn_logf(1.0f + __expf(-fabsf(x))) : x;
    }

    // e^(v - the largest) and their sum; a row of -infinity has zeros
    __device__ __forceinline__ float exponentials(float v, bool in, float most)
    {
        return in ? __expf(v - (most == -INFINITY ? 0.0f : most)) : 0.0f;
    }

    // The largest of a token's logits, and the sum of the exponentials.  (For the choice by score plus bias it comes before the keys: 16384 tokens, 8 of 256, 26.4 -> 29.2 us, by sigmoid 28.2.)
    template <uint32_t V>
    __device__ __forceinline__ void ofAll(const RouteParams& p, const float (&x)[V], uint32_t lane, float& most, float& all)
    {
        most = -INFINITY, all = 0.0f;
#pragma unroll
        for(uint32_t i = 0; i < V; ++i)
            most = fmaxf(most, lane * V + i < p.experts ? x[i] : -INFINITY);
        most = largest(most);
#pragma unroll
        for(uint32_t i = 0; i < V; ++i)
            all += exponentials(x[i], lane * V + i < p.experts, most);
        all = sum(all);
    }

    __device__ __forceinline__ uint32_t maskOf(bool is)
    {
        uint32_t m = is ? ~0u : 0u;
        asm("" : "+v"(m)); // (kept from the compiler, which would take it for a condition again)
        return m;
    }
    __device__ __forceinline__ uint32_t either(uint32_t mask, uint32_t a, uint32_t b)
    {
        return (a & mask) | (b & ~mask);
    }

    // What a lane keeps from token to token: its experts' biases (zeros without), and which of them there are
    template <uint32_t V>
    struct Lane
    {
        float    bias[V];
        uint32_t there[V];
        __device__ __forceinline__ Lane(const RouteParams& p, uint32_t lane)
        {
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
            {
                const uint32_t e = lane * V + i;
                bias[i]          = p.bias && e < p.experts ? p.bias[e] + 0.0f : 0.0f; // (never -0)
                there[i]         = maskOf(e < p.experts);
            }
        }
    };

    // One token a wave: expert V lane + i in x[i] of the lane.  A key orders numbers as integers, NaN below them; every lane sorts its keys, and `top` rounds take the largest of
    // the lanes' first ones, of the lowest lane that has it, which then moves up.  Bound by the vector instructions: of 256 experts
    // and 8 choices 309 a token, 17 of them a round; 16384 tokens 16 us (8.6 of issuing).
    // What is returned lies in lane j for the j-th choice: its expert and its logit.
    template <uint32_t V>
    __device__ __forceinline__ void choose(const RouteParams& p, const float (&x)[V], const Lane<V>& own, uint32_t lane, uint32_t& expert, float& logit)
    {
        uint32_t key[V], of[V]; // keys, and which of the lane's experts they are of
        auto setKey = [&](uint32_t i, float by) __attribute__((always_inline)) {
            key[i] = either(maskOf(by != by), 1u, orderOf(by)) & own.there[i]; // (-infinity: 0x007FFFFF)
            of[i]  = i;
        };
        if(p.scoreBias) // (uniform)
        {
            // (divisions: equal logits aside, what a score is off by decides between experts)
            float most = 0.0f, all = 1.0f;
            if(p.score != R355_ROUTE_SIGMOID)
                ofAll<V>(p, x, lane, most, all);
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
                setKey(i, (p.score == R355_ROUTE_SIGMOID ? 1.0f / (1.0f + __expf(-x[i])) : all == 0.0f ? 0.0f : exponentials(x[i], true, most) / all) + own.bias[i]);
        }
        else
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
                setKey(i, x[i] + own.bias[i]); // (-0 counts as 0)
        // (Neighbours change places only if the later one is larger: equal ones stay in the order of their experts.  Choices by masks, one instruction each: of conditions the
        // compiler makes branches and indices, twice as many.)
#pragma unroll
        for(uint32_t end = V - 1u; end > 0u; --end)
#pragma unroll
            for(uint32_t i = 0; i < end; ++i)
            {
                const uint32_t k = key[i], l = key[i + 1u], o = of[i], swap = maskOf(l > k);
                key[i] = k > l ? k : l, key[i + 1u] = k > l ? l : k;
                of[i] = either(swap, of[i + 1u], o), of[i + 1u] = either(swap, o, of[i + 1u]);
            }
        expert = 0u;
        for(uint32_t j = 0; j < p.top; ++j)
        {
            const uint32_t best = largest(key[0]);
            const uint32_t l    = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(__ballot(key[0] == best)))) - 1u;
            const uint32_t e    = l * V + __builtin_amdgcn_readlane(of[0], l);
            expert              = lane == j ? e : expert;
            const uint32_t moves = maskOf(lane == l);
#pragma unroll
            for(uint32_t i = 0; i + 1u < V; ++i)
                key[i] = either(moves, key[i + 1u], key[i]), of[i] = either(moves, of[i + 1u], of[i]);
            key[V - 1u] &= ~moves;
        }
        // the logit of the lane's choice lies with lane expert / V
        logit = 0.0f;
#pragma unroll
        for(uint32_t i = 0; i < V; ++i)
        {
            const float v = __uint_as_float(__builtin_amdgcn_ds_bpermute(static_cast<int>(expert / V * 4u), static_cast<int>(__float_as_uint(x[i]))));
            logit         = expert % V == i ? v : logit;
        }
    }

    // Weights of the choices, in the lanes that hold them.  (Reciprocals and the logarithm are the hardware's, a step of 32 bits: the weights of 16384 tokens are off by 6.7e-8 of their norm,
    // torch's in 32 bits by 5.9e-8.)
    template <uint32_t V>
    __device__ __forceinline__ float weightOf(const RouteParams& p, const float (&x)[V], uint32_t lane, float logit)
    {
        const bool in = lane < p.top;
        if(p.chosenOnly)
        {
            const float l = logScore(p.score, logit), most = largest(in ? l : -INFINITY);
            const float e = exponentials(l, in, most), all = sum(e);
            return all == 0.0f ? 0.0f : e * __builtin_amdgcn_rcpf(all) * p.scale;
        }
        if(p.score == R355_ROUTE_SIGMOID)
            return p.scale * __builtin_amdgcn_rcpf(1.0f + __expf(-logit));
        float most, all;
        ofAll<V>(p, x, lane, most, all);
        return all == 0.0f ? 0.0f : exponentials(logit, in, most) * __builtin_amdgcn_rcpf(all) * p.scale;
    }

    // experts V lane .. V lane + V - 1 of a token: as vectors where the rows are even (a rule of the host's)
    template <typename T, uint32_t V>
    __device__ __forceinline__ void readLogits(const RouteParams& p, uint32_t token, uint32_t lane, float (&x)[V])
    {
        const T* from = reinterpret_cast<const T*>(p.logits) + (uint64_t)token * p.ldl + lane * V;
        if(V > 1u && p.even)
        {
            constexpr uint32_t PER = V * sizeof(T) > 16u ? 16u / sizeof(T) : V;
#pragma unroll
            for(uint32_t i = 0; i < V; i += PER)
            {
                vec<T, PER> v{};
                if(lane * V + i < p.experts)
                    v = *reinterpret_cast<const vec<T, PER>*>(from + i);
#pragma unroll
                for(uint32_t e = 0; e < PER; ++e)
                    x[i + e] = static_cast<float>(v[e]);
            }
        }
        else
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
                x[i] = lane * V + i < p.experts ? static_cast<float>(from[i]) : 0.0f;
    }
    template <typename T, uint32_t V>
    __device__ __forceinline__ void writeLogits(const RouteParams& p, uint32_t token, uint32_t lane, const float (&d)[V])
    {
        T* to = reinterpret_cast<T*>(p.dlogits) + (uint64_t)token * p.ldd + lane * V;
        if(V > 1u && p.even)
        {
            constexpr uint32_t PER = V * sizeof(T) > 16u ? 16u / sizeof(T) : V;
#pragma unroll
            for(uint32_t i = 0; i < V; i += PER)
            {
                vec<T, PER> v;
#pragma unroll
                for(uint32_t e = 0; e < PER; ++e)
                    v[e] = static_cast<T>(d[i + e]);
                if(lane * V + i < p.experts)
                    *reinterpret_cast<vec<T, PER>*>(to + i) = v;
            }
        }
        else
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
                if(lane * V + i < p.experts)
                    to[i] = static_cast<T>(d[i]);
    }

    // The block's slots (token, choice) in order, a contiguous run of them for each wave: row = base[expert] + how many slots before have the same expert.
    // counts: [WAVES][experts] of LDS, zeros; base: [experts] of LDS; experts of the slots: chosen (LDS or global)
    template <typename Chosen>
    __device__ __forceinline__ void rank(const RouteParams& p, uint32_t slots, uint32_t firstSlot, Chosen&& chosen, const uint32_t* base, uint32_t* counts)
    {
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t each = (slots + WAVES * 64u - 1u) / (WAVES * 64u) * 64u, from = wave * each < slots ? wave * each : slots, to = from + each < slots ? from + each : slots;
        for(uint32_t s = from + lane; s < to; s += 64u)
            atomicAdd(&counts[wave * p.experts + chosen(s)], 1u);
        __syncthreads();
        for(uint32_t e = threadIdx.x; e < p.experts; e += THREADS)
        {
            uint32_t at = base[e];
            for(uint32_t w = 0; w < WAVES; ++w)
            {
                const uint32_t n = counts[w * p.experts + e];
                counts[w * p.experts + e] = at;
                at += n;
            }
        }
        __syncthreads();
        const uint32_t bits = 32u - __builtin_clz(p.experts > 1u ? p.experts - 1u : 1u);
        for(uint32_t s0 = from; s0 < to; s0 += 64u)
        {
            const uint32_t s = s0 + lane;
            const bool     in = s < to;
            const uint32_t e = in ? chosen(s) : 0u;
            uint64_t       same = __ballot(in); // lanes of the same expert
            for(uint32_t b = 0; b < bits; ++b)
            {
                const uint64_t have = __ballot((e >> b) & 1u);
                same &= (e >> b) & 1u ? have : ~have;
            }
            if(in)
            {
                const uint32_t before = static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull)));
                const uint32_t at     = counts[wave * p.experts + e];
                __builtin_amdgcn_wave_barrier(); // (all have read before the last of them writes: LDS is in order within a wave)
                if((same >> lane) == 1ull)
                    counts[wave * p.experts + e] = at + before + 1u;
                p.place[(uint64_t)firstSlot + s]  = static_cast<int32_t>(at + before);
                p.source[(uint64_t)at + before] = static_cast<int32_t>((firstSlot + s) / p.top);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }

    // exclusive sums over the experts of n[e], into base[e] and, for the first block, offsets
    __device__ __forceinline__ void expertBases(const RouteParams& p, const uint32_t* n, uint32_t* base, bool write)
    {
        if(threadIdx.x < 64u)
        {
            uint32_t before = 0u;
            for(uint32_t e0 = 0; e0 < p.experts; e0 += 64u)
            {
                const uint32_t e = e0 + threadIdx.x, mine = e < p.experts ? n[e] : 0u;
                uint32_t       upto = mine;
#pragma unroll
                for(uint32_t d = 1u; d < 64u; d <<= 1)
                {
                    const uint32_t below = __shfl_up(upto, d);
                    upto += threadIdx.x >= d ? below : 0u;
                }
                if(e < p.experts)
                {
                    base[e] = before + upto - mine;
                    if(write)
                        p.offsets[e] = static_cast<int32_t>(before + upto - mine);
                }
                before += __builtin_amdgcn_readlane(upto, 63);
            }
            if(write && threadIdx.x == 0u)
                p.offsets[p.experts] = static_cast<int32_t>(before);
        }
    }

    // (Every form of the order's making waits for memory: of 16384 tokens over 256 experts routeCounts takes 4.0 us, routePlace 6.5.)
    // The choice of a block of tokens, a token a wave at a time; ALL: there is one block, which goes on to the order of the rows.
    template <typename T, uint32_t V, bool ALL>
    __global__ void __launch_bounds__(THREADS) routeChoose(RouteParams p)
    {
        extern __shared__ uint32_t shared[]; // counts [experts]; ALL: base [experts], counts of the waves [WAVES][experts], experts of the slots
        uint32_t* const counts = shared;
        uint32_t* const base   = shared + p.experts;
        uint32_t* const waves  = base + p.experts;
        uint32_t* const slots  = waves + WAVES * p.experts;
        for(uint32_t e = threadIdx.x; e < (ALL ? (2u + WAVES) * p.experts : p.experts); e += THREADS)
            shared[e] = 0u;
        __syncthreads();
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t from = blockIdx.x * p.perBlock, left = p.tokens - from, here = left < p.perBlock ? left : p.perBlock;
        const Lane<V>  own(p, lane);
        float          next[V]; // the following token's, read ahead
        if(wave < here)
            readLogits<T, V>(p, from + wave, lane, next);
        for(uint32_t i = wave; i < here; i += WAVES)
        {
            const uint32_t token = from + i;
            float          x[V], logit;
            uint32_t       expert;
#pragma unroll
            for(uint32_t e = 0; e < V; ++e)
                x[e] = next[e];
            if(i + WAVES < here)
                readLogits<T, V>(p, token + WAVES, lane, next);
            choose<V>(p, x, own, lane, expert, logit);
            const float weight = weightOf<V>(p, x, lane, logit);
            if(lane < p.top)
            {
                p.weights[(uint64_t)token * p.top + lane] = weight;
                p.chosen[(uint64_t)token * p.top + lane]  = static_cast<int32_t>(expert);
                atomicAdd(&counts[expert], 1u);
                if(ALL)
                    slots[i * p.top + lane] = expert;
            }
        }
        __syncthreads();
        if constexpr(ALL)
        {
            expertBases(p, counts, base, true);
            __syncthreads();
            rank(p, here * p.top, 0u, [&](uint32_t s) { return slots[s]; }, base, waves);
        }
        else
            for(uint32_t e = threadIdx.x; e < p.experts; e += THREADS)
                p.counts[(uint64_t)e * p.blocks + blockIdx.x] = counts[e];
    }

    // Of one expert: how many rows the blocks before each have, and the total; a wave, a run of 16 blocks a lane at a time
    __global__ void __launch_bounds__(64) routeCounts(RouteParams p)
    {
        constexpr uint32_t RUN    = 16u;
        uint32_t* const    counts = p.counts + (uint64_t)blockIdx.x * p.blocks;
        uint32_t           before = 0u;
        for(uint32_t b0 = 0; b0 < p.blocks; b0 += 64u * RUN)
        {
            const uint32_t b = b0 + threadIdx.x * RUN;
            uint32_t       mine[RUN], all = 0u;
#pragma unroll
            for(uint32_t i = 0; i < RUN; ++i)
                mine[i] = b + i < p.blocks ? counts[b + i] : 0u;
#pragma unroll
            for(uint32_t i = 0; i < RUN; ++i)
                all += mine[i];
            uint32_t upto = all;
#pragma unroll
            for(uint32_t d = 1u; d < 64u; d <<= 1)
            {
                const uint32_t below = __shfl_up(upto, d);
                upto += threadIdx.x >= d ? below : 0u;
            }
            uint32_t at = before + upto - all;
#pragma unroll
            for(uint32_t i = 0; i < RUN; ++i)
            {
                if(b + i < p.blocks)
                    counts[b + i] = at;
                at += mine[i];
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        if(threadIdx.x == 0u)
            p.totals[blockIdx.x] = before;
    }

    // The rows of a block of tokens
    __global__ void __launch_bounds__(THREADS) routePlace(RouteParams p)
    {
        extern __shared__ uint32_t shared[]; // base [experts], counts of the waves [WAVES][experts]
        uint32_t* const base  = shared;
        uint32_t* const waves = shared + p.experts;
        for(uint32_t e = threadIdx.x; e < WAVES * p.experts; e += THREADS)
            waves[e] = 0u;
        expertBases(p, p.totals, base, blockIdx.x == 0u);
        __syncthreads();
        for(uint32_t e = threadIdx.x; e < p.experts; e += THREADS)
            base[e] += p.counts[(uint64_t)e * p.blocks + blockIdx.x];
        __syncthreads();
        const uint32_t from = blockIdx.x * p.perBlock, left = p.tokens - from, here = left < p.perBlock ? left : p.perBlock;
        const int32_t* chosen = p.chosen + (uint64_t)from * p.top;
        rank(p, here * p.top, from * p.top, [&](uint32_t s) { return static_cast<uint32_t>(chosen[s]); }, base, waves);
    }

    // The gradient of the weights with respect to the logits, a token a wave.  With l_j the logarithms of the scores, d w_j / d x_i = w_j (d l_j / d x_i - what the sum takes off):
    //   g_j = dw_j w_j, over the chosen alone g_j - w_j / scale sum g;  sigmoid: dx_j = g_j (1 - s_j);  softmax: dx_j = g_j, over all experts less p_i sum g for every one.
    // Bound by the exponentials and a wave's way through memory and back: 16001 tokens of 128 experts 6.5 us, 1.3 TB/s.
    template <typename T, uint32_t V>
    __global__ void __launch_bounds__(THREADS) routeGrad(RouteParams p)
    {
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t token = blockIdx.x * WAVES + wave;
        if(token >= p.tokens)
            return;
        float x[V];
        readLogits<T, V>(p, token, lane, x);
        const bool     slot   = lane < p.top;
        const uint32_t expert = slot ? static_cast<uint32_t>(p.given[(uint64_t)token * p.top + lane]) : p.experts;
        const bool     in     = expert < p.experts; // (a number that is no expert's has no part in it)
        const float    logit  = in ? static_cast<float>(reinterpret_cast<const T*>(p.logits)[(uint64_t)token * p.ldl + expert]) : 0.0f;
        const float    dw     = in ? p.dweights[(uint64_t)token * p.top + lane] : 0.0f;
        float          g, off = 0.0f, most = -INFINITY, all = 0.0f;
        if(p.chosenOnly)
        {
            const float l = logScore(p.score, logit);
            most          = largest(in ? l : -INFINITY);
            const float e = exponentials(l, in, most);
            all           = sum(e);
            const float w = all == 0.0f ? 0.0f : e / all;
            g             = in ? dw * w * p.scale : 0.0f;
            g -= w * sum(g);
        }
        else if(p.score == R355_ROUTE_SIGMOID)
            g = in ? dw * p.scale / (1.0f + __expf(-logit)) : 0.0f;
        else
        {
            ofAll<V>(p, x, lane, most, all);
            g   = in && all != 0.0f ? dw * p.scale * exponentials(logit, true, most) / all : 0.0f;
            off = all == 0.0f ? 0.0f : sum(g) / all;
        }
        if(p.score == R355_ROUTE_SIGMOID && in)
            g *= 1.0f / (1.0f + __expf(logit)); // 1 - sigma
        float d[V];
#pragma unroll
        for(uint32_t i = 0; i < V; ++i)
            d[i] = off == 0.0f ? 0.0f : -off * exponentials(x[i], lane * V + i < p.experts, most);
        for(uint32_t j = 0; j < p.top; ++j) // (one after the other: an expert given twice gets both)
        {
            const uint32_t e = __builtin_amdgcn_readlane(expert, j);
            const float    v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
#pragma unroll
            for(uint32_t i = 0; i < V; ++i)
                d[i] += lane * V + i == e ? v : 0.0f;
        }
        writeLogits<T, V>(p, token, lane, d);
    }

    // ---- rows to the experts and back
    struct RowsParams
    {
        const char*    x;      // dispatch: of the tokens; combine: c
        const char*    values; // of the experts' rows
        char*          out;
        const int32_t* place;
        const float*   weights;
        float*         dweights;
        uint32_t       tokens, top, width, rows;
        uint32_t       ldx, ldv, ldo, pieces; // pieces: of EW elements of a row
    };

    // STREAM: nontemporally, as what lies beyond the caches (a rule of the host's)
    template <typename T, uint32_t EW, bool STREAM>
    __device__ __forceinline__ vec<T, EW> readPiece(const char* base, uint64_t row, uint32_t ld, uint32_t col)
    {
        const vec<T, EW>* at = reinterpret_cast<const vec<T, EW>*>(reinterpret_cast<const T*>(base) + row * ld + col);
        if constexpr(STREAM)
            return __builtin_nontemporal_load(at);
        else
            return *at;
    }
    template <typename T, uint32_t EW, bool STREAM>
    __device__ __forceinline__ void writePiece(char* base, uint64_t row, uint32_t ld, uint32_t col, vec<T, EW> v)
    {
        vec<T, EW>* at = reinterpret_cast<vec<T, EW>*>(reinterpret_cast<T*>(base) + row * ld + col);
        if constexpr(STREAM)
            __builtin_nontemporal_store(v, at);
        else
            *at = v;
    }

    // A thread per piece of a token's row; the rows of up to eight of its choices are under way at once.  Bound by HBM: 8192 x 8 x 4096 and a residual 110 us, 6.1 TB/s.
    template <typename T, uint32_t EW, bool STREAM>
    __global__ void __launch_bounds__(THREADS) combineRows(RowsParams p)
    {
        const uint32_t at = blockIdx.x * THREADS + threadIdx.x, token = at / p.pieces; // (a launch has less than 2^32 threads)
        if(token >= p.tokens)
            return;
        const uint32_t col = at % p.pieces * EW;
        float          total[EW];
#pragma unroll
        for(uint32_t e = 0; e < EW; ++e)
            total[e] = 0.0f;
        for(uint32_t j0 = 0; j0 < p.top; j0 += 8u)
        {
            vec<T, EW> v[8];
            float      w[8];
            bool       in[8];
#pragma unroll
            for(uint32_t u = 0; u < 8u; ++u)
                if(j0 + u < p.top) // (uniform)
                {
                    const uint64_t slot = (uint64_t)token * p.top + j0 + u;
                    const uint32_t row  = static_cast<uint32_t>(p.place[slot]);
                    in[u]               = row < p.rows;
                    w[u]                = p.weights ? p.weights[slot] : 1.0f;
                    if(in[u])
                        v[u] = readPiece<T, EW, STREAM>(p.values, row, p.ldv, col);
                }
#pragma unroll
            for(uint32_t u = 0; u < 8u; ++u)
                if(j0 + u < p.top && in[u])
#pragma unroll
                    for(uint32_t e = 0; e < EW; ++e)
                        total[e] = fmaf(w[u], static_cast<float>(v[u][e]), total[e]);
        }
        if(p.x)
        {
            const vec<T, EW> c = readPiece<T, EW, STREAM>(p.x, token, p.ldx, col);
#pragma unroll
            for(uint32_t e = 0; e < EW; ++e)
                total[e] += static_cast<float>(c[e]);
        }
        vec<T, EW> y;
#pragma unroll
        for(uint32_t e = 0; e < EW; ++e)
            y[e] = static_cast<T>(total[e]);
        writePiece<T, EW, STREAM>(p.out, token, p.ldo, col, y);
    }

    // SHARE waves per token take its pieces in turn, 64 at a time; the dot products of up to eight choices at once, joined in the order of the waves.  Bound by memory: 4099 x 2 x 2832 with
    // weights and their gradient 23 us, 5.0 TB/s.
    template <typename T, uint32_t EW, uint32_t SHARE, bool DOTS, bool STREAM>
    __global__ void __launch_bounds__(THREADS) dispatchRows(RowsParams p)
    {
        __shared__ float meet[WAVES][8];
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t token = blockIdx.x * (WAVES / SHARE) + wave / SHARE, part = wave % SHARE;
        const bool     there = token < p.tokens;
        for(uint32_t j0 = 0; j0 < p.top; j0 += 8u)
        {
            uint32_t row[8];
            float    w[8], dot[8];
#pragma unroll
            for(uint32_t u = 0; u < 8u; ++u)
            {
                const uint64_t slot = (uint64_t)token * p.top + j0 + u;
                row[u] = there && j0 + u < p.top ? static_cast<uint32_t>(p.place[slot]) : p.rows;
                w[u]   = p.weights && row[u] < p.rows ? p.weights[slot] : 1.0f;
                dot[u] = 0.0f;
            }
            if(there)
                for(uint32_t at = part * 64u + lane; at < p.pieces; at += SHARE * 64u)
                {
                    const uint32_t   col = at * EW;
                    const vec<T, EW> x   = readPiece<T, EW, false>(p.x, token, p.ldx, col);
                    vec<T, EW>       v[DOTS ? 8 : 1];
                    if constexpr(DOTS)
#pragma unroll
                        for(uint32_t u = 0; u < 8u; ++u)
                            if(row[u] < p.rows)
                                v[u] = readPiece<T, EW, STREAM>(p.values, row[u], p.ldv, col);
#pragma unroll
                    for(uint32_t u = 0; u < 8u; ++u)
                        if(row[u] < p.rows)
                        {
                            vec<T, EW> y;
#pragma unroll
                            for(uint32_t e = 0; e < EW; ++e)
                            {
                                y[e] = p.weights ? static_cast<T>(w[u] * static_cast<float>(x[e])) : x[e];
                                if constexpr(DOTS)
                                    dot[u] = fmaf(static_cast<float>(x[e]), static_cast<float>(v[u][e]), dot[u]);
                            }
                            if(p.out)
                                writePiece<T, EW, false>(p.out, row[u], p.ldo, col, y);
                        }
                }
            if constexpr(DOTS)
            {
#pragma unroll
                for(uint32_t u = 0; u < 8u; ++u)
                    dot[u] = sum(dot[u]);
                if constexpr(SHARE > 1u)
                {
                    if(lane == 0u)
#pragma unroll
                        for(uint32_t u = 0; u < 8u; ++u)
                            meet[wave][u] = dot[u];
                    __syncthreads();
#pragma unroll
                    for(uint32_t u = 0; u < 8u; ++u)
                    {
                        dot[u] = meet[0][u];
#pragma unroll
                        for(uint32_t s = 1; s < SHARE; ++s)
                            dot[u] += meet[s][u];
                    }
                    __syncthreads();
                }
                if(there && part == 0u && lane < 8u && j0 + lane < p.top)
                {
                    float mine = dot[0];
#pragma unroll
                    for(uint32_t u = 1; u < 8u; ++u)
                        mine = lane == u ? dot[u] : mine;
                    p.dweights[(uint64_t)token * p.top + j0 + lane] = mine;
                }
            }
        }
    }

    // blocks of tokens of a routing in three launches: enough to fill the CUs, 16 tokens each at least, up to 2048 slots
    uint32_t tokensPerBlock(uint32_t tokens, uint32_t top)
    {
        uint32_t per = (tokens + 1023u) / 1024u;
        per          = per < 16u ? 16u : (per + 3u) / 4u * 4u;
        const uint32_t most = 2048u / top / 4u * 4u;
        return per < most ? per : most;
    }
    // few enough for one workgroup to do it all
    bool alone(uint32_t tokens, uint32_t top)
    {
        return tokens <= 64u && (uint64_t)tokens * top <= 1024u;
    }

    uint64_t routeScratch(uint32_t tokens, uint32_t experts, uint32_t top)
    {
        if(alone(tokens, top))
            return 0u;
        // (what any number of tokens up to that needs: blocks of 16 tokens, 1024 of them or as many as 2048 slots in each make)
        const uint32_t most = 2048u / top / 4u * 4u, small = (tokens - 1u) / 16u + 1u, large = (tokens - 1u) / most + 1u, few = small < 1024u ? small : 1024u;
        return ((uint64_t)(few > large ? few : large) + 1u) * experts * 4u;
    }

    template <typename T, uint32_t V>
    void launchRoute(const RouteParams& p, hipStream_t s)
    {
        if(p.blocks == 1u)
        {
            hipLaunchKernelGGL((routeChoose<T, V, true>), dim3(1), dim3(THREADS), ((2u + WAVES) * p.experts + p.tokens * p.top) * 4u, s, p);
            return;
        }
        hipLaunchKernelGGL((routeChoose<T, V, false>), dim3(p.blocks), dim3(THREADS), p.experts * 4u, s, p);
        hipLaunchKernelGGL(routeCounts, dim3(p.experts), dim3(64), 0, s, p);
        hipLaunchKernelGGL(routePlace, dim3(p.blocks), dim3(THREADS), (1u + WAVES) * p.experts * 4u, s, p);
    }
    template <typename T, uint32_t V>
    void launchRouteGrad(const RouteParams& p, hipStream_t s)
    {
        hipLaunchKernelGGL((routeGrad<T, V>), dim3((p.tokens + WAVES - 1u) / WAVES), dim3(THREADS), 0, s, p);
    }
    // rows whose lanes read vectors: those of V elements, up to 16 bytes, begin on their boundaries and end with one
    template <typename T>
    bool evenRows(const void* at, uint32_t ld, uint32_t experts)
    {
        const uint32_t v = experts <= 64u ? 1u : experts <= 128u ? 2u : experts <= 256u ? 4u : 16u, per = v * sizeof(T) > 16u ? 16u / sizeof(T) : v;
        return !at || (r355::aligned(at, per * sizeof(T)) && ld % per == 0u && experts % per == 0u);
    }

    template <typename T>
    void launchRouteType(RouteParams p, bool gradient, hipStream_t s)
    {
        p.even = evenRows<T>(p.logits, p.ldl, p.experts) && evenRows<T>(p.dlogits, p.ldd, p.experts);
        if(p.experts <= 64u)
            gradient ? launchRouteGrad<T, 1>(p, s) : launchRoute<T, 1>(p, s);
        else if(p.experts <= 128u)
            gradient ? launchRouteGrad<T, 2>(p, s) : launchRoute<T, 2>(p, s);
        else if(p.experts <= 256u)
            gradient ? launchRouteGrad<T, 4>(p, s) : launchRoute<T, 4>(p, s);
        else
            gradient ? launchRouteGrad<T, 16>(p, s) : launchRoute<T, 16>(p, s);
    }
    void launchRouteAny(int32_t type, const RouteParams& p, bool gradient, hipStream_t s)
    {
        if(type == R355_F16)
            launchRouteType<_Float16>(p, gradient, s);
        else if(type == R355_BF16)
            launchRouteType<__bf16>(p, gradient, s);
        else
            launchRouteType<float>(p, gradient, s);
    }

    int32_t scoreOf(int32_t score)
    {
        return score & ~R355_ROUTE_SCORE_BIAS;
    }
    int checkRoute(const char* what, int32_t type, int32_t score, uint32_t tokens, uint32_t experts, uint32_t top, const void* logits, uint32_t ldl)
    {
        if(type != R355_F16 && type != R355_BF16 && type != R355_F32)
            return r355::fail(R355_ERR_UNSUPPORTED, "%s: logits are f16, bf16 or f32", what);
        if(scoreOf(score) != R355_ROUTE_SOFTMAX && scoreOf(score) != R355_ROUTE_SIGMOID)
            return r355::fail(R355_ERR_BAD_ARG, "%s: unknown score %d", what, score);
        if(experts == 0 || top == 0 || top > experts)
            return r355::fail(R355_ERR_BAD_ARG, "%s: of %u experts %u cannot be chosen", what, experts, top);
        if(experts > MOST_EXPERTS || top > MOST_TOP || (uint64_t)tokens * top > (1u << 30))
            return r355::fail(R355_ERR_BAD_SIZE, "%s: at most %u experts, %u choices and 2^30 rows, got %u, %u and %u tokens", what, MOST_EXPERTS, MOST_TOP, experts, top, tokens);
        if(ldl < experts)
            return r355::fail(R355_ERR_BAD_ARG, "%s: the leading dimension %u is less than a row", what, ldl);
        if(!r355::aligned(logits, r355::dtypeBytes(type)))
            return r355::fail(R355_ERR_MISALIGNED, "%s: logits need the alignment of their elements", what);
        return R355_OK;
    }

    int checkRows(const char* what, int32_t type, uint32_t tokens, uint32_t top, uint32_t width, uint32_t rows)
    {
        if(type != R355_F16 && type != R355_BF16)
            return r355::fail(R355_ERR_UNSUPPORTED, "%s: rows are f16 or bf16", what);
        if(top == 0 || width == 0)
            return r355::fail(R355_ERR_BAD_ARG, "%s: top and width must be non-zero", what);
        if((uint64_t)tokens * top > (1u << 30) || rows > (1u << 30) || width > (1u << 24))
            return r355::fail(R355_ERR_BAD_SIZE, "%s: at most 2^30 rows of 2^24 elements, got %u tokens, %u choices, %u rows and %u elements", what, tokens, top, rows, width);
        return R355_OK;
    }
    // Whether the experts' rows are more than the caches keep.  Combined: 8192 x 8 x 4096 133 -> 112 us nontemporally, 512 x 8 x 4096 7.9 -> 9.7; dispatched, the reads for the weights' gradient: 8192 x 8 x
    // 4096 233 -> 220, 4099 x 2 x 2832 23.9 -> 28.1.
    bool streams(uint32_t tokens, uint32_t top, uint32_t width)
    {
        return (uint64_t)tokens * top * width * 2u > (uint64_t{96} << 20);
    }
    bool pieces16(const void* at, uint32_t ld)
    {
        return !at || (r355::aligned(at, 16) && ld % 8u == 0u);
    }
} // namespace

extern "C" size_t r355_route_workspace_bytes(uint32_t tokens, uint32_t experts, uint32_t top)
{
    if(tokens == 0 || experts == 0 || top == 0 || experts > MOST_EXPERTS || top > MOST_TOP)
        return 0;
    return static_cast<size_t>(routeScratch(tokens, experts, top));
}

extern "C" int r355_route(const r355_route_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "route: null arguments");
    const r355_route_args& a = *args;
    if(const int rc = checkRoute("route", a.type, a.score, a.tokens, a.experts, a.top, a.logits, a.ldl))
        return rc;
    if(!a.offsets || (a.tokens != 0 && (!a.logits || !a.weights || !a.chosen || !a.place || !a.source)))
        return r355::fail(R355_ERR_BAD_ARG, "route: null pointer");
    if(!r355::aligned(a.bias, 4) || !r355::aligned(a.weights, 4) || !r355::aligned(a.chosen, 4) || !r355::aligned(a.place, 4) || !r355::aligned(a.source, 4) || !r355::aligned(a.offsets, 4))
        return r355::fail(R355_ERR_MISALIGNED, "route: bias, weights and indices need the alignment of their elements");
    const uint64_t need = a.tokens ? routeScratch(a.tokens, a.experts, a.top) : 0u;
    if(need != 0u && (!a.workspace || a.workspace_bytes < need))
        return r355::fail(R355_ERR_BAD_SIZE, "route: %u tokens need %llu bytes of workspace, got %llu", a.tokens, static_cast<unsigned long long>(need),
                          static_cast<unsigned long long>(a.workspace ? a.workspace_bytes : 0u));
    if(need != 0u && !r355::aligned(a.workspace, 16))
        return r355::fail(R355_ERR_MISALIGNED, "route: the workspace needs 16-byte alignment");
    RouteParams p{};
    p.logits = static_cast<const char*>(a.logits), p.bias = a.bias, p.weights = a.weights, p.chosen = a.chosen, p.place = a.place, p.source = a.source, p.offsets = a.offsets;
    p.tokens = a.tokens, p.experts = a.experts, p.top = a.top, p.ldl = a.ldl, p.score = scoreOf(a.score), p.chosenOnly = a.chosen_only, p.scale = static_cast<float>(a.scale);
    p.scoreBias = a.bias && (a.score & R355_ROUTE_SCORE_BIAS); // (without a bias the order of the scores is that of the logits)
    p.perBlock = need ? tokensPerBlock(a.tokens, a.top) : a.tokens;
    p.blocks   = need ? (a.tokens - 1u) / p.perBlock + 1u : 1u;
    p.counts   = static_cast<uint32_t*>(a.workspace);
    p.totals   = p.counts + (uint64_t)p.blocks * p.experts;
    r355::beginCall();
    launchRouteAny(a.type, p, false, static_cast<hipStream_t>(stream));
    return r355::checkLaunch("route");
}

extern "C" int r355_route_backward(const r355_route_backward_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "route_backward: null arguments");
    const r355_route_backward_args& a = *args;
    if(const int rc = checkRoute("route_backward", a.type, a.score, a.tokens, a.experts, a.top, a.logits, a.ldl))
        return rc;
    if(a.tokens == 0)
        return R355_OK;
    if(!a.logits || !a.chosen || !a.dweights || !a.dlogits)
        return r355::fail(R355_ERR_BAD_ARG, "route_backward: null pointer");
    if(a.ldd < a.experts)
        return r355::fail(R355_ERR_BAD_ARG, "route_backward: the leading dimension %u is less than a row", a.ldd);
    if(!r355::aligned(a.chosen, 4) || !r355::aligned(a.dweights, 4) || !r355::aligned(a.dlogits, r355::dtypeBytes(a.type)))
        return r355::fail(R355_ERR_MISALIGNED, "route_backward: chosen, dweights and dlogits need the alignment of their elements");
    if((a.tokens - 1u) / WAVES + 1u > r355::MAX_GROUPS)
        return r355::fail(R355_ERR_BAD_SIZE, "route_backward: at most %u tokens, got %u", r355::MAX_GROUPS * WAVES, a.tokens);
    RouteParams p{};
    p.logits = static_cast<const char*>(a.logits), p.given = a.chosen, p.dweights = a.dweights, p.dlogits = static_cast<char*>(a.dlogits);
    p.tokens = a.tokens, p.experts = a.experts, p.top = a.top, p.ldl = a.ldl, p.ldd = a.ldd, p.score = scoreOf(a.score), p.chosenOnly = a.chosen_only, p.scale = static_cast<float>(a.scale);
    r355::beginCall();
    launchRouteAny(a.type, p, true, static_cast<hipStream_t>(stream));
    return r355::checkLaunch("route_backward");
}

extern "C" int r355_combine(const r355_combine_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "combine: null arguments");
    const r355_combine_args& a = *args;
    if(const int rc = checkRows("combine", a.type, a.tokens, a.top, a.width, a.rows))
        return rc;
    if(a.tokens == 0)
        return R355_OK;
    if((a.rows != 0 && !a.values) || !a.place || !a.y)
        return r355::fail(R355_ERR_BAD_ARG, "combine: null pointer");
    if(a.ldv < a.width || a.ldy < a.width || (a.c && a.ldc < a.width))
        return r355::fail(R355_ERR_BAD_ARG, "combine: a leading dimension is less than its row");
    if(!r355::aligned(a.values, 2) || !r355::aligned(a.c, 2) || !r355::aligned(a.y, 2) || !r355::aligned(a.place, 4) || !r355::aligned(a.weights, 4))
        return r355::fail(R355_ERR_MISALIGNED, "combine: rows, place and weights need the alignment of their elements");
    RowsParams p{};
    p.x = static_cast<const char*>(a.c), p.values = static_cast<const char*>(a.values), p.out = static_cast<char*>(a.y), p.place = a.place, p.weights = a.weights;
    p.tokens = a.tokens, p.top = a.top, p.width = a.width, p.rows = a.rows, p.ldx = a.ldc, p.ldv = a.ldv, p.ldo = a.ldy;
    const bool wide = a.width % 8u == 0u && pieces16(a.values, a.ldv) && pieces16(a.c, a.ldc) && pieces16(a.y, a.ldy);
    p.pieces        = wide ? a.width / 8u : a.width;
    const uint64_t groups = ((uint64_t)a.tokens * p.pieces + THREADS - 1u) / THREADS;
    if(groups > r355::MAX_GROUPS)
        return r355::fail(R355_ERR_BAD_SIZE, "combine: %u tokens of %u elements are too many for a launch", a.tokens, a.width);
    const bool f16    = a.type == R355_F16;
    const bool nontemporal = streams(a.tokens, a.top, a.width);
    auto       pick   = [&](auto type) {
        using T = decltype(type);
        return wide ? (nontemporal ? combineRows<T, 8, true> : combineRows<T, 8, false>) : combineRows<T, 1, false>;
    };
    const auto kernel = f16 ? pick(_Float16{}) : pick(__bf16{});
    r355::beginCall();
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), p);
    return r355::checkLaunch("combine");
}

extern "C" int r355_dispatch(const r355_dispatch_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "dispatch: null arguments");
    const r355_dispatch_args& a = *args;
    if(const int rc = checkRows("dispatch", a.type, a.tokens, a.top, a.width, a.rows))
        return rc;
    if(a.tokens == 0)
        return R355_OK;
    if(!a.x || !a.place || (a.rows != 0 && !a.out && !a.dweights) || (a.dweights && a.rows != 0 && !a.values))
        return r355::fail(R355_ERR_BAD_ARG, "dispatch: null pointer");
    if(a.ldx < a.width || (a.out && a.ldo < a.width) || (a.dweights && a.ldv < a.width))
        return r355::fail(R355_ERR_BAD_ARG, "dispatch: a leading dimension is less than its row");
    if(!r355::aligned(a.x, 2) || !r355::aligned(a.values, 2) || !r355::aligned(a.out, 2) || !r355::aligned(a.place, 4) || !r355::aligned(a.weights, 4) || !r355::aligned(a.dweights, 4))
        return r355::fail(R355_ERR_MISALIGNED, "dispatch: rows, place and weights need the alignment of their elements");
    RowsParams p{};
    p.x = static_cast<const char*>(a.x), p.values = static_cast<const char*>(a.dweights ? a.values : nullptr), p.out = static_cast<char*>(a.out), p.place = a.place;
    p.weights = a.weights, p.dweights = a.dweights;
    p.tokens = a.tokens, p.top = a.top, p.width = a.width, p.rows = a.rows, p.ldx = a.ldx, p.ldv = a.ldv, p.ldo = a.ldo;
    const bool wide = a.width % 8u == 0u && pieces16(a.x, a.ldx) && pieces16(p.values, a.ldv) && pieces16(a.out, a.ldo);
    p.pieces        = wide ? a.width / 8u : a.width;
    // a token a wave where its row is short, or a workgroup
    const bool     share  = p.pieces > 128u;
    const uint64_t groups = share ? a.tokens : (a.tokens + WAVES - 1u) / WAVES;
    if(groups > r355::MAX_GROUPS)
        return r355::fail(R355_ERR_BAD_SIZE, "dispatch: %u tokens are too many for a launch", a.tokens);
    auto pick = [&](auto type, auto dots) {
        using T             = decltype(type);
        constexpr bool DOTS = decltype(dots)::value;
        if constexpr(DOTS)
            if(wide && share && streams(a.tokens, a.top, a.width))
                return dispatchRows<T, 8, 4, DOTS, true>;
        return wide ? (share ? dispatchRows<T, 8, 4, DOTS, false> : dispatchRows<T, 8, 1, DOTS, false>) : (share ? dispatchRows<T, 1, 4, DOTS, false> : dispatchRows<T, 1, 1, DOTS, false>);
    };
    const bool f16    = a.type == R355_F16;
    const auto kernel = a.dweights ? (f16 ? pick(_Float16{}, std::true_type{}) : pick(__bf16{}, std::true_type{})) : (f16 ? pick(_Float16{}, std::false_type{}) : pick(__bf16{}, std::false_type{}));
    r355::beginCall();
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), p);
    return r355::checkLaunch("dispatch");
}
