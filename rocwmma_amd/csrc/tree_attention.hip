// Attention of drafted tokens over a paged cache, on gfx950 matrix cores.  No counterpart in the reference.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i),  lse_i = log sum_j exp(scale q_i . k_j)
//
// over the positions j that row i sees: all of the prefix and, of the drafted tokens (whose keys and values are the last rows of the
// cache), those whose bit is set in the row's mask; without a mask those up to the row itself.
//
// The rows of a key head are its query heads times the drafted tokens of a sequence: 16 QB of them per wave.  A wave multiplies
// S^T = K Q^T (16 positions x 16 rows a matrix instruction), so that a lane holds four consecutive positions of one row: the running
// maximum and sum of the softmax stay within a lane's registers but for two exchanges, and P^T is, as it lies, the B operand
// of O^T = V^T P^T.  K and V go to LDS by direct loads, a 16-byte piece of a row in a slot that depends on the row, so that neither the reads
// of K (16 rows at one place) nor the transposing reads of V meet in a bank.
//
// WQ waves of the four take different rows (and share the tiles), 4 / WQ different positions.  With all four on positions every wave fills
// and reads tiles of its own and the loop has no barrier.
// The positions of a sequence are split over workgroups where there are few; partial results (f32) meet in a second kernel, in order.
#include <hip/hip_runtime.h>

#include <cmath>
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

    constexpr uint32_t WAVES = 4;
    constexpr uint32_t LEAST_CHUNK = 256; // positions of a workgroup at least
    constexpr uint32_t ABSENT = 0xFFFFFFFFu; // no such block of the cache
    constexpr uint32_t OUTSIDE = 0x7FFFFFF0u; // a lane's offset past the end of any buffer

    struct TreeParams
    {
        const char*     q;
        const char*     k;
        const char*     v;
        char*           out;
        float*          lse;
        const int32_t*  table;
        const int32_t*  qStart;
        const int32_t*  kvLen;
        const uint64_t* mask;
        float*          partial; // [splits][rows][dim], then [splits][rows][2]: maximum (in powers of two) and sum
        int64_t         qToken, qHead, kSlot, kHead, vSlot, vHead, oToken, oHead; // strides in elements
        uint32_t        batch, heads, kvHeads, group, dim, totalTokens, maxTokens, maxKv;
        uint32_t        pageSize, pages, tableStride, maskWords;
        uint32_t        splits, columns; // columns: (sequence, key head, split) triples
        float           scale2; // |scale| * log2(e), at least the smallest normal number (times minus infinity it is minus infinity)
        uint32_t        signs; // what turns the signs of two elements of q: the scale's
    };

    // the positions of one sequence that a workgroup takes
    __device__ __forceinline__ uint32_t chunkOf(uint32_t length, uint32_t splits)
    {
        const uint32_t even = (length + splits - 1u) / splits;
        const uint32_t most = even > LEAST_CHUNK ? even : LEAST_CHUNK;
        return (most + 127u) / 128u * 128u;
    }

    struct Sequence
    {
        uint32_t first, tokens, length; // first row of q, drafted tokens, cached positions
    };

    // what the arrays say of a sequence, held to what the host was told
    __device__ __forceinline__ Sequence sequenceOf(const TreeParams& p, int32_t from, int32_t to, int32_t len)
    {
        Sequence      s;
        s.first  = from < 0 ? 0u : static_cast<uint32_t>(from);
        s.first  = s.first < p.totalTokens ? s.first : p.totalTokens;
        s.tokens = to > static_cast<int32_t>(s.first) ? static_cast<uint32_t>(to) - s.first : 0u;
        s.tokens = s.tokens < p.maxTokens ? s.tokens : p.maxTokens;
        s.tokens = s.tokens < p.totalTokens - s.first ? s.tokens : p.totalTokens - s.first;
        s.length = len < 0 ? 0u : static_cast<uint32_t>(len);
        s.length = s.length < p.maxKv ? s.length : p.maxKv;
        return s;
    }

    // where block `inChunk` (of 16 positions) of the chunk that begins at block `first` of sequence b lies, in blocks of the cache
    __device__ __forceinline__ uint32_t placeOf(const TreeParams& p, uint32_t b, uint32_t first, uint32_t inChunk, uint32_t blocks, uint32_t pageBlocks)
    {
        if(inChunk >= blocks)
            return ABSENT;
        const uint32_t page = (first + inChunk) / pageBlocks, to = static_cast<uint32_t>(p.table[(uint64_t)b * p.tableStride + page]);
        return to < p.pages ? to * pageBlocks + (first + inChunk - page * pageBlocks) : ABSENT;
    }

    // which of 32 positions a row sees: bit i the one that holds drafted token past + i of the sequence (negative: of the prefix, seen by all);
    // past is less than the number of drafted tokens
    __device__ __forceinline__ uint32_t seenOf(const TreeParams& p, uint32_t row, uint32_t token, int64_t past)
    {
        if(past <= -32)
            return 0xFFFFFFFFu;
        const uint32_t before = past < 0 ? static_cast<uint32_t>(-past) : 0u, from = past < 0 ? 0u : static_cast<uint32_t>(past);
        uint32_t       bits; // of the drafted tokens from .. from + 31
        if(p.mask)
        {
            const uint64_t* words = p.mask + (uint64_t)row * p.maskWords + from / 64u;
            uint64_t        w     = words[0] >> (from % 64u);
            if(from % 64u > 32u && from / 64u + 1u < p.maskWords)
                w |= words[1] << (64u - from % 64u);
            bits = static_cast<uint32_t>(w);
        }
        else
            bits = token < from ? 0u : token - from >= 31u ? 0xFFFFFFFFu : (2u << (token - from)) - 1u;
        return (bits << before) | ((1u << before) - 1u);
    }

    template <uint32_t D>
    __device__ __forceinline__ uint32_t swizzleK(uint32_t row)
    {
        return D == 64u ? (row >> 1) & 7u : row & 15u;
    }
    template <uint32_t D>
    __device__ __forceinline__ uint32_t swizzleV(uint32_t row)
    {
        return D == 64u ? ((row >> 1) & 3u) << 1 : (row & 7u) << 1;
    }

    // of two 16-bit numbers: 1 in each half that holds an infinity or a NaN
    template <typename T>
    __device__ __forceinline__ uint32_t unfitHalves(uint32_t v)
    {
        constexpr uint32_t EXPONENT = std::is_same_v<T, __bf16> ? 0x7F807F80u : 0x7C007C00u, ULP = std::is_same_v<T, __bf16> ? 0x00800080u : 0x04000400u;
        return (((v & EXPONENT) + ULP) >> 15) & 0x00010001u;
    }
    // 1.0 in each half that holds a NaN or the infinity of the given sign, otherwise zero
    template <typename T>
    __device__ __forceinline__ uint32_t unfitOnes(uint32_t v, bool negative)
    {
        constexpr uint32_t INF = std::is_same_v<T, __bf16> ? 0x7F80u : 0x7C00u, ONE = std::is_same_v<T, __bf16> ? 0x3F80u : 0x3C00u;
        const uint32_t     lo = v & 0xFFFFu, hi = v >> 16, want = negative ? INF | 0x8000u : INF;
        return (lo == want || (lo & 0x7FFFu) > INF ? ONE : 0u) | (hi == want || (hi & 0x7FFFu) > INF ? ONE << 16 : 0u);
    }

    __device__ __forceinline__ float maxOverQuads(float x)
    {
        x = fmaxf(x, __shfl_xor(x, 16));
        return fmaxf(x, __shfl_xor(x, 32));
    }
    __device__ __forceinline__ float sumOverQuads(float x)
    {
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    }

    template <typename T, uint32_t D, uint32_t WQ, uint32_t QB>
    __global__ void __launch_bounds__(WAVES * 64, WQ == 1u ? 1 : 2) treeKernel(TreeParams p)
    {
        constexpr uint32_t WK    = WAVES / WQ;
        constexpr uint32_t NP    = D == 256u ? 16u : 32u; // positions of a tile
        constexpr uint32_t PB    = NP / 16u;
        constexpr uint32_t ROWB  = D * 2u, SLOTS = ROWB / 16u; // bytes and 16-byte pieces of a row
        constexpr uint32_t RPL   = 64u / SLOTS; // rows of a direct load
        constexpr uint32_t TILE  = NP * ROWB;
        constexpr uint32_t BUFS  = WQ == 1u ? 2u : 3u;
        constexpr uint32_t LOADS = NP / RPL / WQ; // direct loads of a wave per tile, of K or of V
        constexpr uint32_t LDS   = WK * BUFS * 2u * TILE;
        constexpr uint32_t MERGE = WK > 1u ? WK * QB * 16u * (D + 2u) * 4u : 0u;
        // weights are held relative to 2^-SHIFT of the largest: in f16 those under 2^-14 of it, of which a long row has many, stay normal numbers
        constexpr float SHIFT = std::is_same_v<T, __bf16> ? 0.0f : 10.0f;
        // ... and the maximum is taken as it was until it has grown by more than this: the sums are scaled anew in few tiles, and the largest weight is 2^(SHIFT + SLACK)
        constexpr float SLACK = 4.0f;
        static_assert(LDS <= 160u * 1024u, "LDS");
        __shared__ __attribute__((aligned(1024))) char lds[LDS > MERGE ? LDS : MERGE];

        const uint32_t tile0 = blockIdx.x / p.columns, column = blockIdx.x % p.columns;
        const uint32_t split = column % p.splits, bh = column / p.splits;
        const uint32_t head = bh % p.kvHeads, b = bh / p.kvHeads;
        if(b >= p.batch)
            return;
        const Sequence seq  = sequenceOf(p, __builtin_amdgcn_readfirstlane(p.qStart[b]), __builtin_amdgcn_readfirstlane(p.qStart[b + 1u]), __builtin_amdgcn_readfirstlane(p.kvLen[b]));
        const uint32_t rows = seq.tokens * p.group, row0 = tile0 * WQ * QB * 16u;
        if(row0 >= rows)
            return;
        const uint32_t chunk = chunkOf(seq.length, p.splits), begin = split * chunk;
        if(begin >= seq.length && split != 0u)
            return;
        const uint32_t end = seq.length - begin < chunk ? seq.length : begin + chunk;
        const bool     whole = seq.length <= chunk; // no other workgroup has positions of this sequence

        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t col = lane & 15u, quad = lane >> 4;
        const uint32_t wq = wave / WK, wk = wave % WK;
        const int64_t  prefix = (int64_t)seq.length - seq.tokens;

        // ---- this wave's rows of Q, as B operands: column `col`, d = 32 i + 8 quad + 0..7
        u32x4    qf[QB][D / 32u];
        uint32_t token[QB], qHead[QB]; // of the lane's row in each block
        bool     rowValid[QB];
#pragma unroll
        for(uint32_t a = 0; a < QB; ++a)
        {
            const uint32_t r = row0 + (wq * QB + a) * 16u + col;
            rowValid[a]      = r < rows;
            token[a]         = rowValid[a] ? r / p.group : 0u;
            qHead[a]         = head * p.group + (rowValid[a] ? r % p.group : 0u);
            const T* at      = reinterpret_cast<const T*>(p.q) + (int64_t)(seq.first + token[a]) * p.qToken + (int64_t)qHead[a] * p.qHead;
#pragma unroll
            for(uint32_t i = 0; i < D / 32u; ++i)
            {
                const uint32_t d = i * 32u + quad * 8u;
                qf[a][i]         = rowValid[a] && d < p.dim ? *reinterpret_cast<const u32x4*>(at + d) ^ p.signs : u32x4{0u, 0u, 0u, 0u};
            }
        }

        // ---- direct loads.  A tile is PB blocks of 16 positions, each within one page.  Lane i holds where the blocks 64 g + i of the chunk
        // lie, in blocks of the cache, for GROUPS of 64 at a time: a load of the table within the loop would have the compiler wait for every
        // direct load before it (the positions of a chunk and more are read at the start).
        const uint32_t ldsBase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
        const uint32_t myTiles = wk * BUFS * 2u * TILE;
        const uint32_t pageBlocks = p.pageSize / 16u, lastBlocks = end > begin ? (end - begin + 15u) / 16u : 0u;
        constexpr uint32_t GROUPS = 4;
        uint32_t           group = 0u, here, ahead[GROUPS];
#pragma unroll
        for(uint32_t g = 0; g < GROUPS; ++g)
            ahead[g] = placeOf(p, b, begin / 16u, g * 64u + lane, lastBlocks, pageBlocks);
#pragma unroll
        for(uint32_t g = 0; g < GROUPS; ++g)
            asm volatile("" : "+v"(ahead[g])); // (they are there from here on)
        here = ahead[0];
        // a lane's offsets: RPL rows a load, 16-byte pieces exchanged within the row; past the width of a head: outside the buffer, which loads zeros
        const uint32_t loadRow = lane / SLOTS, loadSlot = lane % SLOTS;
        uint32_t       offK[LOADS], offV[LOADS];
#pragma unroll
        for(uint32_t j = 0; j < LOADS; ++j)
        {
            const uint32_t inTile = (wq * LOADS + j) * RPL + loadRow;
            const uint32_t pieceK = loadSlot ^ swizzleK<D>(inTile), pieceV = loadSlot ^ swizzleV<D>(inTile);
            offK[j] = pieceK * 8u < p.dim ? inTile % 16u * (uint32_t)(p.kSlot * 2) + pieceK * 16u : OUTSIDE;
            offV[j] = pieceV * 8u < p.dim ? inTile % 16u * (uint32_t)(p.vSlot * 2) + pieceV * 16u : OUTSIDE;
        }
        const uint64_t baseK = reinterpret_cast<uint64_t>(p.k) + 2u * (uint64_t)(head * p.kHead), baseV = reinterpret_cast<uint64_t>(p.v) + 2u * (uint64_t)(head * p.vHead);
        auto issue = [&](uint32_t tile, uint32_t buf) __attribute__((always_inline)) {
            if(const uint32_t of = tile * PB / 64u; of != group)
            {
                group = of;
                if(of % GROUPS == 0u)
                {
#pragma unroll
                    for(uint32_t g = 0; g < GROUPS; ++g)
                        ahead[g] = placeOf(p, b, begin / 16u, (of + g) * 64u + lane, lastBlocks, pageBlocks);
#pragma unroll
                    for(uint32_t g = 0; g < GROUPS; ++g)
                        asm volatile("" : "+v"(ahead[g]));
                    here = ahead[0];
                }
                else
                    here = of % GROUPS == 1u ? ahead[1] : of % GROUPS == 2u ? ahead[2] : ahead[3];
            }
#pragma unroll
            for(uint32_t j = 0; j < LOADS; ++j)
            {
                const uint32_t piece = wq * LOADS + j; // which RPL rows of the tile
                const uint32_t block = tile * PB + piece * RPL / 16u; // of the chunk
                const uint32_t at   = __builtin_amdgcn_readlane(here, block % 64u);
                const uint32_t rows = at == ABSENT ? 0u : end - begin - block * 16u < 16u ? end - begin - block * 16u : 16u;
                // (a buffer that ends with the last row that there is: the others load zeros)
                r355::dma_i32x4 bufK = r355::rawBuffer(baseK + (uint64_t)at * (uint32_t)(p.kSlot * 32)), bufV = r355::rawBuffer(baseV + (uint64_t)at * (uint32_t)(p.vSlot * 32));
                bufK[2] = __builtin_amdgcn_readfirstlane(rows * (uint32_t)(p.kSlot * 2)), bufV[2] = __builtin_amdgcn_readfirstlane(rows * (uint32_t)(p.vSlot * 2));
                const uint32_t to = __builtin_amdgcn_readfirstlane(ldsBase + myTiles + buf * 2u * TILE + piece * 1024u);
                r355::loadToLds(bufK, offK[j], 0u, to);
                r355::loadToLds(bufV, offV[j], 0u, to + TILE);
            }
        };

        f32x4 o[QB][D / 16u];
        float top[QB], sum[QB]; // running maximum (of the row: the same in its four lanes) and the lane's share of the sum
#pragma unroll
        for(uint32_t a = 0; a < QB; ++a)
        {
            top[a] = -INFINITY, sum[a] = 0.0f;
#pragma unroll
            for(uint32_t d = 0; d < D / 16u; ++d)
                o[a][d] = f32x4{0, 0, 0, 0};
        }

        // MASKED: some row does not see all of the tile
        auto compute = [&](auto maskedTile, uint32_t pos0, uint32_t buf) __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(maskedTile)::value;
            // LDS addresses of the lane's row: the pieces of a row differ in an exclusive or with a constant (rows start on multiples of their
            // size), the blocks of 16 rows in a constant offset
            const uint32_t tileK = ldsBase + myTiles + buf * 2u * TILE, tileV = tileK + TILE;
            const uint32_t rowV = quad * 4u + (col >> 2);
            const uint32_t fromK = tileK + col * ROWB + (quad ^ swizzleK<D>(col)) * 16u, fromV = tileV + rowV * ROWB + (((col >> 1) & 1u) ^ swizzleV<D>(rowV)) * 16u + (col & 1u) * 8u;
            f32x4          s[QB][PB];
#pragma unroll
            for(uint32_t n = 0; n < PB; ++n)
#pragma unroll
                for(uint32_t a = 0; a < QB; ++a)
                    s[a][n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for(uint32_t i = 0; i < D / 32u; ++i)
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                {
                    const u32x4 kf = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)((fromK ^ (i * 64u)) + n * 16u * ROWB);
#pragma unroll
                    for(uint32_t a = 0; a < QB; ++a)
                        s[a][n] = r355::mfma32<T>(kf, qf[a][i], s[a][n]);
                }
            if constexpr(MASKED)
            {
#pragma unroll
                for(uint32_t a = 0; a < QB; ++a)
                {
                    // bit i: the row sees position pos0 + i
                    const uint32_t seen = rowValid[a] ? seenOf(p, seq.first + token[a], token[a], (int64_t)pos0 - prefix) : 0u;
                    const uint32_t mine = (end - pos0 < 32u ? seen & ((1u << (end - pos0)) - 1u) : seen) >> (quad * 4u);
#pragma unroll
                    for(uint32_t n = 0; n < PB; ++n)
#pragma unroll
                        for(uint32_t j = 0; j < 4; ++j)
                            s[a][n][j] = (mine >> (n * 16u + j)) & 1u ? s[a][n][j] : -INFINITY;
                }
            }
            uint32_t pf[QB][PB][2];
#pragma unroll
            for(uint32_t a = 0; a < QB; ++a)
            {
                float most = -INFINITY;
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                    most = fmaxf(fmaxf(fmaxf(s[a][n][0], s[a][n][1]), fmaxf(s[a][n][2], s[a][n][3])), most);
                most = most == -INFINITY ? most : most * p.scale2;
                most = maxOverQuads(most) - SHIFT;
                if(__any(most > top[a] + SLACK))
                {
                    const float next = fmaxf(most, top[a]);
                    const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[a] - next);
                    top[a]           = next;
                    sum[a] *= keep;
#pragma unroll
                    for(uint32_t d = 0; d < D / 16u; ++d)
                        o[a][d] *= keep;
                }
                const float base = top[a] == -INFINITY ? 0.0f : top[a];
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                {
#pragma unroll
                    for(uint32_t j = 0; j < 4; ++j)
                    {
                        s[a][n][j] = __builtin_amdgcn_exp2f(fmaf(s[a][n][j], p.scale2, -base));
                        sum[a] += s[a][n][j];
                    }
                    pf[a][n][0] = r355::pack2<T>(s[a][n][0], s[a][n][1]), pf[a][n][1] = r355::pack2<T>(s[a][n][2], s[a][n][3]);
                }
            }
            // A position that a row does not see has weight 0, and 0 times an infinity or a NaN is a NaN: where the tile holds one, those are
            // taken out of the product, and the rows that give them weight get them by two more (where (+inf or NaN) and where (-inf or NaN)).
            bool unfit = false;
            if constexpr(MASKED)
            {
                uint32_t found = 0u;
                for(uint32_t at = lane * 16u; at < TILE; at += 1024u)
                {
                    const u32x4 v = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(tileV + at);
                    found |= unfitHalves<T>(v[0]) | unfitHalves<T>(v[1]) | unfitHalves<T>(v[2]) | unfitHalves<T>(v[3]);
                }
                unfit = __any(found != 0u);
            }
            // V^T: lane t of 16 names four consecutive d of position t / 4 and receives four positions of d = t
            using lp = __attribute__((address_space(3))) vec<short, 4>*;
#pragma unroll
            for(uint32_t d = 0; d < D / 16u; ++d)
            {
                u32x2 vf[PB];
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                    vf[n] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)((fromV ^ (d * 32u)) + n * 16u * ROWB)));
                auto times = [&](const u32x2(&v)[PB], uint32_t a, f32x4 c) __attribute__((always_inline)) {
                    if constexpr(PB == 2u)
                        return r355::mfma32<T>(u32x4{v[0][0], v[0][1], v[1][0], v[1][1]}, u32x4{pf[a][0][0], pf[a][0][1], pf[a][1][0], pf[a][1][1]}, c);
                    else
                        return r355::mfma16<T>(v[0], u32x2{pf[a][0][0], pf[a][0][1]}, c);
                };
                if constexpr(MASKED)
                    if(unfit)
                    {
                        u32x2 up[PB], down[PB];
#pragma unroll
                        for(uint32_t n = 0; n < PB; ++n)
#pragma unroll
                            for(uint32_t w = 0; w < 2; ++w)
                            {
                                up[n][w] = unfitOnes<T>(vf[n][w], false), down[n][w] = unfitOnes<T>(vf[n][w], true);
                                vf[n][w] &= ~(unfitHalves<T>(vf[n][w]) * 0xFFFFu);
                            }
#pragma unroll
                        for(uint32_t a = 0; a < QB; ++a)
                        {
                            const f32x4 above = times(up, a, f32x4{0, 0, 0, 0}), below = times(down, a, f32x4{0, 0, 0, 0});
#pragma unroll
                            for(uint32_t e = 0; e < 4; ++e)
                            {
                                o[a][d][e] += above[e] != 0.0f ? INFINITY : 0.0f;
                                o[a][d][e] -= below[e] != 0.0f ? INFINITY : 0.0f;
                            }
                        }
                    }
#pragma unroll
                for(uint32_t a = 0; a < QB; ++a)
                    o[a][d] = times(vf, a, o[a][d]);
            }
        };

        const uint32_t tiles = begin < end ? (end - begin + NP - 1u) / NP : 0u;
        // the tiles that every row sees all of come first
        const int64_t  open = prefix < (int64_t)end ? prefix : (int64_t)end;
        const uint32_t clear = open > (int64_t)begin ? static_cast<uint32_t>(open - begin) / NP : 0u;
        uint32_t       buf = 0u, t = WQ == 1u ? wk : 0u;
        // tile t (of tiles wk, wk + 4, ... where every wave has its own)
        auto step = [&](auto maskedTile) __attribute__((always_inline)) {
            if constexpr(WQ == 1u)
            {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the reads of the buffer that is filled next have returned
                if(t + WK < tiles)
                {
                    issue(t + WK, buf ^ 1u);
                    r355::waitVmcnt<2u * LOADS>();
                }
                else
                    r355::waitVmcnt<0>();
                asm volatile("" ::: "memory");
                compute(maskedTile, begin + t * NP, buf);
                buf ^= 1u;
                t += WK;
            }
            else
            {
                if(t + 1u < tiles)
                    r355::waitVmcnt<2u * LOADS>();
                else
                    r355::waitVmcnt<0>();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                r355::ldsBarrier(); // everyone's part of tile t is there, and everyone is done with the buffer of tile t - 1
                if(t + 2u < tiles)
                    issue(t + 2u, buf == 0u ? 2u : buf - 1u);
                compute(maskedTile, begin + t * NP, buf);
                buf = buf == 2u ? 0u : buf + 1u;
                t += 1u;
            }
        };
        if(t < tiles)
            issue(t, 0u);
        if(WQ > 1u && tiles > 1u)
            issue(1u, 1u);
        while(t < clear)
            step(std::false_type{});
        while(t < tiles)
            step(std::true_type{});
#pragma unroll
        for(uint32_t a = 0; a < QB; ++a)
            sum[a] = sumOverQuads(sum[a]);

        // ---- the waves that took other positions of the same rows
        if constexpr(WK > 1u)
        {
            __syncthreads();
            float* const mine = reinterpret_cast<float*>(lds); // [WK][QB * 16][D], then [WK][QB * 16][2]
            float* const ends = mine + WK * QB * 16u * D;
#pragma unroll
            for(uint32_t a = 0; a < QB; ++a)
            {
                const uint32_t r = a * 16u + col;
#pragma unroll
                for(uint32_t d = 0; d < D / 16u; ++d)
                    *reinterpret_cast<f32x4*>(mine + ((wk * QB * 16u + r) * (D / 4u) + ((d * 4u + quad) ^ (col & 7u))) * 4u) = o[a][d];
                if(quad == 0u)
                    ends[(wk * QB * 16u + r) * 2u] = top[a], ends[(wk * QB * 16u + r) * 2u + 1u] = sum[a];
            }
            __syncthreads();
            // wave w adds up the d blocks w, w + 4, ... of every row
#pragma unroll
            for(uint32_t a = 0; a < QB; ++a)
            {
                const uint32_t r = a * 16u + col;
                float          most = -INFINITY, factor[WK], total = 0.0f;
#pragma unroll
                for(uint32_t w = 0; w < WK; ++w)
                    most = fmaxf(most, ends[(w * QB * 16u + r) * 2u]);
#pragma unroll
                for(uint32_t w = 0; w < WK; ++w)
                {
                    const float theirs = ends[(w * QB * 16u + r) * 2u];
                    factor[w]          = theirs == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(theirs - most);
                    total += factor[w] * ends[(w * QB * 16u + r) * 2u + 1u];
                }
                top[a] = most, sum[a] = total;
#pragma unroll
                for(uint32_t d = 0; d < D / 16u; ++d)
                {
                    if(d % WK != wk)
                        continue;
                    f32x4 all{0, 0, 0, 0};
#pragma unroll
                    for(uint32_t w = 0; w < WK; ++w)
                        all += factor[w] * *reinterpret_cast<const f32x4*>(mine + ((w * QB * 16u + r) * (D / 4u) + ((d * 4u + quad) ^ (col & 7u))) * 4u);
                    o[a][d] = all;
                }
            }
        }

        // ---- results: of the row, or this split's share
#pragma unroll
        for(uint32_t a = 0; a < QB; ++a)
        {
            if(!rowValid[a])
                continue;
            const uint64_t row = (uint64_t)(seq.first + token[a]) * p.heads + qHead[a], allRows = (uint64_t)p.totalTokens * p.heads;
            if(whole)
            {
                const float inverse = sum[a] == 0.0f ? 0.0f : 1.0f / sum[a];
                T* const    to      = reinterpret_cast<T*>(p.out) + (int64_t)(seq.first + token[a]) * p.oToken + (int64_t)qHead[a] * p.oHead;
#pragma unroll
                for(uint32_t d = 0; d < D / 16u; ++d)
                    if(d % WK == wk && d * 16u + quad * 4u < p.dim)
                        *reinterpret_cast<u32x2*>(to + d * 16u + quad * 4u)
                            = u32x2{r355::pack2<T>(o[a][d][0] * inverse, o[a][d][1] * inverse), r355::pack2<T>(o[a][d][2] * inverse, o[a][d][3] * inverse)};
                if(p.lse && wk == 0u && quad == 0u)
                    p.lse[row] = sum[a] == 0.0f ? -INFINITY : (top[a] + __builtin_amdgcn_logf(sum[a])) * 0.693147180559945309f;
            }
            else
            {
                float* const to = p.partial + ((uint64_t)split * allRows + row) * p.dim;
#pragma unroll
                for(uint32_t d = 0; d < D / 16u; ++d)
                    if(d % WK == wk && d * 16u + quad * 4u < p.dim)
                        *reinterpret_cast<f32x4*>(to + d * 16u + quad * 4u) = o[a][d];
                if(wk == 0u && quad == 0u)
                {
                    float* const ends = p.partial + (uint64_t)p.splits * allRows * p.dim + ((uint64_t)split * allRows + row) * 2u;
                    ends[0] = top[a], ends[1] = sum[a];
                }
            }
        }
    }

    // Adds up the splits of a row, in order.  L = D / 4 lanes a row, each four elements; the lanes take the splits' maxima and sums side by side.
    template <typename T, uint32_t D>
    __global__ void __launch_bounds__(256) treeMergeKernel(TreeParams p)
    {
        constexpr uint32_t L = D / 4u;
        const uint32_t     lane = threadIdx.x % L;
        const uint64_t     item = (uint64_t)blockIdx.x * (256u / L) + threadIdx.x / L; // (sequence, drafted token, head)
        const uint32_t     head = static_cast<uint32_t>(item % p.heads);
        const uint64_t     bt = item / p.heads;
        const uint32_t     b = static_cast<uint32_t>(bt / p.maxTokens), t = static_cast<uint32_t>(bt % p.maxTokens);
        if(b >= p.batch)
            return;
        const Sequence seq = sequenceOf(p, p.qStart[b], p.qStart[b + 1u], p.kvLen[b]);
        const uint32_t chunk = chunkOf(seq.length, p.splits);
        if(t >= seq.tokens || seq.length <= chunk)
            return;
        const uint32_t splits = (seq.length + chunk - 1u) / chunk;
        const uint64_t row = (uint64_t)(seq.first + t) * p.heads + head, allRows = (uint64_t)p.totalTokens * p.heads;
        const float*   ends = p.partial + (uint64_t)p.splits * allRows * p.dim + row * 2u;
        const float*   from = p.partial + row * p.dim + lane * 4u;
        float          most = -INFINITY;
        for(uint32_t s = lane; s < splits; s += L)
            most = fmaxf(most, ends[s * allRows * 2u]);
#pragma unroll
        for(uint32_t x = 1u; x < L; x *= 2u)
            most = fmaxf(most, __shfl_xor(most, x));
        float total = 0.0f;
        f32x4 all{0, 0, 0, 0};
        for(uint32_t s0 = 0; s0 < splits; s0 += L)
        {
            float theirs = -INFINITY, sum = 0.0f;
            if(s0 + lane < splits)
                theirs = ends[(s0 + lane) * allRows * 2u], sum = ends[(s0 + lane) * allRows * 2u + 1u];
            const float    factor = theirs == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(theirs - most);
            const uint32_t here   = splits - s0 < L ? splits - s0 : L;
#pragma unroll 8
            for(uint32_t s = 0; s < here; ++s)
            {
                const float f = __shfl(factor, s, L);
                total += f * __shfl(sum, s, L);
                if(lane * 4u < p.dim)
                    all += f * *reinterpret_cast<const f32x4*>(from + (s0 + s) * allRows * p.dim);
            }
        }
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        if(lane * 4u < p.dim)
            *reinterpret_cast<u32x2*>(reinterpret_cast<T*>(p.out) + (int64_t)(seq.first + t) * p.oToken + (int64_t)head * p.oHead + lane * 4u)
                = u32x2{r355::pack2<T>(all[0] * inverse, all[1] * inverse), r355::pack2<T>(all[2] * inverse, all[3] * inverse)};
        if(p.lse && lane == 0u)
            p.lse[row] = total == 0.0f ? -INFINITY : (most + __builtin_amdgcn_logf(total)) * 0.693147180559945309f;
    }

    struct Plan
    {
        uint32_t rowsPerGroup, rowTiles, splits;
    };

    Plan planOf(const r355_tree_attention_args& a, uint32_t mostSplits)
    {
        const uint64_t rows = (uint64_t)a.max_tokens * (a.heads / a.kv_heads);
        Plan           plan;
        plan.rowsPerGroup = rows <= 16u ? 16u : rows <= 32u ? 32u : a.head_dim <= 128u ? (rows <= 64u ? 64u : 128u) : 64u;
        plan.rowTiles     = static_cast<uint32_t>((rows + plan.rowsPerGroup - 1u) / plan.rowsPerGroup);
        const uint64_t groups = (uint64_t)a.batch * a.kv_heads * plan.rowTiles;
        const uint64_t cus    = r355::computeUnits();
        // one row tile for all rows: four workgroups a CU, as sequences differ in length (32 x 1 token of 820..8192 positions, 32 / 8 heads of 128:
        // two 136 us, four 128, eight 136); tiles of 128 rows: two (2 x 64 tokens over 65600: two 207, four 237: more partial results)
        uint64_t       want   = ((plan.rowsPerGroup <= 64u && a.head_dim <= 128u ? 4u : 2u) * cus + groups - 1u) / groups;
        const uint64_t least  = ((uint64_t)a.max_kv + LEAST_CHUNK - 1u) / LEAST_CHUNK;
        want                  = want < least ? want : least;
        want                  = want < mostSplits ? want : mostSplits;
        plan.splits           = static_cast<uint32_t>(want < 1u ? 1u : want > 256u ? 256u : want);
        return plan;
    }

    uint64_t bytesOf(const r355_tree_attention_args& a, uint32_t splits)
    {
        return splits > 1u ? (uint64_t)splits * a.total_tokens * a.heads * (a.head_dim + 2u) * 4u : 0u;
    }

    template <typename T, uint32_t D, uint32_t WQ, uint32_t QB>
    void launchTree(const TreeParams& p, const Plan& plan, hipStream_t s)
    {
        hipLaunchKernelGGL((treeKernel<T, D, WQ, QB>), dim3(p.columns * plan.rowTiles), dim3(WAVES * 64u), 0, s, p);
    }

    template <typename T>
    void launchType(const TreeParams& p, const Plan& plan, hipStream_t s)
    {
        auto byRows = [&](auto width) {
            constexpr uint32_t D = decltype(width)::value;
            if(plan.rowsPerGroup == 16u)
                launchTree<T, D, 1, 1>(p, plan, s);
            else if(plan.rowsPerGroup == 32u)
                launchTree<T, D, 1, 2>(p, plan, s);
            else if constexpr(D == 256u)
                launchTree<T, D, 4, 1>(p, plan, s);
            else if(plan.rowsPerGroup == 64u)
                launchTree<T, D, 1, 4>(p, plan, s);
            else
                launchTree<T, D, 4, 2>(p, plan, s);
            if(plan.splits > 1u)
            {
                const uint64_t items = (uint64_t)p.batch * p.maxTokens * p.heads;
                hipLaunchKernelGGL((treeMergeKernel<T, D>), dim3(static_cast<uint32_t>((items + 1024u / D - 1u) / (1024u / D))), dim3(256), 0, s, p);
            }
        };
        using std::integral_constant;
        if(p.dim <= 64u)
            byRows(integral_constant<uint32_t, 64>{});
        else if(p.dim <= 128u)
            byRows(integral_constant<uint32_t, 128>{});
        else
            byRows(integral_constant<uint32_t, 256>{});
    }

    // everything that the sizes alone decide
    int checkSizes(const r355_tree_attention_args& a)
    {
        if(a.type != R355_F16 && a.type != R355_BF16)
            return r355::fail(R355_ERR_UNSUPPORTED, "tree_attention: f16 and bf16");
        if(a.heads == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.page_size == 0)
            return r355::fail(R355_ERR_BAD_ARG, "tree_attention: heads, kv_heads, head_dim and page_size must be non-zero");
        if(a.heads % a.kv_heads)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: heads=%u must be a multiple of kv_heads=%u", a.heads, a.kv_heads);
        if(a.head_dim % 8u || a.head_dim > 256u)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: head_dim=%u must be a multiple of 8 and at most 256", a.head_dim);
        if(a.page_size % 16u)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: page_size=%u must be a multiple of 16", a.page_size);
        if(a.mask && (uint64_t)a.mask_words * 64u < a.max_tokens)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: %u words of mask are less than %u drafted tokens", a.mask_words, a.max_tokens);
        if(a.max_kv > 0x40000000u || a.total_tokens > 0x40000000u || a.max_tokens > 0x40000000u)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: at most 2^30 positions and tokens");
        if((uint64_t)((uint64_t)a.max_kv + a.page_size - 1u) / a.page_size > a.table_stride && a.batch > 0)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: rows of %u pages hold fewer than max_kv=%u positions", a.table_stride, a.max_kv);
        if((uint64_t)a.max_tokens * (a.heads / a.kv_heads) > 0x40000000u)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: max_tokens=%u times %u heads per key head is over 2^30", a.max_tokens, a.heads / a.kv_heads);
        const uint64_t groups = ((uint64_t)a.batch * a.kv_heads + 8u) * (((uint64_t)a.max_tokens * (a.heads / a.kv_heads) + 15u) / 16u);
        if(groups > r355::MAX_GROUPS || (uint64_t)a.batch * a.max_tokens * a.heads / 4u >= r355::MAX_GROUPS)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: too many sequences, heads and drafted tokens for one launch");
        return R355_OK;
    }
} // namespace

extern "C" size_t r355_tree_attention_workspace_bytes(const r355_tree_attention_args* args)
{
    if(!args || checkSizes(*args) != R355_OK || args->batch == 0 || args->total_tokens == 0 || args->max_tokens == 0)
        return 0;
    return bytesOf(*args, planOf(*args, 256u).splits);
}

extern "C" int r355_tree_attention(const r355_tree_attention_args* args, void* stream)
{
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "tree_attention: null arguments");
    const r355_tree_attention_args& a = *args;
    if(const int rc = checkSizes(a); rc != R355_OK)
        return rc;
    if(a.batch == 0 || a.total_tokens == 0 || a.max_tokens == 0)
        return R355_OK;
    if(!a.q || !a.k || !a.v || !a.out || !a.table || !a.q_start || !a.kv_len)
        return r355::fail(R355_ERR_BAD_ARG, "tree_attention: null pointer");
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.k_slot_stride, a.k_head_stride, a.v_slot_stride, a.v_head_stride};
    for(const int64_t stride : strides)
        if(stride % 8)
            return r355::fail(R355_ERR_MISALIGNED, "tree_attention: strides of q, k and v must be multiples of 8 elements");
    if(a.out_token_stride % 4 || a.out_head_stride % 4)
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: strides of out must be multiples of 4 elements");
    if(!r355::aligned(a.q, 16) || !r355::aligned(a.k, 16) || !r355::aligned(a.v, 16) || !r355::aligned(a.out, 8))
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: q, k and v need 16-byte alignment, out 8-byte alignment");
    if(a.lse && !r355::aligned(a.lse, 4))
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: lse needs 4-byte alignment");
    if(a.mask && !r355::aligned(a.mask, 8))
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: the mask needs 8-byte alignment");
    if(a.k_slot_stride < (int64_t)a.head_dim || a.v_slot_stride < (int64_t)a.head_dim || a.k_slot_stride > (1 << 25) || a.v_slot_stride > (1 << 25))
        return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: slot strides must be head_dim to 2^25 elements");
    if((uint64_t)a.pages * (a.page_size / 16u) >= 0xFFFFFFFFull)
        return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: a cache of 2^36 slots and more");
    if(a.workspace && !r355::aligned(a.workspace, 16))
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: the workspace needs 16-byte alignment");
    const uint64_t perSplit = (uint64_t)a.total_tokens * a.heads * (a.head_dim + 2u) * 4u;
    const uint64_t fit      = a.workspace ? a.workspace_bytes / perSplit : 0u;
    const Plan     plan     = planOf(a, static_cast<uint32_t>(fit < 256u ? fit : 256u));

    TreeParams p;
    p.q = static_cast<const char*>(a.q), p.k = static_cast<const char*>(a.k), p.v = static_cast<const char*>(a.v), p.out = static_cast<char*>(a.out), p.lse = a.lse;
    p.table = a.table, p.qStart = a.q_start, p.kvLen = a.kv_len, p.mask = a.mask, p.partial = static_cast<float*>(a.workspace);
    p.qToken = a.q_token_stride, p.qHead = a.q_head_stride, p.kSlot = a.k_slot_stride, p.kHead = a.k_head_stride, p.vSlot = a.v_slot_stride, p.vHead = a.v_head_stride;
    p.oToken = a.out_token_stride, p.oHead = a.out_head_stride;
    p.batch = a.batch, p.heads = a.heads, p.kvHeads = a.kv_heads, p.group = a.heads / a.kv_heads, p.dim = a.head_dim;
    p.totalTokens = a.total_tokens, p.maxTokens = a.max_tokens, p.maxKv = a.max_kv;
    p.pageSize = a.page_size, p.pages = a.pages, p.tableStride = a.table_stride, p.maskWords = a.mask_words;
    p.splits = plan.splits, p.columns = (a.batch * a.kv_heads * plan.splits + 7u) / 8u * 8u; // (row tiles of one split on one XCD)
    p.scale2 = std::fmax(static_cast<float>(std::fabs(a.scale) * 1.4426950408889634), 1.17549435e-38f);
    p.signs  = a.scale < 0.0 ? 0x80008000u : 0u;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    r355::beginCall();
    if(a.type == R355_F16)
        launchType<_Float16>(p, plan, s);
    else
        launchType<__bf16>(p, plan, s);
    return r355::checkLaunch("tree_attention");
}
