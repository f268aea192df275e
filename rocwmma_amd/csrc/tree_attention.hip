// Attention of drafted tokens over a paged cache, on gfx950 matrix cores.  No counterpart in the reference.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i),  lse_i = log sum_j exp(scale q_i . k_j)
//
// over the positions j that row i sees: all of the prefix and, of the drafted tokens (whose keys and values are the last rows of the
// cache), those whose bit is set in the row's mask; without a mask those up to the row itself.
//
// The rows of a key head are its query heads times the drafted tokens of a sequence, 16 QB of them to a wave.  A wave multiplies
// S^T = K Q^T (16 positions x 16 rows a matrix instruction), so that a lane holds four consecutive positions of one row: the running
// maximum and sum of the softmax stay within a lane's registers but for two exchanges, and P^T is, as it lies, the B operand
// of O^T = V^T P^T.  K and V go to LDS by direct loads, a 16-byte piece of a row in a slot that depends on the row, so that neither the reads
// of K (16 rows at one place) nor the transposing reads of V meet in a bank.
//
// WQ waves of a workgroup take different rows (and share the tiles), the others different positions.  WQ = 1: four waves on positions, each of which fills and
// reads tiles of its own, without a barrier.  WQ = 4 and 8: as many waves, all on rows, with the scores of the next tile made beside the exponentials of this one.
// The positions of all sequences are split into shares of one length; partial results (f32) meet in a second kernel, in order.
//
// What bounds it, 32 / 8 heads of 128: with single tokens the bytes of the cache (32 tokens over 820 .. 8192 positions: 124 us, 4.9 TB/s), with a
// short cache two launches and the first reads' latency (one token over 700: 11.7 us); with 64 tokens over 65600 positions the matrix and vector
// instructions under the power limit (two sequences: 152 us, 675 TFLOP/s; their bytes alone are 62 us at the rate of reads).  A chunk of a prompt takes the
// time of all its positions: every tile of rows goes over those after its last token too, masked (2048 tokens after 6144: 429 us, 561 TFLOP/s of what is seen;
// 8192 without a prefix: 2109 us, 261).
#include <hip/hip_runtime.h>

#include <cmath>
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

    constexpr uint32_t LEAST_CHUNK = 256; // positions of a workgroup at least
    constexpr uint32_t WHOLE = 0xFFFFFF80u; // a chunk that no sequence fills
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
        float*          partial; // [shares][maxTokens * heads][dim], then [shares][maxTokens * heads][2]: maximum (in powers of two) and sum
        int64_t         qToken, qHead, kSlot, kHead, vSlot, vHead, oToken, oHead; // strides in elements
        uint32_t        batch, heads, kvHeads, group, dim, totalTokens, maxTokens, maxKv;
        uint32_t        pageSize, pages, tableStride, maskWords;
        uint32_t        shares, columns; // shares of all sequences' positions (as many as sequences: none is split); (share, key head) pairs, a multiple of eight
        float           scale2; // |scale| * log2(e), at least the smallest normal number (times minus infinity it is minus infinity)
        uint32_t        signs; // what turns the signs of two elements of q: the scale's
    };

    // The positions of all sequences are split into at most `shares` shares of the same length (LEAST_CHUNK at least, a multiple of it), each of one
    // sequence: a long sequence gets as many more of them as it is longer.  With L positions in all and n sequences a share of
    // L / (shares - n) leaves room for the last, shorter share of every sequence.
    struct Share
    {
        uint32_t sequence, split, chunk; // whose share, which of its, positions of a share
    };
    __device__ __forceinline__ uint32_t lengthOf(const TreeParams& p, int32_t length)
    {
        const uint32_t n = length < 0 ? 0u : static_cast<uint32_t>(length);
        return n < p.maxKv ? n : p.maxKv;
    }
    // (by a whole wave)
    __device__ __forceinline__ uint32_t chunkFrom(const TreeParams& p, uint32_t blocks)
    {
#pragma unroll
        for(uint32_t x = 1u; x < 64u; x *= 2u)
            blocks += __shfl_xor(blocks, x);
        const uint32_t each = (blocks + p.shares - p.batch - 1u) / (p.shares - p.batch);
        return __builtin_amdgcn_readfirstlane((each > 1u ? each : 1u) * LEAST_CHUNK);
    }
    // the same of one sequence
    __device__ __forceinline__ uint32_t chunkAlone(const TreeParams& p, uint32_t length)
    {
        const uint32_t each = ((length + LEAST_CHUNK - 1u) / LEAST_CHUNK + p.shares - 1u) / p.shares;
        return (each > 1u ? each : 1u) * LEAST_CHUNK;
    }
    __device__ __forceinline__ uint32_t chunkOf(const TreeParams& p, uint32_t lane)
    {
        if(p.shares <= p.batch)
            return WHOLE;
        if(p.batch == 1u)
            return chunkAlone(p, __builtin_amdgcn_readfirstlane(lengthOf(p, p.kvLen[0])));
        uint32_t blocks = 0u; // of LEAST_CHUNK positions
        for(uint32_t first = 0; first < p.batch; first += 64u)
            if(first + lane < p.batch)
                blocks += (lengthOf(p, p.kvLen[first + lane]) + LEAST_CHUNK - 1u) / LEAST_CHUNK;
        return chunkFrom(p, blocks);
    }
    __device__ __forceinline__ uint32_t splitsOf(uint32_t length, uint32_t chunk)
    {
        return length > chunk ? (length + chunk - 1u) / chunk : 1u; // (a sequence without positions has a share, which writes its zeros)
    }

    struct Sequence
    {
        uint32_t first, tokens, length; // first row of q, drafted tokens, cached positions
    };

    // what the arrays say of a sequence, held to what the host was told
    __device__ __forceinline__ Sequence sequenceOf(const TreeParams& p, int32_t from, int32_t to, int32_t len)
    {
        Sequence s;
        s.first  = from < 0 ? 0u : static_cast<uint32_t>(from);
        s.first  = s.first < p.totalTokens ? s.first : p.totalTokens;
        s.tokens = to > static_cast<int32_t>(s.first) ? static_cast<uint32_t>(to) - s.first : 0u;
        s.tokens = s.tokens < p.maxTokens ? s.tokens : p.maxTokens;
        s.tokens = s.tokens < p.totalTokens - s.first ? s.tokens : p.totalTokens - s.first;
        s.length = lengthOf(p, len);
        return s;
    }

    // The sequence and split of share `share`, and the sequence itself (share.sequence: batch where there is no such share).  The arrays are read by
    // the lanes, all three before anything of them is used.
    __device__ __forceinline__ Share shareOf(const TreeParams& p, uint32_t share, uint32_t lane, Sequence& seq)
    {
        const bool split = p.shares > p.batch;
        if(p.batch == 1u)
        {
            seq = sequenceOf(p, __builtin_amdgcn_readfirstlane(p.qStart[0]), __builtin_amdgcn_readfirstlane(p.qStart[1]), __builtin_amdgcn_readfirstlane(p.kvLen[0]));
            const uint32_t chunk = split ? chunkAlone(p, seq.length) : WHOLE;
            return Share{share < splitsOf(seq.length, chunk) ? 0u : 1u, share, chunk};
        }
        Share      s{p.batch, 0u, WHOLE};
        uint32_t   before = 0u;
        for(uint32_t first = split ? 0u : share; first < p.batch; first += 64u)
        {
            const uint32_t i = first + lane < p.batch ? first + lane : p.batch - 1u;
            const int32_t  from = p.qStart[i], to = p.qStart[i + 1u], len = p.kvLen[i];
            uint32_t       at = 0u;
            if(split)
            {
                const uint32_t length = lengthOf(p, len);
                if(first == 0u)
                    s.chunk = p.batch <= 64u ? chunkFrom(p, lane < p.batch ? (length + LEAST_CHUNK - 1u) / LEAST_CHUNK : 0u) : chunkOf(p, lane);
                const uint32_t own  = first + lane < p.batch ? splitsOf(length, s.chunk) : 0u;
                uint32_t       upTo = own;
#pragma unroll
                for(uint32_t x = 1u; x < 64u; x *= 2u)
                {
                    const uint32_t left = __shfl_up(upTo, x);
                    upTo += lane >= x ? left : 0u;
                }
                const uint64_t holds = __ballot(own != 0u && share < before + upTo);
                if(holds == 0u)
                {
                    before += __builtin_amdgcn_readlane(upTo, 63);
                    continue;
                }
                at      = static_cast<uint32_t>(__builtin_ctzll(holds));
                s.split = share - before - (__builtin_amdgcn_readlane(upTo, at) - __builtin_amdgcn_readlane(own, at));
            }
            s.sequence = first + at;
            seq        = sequenceOf(p, __builtin_amdgcn_readlane(from, at), __builtin_amdgcn_readlane(to, at), __builtin_amdgcn_readlane(len, at));
            break;
        }
        return s;
    }
    // the first share of sequence b
    __device__ __forceinline__ uint32_t firstShareOf(const TreeParams& p, uint32_t b, uint32_t chunk, uint32_t lane)
    {
        uint32_t before = 0u;
        for(uint32_t i = lane; i < b; i += 64u)
            before += splitsOf(lengthOf(p, p.kvLen[i]), chunk);
#pragma unroll
        for(uint32_t x = 1u; x < 64u; x *= 2u)
            before += __shfl_xor(before, x);
        return __builtin_amdgcn_readfirstlane(before);
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
    // ... 1 in each half whose mantissa is not zero
    template <typename T>
    __device__ __forceinline__ uint32_t mantissaHalves(uint32_t v)
    {
        constexpr uint32_t MANTISSA = std::is_same_v<T, __bf16> ? 0x007F007Fu : 0x03FF03FFu, BITS = std::is_same_v<T, __bf16> ? 7u : 10u;
        return (((v & MANTISSA) + MANTISSA) >> BITS) & 0x00010001u;
    }
    template <typename T>
    constexpr uint32_t ONE = std::is_same_v<T, __bf16> ? 0x3F80u : 0x3C00u;

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
    __global__ void __launch_bounds__(WQ == 8u ? 512 : 256, WQ == 4u ? 2 : 1) treeKernel(TreeParams p)
    {
        constexpr uint32_t WAVES = WQ == 8u ? 8u : 4u, WK = WAVES / WQ;
        constexpr uint32_t NP    = D == 256u ? 16u : D == 128u || WQ > 1u ? 32u : 64u; // positions of a tile
        constexpr uint32_t PB    = NP / 16u;
        constexpr uint32_t ROWB  = D * 2u, SLOTS = ROWB / 16u; // bytes and 16-byte pieces of a row
        constexpr uint32_t RPL   = 64u / SLOTS; // rows of a direct load
        constexpr uint32_t TILE  = NP * ROWB;
        constexpr uint32_t BUFS  = WQ == 1u ? 2u : 4u;
        constexpr uint32_t LOADS = 2u * NP / RPL / WQ; // direct loads of a wave per tile: those of K, then those of V, shared out
        constexpr uint32_t LDS   = WK * BUFS * 2u * TILE;
        constexpr uint32_t MERGE = WK > 1u ? WK * QB * 16u * (D + 2u) * 4u : 0u;
        // weights are held relative to 2^-SHIFT of the largest: in f16 those under 2^-14 of it, of which a long row has many, stay normal numbers
        constexpr float SHIFT = std::is_same_v<T, __bf16> ? 0.0f : 10.0f;
        // ... and the maximum is taken as it was until it has grown by more than this: the sums are scaled anew in few tiles, and the largest weight is 2^(SHIFT + SLACK)
        constexpr float SLACK = 4.0f;
        static_assert(LDS <= 160u * 1024u, "LDS");
        __shared__ __attribute__((aligned(1024))) char lds[LDS > MERGE ? LDS : MERGE];

        const uint32_t tile0 = blockIdx.x / p.columns, column = blockIdx.x % p.columns, head = column % p.kvHeads, index = column / p.kvHeads;
        if(index >= p.shares)
            return;
        Sequence       seq;
        const Share    share = shareOf(p, index, threadIdx.x & 63u, seq);
        const uint32_t b     = share.sequence;
        if(b >= p.batch)
            return;
        const uint32_t rows = seq.tokens * p.group, row0 = tile0 * WQ * QB * 16u;
        if(row0 >= rows)
            return;
        const bool     whole = seq.length <= share.chunk; // no other workgroup has positions of this sequence
        const uint32_t begin = whole ? 0u : share.split * share.chunk;
        const uint32_t end   = seq.length - begin < share.chunk ? seq.length : begin + share.chunk;

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
        constexpr uint32_t GROUPS = WQ == 1u ? 4u : 2u;
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
        uint32_t       off[LOADS];
#pragma unroll
        for(uint32_t j = 0; j < LOADS; ++j)
        {
            const uint32_t item = wq * LOADS + j, inTile = item % (NP / RPL) * RPL + loadRow;
            const uint32_t piece = loadSlot ^ (item < NP / RPL ? swizzleK<D>(inTile) : swizzleV<D>(inTile));
            off[j] = piece * 8u < p.dim ? inTile % 16u * (uint32_t)((item < NP / RPL ? p.kSlot : p.vSlot) * 2) + piece * 16u : OUTSIDE;
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
                    here = of % GROUPS == 1u ? ahead[1] : of % GROUPS == 2u ? ahead[GROUPS - 2u] : ahead[GROUPS - 1u];
            }
#pragma unroll
            for(uint32_t j = 0; j < LOADS; ++j)
            {
                const uint32_t item = wq * LOADS + j, piece = item % (NP / RPL); // K or V, and which RPL rows of the tile
                const bool     isK  = item < NP / RPL;
                const uint32_t block = tile * PB + piece * RPL / 16u; // of the chunk
                const uint32_t at    = __builtin_amdgcn_readlane(here, block % 64u);
                const uint32_t rows  = at == ABSENT ? 0u : end - begin - block * 16u < 16u ? end - begin - block * 16u : 16u;
                const uint32_t slot  = static_cast<uint32_t>(isK ? p.kSlot : p.vSlot);
                // (a buffer that ends with the last row that there is: the others load zeros)
                r355::dma_i32x4 rsrc = r355::rawBuffer((isK ? baseK : baseV) + (uint64_t)at * (slot * 32u));
                rsrc[2]              = __builtin_amdgcn_readfirstlane(rows * slot * 2u);
                r355::loadToLds(rsrc, off[j], 0u, __builtin_amdgcn_readfirstlane(ldsBase + myTiles + buf * 2u * TILE + (isK ? 0u : TILE) + piece * 1024u));
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

        // S^T of a tile.  LDS addresses of the lane's row: the pieces of a row differ in an exclusive or with a constant (rows start on multiples of their
        // size), the blocks of 16 rows in a constant offset.
        uint32_t atK[D / 32u], atV[D / 16u]; // in the first buffer
        {
            const uint32_t rowV = quad * 4u + (col >> 2), tile = ldsBase + myTiles;
#pragma unroll
            for(uint32_t i = 0; i < D / 32u; ++i)
                atK[i] = (tile + col * ROWB + (quad ^ swizzleK<D>(col)) * 16u) ^ (i * 64u);
#pragma unroll
            for(uint32_t d = 0; d < D / 16u; ++d)
                atV[d] = (tile + TILE + rowV * ROWB + (((col >> 1) & 1u) ^ swizzleV<D>(rowV)) * 16u + (col & 1u) * 8u) ^ (d * 32u);
        }
        auto scores = [&](auto buf, f32x4(&s)[QB][PB]) __attribute__((always_inline)) {
#pragma unroll
            for(uint32_t i = 0; i < D / 32u; ++i)
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                {
                    const u32x4 kf = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(atK[i] + (buf * 2u * TILE + n * 16u * ROWB));
#pragma unroll
                    for(uint32_t a = 0; a < QB; ++a)
                        s[a][n] = r355::mfma32<T>(kf, qf[a][i], i != 0u ? s[a][n] : f32x4{0, 0, 0, 0});
                }
        };
        // The weights of a tile and their product with V.  masked: some row does not see all of the tile.  between(): what can go on beside the exponentials.
        // (With few rows one copy of the code for both: a call over few positions takes about as long as its instructions take to arrive, some 25 ns for 64 bytes.)
        auto weigh = [&](auto ahead, auto masked, uint32_t pos0, auto buf, f32x4(&s)[QB][PB], auto&& between) __attribute__((always_inline)) {
            if(masked)
            {
#pragma unroll
                for(uint32_t a = 0; a < QB; ++a)
                {
#pragma unroll
                    for(uint32_t w = 0; w < PB; w += 2u)
                    {
                        // bit i: the row sees position from + i
                        const uint32_t from = pos0 + w * 16u;
                        const uint32_t seen = rowValid[a] && from < end ? seenOf(p, seq.first + token[a], token[a], (int64_t)from - prefix) : 0u;
                        const uint32_t mine = (from < end && end - from < 32u ? seen & ((1u << (end - from)) - 1u) : seen) >> (quad * 4u);
#pragma unroll
                        for(uint32_t n = w; n < w + 2u && n < PB; ++n)
#pragma unroll
                            for(uint32_t j = 0; j < 4; ++j)
                                s[a][n][j] = (mine >> ((n - w) * 16u + j)) & 1u ? s[a][n][j] : -INFINITY;
                    }
                }
            }
#pragma unroll
            for(uint32_t a = 0; a < QB; ++a)
            {
                // the lane's largest score; what the row's four lanes have is compared only where one has grown too large
                float most = -INFINITY;
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                    most = fmaxf(fmaxf(fmaxf(s[a][n][0], s[a][n][1]), fmaxf(s[a][n][2], s[a][n][3])), most);
                most = most == -INFINITY ? most : most * p.scale2 - SHIFT;
                if(__any(most > top[a] + SLACK))
                {
                    const float next = fmaxf(maxOverQuads(most), top[a]);
                    const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[a] - next);
                    top[a]           = next;
                    sum[a] *= keep;
#pragma unroll
                    for(uint32_t d = 0; d < D / 16u; ++d)
                        o[a][d] *= keep;
                }
            }
            // V^T: lane t of 16 names four consecutive d of position t / 4 and receives four positions of d = t.  (ahead: all of it is asked for
            // before the exponentials; next to the product each read is waited for.)
            using lp = __attribute__((address_space(3))) vec<short, 4>*;
            auto v   = [&](uint32_t d, u32x2(&to)[PB]) __attribute__((always_inline)) {
#pragma unroll
                for(uint32_t n = 0; n < PB; ++n)
                    to[n] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)(atV[d] + (buf * 2u * TILE + n * 16u * ROWB))));
            };
            constexpr uint32_t EARLY = decltype(ahead)::value ? D / 16u : 0u;
            u32x2              early[EARLY + 1u][PB];
#pragma unroll
            for(uint32_t d = 0; d < EARLY; ++d)
                v(d, early[d]);
            if constexpr(EARLY != 0u)
                __builtin_amdgcn_sched_barrier(0);
            uint32_t pf[QB][PB][2];
            between();
            // (shared tiles that are masked: nothing is moved up here, for want of registers)
            constexpr bool TIGHT = WQ > 1u && !decltype(ahead)::value;
            if constexpr(TIGHT)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for(uint32_t a = 0; a < QB; ++a)
            {
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
                    // (Rounded to 16 bits, as the second operand of the product with V has to be: at most what the rounding of the result is, and averaged over the
                    // positions.  Relative error of results in all, against 64 bits, 32 tokens over 820 .. 8192 positions: bf16 0.0020, of which the result's own
                    // rounding is 0.0017; f16 0.00025 and 0.00021.  The sum takes them unrounded, so lse has none of it.)
                    pf[a][n][0] = r355::pack2<T>(s[a][n][0], s[a][n][1]), pf[a][n][1] = r355::pack2<T>(s[a][n][2], s[a][n][3]);
                }
            }
            auto times = [&](const u32x2(&of)[PB], uint32_t a, f32x4 c) __attribute__((always_inline)) {
                if constexpr(PB == 1u)
                    return r355::mfma16<T>(of[0], u32x2{pf[a][0][0], pf[a][0][1]}, c);
                else
                {
#pragma unroll
                    for(uint32_t n = 0; n < PB; n += 2u)
                        c = r355::mfma32<T>(u32x4{of[n][0], of[n][1], of[n + 1u][0], of[n + 1u][1]}, u32x4{pf[a][n][0], pf[a][n][1], pf[a][n + 1u][0], pf[a][n + 1u][1]}, c);
                    return c;
                }
            };
            // A position that a row does not see has weight 0, and 0 times an infinity or a NaN is a NaN.  Where the tile holds one, the product is made with zeros in
            // their place; two more, with ones in the place of each sign's (a NaN: of both) and zeros elsewhere, are more than 0 where a row gives one a weight.
            if(masked)
            {
                uint32_t found = 0u;
#pragma unroll 1
                for(uint32_t at = lane * 16u; at < TILE; at += 1024u)
                {
                    const u32x4 x = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(ldsBase + myTiles + buf * 2u * TILE + TILE + at);
                    found |= unfitHalves<T>(x[0]) | unfitHalves<T>(x[1]) | unfitHalves<T>(x[2]) | unfitHalves<T>(x[3]);
                }
                if(__any(found != 0u))
                {
#pragma unroll
                    for(uint32_t d = 0; d < D / 16u; ++d)
                    {
#pragma unroll
                        for(uint32_t of = 0; of < 3u; ++of) // the numbers, the positive ones, the negative ones
                        {
                            u32x2 x[PB];
                            asm volatile("" ::: "memory"); // (read again each time: kept, they would not fit)
                            if constexpr(TIGHT)
                                __builtin_amdgcn_sched_barrier(0);
                            v(d, x);
#pragma unroll
                            for(uint32_t n = 0; n < PB; ++n)
#pragma unroll
                                for(uint32_t w = 0; w < 2u; ++w)
                                {
                                    const uint32_t was = x[n][w], unfit = unfitHalves<T>(was);
                                    x[n][w] = of == 0u ? was & ~(unfit * 0xFFFFu) : (unfit & ((of == 1u ? ~was : was) >> 15 | mantissaHalves<T>(was))) * ONE<T>;
                                }
#pragma unroll
                            for(uint32_t a = 0; a < QB; ++a)
                                if(of == 0u)
                                    o[a][d] = times(x, a, o[a][d]);
                                else
                                {
                                    const f32x4 seen = times(x, a, f32x4{0, 0, 0, 0});
#pragma unroll
                                    for(uint32_t e = 0; e < 4u; ++e)
                                        o[a][d][e] += seen[e] > 0.0f ? of == 1u ? INFINITY : -INFINITY : 0.0f;
                                }
                        }
                    }
                    return;
                }
            }
#pragma unroll
            for(uint32_t d = 0; d < D / 16u; ++d)
            {
                u32x2 vf[PB];
                if constexpr(EARLY != 0u)
#pragma unroll
                    for(uint32_t n = 0; n < PB; ++n)
                        vf[n] = early[d < EARLY ? d : 0u][n];
                else
                {
                    if constexpr(TIGHT)
                        if(d % 4u == 0u)
                            __builtin_amdgcn_sched_barrier(0);
                    v(d, vf);
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
        f32x4 held[QB][PB];
        // WQ > 1: the scores of tile t + 1 are made beside the exponentials of tile t (after the last tile: of what the buffer holds, and not used)
        [[maybe_unused]] f32x4 other[QB][PB];
        auto arrive = [&]() __attribute__((always_inline)) {
            if(t + 2u < tiles)
                r355::waitVmcnt<LOADS>();
            else
                r355::waitVmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            r355::ldsBarrier(); // everyone's part of tile t + 1 is there, and everyone is done with the buffer of tile t - 1
        };
        auto step = [&](auto ahead, auto masked) __attribute__((always_inline)) {
            if constexpr(WQ == 1u)
            {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the reads of the buffer that is filled next have returned
                if(t + WK < tiles)
                {
                    issue(t + WK, buf ^ 1u);
                    r355::waitVmcnt<LOADS>();
                }
                else
                    r355::waitVmcnt<0>();
                asm volatile("" ::: "memory");
                scores(buf, held);
                weigh(ahead, masked, begin + t * NP, buf, held, [] {});
                buf ^= 1u;
                t += WK;
            }
            else
            {
                arrive();
                if(t + 3u < tiles)
                    issue(t + 3u, (buf + 3u) % BUFS);
                if constexpr(decltype(ahead)::value)
                {
                    weigh(ahead, masked, begin + t * NP, buf, held, [&]() __attribute__((always_inline)) { scores((buf + 1u) % BUFS, other); });
#pragma unroll
                    for(uint32_t a = 0; a < QB; ++a)
#pragma unroll
                        for(uint32_t n = 0; n < PB; ++n)
                            held[a][n] = other[a][n];
                }
                else // (the few masked tiles: one after the other, for want of registers)
                {
                    weigh(ahead, masked, begin + t * NP, buf, held, [] {});
                    scores((buf + 1u) % BUFS, held);
                }
                buf = (buf + 1u) % BUFS;
                t += 1u;
            }
        };
        if(t < tiles)
            issue(t, 0u);
        if constexpr(WQ > 1u)
        {
            if(tiles > 1u)
                issue(1u, 1u);
            if(tiles > 2u)
                issue(2u, 2u);
            if(tiles > 2u)
                r355::waitVmcnt<2u * LOADS>();
            else if(tiles > 1u)
                r355::waitVmcnt<LOADS>();
            else
                r355::waitVmcnt<0>();
            r355::ldsBarrier();
            scores(0u, held);
            // Long caches: four tiles at a time, so that LDS addresses and the places of the scores are the same each time around (2 x 64 tokens over 65600:
            // 163 -> 154 us; where a workgroup has few tiles the code takes longer to arrive: 8 trees of up to 48 tokens over 4099 28 -> 33 us)
            static_assert(BUFS == 4u, "one tile of a turn for each buffer");
            while(WQ == 8u && t + 3u < clear)
                each<WQ == 8u ? 4u : 0u>([&](auto at) __attribute__((always_inline)) {
                    constexpr uint32_t i = decltype(at)::value;
                    arrive();
                    if(t + 3u < tiles)
                        issue(t + 3u, (i + 3u) % 4u);
                    const std::integral_constant<uint32_t, i> here;
                    const std::integral_constant<uint32_t, (i + 1u) % 4u> next;
                    if constexpr(i % 2u == 0u)
                        weigh(std::true_type{}, std::false_type{}, begin + t * NP, here, held, [&]() __attribute__((always_inline)) { scores(next, other); });
                    else
                        weigh(std::true_type{}, std::false_type{}, begin + t * NP, here, other, [&]() __attribute__((always_inline)) { scores(next, held); });
                    t += 1u;
                });
        }
        if constexpr(WQ == 1u)
            while(t < tiles)
                step(std::false_type{}, t >= clear);
        else
        {
            while(t < clear)
                step(std::true_type{}, std::false_type{});
            while(t < tiles)
                step(std::false_type{}, std::true_type{});
        }
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
            const uint64_t row = (uint64_t)(seq.first + token[a]) * p.heads + qHead[a];
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
                const uint64_t all = (uint64_t)p.maxTokens * p.heads, at = index * all + token[a] * p.heads + qHead[a];
                float* const   to  = p.partial + at * p.dim;
#pragma unroll
                for(uint32_t d = 0; d < D / 16u; ++d)
                    if(d % WK == wk && d * 16u + quad * 4u < p.dim)
                        *reinterpret_cast<f32x4*>(to + d * 16u + quad * 4u) = o[a][d];
                if(wk == 0u && quad == 0u)
                {
                    float* const ends = p.partial + p.shares * all * p.dim + at * 2u;
                    ends[0] = top[a], ends[1] = sum[a];
                }
            }
        }
    }

    // Adds up the shares of a row.  L = D / 4 lanes take four elements each, of four shares at once.  A workgroup has 256 / L sets of such lanes: one set a row, or
    // (ALL: few rows) all of them for one row, each every (256 / L)-th share, and their sums meet in LDS, in order.  (64 rows of 16 shares: 8.0 us with a set a
    // row, 4.0 with all; 4600 rows of 9 shares: 5 and 14 us.)  blockIdx.x: drafted tokens and heads, blockIdx.y: the sequence.
    template <typename T, uint32_t D, bool ALL>
    __global__ void __launch_bounds__(256) treeMergeKernel(TreeParams p)
    {
        constexpr uint32_t L = D / 4u, SETS = 256u / L, UNROLL = 4, STEP = ALL ? SETS : 1u;
        __shared__ __attribute__((aligned(16))) f32x4 sums[SETS][L];
        __shared__ float ends[SETS][2];
        const uint32_t   lane = threadIdx.x % L, set = threadIdx.x / L, item = ALL ? blockIdx.x : blockIdx.x * SETS + set;
        const uint32_t   b = blockIdx.y, t = item / p.heads, head = item % p.heads;
        const Sequence   seq = sequenceOf(p, p.qStart[b], p.qStart[b + 1u], p.kvLen[b]);
        const uint32_t   chunk = chunkOf(p, threadIdx.x & 63u);
        if(seq.length <= chunk)
            return;
        const uint32_t splits = splitsOf(seq.length, chunk), begin = ALL ? set : 0u;
        const uint64_t all = (uint64_t)p.maxTokens * p.heads, at = firstShareOf(p, b, chunk, threadIdx.x & 63u) * all + item;
        if(t >= seq.tokens)
            return;
        const float*   endsOf = p.partial + p.shares * all * p.dim + at * 2u;
        const float*   sumsOf = p.partial + at * p.dim + lane * 4u;
        float          top = -INFINITY, total = 0.0f;
        f32x4          sum{0, 0, 0, 0};
        for(uint32_t first = begin; first < splits; first += STEP * UNROLL)
        {
            float theirs[UNROLL], weight[UNROLL], next = top;
            f32x4 v[UNROLL];
#pragma unroll
            for(uint32_t u = 0; u < UNROLL; ++u)
            {
                const uint32_t s = first + u * STEP, i = s < splits ? s : begin; // (those past the last: the first again, without weight)
                theirs[u]        = endsOf[i * all * 2u], weight[u] = endsOf[i * all * 2u + 1u];
                v[u]             = lane * 4u < p.dim ? *reinterpret_cast<const f32x4*>(sumsOf + i * all * p.dim) : f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for(uint32_t u = 0; u < UNROLL; ++u)
            {
                theirs[u] = first + u * STEP < splits ? theirs[u] : -INFINITY;
                next      = fmaxf(next, theirs[u]);
            }
            const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
            total *= keep, sum *= keep, top = next;
#pragma unroll
            for(uint32_t u = 0; u < UNROLL; ++u)
            {
                const float factor = theirs[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(theirs[u] - next);
                total += factor * weight[u];
                sum += factor * v[u];
            }
        }
        if constexpr(ALL)
        {
            sums[set][lane] = sum;
            if(lane == 0u)
                ends[set][0] = top, ends[set][1] = total;
            __syncthreads();
            if(set != 0u)
                return;
            for(uint32_t s = 1u; s < SETS; ++s)
                top = fmaxf(top, ends[s][0]);
            total = 0.0f, sum = f32x4{0, 0, 0, 0};
            for(uint32_t s = 0; s < SETS; ++s)
            {
                const float factor = ends[s][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ends[s][0] - top);
                total += factor * ends[s][1];
                sum += factor * sums[s][lane];
            }
        }
        const float    inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const uint64_t row = seq.first + t;
        if(lane * 4u < p.dim)
            *reinterpret_cast<u32x2*>(reinterpret_cast<T*>(p.out) + (int64_t)row * p.oToken + (int64_t)head * p.oHead + lane * 4u)
                = u32x2{r355::pack2<T>(sum[0] * inverse, sum[1] * inverse), r355::pack2<T>(sum[2] * inverse, sum[3] * inverse)};
        if(p.lse && lane == 0u)
            p.lse[row * p.heads + head] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.693147180559945309f;
    }

    struct Plan
    {
        uint32_t rowsPerGroup, rowTiles, shares;
    };

    uint64_t bytesOfShare(const r355_tree_attention_args& a)
    {
        return (uint64_t)a.max_tokens * a.heads * (a.head_dim + 2u) * 4u;
    }

    Plan planOf(const r355_tree_attention_args& a, uint64_t workspaceBytes)
    {
        const uint64_t rows = (uint64_t)a.max_tokens * (a.heads / a.kv_heads), cus = r355::computeUnits();
        const uint64_t cache = (uint64_t)a.batch * a.max_kv * a.kv_heads * a.head_dim * 4u; // bytes, at most
        Plan           plan;
        // 16 and 32 rows: all four waves on positions; 64 and 128: on rows (64 rows, 4 x 16 tokens over 16000, 32 / 8 heads of 128: 50 us, with the waves on positions 133).
        plan.rowsPerGroup = rows <= 16u ? 16u : rows <= 32u && a.head_dim <= 128u ? 32u : a.head_dim <= 128u ? (rows <= 64u ? 64u : 128u) : 64u;
        // More than 128 rows over a cache that the memory-side cache does not hold: one workgroup of eight waves reads it instead of two of four, which drift apart further than
        // an XCD's L2 reaches (2 x 64 tokens over 65600, 32 / 8 heads of 128: 890 instead of 450 MB past the L2, 180 and 163 us).  (Heads over 128 have tiles of 64 rows on
        // four waves and would gain from 65 rows on: 4 x 17 .. 32 tokens over 32768, 16 / 4 heads of 256: 193 .. 205 and 129 .. 137 us; 8 x 17 over up to 16000, 32 / 8
        // of 192: 196 and 170.)
        if(rows > 128u && cache >= 192ull << 20)
            plan.rowsPerGroup = a.head_dim <= 128u ? 256u : 128u;
        plan.rowTiles         = static_cast<uint32_t>((rows + plan.rowsPerGroup - 1u) / plan.rowsPerGroup);
        const uint64_t groups = (uint64_t)a.kv_heads * plan.rowTiles; // workgroups of a share
        // Workgroups a CU that are aimed at.  Eight waves: one (1 x 64 tokens over 65600, 32 / 8 heads of 128: 100 us, two 127).  Waves on positions, of which a CU holds
        // one workgroup: one, where that makes eight shares of a sequence and more, so that the last share of each, which is shorter, weighs little (one token, 32 / 8 heads of 128:
        // 1 x 16000 18.8 us, two 23.7, four 23.7; 4 x 16000 56, 61, 64; 8 tokens, 1 x 65536: 59, 66, 81).  With more sequences the lengths decide, which are not known here.
        // Of 8 to 100 sequences of up to 2048 and 8192 positions, all equal, evenly spread or a few eight times as long as the rest, as many as a CU takes
        // over the best of one to eight, mean and most, single tokens: 32 / 8 heads of 128 one 1.09 and 1.81, two 1.10 and 1.53, four 1.11 and 1.51; 16 / 4 of 128
        // 1.07 and 2.28, 1.11 and 1.44, 1.14 and 1.52; 32 / 8 of 64 1.05 and 1.63, 1.12 and 1.63, 1.15 and 1.62; 16 / 2 of 256 1.06 and 1.92, 1.09 and 1.36, 1.12 and 1.45.  So
        // not one, which leaves the longest sequence to run by itself, though with lengths that are near each other it is the best (8 x 8192 evenly spread, 32 / 8 heads of 128:
        // 34, 37, 42 us; 32 x 820 .. 8192: 134, 145, 122): two, and four for single tokens with heads of 128, which differ by 3 % in the mean.
        // Several tiles, of which shorter sequences have fewer: four (8 trees of up to 48 tokens over 4099, 24 / 4 heads of 64: two 34 us, three 33, four 25; 4 x 64 tokens over
        // 2500 .. 8000, 16 / 4 of 64: 29 each; of 128: two 38, three 49, four 48), three of heads of 256 (4 x 64 tokens over 8000: two 69 us, three 60, four 74).
        const bool     eight  = plan.rowsPerGroup == 256u || (a.head_dim > 128u && plan.rowsPerGroup == 128u);
        const bool     one    = eight || (plan.rowsPerGroup <= 32u && (a.batch == 1u || a.batch * 8u <= cus / groups));
        const uint64_t target = one ? 1u : rows <= 16u && a.head_dim > 64u && a.head_dim <= 128u ? 4u : plan.rowTiles == 1u ? 2u : a.head_dim > 128u ? 3u : 4u;
        uint64_t       shares = (target * cus + groups - 1u) / groups;
        const uint64_t most   = (uint64_t)a.batch * (((uint64_t)a.max_kv + LEAST_CHUNK - 1u) / LEAST_CHUNK);
        shares                = shares < most ? shares : most;
        const uint64_t fit    = workspaceBytes / bytesOfShare(a);
        shares                = shares < fit ? shares : fit;
        plan.shares           = static_cast<uint32_t>(shares > a.batch ? shares : a.batch);
        return plan;
    }

    // shares times key heads, a multiple of the XCDs (the row tiles of a share on one of them)
    uint64_t columnsOf(const r355_tree_attention_args& a, const Plan& plan)
    {
        return ((uint64_t)plan.shares * a.kv_heads + 7u) / 8u * 8u;
    }
    // of a workgroup: eight waves on 256 rows, with heads over 128 on 128; else four
    uint32_t threadsOf(const r355_tree_attention_args& a, const Plan& plan)
    {
        return plan.rowsPerGroup == 256u || (a.head_dim > 128u && plan.rowsPerGroup == 128u) ? 512u : 256u;
    }

    template <typename T, uint32_t D, uint32_t WQ, uint32_t QB>
    void launchTree(const TreeParams& p, const Plan& plan, hipStream_t s)
    {
        hipLaunchKernelGGL((treeKernel<T, D, WQ, QB>), dim3(p.columns * plan.rowTiles), dim3(WQ == 8u ? 512u : 256u), 0, s, p);
    }

    template <typename T>
    void launchType(const TreeParams& p, const Plan& plan, hipStream_t s)
    {
        auto byRows = [&](auto width) {
            constexpr uint32_t D = decltype(width)::value;
            if(plan.rowsPerGroup == 16u)
                launchTree<T, D, 1, 1>(p, plan, s);
            else if constexpr(D == 256u)
            {
                if(plan.rowsPerGroup == 64u)
                    launchTree<T, D, 4, 1>(p, plan, s);
                else
                    launchTree<T, D, 8, 1>(p, plan, s);
            }
            else if(plan.rowsPerGroup == 32u)
                launchTree<T, D, 1, 2>(p, plan, s);
            else if(plan.rowsPerGroup == 64u)
                launchTree<T, D, 4, 1>(p, plan, s);
            else if(plan.rowsPerGroup == 128u)
                launchTree<T, D, 4, 2>(p, plan, s);
            else
                launchTree<T, D, 8, 2>(p, plan, s);
            if(plan.shares > p.batch) // (planOf: batch * kv_heads * row tiles of up to 256 rows are fewer than four times the CUs then)
            {
                const uint32_t rows = p.maxTokens * p.heads;
                if((uint64_t)p.batch * rows <= 2048u)
                    hipLaunchKernelGGL((treeMergeKernel<T, D, true>), dim3(rows, p.batch), dim3(256), 0, s, p);
                else
                    hipLaunchKernelGGL((treeMergeKernel<T, D, false>), dim3((rows + 1024u / D - 1u) / (1024u / D), p.batch), dim3(256), 0, s, p);
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
        if(a.batch > 65535u)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: batch=%u is over 65535", a.batch);
        if(a.batch == 0 || a.total_tokens == 0 || a.max_tokens == 0)
            return R355_OK;
        // (the most workgroups that there can be: those with all of the workspace asked for)
        const Plan     plan   = planOf(a, ~0ull);
        const uint64_t groups = columnsOf(a, plan) * plan.rowTiles;
        if(groups * (threadsOf(a, plan) / 256u) > r355::MAX_GROUPS)
            return r355::fail(R355_ERR_BAD_SIZE, "tree_attention: %llu workgroups of %u threads for the sequences, heads and drafted tokens are too many for one launch",
                              (unsigned long long)groups, threadsOf(a, plan));
        return R355_OK;
    }
} // namespace

extern "C" size_t r355_tree_attention_workspace_bytes(const r355_tree_attention_args* args)
{
    if(!args || checkSizes(*args) != R355_OK || args->batch == 0 || args->total_tokens == 0 || args->max_tokens == 0)
        return 0;
    const Plan plan = planOf(*args, ~0ull);
    return plan.shares > args->batch ? plan.shares * bytesOfShare(*args) : 0u;
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
    if(!std::isfinite(static_cast<float>(a.scale)))
        return r355::fail(R355_ERR_BAD_ARG, "tree_attention: the scale must be finite");
    if(!r355::aligned(a.table, 4) || !r355::aligned(a.q_start, 4) || !r355::aligned(a.kv_len, 4))
        return r355::fail(R355_ERR_MISALIGNED, "tree_attention: table, q_start and kv_len need 4-byte alignment");
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
    const Plan plan = planOf(a, a.workspace ? a.workspace_bytes : 0u);

    TreeParams p;
    p.q = static_cast<const char*>(a.q), p.k = static_cast<const char*>(a.k), p.v = static_cast<const char*>(a.v), p.out = static_cast<char*>(a.out), p.lse = a.lse;
    p.table = a.table, p.qStart = a.q_start, p.kvLen = a.kv_len, p.mask = a.mask, p.partial = static_cast<float*>(a.workspace);
    p.qToken = a.q_token_stride, p.qHead = a.q_head_stride, p.kSlot = a.k_slot_stride, p.kHead = a.k_head_stride, p.vSlot = a.v_slot_stride, p.vHead = a.v_head_stride;
    p.oToken = a.out_token_stride, p.oHead = a.out_head_stride;
    p.batch = a.batch, p.heads = a.heads, p.kvHeads = a.kv_heads, p.group = a.heads / a.kv_heads, p.dim = a.head_dim;
    p.totalTokens = a.total_tokens, p.maxTokens = a.max_tokens, p.maxKv = a.max_kv;
    p.pageSize = a.page_size, p.pages = a.pages, p.tableStride = a.table_stride, p.maskWords = a.mask_words;
    p.shares = plan.shares, p.columns = static_cast<uint32_t>(columnsOf(a, plan));
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
