// What the kernels of the layers' products share (linear.hip, linear_tiles.hip): their parameters, the activations, the way from a workgroup to its group of rows.
#ifndef R355_LINEAR_HPP
#define R355_LINEAR_HPP

#include <cmath>
#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "half_types.hpp"
#include "tile_map.hpp"

namespace r355
{
    // One launch of Y = A B for each group of rows.  Three forms of a layer's product, w: [groups][n][k]:
    //   forward           A: rows of x (m ragged),            B: w, contiguous along the sum         Y: [rows][n]
    //   input's gradient  A: rows of dz (m ragged),           B: w, contiguous along the columns     Y: [rows][k]
    //   weights' gradient A: dz, contiguous along its columns, B: x likewise; the sum is ragged      Y: [groups][n][k]
    struct LinearParams
    {
        const char*    a;
        const char*    b;
        const char*    bias; // [groups][n]
        const char*    gate;
        const char*    c; // what is added to the result, of its type
        char*          y;
        char*          z; // what the activation is taken of
        const int32_t* offsets; // [groups + 1] or NULL: one group of all rows
        const int32_t* source;  // row of A of each row, or NULL
        uint32_t       rows, m, n, k; // m: rows of Y of the weights' gradient; k: length of the sum (forward, input's gradient)
        uint32_t       groups, sourceRows;
        uint32_t       lda, ldb, ldy, ldz, ldg, ldc;
        uint64_t       strideB, strideY, strideC; // bytes from group to group
        uint64_t       strideSplit; // ... from one share of the sum to the next
        uint32_t       tilesM, tilesN; // tilesM: of a group's Y (weights' gradient)
        uint32_t       splits; // workgroups along the sum, each writes its own f32 sums (workspace [splits][rows of Y][n]); 1: none
        int32_t        activation;
        uint32_t       outF32, linesY, linesZ; // lines: rows begin with a cache line
    };

    constexpr uint32_t OUTSIDE = 0x80000000u; // a lane's offset past the end of any buffer here: loads zeros, stores nothing

    struct Rows
    {
        uint32_t first, count;
    };
    // The rows of a group.  What offsets holds is only known here: whatever it is, the rows are rows of the matrix.
    __device__ __forceinline__ Rows rowsOf(const LinearParams& p, uint32_t group)
    {
        if(!p.offsets)
            return Rows{0u, p.rows};
        const int32_t  from = p.offsets[group], to = p.offsets[group + 1u];
        const uint32_t first = from < 0 ? 0u : static_cast<uint32_t>(from) < p.rows ? static_cast<uint32_t>(from) : p.rows;
        const uint32_t end   = to < 0 ? 0u : static_cast<uint32_t>(to) < p.rows ? static_cast<uint32_t>(to) : p.rows;
        return Rows{first, end > first ? end - first : 0u};
    }

    __device__ __forceinline__ uint32_t lanesUpTo(uint32_t v) // sum over the lanes up to this one
    {
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
        for(uint32_t d = 1u; d < 64u; d <<= 1)
        {
            const uint32_t below = __shfl_up(v, d);
            v += lane >= d ? below : 0u;
        }
        return v;
    }

    // A tile of a ragged Y: the group it belongs to, its first row and how many of its rows there are.
    struct GroupTile
    {
        uint32_t group, first, count;
    };
    // Walks the groups' tiles of TM rows, 64 groups at a time, a group a lane: total() counts them, at() finds one.  The host does not know the groups' sizes;
    // a launch has as many workgroups as any division of the rows could need, and those without a tile end at once.  (Offsets that are no division of the rows can name more tiles than
    // that: the count stops at MOST, which keeps it from passing 32 bits, and tiles past the launch's workgroups are left out.)
    template <uint32_t TM>
    struct GroupTiles
    {
        static constexpr uint32_t MOST = 1u << 31; // (64 groups have 2^30 tiles at most: 2^30 rows, TM >= 64 or few rows)
        const LinearParams&       p;
        uint32_t                  base = 0u, tiles = 0u, upto = 0u, all = 0u;
        Rows                      rows{0u, 0u};

        __device__ __forceinline__ void block(uint32_t first, uint32_t before)
        {
            const uint32_t g = first + (threadIdx.x & 63u);
            rows             = g < p.groups ? rowsOf(p, g) : Rows{0u, 0u};
            tiles            = rows.count / TM + (rows.count % TM != 0u ? 1u : 0u);
            base             = first;
            upto             = before + lanesUpTo(tiles);
        }
        __device__ __forceinline__ uint32_t upToHere() const
        {
            const uint32_t n = __builtin_amdgcn_readlane(upto, 63);
            return n < MOST ? n : MOST;
        }
        __device__ __forceinline__ uint32_t total()
        {
            if(!p.offsets)
                return p.rows / TM + (p.rows % TM != 0u ? 1u : 0u);
            all = 0u;
            for(uint32_t first = 0; first < p.groups; first += 64u)
            {
                block(first, all);
                all = upToHere();
            }
            return all;
        }
        __device__ __forceinline__ GroupTile at(uint32_t tile) // tile < total()
        {
            if(!p.offsets)
            {
                const uint32_t left = p.rows - tile * TM;
                return GroupTile{0u, tile * TM, left < TM ? left : TM};
            }
            if(p.groups > 64u)
                for(uint32_t first = 0, before = 0; first < p.groups; first += 64u)
                {
                    block(first, before);
                    before = upToHere();
                    if(before > tile)
                        break;
                }
            const uint32_t l    = static_cast<uint32_t>(__ffsll(__ballot(upto > tile))) - 1u;
            const uint32_t in   = tile - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l));
            const uint32_t left = __builtin_amdgcn_readlane(rows.count, l) - in * TM;
            return GroupTile{base + l, __builtin_amdgcn_readlane(rows.first, l) + in * TM, left < TM ? left : TM};
        }
    };

    // sigma(z) = 1 / (1 + e^-z); e^-z = infinity gives 0
    __device__ __forceinline__ float sigmoid(float z)
    {
        return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    }
    // The normal distribution function, erfc(x) / 2 beyond x = |z| / sqrt 2.  e^(x^2) erfc(x) / 2 is smooth and falls like 1 / x: t P(t) with t = 1 / (1 + x / 2) and P of degree 8, the
    // minimax polynomial of the relative error (Remez' exchange over 0 <= x <= 9.6, where e^(-x^2) leaves 32 bits): 4.7e-8.  So the lower tail keeps its digits: it is off by the
    // rounding of z^2 / 2, (1.5 z^2 + 16) 2^-24 of itself at most.  (A polynomial of degree 5 with a bound on the absolute error was off by 0.05 % at -4 and 1 % at -8, and took 3 of 210 us
    // less in 4000 x 8192 x 4096; erff, with its cases, takes 20 us more for the 256 values of a thread of a 256 x 256 tile.)  e = e^(-z^2 / 2)
    __device__ __forceinline__ float normalCdf(float z, float& e)
    {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.353553391f, fabsf(z), 1.0f));
        e             = __builtin_amdgcn_exp2f(z * z * -0.721347520f); // (log2 e / 2)
        float p       = -0.029465685f;
        p             = fmaf(p, t, 0.141950533f);
        p             = fmaf(p, t, -0.242899194f);
        p             = fmaf(p, t, 0.138227910f);
        p             = fmaf(p, t, -0.012754682f);
        p             = fmaf(p, t, 0.101105735f);
        p             = fmaf(p, t, 0.121612407f);
        p             = fmaf(p, t, 0.141179264f);
        p             = fmaf(p, t, 0.141043693f);
        const float upper = e * (t * p); // beyond |z|
        return z < 0.0f ? upper : 1.0f - upper;
    }
    // (1 + tanh(u / 2)) / 2 is sigma(u): the tanh form of GELU is z sigma(u) with u = 2 sqrt(2 / pi) (z + 0.044715 z^3)
    constexpr float GELU_U = 1.5957691216057308f, GELU_U3 = 0.044715f;

    template <int32_t ACT>
    __device__ __forceinline__ float activate(float z)
    {
        if constexpr(ACT == R355_ACT_RELU)
            return z < 0.0f ? 0.0f : z; // (a NaN stays one)
        else if constexpr(ACT == R355_ACT_GELU)
        {
            float e;
            return z * normalCdf(z, e);
        }
        else if constexpr(ACT == R355_ACT_GELU_TANH)
            return z * sigmoid(GELU_U * z * fmaf(GELU_U3 * z, z, 1.0f));
        else if constexpr(ACT == R355_ACT_SILU)
            return z * sigmoid(z);
        else
            return z;
    }
    // value and derivative
    template <int32_t ACT>
    __device__ __forceinline__ void activateBoth(float z, float& value, float& slope)
    {
        if constexpr(ACT == R355_ACT_RELU)
        {
            value = z < 0.0f ? 0.0f : z;
            slope = z > 0.0f ? 1.0f : 0.0f;
        }
        else if constexpr(ACT == R355_ACT_GELU)
        {
            float       e;
            const float cdf = normalCdf(z, e);
            value           = z * cdf;
            slope           = fmaf(z, 0.39894228040143268f * e, cdf);
        }
        else if constexpr(ACT == R355_ACT_GELU_TANH)
        {
            const float s = sigmoid(GELU_U * z * fmaf(GELU_U3 * z, z, 1.0f)), t = s * (1.0f - s);
            value         = z * s;
            // s + z s (1 - s) u': where u' z overflows s (1 - s) is 0
            slope = t == 0.0f ? s : fmaf(z * t, GELU_U * fmaf(3.0f * GELU_U3 * z, z, 1.0f), s);
        }
        else if constexpr(ACT == R355_ACT_SILU)
        {
            const float s = sigmoid(z), t = s * (1.0f - s);
            value = z * s;
            slope = t == 0.0f ? s : fmaf(z, t, s);
        }
        else
            value = z, slope = 1.0f;
    }
    // calls f with the activation as a constant.  (Around whole batches of values: a choice for each value keeps their chains of instructions from running side by
    // side, 27 us instead of 10 for the 256 values that a thread of a 256 x 256 tile has.)
    template <typename F>
    __device__ __forceinline__ void withActivation(int32_t activation, F&& f)
    {
        switch(activation)
        {
        case R355_ACT_RELU: return f(std::integral_constant<int32_t, R355_ACT_RELU>{});
        case R355_ACT_GELU: return f(std::integral_constant<int32_t, R355_ACT_GELU>{});
        case R355_ACT_GELU_TANH: return f(std::integral_constant<int32_t, R355_ACT_GELU_TANH>{});
        case R355_ACT_SILU: return f(std::integral_constant<int32_t, R355_ACT_SILU>{});
        default: return f(std::integral_constant<int32_t, R355_ACT_NONE>{});
        }
    }

    // Macro tiles (linear_tiles.hip); ANY is 64 x 64, element by element, whatever the alignment
    enum LinearTile : uint32_t
    {
        TILE_256 = 0,
        TILE_192_256,
        TILE_256_128,
        TILE_192_128,
        TILE_128_256,
        TILE_128,
        TILE_64,
        TILE_ANY
    };
    constexpr uint32_t LINEAR_TILES = 8u, LINEAR_ROWS[LINEAR_TILES] = {256u, 192u, 256u, 192u, 128u, 128u, 64u, 64u}, LINEAR_COLS[LINEAR_TILES] = {256u, 256u, 128u, 128u, 256u, 128u, 64u, 64u};
    // the forms, one set of kernels per type; aK, bK: A, B contiguous along the sum
    void linearTilesF16(const LinearParams& p, bool aK, bool bK, LinearTile tile, uint32_t workgroups, hipStream_t s);
    void linearTilesBF16(const LinearParams& p, bool aK, bool bK, LinearTile tile, uint32_t workgroups, hipStream_t s);
    // both gradients, input's and weights', on tiles of 64 x 64 in one launch
    void linearBothF16(const LinearParams& px, const LinearParams& pw, uint32_t workgroupsX, uint32_t workgroupsW, hipStream_t s);
    void linearBothBF16(const LinearParams& px, const LinearParams& pw, uint32_t workgroupsX, uint32_t workgroupsW, hipStream_t s);
} // namespace r355

#endif // R355_LINEAR_HPP
