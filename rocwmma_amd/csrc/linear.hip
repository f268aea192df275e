// Products of a layer with bias, activation, gate and residual, and their gradients, for one matrix of weights or one per group of rows: the entry points, the kernel
// for few rows, what the gradient does element by element, and the sums of split products.  The macro tiles are in linear_tiles.hip.
//
//   forward    z = x W^T + b;  y = act(z) gate + c
//   backward   dz = dy gate act'(z);  dgate = dy act(z);  dx = dz W;  dW = dz^T x;  db = sum of dz over the rows
//
// No counterpart in the reference.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "linear.hpp"

#define R355_TRY(call)          \
    do                          \
    {                           \
        const int rc_ = (call); \
        if(rc_ != R355_OK)      \
            return rc_;         \
    } while(0)

namespace
{
    using r355::each;
    using r355::f32x4;
    using r355::GroupTile;
    using r355::GroupTiles;
    using r355::LinearParams;
    using r355::OUTSIDE;
    using r355::Rows;
    using r355::u32x4;
    using r355::vec;

    constexpr uint32_t WAVES = 8u;

    // ---- One or two rows of each group: dot products.  A wave takes 16 weight rows, each lane 16 bytes of every row at a time, so that an access is 1 KiB of one row (the matrix instructions'
    // operands are 64 bytes of each of 16 rows: 16 experts of 4096 x 4096 105 us instead of 84).  Pieces of 512 of the sum go to WK waves in turn, other
    // waves have other rows.  Bound by HBM: 16 rows of 16 experts of 4096 x 4096 83 us, 6.5 TB/s; 1024 x 2048 4.0, a launch and two accesses' latency.
    //
    // A lane's 16 T sums become one sum of the wave in each lane: of a pair of sums each half of the lanes keeps one and adds the other half's part of it, and so on by halves,
    // about 16 T additions instead of 6 for each sum.  After the steps over lanes 32, 16, 8 and 4 apart lane l has sum 8 (l / 4 % 2) + 4 (l / 8 % 2) + 2 (l / 16 % 2) + l / 32 of 16.
    __device__ __forceinline__ float other(float v, uint32_t distance) // the lane's that is so far away
    {
        if(distance == 8u)
            return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), 0x128, 0xF, 0xF, true))); // row_ror:8
        if(distance == 2u)
            return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), 0x4E, 0xF, 0xF, true))); // quad_perm [2, 3, 0, 1]
        if(distance == 1u)
            return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), 0xB1, 0xF, 0xF, true))); // quad_perm [1, 0, 3, 2]
        return __shfl_xor(v, static_cast<int>(distance));
    }
    template <uint32_t N>
    __device__ __forceinline__ void halve(float (&v)[N], uint32_t lane)
    {
        static_assert(N == 16u || N == 32u, "one or two rows");
        auto step = [&](auto countOf, auto distanceOf) __attribute__((always_inline)) {
            constexpr uint32_t COUNT = decltype(countOf)::value, D = decltype(distanceOf)::value;
#pragma unroll
            for(uint32_t i = 0; i < COUNT; ++i)
            {
                const uint32_t a = __float_as_uint(v[2u * i]), b = __float_as_uint(v[2u * i + 1u]);
                if constexpr(D == 32u)
                {
                    const auto s = __builtin_amdgcn_permlane32_swap(a, b, false, false);
                    v[i]         = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                }
                else if constexpr(D == 16u)
                {
                    const auto s = __builtin_amdgcn_permlane16_swap(a, b, false, false);
                    v[i]         = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                }
                else
                {
                    const bool  high = (lane & D) != 0u;
                    const float keep = high ? v[2u * i + 1u] : v[2u * i], give = high ? v[2u * i] : v[2u * i + 1u];
                    v[i]             = keep + other(give, D);
                }
            }
        };
        using std::integral_constant;
        step(integral_constant<uint32_t, N / 2u>{}, integral_constant<uint32_t, 32>{});
        step(integral_constant<uint32_t, N / 4u>{}, integral_constant<uint32_t, 16>{});
        step(integral_constant<uint32_t, N / 8u>{}, integral_constant<uint32_t, 8>{});
        step(integral_constant<uint32_t, N / 16u>{}, integral_constant<uint32_t, 4>{});
        if constexpr(N == 32u)
            step(integral_constant<uint32_t, 1>{}, integral_constant<uint32_t, 2>{});
        else
            v[0] += other(v[0], 2u);
        v[0] += other(v[0], 1u);
    }
    // the sum that a lane has after halve()
    __device__ __forceinline__ uint32_t sumOf(uint32_t lane)
    {
        return __brev(lane) >> 26;
    }

    // acc + a0 b0 + ... + a7 b7
    template <typename T>
    __device__ __forceinline__ float dot8(u32x4 a, u32x4 b, float acc)
    {
#pragma unroll
        for(uint32_t i = 0; i < 4u; ++i)
        {
            const uint32_t x = a[i], y = b[i]; // (a cast of a vector's element itself takes the first one's bits)
            if constexpr(__is_same(T, __bf16))
                acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(vec<__bf16, 2>, x), __builtin_bit_cast(vec<__bf16, 2>, y), acc, false);
            else
                acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(vec<_Float16, 2>, x), __builtin_bit_cast(vec<_Float16, 2>, y), acc, false);
        }
        return acc;
    }

    // y of one row and column, from its sum: z = sum + bias; y = act(z) gate + c
    template <typename T>
    __device__ __forceinline__ void finishOne(const LinearParams& p, uint32_t group, uint64_t row, uint32_t col, float sum)
    {
        float gate = 1.0f, add = 0.0f; // (asked for before anything waits)
        if(p.gate)
            gate = static_cast<float>(reinterpret_cast<const T*>(p.gate)[row * p.ldg + col]);
        if(p.c)
            add = p.outF32 ? reinterpret_cast<const float*>(p.c)[row * p.ldc + col] : static_cast<float>(reinterpret_cast<const T*>(p.c)[row * p.ldc + col]);
        if(p.bias)
            sum += static_cast<float>(reinterpret_cast<const T*>(p.bias)[(uint64_t)group * p.n + col]);
        if(p.z)
            reinterpret_cast<T*>(p.z)[row * p.ldz + col] = static_cast<T>(sum);
        r355::withActivation(p.activation, [&](auto act) { sum = r355::activate<decltype(act)::value>(sum); });
        if(p.gate)
            sum *= gate;
        if(p.c)
            sum += add;
        if(p.outF32)
            reinterpret_cast<float*>(p.y)[row * p.ldy + col] = sum;
        else
            reinterpret_cast<T*>(p.y)[row * p.ldy + col] = static_cast<T>(sum);
    }

    // the sums of ROWS rows (count of them there) and a wave's 16 columns: sums[16 t + column]
    template <typename T, uint32_t ROWS, bool STREAM>
    __device__ __forceinline__ void dotWave(const LinearParams& p, const GroupTile& t, uint32_t col0, uint32_t waveK, uint32_t wavesK, float* sums)
    {
        const uint32_t lane = threadIdx.x & 63u, pieces = (p.k + 511u) / 512u;
        const uint32_t last = p.n - col0 < 16u ? p.n - col0 - 1u : 15u; // (columns past the last read it again)
        const auto bufW = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.b) + (uint64_t)t.group * p.strideB + (uint64_t)col0 * p.ldb * 2u, 0,
                                                            static_cast<int>((last * p.ldb + p.k) * 2u), 0x00020000);
        const char* x[ROWS];
        bool        in[ROWS];
#pragma unroll
        for(uint32_t r = 0; r < ROWS; ++r)
        {
            uint64_t row = t.first + (r < t.count ? r : t.count - 1u);
            in[r]        = true;
            if(p.source)
            {
                row   = static_cast<uint32_t>(p.source[row]);
                in[r] = row < p.sourceRows;
            }
            x[r] = p.a + (in[r] ? row * p.lda * 2u : 0u);
        }
        float acc[16u * ROWS];
#pragma unroll
        for(uint32_t i = 0; i < 16u * ROWS; ++i)
            acc[i] = 0.0f;
        u32x4 w[16], xs[ROWS];
        auto  offset = [&](uint32_t piece) { return piece * 512u + lane * 8u < p.k ? lane * 16u : OUTSIDE; };
        auto  loadX = [&](uint32_t piece) __attribute__((always_inline)) {
#pragma unroll
            for(uint32_t r = 0; r < ROWS; ++r)
                xs[r] = in[r] && piece * 512u + lane * 8u < p.k ? *reinterpret_cast<const u32x4*>(x[r] + ((uint64_t)piece * 512u + lane * 8u) * 2u) : u32x4{0u, 0u, 0u, 0u};
        };
        auto loadW = [&](uint32_t piece, uint32_t c) __attribute__((always_inline)) {
            return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bufW, offset(piece), (c < last ? c : last) * p.ldb * 2u + piece * 1024u, STREAM ? 2 : 0));
        };
        if(waveK < pieces)
        {
#pragma unroll
            for(uint32_t c = 0; c < 16u; ++c)
                w[c] = loadW(waveK, c);
            loadX(waveK);
        }
        for(uint32_t piece = waveK; piece < pieces; piece += wavesK)
        {
            const uint32_t next = piece + wavesK;
#pragma unroll
            for(uint32_t c = 0; c < 16u; ++c)
            {
#pragma unroll
                for(uint32_t r = 0; r < ROWS; ++r)
                    acc[16u * r + c] = dot8<T>(w[c], xs[r], acc[16u * r + c]);
                if(next < pieces) // (uniform)
                    w[c] = loadW(next, c);
            }
            if(next < pieces)
                loadX(next);
        }
        halve<16u * ROWS>(acc, lane);
        constexpr uint32_t SAME = 64u / (16u * ROWS); // lanes that have the same sum
        if((lane & (SAME - 1u)) == 0u)
            sums[sumOf(lane) & (16u * ROWS - 1u)] = acc[0];
    }

    // ROWS: of a tile.  Workgroups of wavesK x (waves / wavesK) waves.
    template <typename T, uint32_t ROWS, bool STREAM>
    __global__ void __launch_bounds__(64 * WAVES, 2) linearDots(LinearParams p, uint32_t wavesK)
    {
        __shared__ float sums[WAVES][16u * ROWS];
        GroupTiles<ROWS> tiles{p};
        const uint32_t   tilesM = tiles.total(), count = tilesM * p.tilesN, perXcd = (count + 7u) / 8u;
        const uint32_t   id = blockIdx.x % 8u * perXcd + blockIdx.x / 8u;
        if(blockIdx.x / 8u >= perXcd || id >= count)
            return;
        GroupTile t = tiles.at(id % tilesM);
        t.group = __builtin_amdgcn_readfirstlane(t.group), t.first = __builtin_amdgcn_readfirstlane(t.first), t.count = __builtin_amdgcn_readfirstlane(t.count);
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sets = (blockDim.x >> 6) / wavesK, set = wave / wavesK;
        const uint32_t col0 = id / tilesM * 16u * sets, mine = col0 + set * 16u;
        if(mine < p.n)
        {
            if(ROWS == 1u || t.count == 1u)
                dotWave<T, 1, STREAM>(p, t, mine, wave % wavesK, wavesK, sums[wave]);
            else
                dotWave<T, ROWS, STREAM>(p, t, mine, wave % wavesK, wavesK, sums[wave]);
        }
        __syncthreads();
        for(uint32_t i = threadIdx.x; i < 16u * sets * t.count; i += blockDim.x)
        {
            const uint32_t row = i / (16u * sets), col = i % (16u * sets), of = col / 16u * wavesK;
            if(col0 + col >= p.n)
                continue;
            float sum = 0.0f;
            for(uint32_t v = 0; v < wavesK; ++v)
                sum += sums[of + v][row * 16u + col % 16u];
            finishOne<T>(p, t.group, (uint64_t)t.first + row, col0 + col, sum);
        }
    }

    // ---- Few rows of each group.  A workgroup's eight waves share 16 RB weight rows x 16 CB rows of x and take DEPTH neighbouring pieces of 64 of the sum in turn, both
    // straight from global memory; their sums meet in LDS in the order of the waves.  The weights are the first operand: a lane then holds four of them of one row of x.
    // Bound by HBM: two rows of each of 16 experts of 1326 x 6520 50 us, 5.5 TB/s.  (Single pieces in turn: rows that do not begin with a cache line have lines of two waves, 30 rows of 8 experts
    // of 8192 x 4104 167 instead of 162 us; and such lines come twice where they are read nontemporally, 162 instead of 125.)
    template <typename T>
    __global__ void __launch_bounds__(64 * WAVES, 2) linearFew(LinearParams p)
    {
        constexpr uint32_t RB = 1u, CB = 1u, DEPTH = 4u; // (written out for one block the loads are scheduled worse: 16 x 16384 x 4096 38.7 us instead of 35.7)
        constexpr uint32_t ROWS = 16u * CB, COLS = 16u * RB, PITCH = COLS + 4u;
        __shared__ __attribute__((aligned(16))) float sums[WAVES * ROWS * PITCH];
        GroupTiles<ROWS> tiles{p};
        const uint32_t   tilesM = tiles.total(), count = tilesM * p.tilesN, perXcd = (count + 7u) / 8u;
        // (a group's tiles of rows one after another on one XCD: they read the same weights)
        const uint32_t id = blockIdx.x % 8u * perXcd + blockIdx.x / 8u;
        if(blockIdx.x / 8u >= perXcd || id >= count)
            return;
        const uint32_t  tn = id / tilesM;
        const GroupTile t  = tiles.at(id % tilesM);
        const uint32_t  group = __builtin_amdgcn_readfirstlane(t.group), first = __builtin_amdgcn_readfirstlane(t.first), rows = __builtin_amdgcn_readfirstlane(t.count);
        const uint32_t  lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15u, quad = lane >> 4;
        const uint32_t  col0 = tn * COLS, cols = p.n - col0 < COLS ? p.n - col0 : COLS;

        // (buffers that end with the last element; rows that are not there lie outside)
        const auto bufW = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.b) + (uint64_t)group * p.strideB + (uint64_t)col0 * p.ldb * 2u, 0,
                                                            static_cast<int>(((cols - 1u) * p.ldb + p.k) * 2u), 0x00020000);
        const auto bufX = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p.a) + (p.source ? 0u : (uint64_t)first * p.lda * 2u), 0,
                                                            static_cast<int>(((p.source ? p.sourceRows : rows) - 1u) * p.lda * 2u + p.k * 2u), 0x00020000);
        uint32_t offW[RB], offX[CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
            offW[r] = r * 16u + r16 < cols ? (r * 16u + r16) * p.ldb * 2u + quad * 16u : OUTSIDE;
#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
        {
            const uint32_t row  = c * 16u + r16;
            uint32_t       from = row;
            bool           in   = row < rows;
            if(in && p.source)
            {
                from = static_cast<uint32_t>(p.source[(uint64_t)first + row]);
                in   = from < p.sourceRows;
            }
            offX[c] = in ? from * p.lda * 2u + quad * 16u : OUTSIDE;
        }
        f32x4 acc[RB][CB];
#pragma unroll
        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
            for(uint32_t c = 0; c < CB; ++c)
                acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        struct Stage
        {
            u32x4 w[RB][2], x[CB][2];
        };
        const uint32_t pieces = (p.k + 63u) / 64u;
        auto load = [&](uint32_t piece) __attribute__((always_inline)) {
            Stage s;
#pragma unroll
            for(uint32_t i = 0; i < 2u; ++i)
            {
                const bool in = piece * 64u + i * 32u + quad * 8u < p.k; // (what lies past the sum's end is another row's)
#pragma unroll
                for(uint32_t r = 0; r < RB; ++r)
                    s.w[r][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bufW, in ? offW[r] + i * 64u : OUTSIDE, piece * 128u, 0));
#pragma unroll
                for(uint32_t c = 0; c < CB; ++c)
                    s.x[c][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bufX, in ? offX[c] + i * 64u : OUTSIDE, piece * 128u, 0));
            }
            return s;
        };
        Stage stage[DEPTH];
        each<DEPTH>([&](auto at) __attribute__((always_inline)) {
            constexpr uint32_t d = decltype(at)::value;
            if(wave * DEPTH + d < pieces)
                stage[d] = load(wave * DEPTH + d);
        });
        for(uint32_t from = wave * DEPTH; from < pieces; from += DEPTH * WAVES)
            each<DEPTH>([&](auto at) __attribute__((always_inline)) {
                constexpr uint32_t d     = decltype(at)::value;
                const uint32_t     piece = from + d;
                if(piece < pieces)
                {
#pragma unroll
                    for(uint32_t i = 0; i < 2u; ++i)
#pragma unroll
                        for(uint32_t r = 0; r < RB; ++r)
#pragma unroll
                            for(uint32_t c = 0; c < CB; ++c)
                                acc[r][c] = r355::mfma32<T>(stage[d].w[r][i], stage[d].x[c][i], acc[r][c]);
                    if(piece + DEPTH * WAVES < pieces)
                        stage[d] = load(piece + DEPTH * WAVES);
                }
            });
#pragma unroll
        for(uint32_t c = 0; c < CB; ++c)
#pragma unroll
            for(uint32_t r = 0; r < RB; ++r)
                *reinterpret_cast<f32x4*>(&sums[(wave * ROWS + c * 16u + r16) * PITCH + r * 16u + quad * 4u]) = acc[r][c];
        __syncthreads();
        for(uint32_t i = threadIdx.x; i < rows * COLS; i += 64u * WAVES)
        {
            const uint32_t row = i / COLS, col = i % COLS;
            if(col >= cols)
                continue;
            float sum = 0.0f;
#pragma unroll
            for(uint32_t v = 0; v < WAVES; ++v)
                sum += sums[(v * ROWS + row) * PITCH + col];
            finishOne<T>(p, group, (uint64_t)first + row, col0 + col, sum);
        }
    }

    // ---- Sums of a split product: [splits][rows][pitch] of f32, added in order, then the epilogue of linear_tiles.hip.  Result rows are `p.m` to a group (weights' gradient), or
    // by offsets; those of no group are left.  Four columns a thread; what is not four columns wide, or past a row's end, goes element by element.  4 to 5 us: a launch, and the shares out of the caches.
    template <typename T, typename Out>
    __global__ void __launch_bounds__(256) linearReduce(LinearParams p, const float* sums, uint64_t rows, uint32_t pitch)
    {
        const uint32_t mine = (blockIdx.x * 256u + threadIdx.x) * 4u, left = mine < p.n ? p.n - mine : 0u, col = left ? mine : 0u;
        if(__ballot(left != 0u) == 0u)
            return; // (whole waves: the lanes find a row's group together)
        // (rows anywhere: vectors of an element's alignment)
        typedef T    TU __attribute__((ext_vector_type(4), aligned(2)));
        typedef Out  OutU __attribute__((ext_vector_type(4), aligned(sizeof(Out))));
        auto read = [&](const auto* from, float (&v)[4]) {
            using E = std::remove_cv_t<std::remove_pointer_t<decltype(from)>>;
            using U = std::conditional_t<std::is_same_v<E, T>, TU, OutU>;
            if(left >= 4u)
            {
                const U w = *reinterpret_cast<const U*>(from);
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    v[e] = static_cast<float>(w[e]);
            }
            else
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    v[e] = e < left ? static_cast<float>(from[e]) : 0.0f;
        };
        auto write = [&](auto* to, const float (&v)[4]) {
            using E = std::remove_pointer_t<decltype(to)>;
            using U = std::conditional_t<std::is_same_v<E, T>, TU, OutU>;
            if(left >= 4u)
                *reinterpret_cast<U*>(to) = U{static_cast<E>(v[0]), static_cast<E>(v[1]), static_cast<E>(v[2]), static_cast<E>(v[3])};
            else
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    if(e < left)
                        to[e] = static_cast<E>(v[e]);
        };
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if(p.bias && !p.offsets)
            read(reinterpret_cast<const T*>(p.bias) + col, bias);
        const uint64_t share = rows * pitch;
        for(uint64_t row = blockIdx.y; row < rows; row += gridDim.y)
        {
            const uint64_t group = p.m ? row / p.m : 0u, in = p.m ? row % p.m : row;
            if(p.m == 0u && p.offsets)
            {
                // a row's group is the last one that begins at or before it: as many offsets are no larger, less one
                uint32_t begun = 0u;
                for(uint32_t g = threadIdx.x & 63u; g - (threadIdx.x & 63u) <= p.groups; g += 64u)
                    begun += static_cast<uint32_t>(__popcll(__ballot(g <= p.groups && p.offsets[g <= p.groups ? g : 0u] <= static_cast<int64_t>(row))));
                if(begun == 0u || begun > p.groups)
                    continue; // no group's
                const Rows its = r355::rowsOf(p, begun - 1u);
                if(row < its.first || row - its.first >= its.count)
                    continue; // (offsets that are no division)
                if(p.bias)
                    read(reinterpret_cast<const T*>(p.bias) + (uint64_t)(begun - 1u) * p.n + col, bias);
            }
            const float*   from = sums + row * pitch + col;
            float          sum[4], more[4];
            f32x4          all{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for(uint32_t s = 0; s < p.splits; ++s)
                all += *reinterpret_cast<const f32x4*>(from + s * share);
#pragma unroll
            for(uint32_t e = 0; e < 4u; ++e)
                sum[e] = all[e] + bias[e];
            if(p.z)
                write(reinterpret_cast<T*>(p.z) + row * p.ldz + col, sum);
            r355::withActivation(p.activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    sum[e] = r355::activate<decltype(act)::value>(sum[e]);
            });
            if(p.gate)
            {
                read(reinterpret_cast<const T*>(p.gate) + row * p.ldg + col, more);
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    sum[e] *= more[e];
            }
            if(p.c)
            {
                read(reinterpret_cast<const Out*>(p.c + group * p.strideC) + in * p.ldc + col, more);
#pragma unroll
                for(uint32_t e = 0; e < 4u; ++e)
                    sum[e] += more[e];
            }
            write(reinterpret_cast<Out*>(p.y + group * p.strideY) + in * p.ldy + col, sum);
        }
    }

    // ---- The gradient's part element by element: dz, dgate and the bias's gradient, one pass over dy, z and gate.  Bound by HBM: three operands and two results of 4099 x 4096 in bf16 31 us,
    // 5.4 TB/s.  (Made once and read by both products: in their loads it would be made anew for each tile that a row is part of, and dz would have to lie somewhere for the transposed reads anyway.  dz is rounded to 16
    // bits, as the matrix instructions take no more; a product of its f32 value in two parts would take twice as many.  With it dx and dW are off by 0.0023 of their norm in bf16, of which a result's own
    // rounding is 0.0017.)
    struct GradParams
    {
        const char*    dy;
        const char*    z;
        const char*    gate;
        char*          dz;    // NULL: dz is dy
        char*          dgate; // or NULL
        float*         sums;  // [groups][parts][n]; parts = 1: the gradient itself; NULL: none
        const int32_t* offsets;
        uint32_t       rows, n, groups, parts;
        uint32_t       lddy, ldz, ldg, lddz, lddg;
        int32_t        activation, accumulate;
    };

    // A workgroup takes EW columns a lane and one of `parts` shares of a group's rows, its four waves every fourth of them.
    template <typename T, uint32_t EW>
    __global__ void __launch_bounds__(256) linearGrad(GradParams p)
    {
        __shared__ float meet[4][64 * EW];
        LinearParams     rowsArg{};
        rowsArg.offsets = p.offsets, rowsArg.rows = p.rows;
        const uint32_t group = blockIdx.z, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        const Rows     all   = r355::rowsOf(rowsArg, group);
        const uint32_t from = all.first + static_cast<uint32_t>((uint64_t)all.count * blockIdx.y / p.parts);
        const uint32_t to   = all.first + static_cast<uint32_t>((uint64_t)all.count * (blockIdx.y + 1u) / p.parts);
        const uint32_t col  = (blockIdx.x * 64u + lane) * EW;
        using V             = vec<T, EW>;
        float total[EW];
#pragma unroll
        for(uint32_t e = 0; e < EW; ++e)
            total[e] = 0.0f;
        auto read = [&](const char* base, uint64_t row, uint32_t ld, float (&v)[EW]) {
            const T* at = reinterpret_cast<const T*>(base) + row * ld + col;
            if constexpr(EW == 1u)
                v[0] = static_cast<float>(*at);
            else
            {
                const V w = *reinterpret_cast<const V*>(at);
#pragma unroll
                for(uint32_t e = 0; e < EW; ++e)
                    v[e] = static_cast<float>(w[e]);
            }
        };
        auto write = [&](char* base, uint64_t row, uint32_t ld, const float (&v)[EW]) {
            T* at = reinterpret_cast<T*>(base) + row * ld + col;
            if constexpr(EW == 1u)
                *at = static_cast<T>(v[0]);
            else
            {
                V w;
#pragma unroll
                for(uint32_t e = 0; e < EW; ++e)
                    w[e] = static_cast<T>(v[e]);
                *reinterpret_cast<V*>(at) = w;
            }
        };
        if(col < p.n)
#pragma unroll 2
            for(uint32_t row = from + wave; row < to; row += 4u)
            {
                float d[EW];
                read(p.dy, row, p.lddy, d);
                if(p.dz)
                {
                    float z[EW], value[EW], slope[EW];
                    if(p.z)
                    {
                        read(p.z, row, p.ldz, z);
                        r355::withActivation(p.activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
                            for(uint32_t e = 0; e < EW; ++e)
                                r355::activateBoth<decltype(act)::value>(z[e], value[e], slope[e]);
                        });
                    }
                    else
#pragma unroll
                        for(uint32_t e = 0; e < EW; ++e)
                            value[e] = 0.0f, slope[e] = 1.0f;
                    if(p.dgate)
                    {
                        float g[EW];
#pragma unroll
                        for(uint32_t e = 0; e < EW; ++e)
                            g[e] = d[e] * value[e];
                        write(p.dgate, row, p.lddg, g);
                    }
                    if(p.gate)
                    {
                        float g[EW];
                        read(p.gate, row, p.ldg, g);
#pragma unroll
                        for(uint32_t e = 0; e < EW; ++e)
                            d[e] *= g[e];
                    }
#pragma unroll
                    for(uint32_t e = 0; e < EW; ++e)
                        d[e] = p.activation == R355_ACT_RELU && slope[e] == 0.0f ? 0.0f : d[e] * slope[e];
                    write(p.dz, row, p.lddz, d);
                }
#pragma unroll
                for(uint32_t e = 0; e < EW; ++e)
                    total[e] += d[e];
            }
        if(!p.sums)
            return;
#pragma unroll
        for(uint32_t e = 0; e < EW; ++e)
            meet[wave][lane * EW + e] = total[e];
        __syncthreads();
        for(uint32_t i = threadIdx.x; i < 64u * EW; i += 256u)
        {
            const uint32_t c = blockIdx.x * 64u * EW + i;
            if(c < p.n)
            {
                const float sum = ((meet[0][i] + meet[1][i]) + meet[2][i]) + meet[3][i];
                float*      to_ = p.sums + ((uint64_t)group * p.parts + blockIdx.y) * p.n + c;
                *to_            = p.parts == 1u && p.accumulate ? *to_ + sum : sum;
            }
        }
    }

    // The shares of the bias's gradient: 64 columns a workgroup, a quarter of the shares a wave (of 128 shares of 4096 columns 38 us with one thread a column)
    __global__ void __launch_bounds__(256) linearGradSums(const float* sums, float* dbias, uint32_t parts, uint32_t n, int32_t accumulate)
    {
        __shared__ float meet[4][64];
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, col = blockIdx.x * 64u + lane;
        const float*   from = sums + (uint64_t)blockIdx.y * parts * n + col;
        float          sum  = 0.0f;
        if(col < n)
#pragma unroll 8
            for(uint32_t s = wave; s < parts; s += 4u)
                sum += from[(uint64_t)s * n];
        meet[wave][lane] = sum;
        __syncthreads();
        if(wave == 0u && col < n)
        {
            sum       = ((meet[0][lane] + meet[1][lane]) + meet[2][lane]) + meet[3][lane];
            float* to = dbias + (uint64_t)blockIdx.y * n + col;
            *to       = accumulate ? *to + sum : sum;
        }
    }

    // ---- An operand whose rows do not begin on 16-byte boundaries, or end inside 16 bytes, laid out in the workspace so that they do, with zeros behind them; the macro tiles' loads
    // are 16 bytes.  A thread moves 16 of them.  Bound by memory.
    struct Copy
    {
        const char* from;
        uint64_t    stride; // bytes from group to group
        uint32_t    groups, rows, cols, ld;
        uint32_t    toRows, toCols;

        uint64_t bytes() const
        {
            return (uint64_t)groups * toRows * toCols * 2u;
        }
    };
    __global__ void __launch_bounds__(256) linearEven(Copy c, char* to)
    {
        typedef uint16_t Unaligned __attribute__((ext_vector_type(8), aligned(2)));
        const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
        const uint32_t pieces = c.toCols / 8u;
        const uint64_t row = at / pieces, group = row / c.toRows;
        if(group >= c.groups)
            return;
        const uint32_t  in = static_cast<uint32_t>(row % c.toRows), col = static_cast<uint32_t>(at % pieces) * 8u, left = in < c.rows && col < c.cols ? c.cols - col : 0u;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(c.from + group * c.stride) + (uint64_t)in * c.ld + col;
        Unaligned       v{};
        if(left >= 8u)
            v = *reinterpret_cast<const Unaligned*>(from);
        else
#pragma unroll
            for(uint32_t e = 0; e < 7u; ++e)
                if(e < left)
                    v[e] = from[e];
        *reinterpret_cast<u32x4*>(to + at * 16u) = __builtin_bit_cast(u32x4, v);
    }

    constexpr uint64_t FAR = 0x7FFFFFF0u; // bytes of a buffer that rows are taken from by their numbers
    constexpr uint32_t MOST_ROWS = 1u << 30, MOST_LENGTH = (1u << 22) - 8u, MOST_GROUPS = 1024u;

    uint64_t tilesOf(uint64_t n, uint32_t edge)
    {
        return (n + edge - 1u) / edge;
    }
    // tiles of `edge` rows that any division of the rows into groups fits in
    uint64_t mostTiles(const LinearParams& p, uint32_t edge)
    {
        if(!p.offsets)
            return tilesOf(p.rows, edge);
        const uint64_t most = p.rows / edge + p.groups;
        return most < p.rows ? most : p.rows;
    }

    // Workgroups of a product on macro tiles (of a share of the sum): every XCD has as many
    uint64_t workgroupsOf(const LinearParams& p, bool aK, uint32_t tile)
    {
        const uint64_t across = tilesOf(p.n, r355::LINEAR_COLS[tile]);
        // (of a weights' gradient: an eighth of a group's tiles for each XCD may be a tile more)
        return aK ? tilesOf(mostTiles(p, r355::LINEAR_ROWS[tile]) * across, 8u) * 8u : tilesOf(tilesOf(p.m, r355::LINEAR_ROWS[tile]) * across, 8u) * 8u * p.groups;
    }

    // How a product on macro tiles is launched: `splits` workgroups along the sum; the first `tall` rows alone where the rest goes out by a plan of its own.
    struct Plan
    {
        r355::LinearTile tile;
        uint32_t         splits, tall;
        double           us;
    };

    // What a launch takes, in us, of `tiles` with `stages` of 64 of the sum each (bf16, 256 CUs): rounds of as many tiles as the CUs hold at a time, the last one of fewer.  Per tile:
    // how many a CU holds; a round's start and end; a stage with one, two, three, four of them on a CU (the large tile, which the power limit slows: on few CUs, on all).
    struct TileTimes
    {
        uint32_t held;
        double   ends, stage[4];
    };
    constexpr TileTimes TILE_TIMES[r355::LINEAR_TILES] = {{1u, 11.0, {1.05, 1.34}}, {1u, 9.0, {0.85, 1.10}}, {1u, 6.0, {0.63, 0.80}}, {1u, 5.0, {0.55, 0.68}}, {1u, 6.0, {0.63, 0.80}}, {2u, 4.5, {0.45, 0.88}},
                                                          {4u, 3.0, {0.37, 0.42, 0.56, 0.70}}, {2u, 2.0, {1.40, 2.60}}};
    double launchTime(uint32_t tile, double tiles, double stages)
    {
        const TileTimes& t    = TILE_TIMES[tile];
        const double     cus  = r355::computeUnits(), round = cus * t.held;
        const double     full = static_cast<double>(static_cast<uint64_t>(tiles / round)), rest = tiles - full * round;
        double           us   = 2.0 + full * (t.ends + stages * t.stage[t.held == 1u ? 1u : t.held - 1u]);
        if(rest > 0.0)
        {
            const uint32_t a = static_cast<uint32_t>((rest - 1e-9) / cus); // a + 1 tiles on a CU
            us += t.ends + stages * (t.held == 1u ? t.stage[rest > 0.4 * cus ? 1u : 0u] : t.stage[a]);
        }
        return us;
    }

    // What tiles of groups, each with weights of its own, take to read them from memory (those of a group's other rows find them in the caches): 5.8 TB/s in whole rounds, of fewer tiles as much
    // as each has under way, 24 bytes a ns of 256 columns, 22 of 128 with two tiles on a CU, otherwise 12 (96 tiles of 256 columns of 6520 119 us, 176 of 128 74, 336 of 64 71).
    double weightsTime(uint32_t tile, double tiles, double k)
    {
        const uint32_t held = TILE_TIMES[tile].held;
        const double   round = static_cast<double>(r355::computeUnits()) * held, bytes = r355::LINEAR_COLS[tile] * k * 2.0, full = static_cast<double>(static_cast<uint64_t>(tiles / round)),
                     rest = tiles - full * round, each = held == 2u ? 22e3 : held == 4u || r355::LINEAR_COLS[tile] < 256u ? 12e3 : 24e3;
        return full * round * bytes / 5.8e6 + (rest > 0.0 ? bytes / (each * rest < 5.8e6 ? each : 5.8e6 / rest) : 0.0);
    }

    // floats between the rows of the sums of a split product
    uint32_t pitchOf(uint32_t n)
    {
        return (n + 3u) / 4u * 4u;
    }

    constexpr double NEVER = 1e30; // us of a plan that there is none of

    // The plan that takes the least by launchTime() of those that a launch holds (none: NEVER), with as many splits as the workspace holds.
    Plan planOf(const LinearParams& p, bool aK, bool any, uint64_t workspaceBytes)
    {
        using namespace r355;
        // (of ragged groups on average: half a tile of each is empty, of the largest tile, whose last one is as high as it has to be, a fifth; a weights' gradient has their rows for its sum)
        const double   stages = aK ? static_cast<double>(tilesOf(p.k, 64u)) : p.offsets ? static_cast<double>(p.rows) / p.groups / 64.0 + 0.5 : static_cast<double>(tilesOf(p.rows, 64u));
        const uint64_t rowsY  = aK ? p.rows : (uint64_t)p.m * p.groups;
        auto tiles = [&](uint32_t tile, uint64_t rows) {
            const double across = static_cast<double>(tilesOf(p.n, LINEAR_COLS[tile]));
            if(!aK)
                return static_cast<double>(tilesOf(p.m, LINEAR_ROWS[tile])) * p.groups * across;
            if(!p.offsets)
                return static_cast<double>(tilesOf(rows, LINEAR_ROWS[tile])) * across;
            const double met = p.groups < rows ? p.groups : static_cast<double>(rows);
            return (static_cast<double>(rows) / LINEAR_ROWS[tile] + (tile == TILE_256 ? 0.2 : 0.5) * met) * across;
        };
        // (A sum that finds its rows' groups again costs more than one that does not.)
        const double sums = aK && p.offsets ? 10.0 : 5.0;
        // (the largest tile is as high as its rows, by quarters: of groups with few rows a quarter high, which takes half the time)
        const double rowsMet = aK && p.offsets ? static_cast<double>(p.rows) / (p.groups < p.rows ? p.groups : p.rows) : 256.0, height = rowsMet < 40.0 ? 0.5 : rowsMet < 80.0 ? 0.75 : 1.0;
        Plan         best{any ? TILE_ANY : TILE_64, 1u, 0u, NEVER};
        for(uint32_t tile = any ? TILE_ANY : TILE_256; tile < (any ? LINEAR_TILES : TILE_ANY); ++tile)
        {
            if(workgroupsOf(p, aK, tile) > MAX_GROUPS)
                continue;
            // (each group that is met has a tile, whatever part of it is there)
            const double all = tiles(tile, p.rows), least = aK && p.offsets ? static_cast<double>(p.groups < p.rows ? p.groups : p.rows) * static_cast<double>(tilesOf(p.n, LINEAR_COLS[tile])) : 0.0,
                         there = all > least ? all : least;
            for(uint32_t splits = 1u; splits <= 64u; splits += splits < 4u ? 1u : splits / 2u)
            {
                // (a sum is split in whole stages, four of them at least)
                if(splits > 1u && (stages < 4.0 * splits || rowsY * pitchOf(p.n) * 4u * splits > workspaceBytes || there > computeUnits()))
                    break;
                const double launch = launchTime(tile, all * splits, stages / splits) * (tile == TILE_256 ? height : 1.0);
                // (a third more where many groups have rows of a second tile, which does not find all of the weights in the caches)
                const double again = 0.5 + rowsMet / LINEAR_ROWS[tile], reads = aK && p.offsets ? weightsTime(tile, there * splits, static_cast<double>(p.k) / splits * least / there) * (again < 1.0 ? 1.0 : again < 1.3 ? again : 1.3) : 0.0;
                const double us     = (launch > reads ? launch : reads) + (splits > 1u ? sums + static_cast<double>(rowsY) * p.n * 4.0 * (2u * splits + 1u) / 5e6 : 0.0);
                if(us < best.us)
                    best = Plan{static_cast<LinearTile>(tile), splits, 0u, us};
            }
            // whole rounds of large tiles, then the rest
            if(tile == TILE_256 && aK && !p.offsets)
            {
                const uint64_t across = tilesOf(p.n, 256u), rounds = static_cast<uint64_t>(all) / computeUnits(), tall = rounds * computeUnits() / across * 256u;
                if(tall > 0u && tall < p.rows)
                {
                    LinearParams rest = p;
                    rest.rows         = static_cast<uint32_t>(p.rows - tall);
                    const double us   = launchTime(TILE_256, tiles(TILE_256, tall), stages) + planOf(rest, aK, any, workspaceBytes).us;
                    if(us < best.us)
                        best = Plan{TILE_256, 1u, static_cast<uint32_t>(tall), us};
                }
            }
        }
        return best;
    }

    // One or two rows: weights that no cache keeps from one call to the next are read nontemporally (16 experts of 4096 x 4096 95 -> 85 us, 8192 x 8192 29.8 -> 26.0; three matrices of
    // 2048 x 8192 in turn, which the 256 MiB of the memory-side cache hold: 8.1 -> 9.1).
    bool streams(const LinearParams& p)
    {
        const uint64_t met = p.offsets && p.groups < p.rows ? p.groups : p.offsets ? p.rows : 1u;
        return met * p.n * p.k * 2u > (uint64_t{96} << 20);
    }

    template <typename T, uint32_t ROWS>
    void launchDots(LinearParams p, hipStream_t s)
    {
        // Few waves along the sum, each with a long stretch of 16 rows, as long as there are enough workgroups (32 experts of 4096 x 4096, 16 of them met, one, two, four, eight waves: 84, 95, 93, 105 us;
        // 16384 x 4096 29, 27, 25, 27; 8192 x 8192 38, 28, 26, 26); of small layers one set of them a workgroup.
        const uint32_t pieces = static_cast<uint32_t>(tilesOf(p.k, 512u)), enough = r355::computeUnits() * 5u / 4u;
        uint32_t       wavesK = 1u;
        while(wavesK < WAVES && 2u * wavesK <= pieces && tilesOf(p.n, 16u * (WAVES / wavesK)) * mostTiles(p, ROWS) < enough)
            wavesK *= 2u;
        const uint32_t sets = tilesOf(p.n, 16u * (WAVES / wavesK)) * mostTiles(p, ROWS) >= enough ? WAVES / wavesK : 1u;
        p.tilesN              = static_cast<uint32_t>(tilesOf(p.n, 16u * sets));
        const uint64_t groups = (mostTiles(p, ROWS) * p.tilesN + 7u) / 8u * 8u;
        const auto     kernel = streams(p) ? linearDots<T, ROWS, true> : linearDots<T, ROWS, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(64 * wavesK * sets), 0, s, p, wavesK);
    }
    template <typename T>
    void launchFew(LinearParams p, hipStream_t s)
    {
        p.tilesN             = static_cast<uint32_t>(tilesOf(p.n, 16u));
        const uint64_t groups = (mostTiles(p, 16u) * p.tilesN + 7u) / 8u * 8u;
        hipLaunchKernelGGL(linearFew<T>, dim3(static_cast<uint32_t>(groups)), dim3(64 * WAVES), 0, s, p);
    }

    int tooMany(const char* what)
    {
        return r355::fail(R355_ERR_BAD_SIZE, "%s: more than 2^24 tiles of the result", what);
    }

    // whether rows begin with a cache line
    bool lines(const void* at, uint32_t ld, uint32_t bytes)
    {
        return r355::aligned(at, 128) && (uint64_t)ld * bytes % 128u == 0u;
    }

    // The tiles of a launch: sets them in p, returns the workgroups
    uint32_t tilesOfLaunch(LinearParams& p, bool aK, r355::LinearTile tile)
    {
        // (shares of a split sum are read again at once)
        p.linesY = p.splits == 1u && lines(p.y, p.ldy, p.outF32 ? 4u : 2u), p.linesZ = lines(p.z, p.ldz, 2u);
        p.tilesN = static_cast<uint32_t>(tilesOf(p.n, r355::LINEAR_COLS[tile])), p.tilesM = static_cast<uint32_t>(tilesOf(p.m, r355::LINEAR_ROWS[tile]));
        return static_cast<uint32_t>(workgroupsOf(p, aK, tile));
    }
    void launchTile(int32_t type, LinearParams p, bool aK, bool bK, r355::LinearTile tile, hipStream_t s)
    {
        const uint32_t workgroups = tilesOfLaunch(p, aK, tile);
        if(type == R355_F16)
            r355::linearTilesF16(p, aK, bK, tile, workgroups, s);
        else
            r355::linearTilesBF16(p, aK, bK, tile, workgroups, s);
    }

    uint64_t usable(const void* workspace, uint64_t bytes)
    {
        return workspace && r355::aligned(workspace, 16) ? bytes : 0u;
    }

    uint64_t rowsOfResult(const LinearParams& p, bool aK)
    {
        return aK ? p.rows : (uint64_t)p.m * p.groups;
    }
    uint64_t sumsBytes(const LinearParams& p, bool aK, uint32_t splits) // of a split product
    {
        return splits > 1u ? rowsOfResult(p, aK) * pitchOf(p.n) * 4u * splits : 0u;
    }
    // a product whose shares of the sum go to `sums`
    LinearParams sharesOf(const LinearParams& p, bool aK, uint32_t splits, void* sums)
    {
        const uint32_t pitch = pitchOf(p.n);
        LinearParams   d     = p;
        d.splits = splits, d.y = static_cast<char*>(sums), d.ldy = pitch, d.strideY = (uint64_t)p.m * pitch * 4u, d.strideSplit = rowsOfResult(p, aK) * pitch * 4u, d.outF32 = 1u;
        d.bias = d.gate = d.c = nullptr, d.z = nullptr, d.activation = R355_ACT_NONE;
        return d;
    }
    void launchReduce(int32_t type, const LinearParams& p, bool aK, uint32_t splits, const void* sums, hipStream_t s)
    {
        const uint64_t rowsY = rowsOfResult(p, aK);
        LinearParams   r     = p;
        r.splits             = splits;
        const dim3 grid(static_cast<uint32_t>(tilesOf(p.n, 1024u)), static_cast<uint32_t>(rowsY < 32768u ? rowsY : 32768u));
        const auto kernel = type == R355_F16 ? (p.outF32 ? linearReduce<_Float16, float> : linearReduce<_Float16, _Float16>)
                                             : (p.outF32 ? linearReduce<__bf16, float> : linearReduce<__bf16, __bf16>);
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, r, static_cast<const float*>(sums), rowsY, pitchOf(p.n));
    }

    // one product on macro tiles, by its plan
    void launchTiles(int32_t type, const LinearParams& p, bool aK, bool bK, bool any, const Plan& plan, void* workspace, uint64_t workspaceBytes, hipStream_t s)
    {
        if(plan.splits > 1u)
        {
            launchTile(type, sharesOf(p, aK, plan.splits, workspace), aK, bK, plan.tile, s);
            return launchReduce(type, p, aK, plan.splits, workspace, s);
        }
        if(plan.tall == 0u)
            return launchTile(type, p, aK, bK, plan.tile, s);
        LinearParams first = p, rest = p;
        first.rows = plan.tall, rest.rows = p.rows - plan.tall;
        const uint64_t outBytes = p.outF32 ? 4u : 2u, by = plan.tall;
        if(p.source)
            rest.source += by;
        else
            rest.a += by * p.lda * 2u;
        rest.y += by * p.ldy * outBytes;
        rest.c = p.c ? p.c + by * p.ldc * outBytes : nullptr, rest.gate = p.gate ? p.gate + by * p.ldg * 2u : nullptr, rest.z = p.z ? p.z + by * p.ldz * 2u : nullptr;
        launchTile(type, first, aK, bK, plan.tile, s);
        launchTiles(type, rest, aK, bK, any, planOf(rest, aK, any, usable(workspace, workspaceBytes)), workspace, workspaceBytes, s);
    }

    // Both gradients in one launch of small tiles: how their sums are split, and what it takes (as launchTime(), with tiles of two lengths).
    struct PlanBoth
    {
        uint32_t splitsX, splitsW;
        double   us;
    };
    PlanBoth planBoth(const LinearParams& px, const LinearParams& pw, uint64_t workspaceBytes)
    {
        using namespace r355;
        const TileTimes& t    = TILE_TIMES[TILE_64];
        const double     cus  = computeUnits(), stagesX = static_cast<double>(tilesOf(px.k, 64u)), last = t.stage[3];
        const double     stagesW = pw.offsets ? static_cast<double>(pw.rows) / pw.groups / 64.0 + 0.5 : static_cast<double>(tilesOf(pw.rows, 64u));
        const double     met = px.groups < px.rows ? px.groups : px.rows;
        const double     tilesX = (px.offsets ? px.rows / 64.0 + 0.5 * met : static_cast<double>(tilesOf(px.rows, 64u))) * static_cast<double>(tilesOf(px.n, 64u));
        const double     tilesW = static_cast<double>(tilesOf(pw.m, 64u) * tilesOf(pw.n, 64u)) * pw.groups;
        PlanBoth         best{1u, 1u, NEVER};
        const uint64_t   workgroupsX = workgroupsOf(px, true, TILE_64), workgroupsW = workgroupsOf(pw, false, TILE_64);
        auto reduced = [](const LinearParams& p, bool aK, uint32_t splits) { return splits > 1u ? 5.0 + static_cast<double>(rowsOfResult(p, aK)) * p.n * 4.0 * (2u * splits + 1u) / 5e6 : 0.0; };
        for(uint32_t sx = 1u; sx <= 16u && (sx == 1u || (stagesX >= 4.0 * sx && tilesX <= cus)); sx *= 2u)
            for(uint32_t sw = 1u; sw <= 16u && (sw == 1u || (stagesW >= 4.0 * sw && tilesW <= cus)); sw *= 2u)
            {
                if(sumsBytes(px, true, sx) + sumsBytes(pw, false, sw) > workspaceBytes || workgroupsX * sx + workgroupsW * sw > MAX_GROUPS)
                    continue;
                const double nx = tilesX * sx, nw = tilesW * sw, lx = stagesX / sx, lw = stagesW / sw, n = nx + nw, longer = lx > lw ? nx : nw, shorter = lx < lw ? lx : lw, rest = (lx > lw ? lx : lw) - shorter;
                auto         stage = [&](double tiles) { return t.stage[tiles > 3.0 * cus ? 3u : tiles > 2.0 * cus ? 2u : tiles > cus ? 1u : 0u]; };
                const double us = 2.0 + reduced(px, true, sx) + reduced(pw, false, sw)
                                  + (n <= 4.0 * cus ? t.ends + shorter * stage(n) + rest * stage(longer)
                                                    : (nx * (t.ends + lx * last) + nw * (t.ends + lw * last)) / (4.0 * cus) + 0.5 * (t.ends + (shorter + rest) * last));
                if(us < best.us)
                    best = PlanBoth{sx, sw, us};
            }
        return best;
    }

    bool evenRows(const void* at, uint32_t ld, uint32_t bytes) // rows on 16-byte boundaries
    {
        return !at || (r355::aligned(at, 16) && (uint64_t)ld * bytes % 16u == 0u);
    }

    // ... of a product's operand, whose rows are there whatever their address says (a query may come before there is one)
    bool evenOperand(const void* at, uint32_t ld)
    {
        return r355::aligned(at, 16) && ld % 8u == 0u;
    }

    int checkCommon(const char* what, int32_t type, int32_t activation, uint32_t rows, uint32_t n, uint32_t k, uint32_t groups, const int32_t* offsets)
    {
        if(type != R355_F16 && type != R355_BF16)
            return r355::fail(R355_ERR_UNSUPPORTED, "%s: operands are f16 or bf16", what);
        if(activation < R355_ACT_NONE || activation > R355_ACT_SILU)
            return r355::fail(R355_ERR_BAD_ARG, "%s: unknown activation %d", what, activation);
        if(n == 0 || k == 0 || groups == 0)
            return r355::fail(R355_ERR_BAD_ARG, "%s: n, k and groups must be non-zero", what);
        if(rows > MOST_ROWS || n > MOST_LENGTH || k > MOST_LENGTH || groups > MOST_GROUPS)
            return r355::fail(R355_ERR_BAD_SIZE, "%s: at most %u rows, n and k of %u and %u groups, got %u, %u, %u and %u", what, MOST_ROWS, MOST_LENGTH, MOST_GROUPS, rows, n, k, groups);
        if(groups > 1u && !offsets)
            return r355::fail(R355_ERR_BAD_ARG, "%s: %u groups of rows need offsets", what, groups);
        if(!r355::aligned(offsets, 4))
            return r355::fail(R355_ERR_MISALIGNED, "%s: offsets need the alignment of their elements", what);
        return R355_OK;
    }
    int checkMatrix(const char* what, const char* name, const void* at, uint32_t ld, uint32_t width, uint32_t bytes)
    {
        if(!at)
            return R355_OK;
        if(ld < width || ld > MOST_LENGTH)
            return r355::fail(R355_ERR_BAD_ARG, "%s: the leading dimension %u of %s must be %u (its row) to %u", what, ld, name, width, MOST_LENGTH);
        if(!r355::aligned(at, bytes))
            return r355::fail(R355_ERR_MISALIGNED, "%s: %s needs the alignment of its elements", what, name);
        return R355_OK;
    }
    int checkStride(const char* what, const char* name, int64_t stride, uint32_t groups, uint64_t least)
    {
        if(groups > 1u && (stride < 0 || static_cast<uint64_t>(stride) < least || stride > (int64_t{1} << 46)))
            return r355::fail(R355_ERR_BAD_ARG, "%s: %s=%lld is less than the %llu elements of a group", what, name, static_cast<long long>(stride), static_cast<unsigned long long>(least));
        return R355_OK;
    }

    // Shares of a group's rows in the gradient's pass: four workgroups a CU, 16 rows each at least
    uint64_t gradParts(const r355_linear_backward_args& a, uint32_t strips)
    {
        const uint64_t parts = tilesOf(4u * r355::computeUnits(), strips * a.groups), most = tilesOf(a.rows, 16u * a.groups);
        return most == 0u ? 1u : parts < most ? parts : most;
    }

    LinearParams forwardParams(const r355_linear_args& a)
    {
        LinearParams p{};
        p.a = static_cast<const char*>(a.x), p.b = static_cast<const char*>(a.w), p.bias = static_cast<const char*>(a.bias), p.gate = static_cast<const char*>(a.gate);
        p.c = static_cast<const char*>(a.c), p.y = static_cast<char*>(a.y), p.z = static_cast<char*>(a.z);
        p.offsets = a.offsets, p.source = a.source, p.rows = a.rows, p.n = a.n, p.k = a.k, p.groups = a.groups, p.sourceRows = a.x_rows;
        p.lda = a.ldx, p.ldb = a.ldw, p.ldy = a.ldy, p.ldz = a.ldz, p.ldg = a.ldg, p.ldc = a.ldc;
        p.strideB = static_cast<uint64_t>(a.groups > 1u ? a.w_stride : 0) * 2u, p.splits = 1u, p.activation = a.activation, p.outF32 = a.out_type == R355_F32;
        return p;
    }
    bool evenForward(const r355_linear_args& a)
    {
        return a.k % 8u == 0u && evenOperand(a.x, a.ldx) && evenOperand(a.w, a.ldw) && (a.groups == 1u || a.w_stride % 8 == 0);
    }
    // The kernel of a forward product by its rows: us of dot products, of the kernel for few rows and of tiles for 4096 x 4096: one row 7.3, 8.0, 14; two 7.8, 8.2, 14; four 8.8, 8.3, 14; sixteen
    // -, 10, 15; 24 -, 17, 14.  Of experts with about one row each (32 of 4096 x 4096, 128 of 1024 x 1024) the first two 84, 105 and 49, 75; with four (8, 32, 64 experts of 2048 x 2048) 21, 15, 16; 79,
    // 54, 48 and 143, 105, 95; with twelve 37, 21, 17; 166, 73, 48 and 321, 143, 95: the kernel for few rows reads the weights at 5.7 TB/s, and once more for every 20 rows or so, after 4 us, whatever their
    // lengths; where the tiles' plan takes more, as of few groups, it wins (4 of 1024 x 1024 with four 5.6, 4.9, 6.7; 16 of 1326 x 6520 with two -, 51, 71).
    // The host knows the average alone.  Rows that meet in fewer groups take less time than rows of all of them, if more than a choice by the rows themselves would: 128 rows over 128 groups of
    // 2048 x 2048, one each 182, in an eighth of the groups 65, in one 48 (one matrix of as many rows 10); 256 over 64, four each 95, in an eighth 21, in one 43 (9); 2048 over 64 97, 44, 44 (23).
    enum class Kernel
    {
        DOTS,
        FEW,
        TILES
    };
    Kernel kernelOf(const r355_linear_args& a, bool even, uint64_t room)
    {
        const LinearParams p = forwardParams(a);
        // (both have a workgroup of up to 512 threads for 16 columns of one row and more, of 16 rows and less: as many for every XCD as a launch holds)
        auto held = [&](uint32_t rows) { return tilesOf(mostTiles(p, rows) * tilesOf(p.n, 16u), 8u) * 8u <= r355::MAX_GROUPS / 2u; };
        if(!even)
            return Kernel::TILES;
        if(a.groups == 1u)
            return a.rows <= 2u ? Kernel::DOTS : a.rows <= 16u ? Kernel::FEW : Kernel::TILES; // (of 2^22 columns a launch holds them)
        if(a.rows <= a.groups && held(1u))
            return Kernel::DOTS;
        const double few = 4.0 + static_cast<double>(a.groups) * a.n * a.k * 2.0 / 5.7e6 * (1.0 + 0.05 * a.rows / a.groups);
        return a.rows / a.groups < 9u && held(16u) && few < planOf(p, true, false, room).us ? Kernel::FEW : Kernel::TILES;
    }
    LinearParams inputParams(const r355_linear_backward_args& a, const char* dz, uint32_t lddz)
    {
        LinearParams p{};
        p.offsets = a.offsets, p.rows = a.rows, p.groups = a.groups, p.splits = 1u;
        p.a = dz, p.lda = lddz, p.b = static_cast<const char*>(a.w), p.ldb = a.ldw, p.strideB = static_cast<uint64_t>(a.groups > 1u ? a.w_stride : 0) * 2u;
        p.y = static_cast<char*>(a.dx), p.ldy = a.lddx, p.n = a.k, p.k = a.n;
        return p;
    }
    LinearParams weightParams(const r355_linear_backward_args& a, const char* dz, uint32_t lddz)
    {
        LinearParams p{};
        p.offsets = a.offsets, p.rows = a.rows, p.groups = a.groups, p.splits = 1u;
        p.a = dz, p.lda = lddz, p.b = static_cast<const char*>(a.x), p.ldb = a.ldx, p.m = a.n, p.n = a.k;
        p.y = static_cast<char*>(a.dw), p.ldy = a.lddw, p.strideY = static_cast<uint64_t>(a.groups > 1u ? a.dw_stride : 0) * r355::dtypeBytes(a.grad_type);
        p.c = a.accumulate ? static_cast<const char*>(a.dw) : nullptr, p.ldc = a.lddw, p.strideC = p.strideY, p.outF32 = a.grad_type == R355_F32;
        return p;
    }
    bool evenInput(const r355_linear_backward_args& a, const char* dz, uint32_t lddz)
    {
        return a.n % 8u == 0u && evenOperand(dz, lddz) && evenOperand(a.w, a.ldw) && (a.groups == 1u || a.w_stride % 8 == 0);
    }
    bool evenWeight(const r355_linear_backward_args& a, const char* dz, uint32_t lddz)
    {
        return evenOperand(dz, lddz) && evenOperand(a.x, a.ldx);
    }
    // Operands to be laid out anew in a workspace, one after the other, and what that takes
    struct Copies
    {
        Copy     copy[3] = {};
        uint32_t count   = 0u;
        uint64_t bytes   = 0u;
        double   us      = 0.0;

        // where `what` will lie
        const char* add(const Copy& what, const void* workspace)
        {
            const char* at = static_cast<const char*>(workspace) + bytes;
            copy[count++]  = what;
            bytes += what.bytes();
            us += 3.0 + 2.0 * static_cast<double>(what.bytes()) / 4.5e6;
            return at;
        }
        void launch(void* workspace, hipStream_t s) const
        {
            char* at = static_cast<char*>(workspace);
            for(uint32_t i = 0; i < count; ++i)
            {
                hipLaunchKernelGGL(linearEven, dim3(static_cast<uint32_t>((copy[i].bytes() / 16u + 255u) / 256u)), dim3(256), 0, s, copy[i], at);
                at += copy[i].bytes();
            }
        }
        bool fit(uint64_t room) const // (and a launch holds the largest)
        {
            return bytes <= room && bytes / 4096u < r355::MAX_GROUPS;
        }
    };
    uint32_t eights(uint32_t n)
    {
        return (n + 7u) / 8u * 8u;
    }
    // The forward product with even operands.  (Both gradients of 1500 x 1500 x 1496, whose rows of 1500 are 3000 bytes: 152 us on tiles of single elements, 42 so, 35 of 1504.)
    Copies evened(const r355_linear_args& a, const void* workspace, LinearParams& p)
    {
        Copies         c;
        const uint32_t rows = a.source ? a.x_rows : a.rows;
        if(a.k % 8u != 0u || !evenOperand(a.x, a.ldx))
            p.a = c.add(Copy{p.a, 0u, 1u, rows, a.k, a.ldx, rows, eights(a.k)}, workspace), p.lda = eights(a.k);
        if(a.k % 8u != 0u || !evenOperand(a.w, a.ldw) || (a.groups > 1u && a.w_stride % 8 != 0))
            p.b = c.add(Copy{p.b, p.strideB, a.groups, a.n, a.k, a.ldw, a.n, eights(a.k)}, workspace), p.ldb = eights(a.k), p.strideB = (uint64_t)a.n * eights(a.k) * 2u;
        p.k = eights(a.k);
        if(a.source && (uint64_t)rows * p.lda * 2u > FAR)
            c.bytes = ~0ull; // (rows taken by their numbers must lie within a buffer's reach)
        return c;
    }
    // Both gradients with even operands: dz (with zeros behind its rows, and as many rows of zeros behind those of w: the sum of dx goes over them), w, x
    Copies evened(const r355_linear_backward_args& a, const char* dz, uint32_t lddz, bool wantX, bool wantW, const void* workspace, LinearParams& px, LinearParams& pw)
    {
        Copies         c;
        const uint32_t n8 = eights(a.n), k8 = eights(a.k);
        if((wantX && a.n % 8u != 0u) || !evenOperand(dz, lddz))
            px.a = pw.a = c.add(Copy{dz, 0u, 1u, a.rows, a.n, lddz, a.rows, n8}, workspace), px.lda = pw.lda = n8;
        if(wantX && (a.n % 8u != 0u || !evenOperand(a.w, a.ldw) || (a.groups > 1u && a.w_stride % 8 != 0)))
            px.b = c.add(Copy{px.b, px.strideB, a.groups, a.n, a.k, a.ldw, n8, k8}, workspace), px.ldb = k8, px.strideB = (uint64_t)n8 * k8 * 2u;
        if(wantW && !evenOperand(a.x, a.ldx))
            pw.b = c.add(Copy{pw.b, 0u, 1u, a.rows, a.k, a.ldx, a.rows, k8}, workspace), pw.ldb = k8;
        px.k = n8;
        return c;
    }

    // what the sums of a split product take
    size_t splitBytes(LinearParams p, bool aK, bool any)
    {
        Plan plan = planOf(p, aK, any, ~0ull);
        while(plan.tall != 0u) // (the rest may be split)
        {
            p.rows -= plan.tall;
            plan = planOf(p, aK, any, ~0ull);
        }
        return static_cast<size_t>(sumsBytes(p, aK, plan.splits));
    }

    // How the products of the gradients go out
    struct BackwardPlan
    {
        Plan     x, w;
        PlanBoth both;
        bool     together;
        double   us;
    };
    BackwardPlan planBackward(const LinearParams& px, const LinearParams& pw, bool wantX, bool wantW, bool anyX, bool anyW, uint64_t room)
    {
        BackwardPlan plan{wantX ? planOf(px, true, anyX, room) : Plan{}, wantW ? planOf(pw, false, anyW, room) : Plan{}, {}, false, 0.0};
        plan.us = plan.x.us + plan.w.us;
        if(wantX && wantW && !anyX && !anyW)
        {
            plan.both     = planBoth(px, pw, room);
            plan.together = plan.both.us < plan.us;
            plan.us       = plan.together ? plan.both.us : plan.us;
        }
        return plan;
    }
    size_t backwardBytes(const BackwardPlan& plan, const LinearParams& px, const LinearParams& pw, bool wantX, bool wantW, bool anyX, bool anyW)
    {
        if(plan.together)
            return static_cast<size_t>(sumsBytes(px, true, plan.both.splitsX) + sumsBytes(pw, false, plan.both.splitsW));
        const size_t x = wantX ? splitBytes(px, true, anyX) : 0u, w = wantW ? splitBytes(pw, false, anyW) : 0u;
        return x > w ? x : w;
    }

    // What a call launches, by its arguments and the workspace offered; the entry points launch it, the queries report it.
    struct ForwardChoice
    {
        Kernel       kernel;
        bool         any; // element by element
        LinearParams p;
        Plan         plan; // TILES
        Copies       copies;

        bool held() const // whether there are launches of as many tiles
        {
            return kernel != Kernel::TILES || plan.us < NEVER;
        }
    };
    ForwardChoice chooseForward(const r355_linear_args& a, const void* workspace, uint64_t room)
    {
        ForwardChoice c{};
        const bool    even = evenForward(a);
        c.p = forwardParams(a), c.kernel = kernelOf(a, even, room);
        if(c.kernel != Kernel::TILES)
            return c;
        c.any = !even, c.plan = planOf(c.p, true, c.any, room);
        if(!even)
        {
            LinearParams q      = c.p;
            const Copies copies = evened(a, workspace, q);
            if(copies.fit(room))
                if(const Plan other = planOf(q, true, false, room - copies.bytes); other.us + copies.us < c.plan.us)
                    c.p = q, c.plan = other, c.copies = copies, c.any = false;
        }
        return c;
    }
    struct BackwardChoice
    {
        bool         element, wantX, wantW, anyX, anyW; // element: dz is made first
        LinearParams px, pw;
        BackwardPlan plan;
        Copies       copies;

        bool held() const
        {
            return plan.us < NEVER;
        }
    };
    BackwardChoice chooseBackward(const r355_linear_backward_args& a, const void* workspace, uint64_t room)
    {
        BackwardChoice c{};
        c.element              = a.activation != R355_ACT_NONE || a.gate;
        const char*    dz      = static_cast<const char*>(c.element ? a.dz : a.dy);
        const uint32_t lddz    = c.element ? a.lddz : a.lddy;
        c.wantX = a.dx && a.rows, c.wantW = a.dw != nullptr, c.anyX = c.wantX && !evenInput(a, dz, lddz), c.anyW = c.wantW && !evenWeight(a, dz, lddz);
        c.px = inputParams(a, dz, lddz), c.pw = weightParams(a, dz, lddz);
        c.plan = planBackward(c.px, c.pw, c.wantX, c.wantW, c.anyX, c.anyW, room);
        if((c.anyX || c.anyW) && a.rows)
        {
            LinearParams x = c.px, w = c.pw;
            const Copies copies = evened(a, dz, lddz, c.wantX, c.wantW, workspace, x, w);
            if(copies.fit(room))
                if(const BackwardPlan other = planBackward(x, w, c.wantX, c.wantW, false, false, room - copies.bytes); other.us + copies.us < c.plan.us)
                    c.px = x, c.pw = w, c.plan = other, c.copies = copies, c.anyX = c.anyW = false;
        }
        return c;
    }

    r355_linear_plan reported(Kernel kernel, bool any, const Plan& plan, const Copies& copies)
    {
        r355_linear_plan r{};
        r.kernel = kernel == Kernel::DOTS ? R355_LINEAR_DOTS : kernel == Kernel::FEW ? R355_LINEAR_FEW : any ? R355_LINEAR_ELEMENTS : R355_LINEAR_TILES;
        if(kernel == Kernel::TILES)
            r.tile_rows = r355::LINEAR_ROWS[plan.tile], r.tile_cols = r355::LINEAR_COLS[plan.tile], r.splits = plan.splits, r.first_rows = plan.tall, r.copies = copies.count;
        return r;
    }

    int checkForward(const r355_linear_args& a)
    {
        constexpr const char* what = "linear";
        R355_TRY(checkCommon(what, a.in_type, a.activation, a.rows, a.n, a.k, a.groups, a.offsets));
        if(a.out_type != a.in_type && a.out_type != R355_F32)
            return r355::fail(R355_ERR_UNSUPPORTED, "linear: the result has the type of x or is f32");
        if(a.rows == 0)
            return R355_OK; // (nothing is read or written)
        if(!a.x || !a.w || !a.y)
            return r355::fail(R355_ERR_BAD_ARG, "linear: null pointer");
        const uint32_t outBytes = r355::dtypeBytes(a.out_type);
        R355_TRY(checkMatrix(what, "x", a.x, a.ldx, a.k, 2));
        R355_TRY(checkMatrix(what, "w", a.w, a.ldw, a.k, 2));
        R355_TRY(checkMatrix(what, "bias", a.bias, a.n, a.n, 2));
        R355_TRY(checkMatrix(what, "gate", a.gate, a.ldg, a.n, 2));
        R355_TRY(checkMatrix(what, "z", a.z, a.ldz, a.n, 2));
        R355_TRY(checkMatrix(what, "c", a.c, a.ldc, a.n, outBytes));
        R355_TRY(checkMatrix(what, "y", a.y, a.ldy, a.n, outBytes));
        R355_TRY(checkStride(what, "w_stride", a.w_stride, a.groups, (uint64_t)(a.n - 1u) * a.ldw + a.k));
        if(a.source)
        {
            if(!r355::aligned(a.source, 4))
                return r355::fail(R355_ERR_MISALIGNED, "linear: source needs the alignment of its elements");
            if(a.x_rows == 0 || (uint64_t)a.x_rows * a.ldx * 2u > FAR)
                return r355::fail(R355_ERR_BAD_SIZE, "linear: rows taken by their numbers must be of 1 to 2^31 bytes of x, got %u rows %u elements apart", a.x_rows, a.ldx);
        }
        return R355_OK;
    }
    int checkBackward(const r355_linear_backward_args& a)
    {
        constexpr const char* what = "linear_backward";
        R355_TRY(checkCommon(what, a.in_type, a.activation, a.rows, a.n, a.k, a.groups, a.offsets));
        if(a.grad_type != a.in_type && a.grad_type != R355_F32)
            return r355::fail(R355_ERR_UNSUPPORTED, "linear_backward: dw has the type of x or is f32");
        const bool slope = a.activation != R355_ACT_NONE, element = slope || a.gate;
        if(a.rows != 0 && (!a.dy || (a.dx && !a.w) || (a.dw && !a.x)))
            return r355::fail(R355_ERR_BAD_ARG, "linear_backward: null pointer");
        if(a.rows != 0 && slope && !a.z)
            return r355::fail(R355_ERR_BAD_ARG, "linear_backward: an activation's gradient needs z");
        if(a.dgate && (!a.gate || !a.z))
            return r355::fail(R355_ERR_BAD_ARG, "linear_backward: dgate needs gate and z");
        if(element && !a.dz)
            return r355::fail(R355_ERR_BAD_ARG, "linear_backward: with an activation or a gate dz is needed");
        const uint32_t gradBytes = r355::dtypeBytes(a.grad_type);
        R355_TRY(checkMatrix(what, "dy", a.dy, a.lddy, a.n, 2));
        R355_TRY(checkMatrix(what, "x", a.x, a.ldx, a.k, 2));
        R355_TRY(checkMatrix(what, "w", a.w, a.ldw, a.k, 2));
        R355_TRY(checkMatrix(what, "z", a.z, a.ldz, a.n, 2));
        R355_TRY(checkMatrix(what, "gate", a.gate, a.ldg, a.n, 2));
        R355_TRY(checkMatrix(what, "dz", element ? a.dz : nullptr, a.lddz, a.n, 2));
        R355_TRY(checkMatrix(what, "dgate", a.dgate, a.lddg, a.n, 2));
        R355_TRY(checkMatrix(what, "dx", a.dx, a.lddx, a.k, 2));
        R355_TRY(checkMatrix(what, "dw", a.dw, a.lddw, a.k, gradBytes));
        R355_TRY(checkMatrix(what, "dbias", a.dbias, a.n, a.n, 4));
        if(a.dx)
            R355_TRY(checkStride(what, "w_stride", a.w_stride, a.groups, (uint64_t)(a.n - 1u) * a.ldw + a.k));
        if(a.dw)
            R355_TRY(checkStride(what, "dw_stride", a.dw_stride, a.groups, (uint64_t)(a.n - 1u) * a.lddw + a.k));
        return R355_OK;
    }
} // namespace

extern "C" int r355_linear(const r355_linear_args* args, void* stream)
{
    constexpr const char* what = "linear";
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "linear: null arguments");
    const r355_linear_args& a = *args;
    R355_TRY(checkForward(a));
    if(a.rows == 0)
        return R355_OK;
    const uint64_t      room = usable(a.workspace, a.workspace_bytes);
    const ForwardChoice c    = chooseForward(a, a.workspace, room);
    const hipStream_t   s    = static_cast<hipStream_t>(stream);
    const bool          f16  = a.in_type == R355_F16;
    if(!c.held())
        return tooMany(what);
    r355::beginCall();
    switch(c.kernel)
    {
    case Kernel::DOTS:
        if(a.rows == 1u)
            f16 ? launchDots<_Float16, 1>(c.p, s) : launchDots<__bf16, 1>(c.p, s);
        else
            f16 ? launchDots<_Float16, 2>(c.p, s) : launchDots<__bf16, 2>(c.p, s);
        break;
    case Kernel::FEW: f16 ? launchFew<_Float16>(c.p, s) : launchFew<__bf16>(c.p, s); break;
    default:
        c.copies.launch(a.workspace, s);
        launchTiles(a.in_type, c.p, true, true, c.any, c.plan, static_cast<char*>(a.workspace) + c.copies.bytes, room - c.copies.bytes, s);
    }
    return r355::checkLaunch(what);
}

extern "C" int r355_linear_launch_plan(const r355_linear_args* args, r355_linear_plan* plan)
{
    if(!args || !plan)
        return r355::fail(R355_ERR_BAD_ARG, "linear_launch_plan: null arguments");
    R355_TRY(checkForward(*args));
    *plan = r355_linear_plan{};
    if(args->rows == 0)
        return R355_OK;
    const ForwardChoice c = chooseForward(*args, args->workspace, usable(args->workspace, args->workspace_bytes));
    if(!c.held())
        return tooMany("linear");
    *plan = reported(c.kernel, c.any, c.plan, c.copies);
    return R355_OK;
}

extern "C" size_t r355_linear_workspace_bytes(const r355_linear_args* args)
{
    if(!args || args->rows == 0 || args->n == 0 || args->k == 0 || args->groups == 0)
        return 0;
    const ForwardChoice c = chooseForward(*args, nullptr, ~0ull);
    return c.kernel == Kernel::TILES ? static_cast<size_t>(c.copies.bytes) + splitBytes(c.p, true, c.any) : 0u;
}

extern "C" size_t r355_linear_backward_workspace_bytes(const r355_linear_backward_args* args)
{
    if(!args || args->rows == 0 || args->n == 0 || args->k == 0 || args->groups == 0)
        return 0;
    const r355_linear_backward_args& a = *args;
    size_t                           most = 0u; // (one after the other)
    if(a.dbias)
        if(const uint64_t parts = gradParts(a, static_cast<uint32_t>(tilesOf(a.n, 512u))); parts > 1u)
            most = static_cast<size_t>(parts * a.groups * a.n * 4u);
    const BackwardChoice c     = chooseBackward(a, nullptr, ~0ull);
    const size_t         bytes = static_cast<size_t>(c.copies.bytes) + backwardBytes(c.plan, c.px, c.pw, c.wantX, c.wantW, c.anyX, c.anyW);
    return most > bytes ? most : bytes;
}

extern "C" int r355_linear_backward_launch_plan(const r355_linear_backward_args* args, r355_linear_plan* dx, r355_linear_plan* dw)
{
    if(!args || !dx || !dw)
        return r355::fail(R355_ERR_BAD_ARG, "linear_backward_launch_plan: null arguments");
    R355_TRY(checkBackward(*args));
    const BackwardChoice c = chooseBackward(*args, args->workspace, usable(args->workspace, args->workspace_bytes));
    if(!c.held())
        return tooMany("linear_backward");
    *dx = c.wantX ? reported(Kernel::TILES, c.anyX, c.plan.x, c.copies) : r355_linear_plan{};
    *dw = c.wantW ? reported(Kernel::TILES, c.anyW, c.plan.w, c.copies) : r355_linear_plan{};
    if(c.plan.together)
    {
        dx->tile_rows = dx->tile_cols = dw->tile_rows = dw->tile_cols = 64u, dx->first_rows = 0u, dx->together = dw->together = 1u;
        dx->splits = c.plan.both.splitsX, dw->splits = c.plan.both.splitsW;
    }
    return R355_OK;
}

extern "C" int r355_linear_backward(const r355_linear_backward_args* args, void* stream)
{
    constexpr const char* what = "linear_backward";
    if(!args)
        return r355::fail(R355_ERR_BAD_ARG, "linear_backward: null arguments");
    const r355_linear_backward_args& a = *args;
    R355_TRY(checkBackward(a));
    uint64_t             room = usable(a.workspace, a.workspace_bytes);
    const BackwardChoice c    = chooseBackward(a, a.workspace, room);
    const hipStream_t    s    = static_cast<hipStream_t>(stream);
    if(!c.held())
        return tooMany(what);
    r355::beginCall();

    if(c.element || a.dbias)
    {
        GradParams g{};
        g.dy = static_cast<const char*>(a.dy), g.z = static_cast<const char*>(a.z), g.gate = static_cast<const char*>(a.gate);
        g.dz = c.element ? static_cast<char*>(a.dz) : nullptr, g.dgate = static_cast<char*>(a.dgate), g.offsets = a.offsets;
        g.rows = a.rows, g.n = a.n, g.groups = a.groups, g.lddy = a.lddy, g.ldz = a.ldz, g.ldg = a.ldg, g.lddz = a.lddz, g.lddg = a.lddg;
        g.activation = a.activation, g.accumulate = a.accumulate;
        const bool     wide   = a.n % 8u == 0u && evenRows(a.dy, a.lddy, 2) && evenRows(a.z, a.ldz, 2) && evenRows(a.gate, a.ldg, 2) && evenRows(g.dz, a.lddz, 2) && evenRows(a.dgate, a.lddg, 2);
        const uint32_t strips = static_cast<uint32_t>(tilesOf(a.n, wide ? 512u : 64u));
        const uint64_t wanted = gradParts(a, strips);
        const uint64_t fit    = a.dbias ? usable(a.workspace, a.workspace_bytes) / ((uint64_t)a.groups * a.n * 4u) : wanted;
        const uint64_t parts  = wanted < fit ? wanted : fit ? fit : 1u;
        g.parts = static_cast<uint32_t>(parts);
        g.sums  = !a.dbias ? nullptr : parts > 1u ? static_cast<float*>(a.workspace) : a.dbias;
        const dim3 grid(strips, g.parts, a.groups), block(256);
        const bool f16 = a.in_type == R355_F16;
        const auto kernel = wide ? (f16 ? linearGrad<_Float16, 8> : linearGrad<__bf16, 8>) : (f16 ? linearGrad<_Float16, 1> : linearGrad<__bf16, 1>);
        hipLaunchKernelGGL(kernel, grid, block, 0, s, g);
        if(a.dbias && parts > 1u)
            hipLaunchKernelGGL(linearGradSums, dim3(static_cast<uint32_t>(tilesOf(a.n, 64u)), a.groups), block, 0, s, static_cast<const float*>(a.workspace), a.dbias, g.parts, a.n,
                               a.accumulate);
    }
    char* work = static_cast<char*>(a.workspace);
    c.copies.launch(work, s);
    work += c.copies.bytes, room -= c.copies.bytes;
    if(c.plan.together)
    {
        const PlanBoth& both  = c.plan.both;
        const uint64_t  sumsX = sumsBytes(c.px, true, both.splitsX);
        LinearParams    x = both.splitsX > 1u ? sharesOf(c.px, true, both.splitsX, work) : c.px, w = both.splitsW > 1u ? sharesOf(c.pw, false, both.splitsW, work + sumsX) : c.pw;
        const uint32_t  workgroupsX = tilesOfLaunch(x, true, r355::TILE_64), workgroupsW = tilesOfLaunch(w, false, r355::TILE_64);
        (a.in_type == R355_F16 ? r355::linearBothF16 : r355::linearBothBF16)(x, w, workgroupsX, workgroupsW, s);
        if(both.splitsX > 1u)
            launchReduce(a.in_type, c.px, true, both.splitsX, work, s);
        if(both.splitsW > 1u)
            launchReduce(a.in_type, c.pw, false, both.splitsW, work + sumsX, s);
        return r355::checkLaunch(what);
    }
    if(c.wantX)
        launchTiles(a.in_type, c.px, true, false, c.anyX, c.plan.x, work, room, s);
    if(c.wantW)
        launchTiles(a.in_type, c.pw, false, false, c.anyW, c.plan.w, work, room, s);
    return r355::checkLaunch(what);
}
