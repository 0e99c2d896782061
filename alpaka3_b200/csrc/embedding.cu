// Rows of a table by tokens, and the gradient of the table: a sum by keys.
//
//   out_i = scale * W[t_i],      dW_v = add_v + scale * sum of g_i over the positions i with t_i = v
//
// Both move memory and compute next to nothing. The gradient first sorts the tokens (stably: the positions of one token
// stay in their order), then sums the sorted list in chunks of a fixed number of positions, whatever the tokens are: a token
// that fills half of a batch is as well spread over the SMs as many rare ones. A run of one token within a chunk goes
// straight to its row; one that crosses chunks leaves partial sums that a last kernel joins in order. So the bits depend on
// the sizes alone, never on which block comes first. The kernels of a call follow one another by dependent launches: 65536
// tokens 105 us in a stream, 113 without; 512 27, without 31.
#include <algorithm>

#include "layout.cuh"
#include "rows.cuh"

namespace a3b
{
    namespace
    {
        constexpr int kThreads = 128;

        // E elements of T as 32-bit floats: whole 16-byte packs, or one element
        template<typename T, int E>
        struct Lot
        {
            static constexpr int words = E == 1 ? 1 : E * static_cast<int>(sizeof(T)) / 4;

            static __device__ __forceinline__ void load(unsigned* w, T const* p)
            {
                if constexpr(E == 1)
                {
                    if constexpr(sizeof(T) == 4)
                        w[0] = *reinterpret_cast<unsigned const*>(p);
                    else
                        w[0] = *reinterpret_cast<unsigned short const*>(p);
                }
                else
#pragma unroll
                    for(int k = 0; k < words / 4; ++k)
                    {
                        uint4 const v = reinterpret_cast<uint4 const*>(p)[k];
                        w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
                    }
            }
            static __device__ __forceinline__ void unpack(float* v, unsigned const* w)
            {
                if constexpr(std::is_same_v<T, float>)
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        v[e] = __uint_as_float(w[e]);
                else if constexpr(E == 1)
                    v[0] = PackOf<T>::pair(w, 0).x;
                else
#pragma unroll
                    for(int k = 0; k < E / 2; ++k)
                    {
                        float2 const f = PackOf<T>::pair(w, k);
                        v[2 * k] = f.x, v[2 * k + 1] = f.y;
                    }
            }
            // rounded to the nearest value of T and stored
            static __device__ __forceinline__ void store(T* p, float const* v)
            {
                if constexpr(E == 1)
                    *p = fromFloat<T>(v[0]);
                else
#pragma unroll
                    for(int k = 0; k < words / 4; ++k)
                    {
                        constexpr int per = PackOf<T>::E;
                        unsigned w[4];
#pragma unroll
                        for(int j = 0; j < per / 2; ++j)
                            PackOf<T>::setPair(w, j, make_float2(v[per * k + 2 * j], v[per * k + 2 * j + 1]));
                        reinterpret_cast<uint4*>(p)[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
            }
        };

        // elements a lane takes at once where both types come in whole packs
        template<typename T, typename U>
        constexpr int kLot = PackOf<T>::E > PackOf<U>::E ? PackOf<T>::E : PackOf<U>::E;

        // the row of the table that token i names; `vocab` if none
        struct Tokens
        {
            void const* data;
            bool wide; // int64
            int64_t first; // the token of the table's first row
            uint32_t vocab;

            __device__ __forceinline__ uint32_t operator()(uint32_t i) const
            {
                int64_t const t = wide ? static_cast<int64_t const*>(data)[i] : static_cast<int32_t const*>(data)[i];
                uint64_t const v = static_cast<uint64_t>(t) - static_cast<uint64_t>(first);
                return t >= first && v < vocab ? static_cast<uint32_t>(v) : vocab;
            }
        };

        // ---------------------------------------------------------------------------------------------- lookup
        struct LookupArgs
        {
            void const* table;
            int64_t stride;
            Tokens tokens;
            void* out;
            RowStep os;
            uint32_t count, inner, n;
            bool one;
            float scale;
            int shift; // lanes of a team: 1 << shift
        };

        template<typename T, typename U, int E, int P>
        __global__ void __launch_bounds__(kThreads) embeddingKernel(LookupArgs a)
        {
            uint32_t const lanes = 1u << a.shift, lane = threadIdx.x & (lanes - 1u);
            uint64_t const i = static_cast<uint64_t>(blockIdx.x) * (kThreads >> a.shift) + (threadIdx.x >> a.shift);
            if(i >= a.count)
                return;
            auto const row = static_cast<uint32_t>(i);
            uint32_t const token = a.tokens(row), lots = a.n / E, first = blockIdx.y * P * lanes + lane;
            bool const known = token < a.tokens.vocab;
            T const* from = static_cast<T const*>(a.table) + (known ? static_cast<int64_t>(token) * a.stride : 0);
            U* to = static_cast<U*>(a.out) + a.os.at(row, a.inner, a.one);
            unsigned raw[P][Lot<T, E>::words];
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(uint32_t const k = first + p * lanes; known && k < lots)
                    Lot<T, E>::load(raw[p], from + static_cast<size_t>(k) * E);
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(uint32_t const k = first + p * lanes; k < lots)
                {
                    float v[E];
                    Lot<T, E>::unpack(v, raw[p]);
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        v[e] = known ? v[e] * a.scale : 0.f;
                    Lot<U, E>::store(to + static_cast<size_t>(k) * E, v);
                }
        }

        int teamShift(uint32_t lots)
        {
            int s = 0;
            while(s < 7 && (1u << s) < lots)
                ++s;
            return s;
        }

        template<typename T, typename U, int E>
        int launchLookup(cudaStream_t stream, DeviceProps const* props, LookupArgs a)
        {
            uint32_t const lots = a.n / E;
            // four loads under way a lane, unless that leaves SMs with few blocks
            bool const deep = static_cast<uint64_t>(a.count) * lots >= 16ull * kThreads * static_cast<unsigned>(props->smCount);
            uint32_t const depth = deep ? 4 : 1;
            a.shift = teamShift((lots + depth - 1) / depth);
            uint32_t const teams = kThreads >> a.shift, lanes = 1u << a.shift;
            uint32_t const blocks = (a.count + teams - 1) / teams, slices = (lots + depth * lanes - 1) / (depth * lanes);
            if(slices > 65535)
            {
                setError("rows of %u elements are more than one launch holds", a.n);
                return A3B_ERR_TOO_LARGE;
            }
            if(deep)
                embeddingKernel<T, U, E, 4><<<dim3(blocks, slices), kThreads, 0, stream>>>(a);
            else
                embeddingKernel<T, U, E, 1><<<dim3(blocks, slices), kThreads, 0, stream>>>(a);
            A3B_CHECK_LAUNCH("embeddingKernel");
            return A3B_OK;
        }

        // ------------------------------------------------------------------------------------ rows of the gradient
        struct SumArgs
        {
            void const* g;
            RowStep gs;
            uint32_t const* keys; // sorted, `vocab` behind the last known token
            uint32_t const* places;
            float* partial; // [chunk][2][n]: the run that reaches in from the chunk before, and the one that reaches out
            uint32_t* runs; // chunks in which a run begins that reaches out, in any order; in front of them their number
            void const* add; // may be null
            int64_t addStride;
            void* out;
            int64_t stride;
            uint32_t count, inner, n, vocab, chunk, chunks, slices, sumBlocks;
            bool one, fill, flat; // fill: rows without a token are written; flat: they are zeros, and the table is one stretch
            float scale;
            int shift;
        };

        template<typename U, int E>
        __device__ __forceinline__ void loadAdd(SumArgs const& a, uint32_t row, uint32_t k, unsigned* raw)
        {
            Lot<U, E>::load(raw, static_cast<U const*>(a.add) + static_cast<int64_t>(row) * a.addStride + k);
        }

        // add: the words of what is added, if the call adds
        template<typename U, int E>
        __device__ __forceinline__ void writeRow(SumArgs const& a, uint32_t row, uint32_t k, float* v, unsigned const* add)
        {
#pragma unroll
            for(int e = 0; e < E; ++e)
                v[e] *= a.scale;
            if(add)
            {
                float more[E];
                Lot<U, E>::unpack(more, add);
#pragma unroll
                for(int e = 0; e < E; ++e)
                    v[e] += more[e];
            }
            Lot<U, E>::store(static_cast<U*>(a.out) + static_cast<int64_t>(row) * a.stride + k, v);
        }

        constexpr uint32_t kFillRows = 16; // rows that a block looks for
        constexpr uint32_t kFillLots = 1024; // lots of a block that looks for none

        // Lots of rows without a token: what is added, or zero. place(u, &row, &k) gives the thread's u-th of four; what is
        // added is loaded for all of them first.
        template<typename U, int E, bool Add, typename F>
        __device__ __forceinline__ void fillLots(SumArgs const& a, F&& place)
        {
            uint32_t row[4], k[4];
            bool in[4];
            unsigned add[Add ? 4 : 1][Lot<U, E>::words];
#pragma unroll
            for(int u = 0; u < 4; ++u)
            {
                in[u] = place(u, row + u, k + u);
                if(Add && in[u])
                    loadAdd<U, E>(a, row[u], k[u] * E, add[Add ? u : 0]);
            }
#pragma unroll
            for(int u = 0; u < 4; ++u)
                if(in[u])
                {
                    float v[E];
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        v[e] = 0.f;
                    writeRow<U, E>(a, row[u], k[u] * E, v, Add ? add[Add ? u : 0] : nullptr);
                }
        }

        // ------------------------------------------------------------------------------------- sorting the tokens
        // Up to kRankMax tokens: the place of each is the number of those that come before it, by comparing all pairs. A
        // block ranks 32 tokens, each of its warps against an eighth of the list. Quadratic, but one short launch.
        constexpr uint32_t kRankMax = 4096;

        // Where tokens are few beside the table's rows, blocks behind those that rank write every row as if its token did not
        // occur; the sums then write over those that do. So the table is filled while the tokens are ranked, and no row needs
        // a search (512 tokens into 32000 x 1024 fp32 27.3 us, 29.2 with the rows searched behind the sort).
        template<typename U, int E, bool Add>
        __global__ void __launch_bounds__(256) rankKernel(Tokens tokens, uint32_t count, uint32_t* keys, uint32_t* places, SumArgs a)
        {
            uint32_t const ranking = (count + 31) / 32;
            signalNext();
            if(blockIdx.x >= ranking)
            {
                uint32_t const lots = a.n / E;
                if(a.flat)
                {
                    // one stretch of zeros, rows of any length
                    constexpr uint32_t per = PackOf<U>::E;
                    uint64_t const all = static_cast<uint64_t>(a.vocab) * a.n, packs = all / per;
                    U* out = static_cast<U*>(a.out);
#pragma unroll
                    for(uint32_t u = 0; u < kFillLots; u += 256)
                    {
                        uint64_t const i = static_cast<uint64_t>(blockIdx.x - ranking) * kFillLots + u + threadIdx.x;
                        if(i < packs)
                            reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
                        else if(i == packs)
                            for(uint64_t k = packs * per; k < all; ++k)
                                out[k] = fromFloat<U>(0.f);
                    }
                    return;
                }
                static_assert(kFillLots == 4 * 256);
                fillLots<U, E, Add>(a, [&](int u, uint32_t* row, uint32_t* k)
                {
                    uint32_t const i = (blockIdx.x - ranking) * kFillLots + u * 256 + threadIdx.x;
                    *row = i / lots;
                    *k = i - *row * lots;
                    return *row < a.vocab;
                });
                return;
            }
            if(blockIdx.x == 0 && threadIdx.x == 0)
                *a.runs = 0;
            extern __shared__ __align__(16) uint32_t all[];
            __shared__ uint32_t part[8][32];
            uint32_t const warp = threadIdx.x / 32, lane = threadIdx.x % 32, base = blockIdx.x * 32, i = base + lane;
            uint32_t const span = ((count + 7) / 8 + 31) / 32 * 32, low = warp * span;
            uint32_t const high = min(low + span, (count + 31) / 32 * 32);
#pragma unroll 8
            for(uint32_t j = low + lane; j < high; j += 32) // behind the last: a key above all others
                all[j] = j < count ? tokens(j) : 0xffffffffu;
            uint32_t const key = i < count ? tokens(i) : 0xfffffffeu;
            __syncwarp();
            uint32_t before = 0;
            auto run = [&](uint32_t from, uint32_t to, uint32_t limit) // keys below `limit`
            {
#pragma unroll 4
                for(uint32_t j = from; j < to; j += 4)
                {
                    uint4 const k = *reinterpret_cast<uint4 const*>(all + j);
                    before += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
                }
            };
            uint32_t const from = min(max(low, base), high), to = min(max(low, base + 32), high);
            run(low, from, key + 1); // in front of the block's own tokens an equal key comes first
            for(uint32_t j = from; j < to; ++j)
                before += all[j] < key || (all[j] == key && j < i);
            run(to, high, key);
            part[warp][lane] = before;
            __syncthreads();
            if(warp == 0 && i < count)
            {
#pragma unroll
                for(int w = 1; w < 8; ++w)
                    before += part[w][lane];
                keys[before] = key;
                places[before] = i;
            }
        }

        // Up to kClusterMax tokens: radix sort in one launch, by a cluster of eight blocks that hold the list in their shared
        // memory; each has an eighth, each of its warps a contiguous part of that, so equal digits keep their order. A digit
        // takes a count by every warp, one exchange of the blocks' counts and one of the tokens themselves.
        constexpr uint32_t kClusterMax = 16384, kSortBlocks = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
        constexpr int kBins = 512;

        struct ClusterSort
        {
            uint2 list[2][kClusterMax / kSortBlocks]; // key and place
            uint32_t at[kSortWarps][kBins]; // counts of a warp, then where its next token of a digit goes
            uint32_t total[kBins]; // of the block, read by the others
            uint32_t sums[kBins / 32];
        };

        __global__ void __cluster_dims__(kSortBlocks, 1, 1) __launch_bounds__(kSortThreads)
            clusterSortKernel(Tokens tokens, uint32_t count, int log2Each, int digits, int bits, uint32_t* keys, uint32_t* places,
                              uint32_t* runs)
        {
            extern __shared__ __align__(16) unsigned char memory[];
            auto& sh = *reinterpret_cast<ClusterSort*>(memory);
            uint32_t const t = threadIdx.x, warp = t / 32, lane = t % 32, rank = clusterRank(), bins = 1u << bits;
            uint32_t const own = kSortThreads << log2Each, span = own / kSortWarps; // tokens of a block and of a warp
            signalNext();
            if(rank == 0 && t == 0)
                *runs = 0;
            // A warp reads its own part in its own order, here and below.
#pragma unroll 8
            for(uint32_t i = lane; i < span; i += 32)
            {
                uint32_t const place = rank * own + warp * span + i;
                if(place < count)
                    sh.list[0][warp * span + i] = make_uint2(tokens(place), place);
            }
            uint32_t const mine = min(span, count - min(count, rank * own + warp * span)); // live tokens of this warp
            for(int d = 0; d < digits; ++d)
            {
                uint2 const* from = sh.list[d & 1];
                for(uint32_t b = lane; b < bins; b += 32)
                    sh.at[warp][b] = 0;
                __syncwarp();
#pragma unroll 4
                for(uint32_t i = lane; i < mine; i += 32)
                    atomicAdd(&sh.at[warp][(from[warp * span + i].x >> (d * bits)) & (bins - 1u)], 1u);
                __syncthreads();
                // of a digit: how many of it the warps in front have, and the block
                uint32_t all = 0;
                if(t < bins)
                {
#pragma unroll 8
                    for(uint32_t w = 0; w < kSortWarps; ++w)
                    {
                        uint32_t const c = sh.at[w][t];
                        sh.at[w][t] = all;
                        all += c;
                    }
                    sh.total[t] = all;
                }
                clusterArrive();
                clusterWait();
                // how many of it the blocks in front have, and all blocks; then how many smaller digits there are
                uint32_t front = 0, v = 0;
                if(t < bins)
#pragma unroll
                    for(uint32_t b = 0; b < kSortBlocks; ++b)
                    {
                        uint32_t const c = *inBlock(&sh.total[t], b);
                        front += b < rank ? c : 0u;
                        v += c;
                    }
                all = v;
#pragma unroll
                for(int step = 1; step < 32; step *= 2)
                {
                    uint32_t const up = __shfl_up_sync(kFullMask, v, step);
                    if(lane >= static_cast<uint32_t>(step))
                        v += up;
                }
                if(lane == 31 && warp < kBins / 32)
                    sh.sums[warp] = v;
                __syncthreads();
                if(t < bins)
                {
                    uint32_t base = v - all + front;
                    for(uint32_t w = 0; w < warp; ++w)
                        base += sh.sums[w];
#pragma unroll 8
                    for(uint32_t w = 0; w < kSortWarps; ++w)
                        sh.at[w][t] += base;
                }
                __syncthreads();
                for(uint32_t first = 0; first < mine; first += 32)
                {
                    bool const live = first + lane < mine;
                    unsigned const here = __ballot_sync(kFullMask, live);
                    if(live)
                    {
                        uint2 const e = from[warp * span + first + lane];
                        uint32_t const digit = (e.x >> (d * bits)) & (bins - 1u);
                        unsigned const same = __match_any_sync(here, digit);
                        uint32_t const before = __popc(same & ((1u << lane) - 1u)), to = sh.at[warp][digit] + before;
                        __syncwarp(here);
                        if(before == 0)
                            sh.at[warp][digit] += __popc(same);
                        if(d + 1 < digits)
                            *inBlock(&sh.list[(d + 1) & 1][to & (own - 1u)], to / own) = e;
                        else
                            keys[to] = e.x, places[to] = e.y;
                    }
                    __syncwarp();
                }
                // the other blocks' tokens have come, and nobody reads `total` any more
                clusterArrive();
                clusterWait();
            }
        }

        // More tokens: radix sort, digits of at most nine bits from the lowest, three kernels a digit. A block counts and
        // later places one contiguous tile, its warps contiguous parts of it, so equal digits keep their order.
        constexpr int kTileWarps = 8;

        struct RadixArgs
        {
            Tokens tokens; // first digit
            uint32_t const* keysIn; // later digits
            uint32_t const* placesIn;
            uint32_t* keys;
            uint32_t* places;
            uint32_t* counts; // [bin][tile]
            uint32_t* totals; // [bin]
            uint32_t* runs; // set to zero for the sums
            uint32_t count, tile, tiles; // tile: a multiple of 32 * kTileWarps
            int shift, bits;
            bool initial;

            __device__ __forceinline__ uint32_t key(uint32_t i) const
            {
                return initial ? tokens(i) : keysIn[i];
            }
            __device__ __forceinline__ uint32_t digit(uint32_t k) const
            {
                return (k >> shift) & ((1u << bits) - 1u);
            }
        };

        __global__ void __launch_bounds__(256) radixCountKernel(RadixArgs a)
        {
            __shared__ uint32_t bin[kBins];
            for(uint32_t b = threadIdx.x; b < kBins; b += 256)
                bin[b] = 0;
            signalNext();
            if(!a.initial)
                waitForPrevious();
            else if(blockIdx.x == 0 && threadIdx.x == 0)
                *a.runs = 0;
            __syncthreads();
            uint32_t const low = blockIdx.x * a.tile, high = min(low + a.tile, a.count);
            for(uint32_t i = low + threadIdx.x; i < high; i += 256)
                atomicAdd(bin + a.digit(a.key(i)), 1u);
            __syncthreads();
            for(uint32_t b = threadIdx.x; b < (1u << a.bits); b += 256)
                a.counts[static_cast<size_t>(b) * a.tiles + blockIdx.x] = bin[b];
        }

        // counts of a digit in the tiles -> how many of it the tiles in front have; a warp a digit
        __global__ void __launch_bounds__(128) radixScanKernel(uint32_t* counts, uint32_t* totals, uint32_t tiles, uint32_t bins)
        {
            uint32_t const b = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
            signalNext();
            waitForPrevious();
            if(b >= bins)
                return;
            uint32_t* row = counts + static_cast<size_t>(b) * tiles;
            uint32_t sum = 0;
            for(uint32_t first = 0; first < tiles; first += 32)
            {
                uint32_t const t = first + lane, own = t < tiles ? row[t] : 0u;
                uint32_t v = own;
#pragma unroll
                for(int d = 1; d < 32; d *= 2)
                {
                    uint32_t const up = __shfl_up_sync(kFullMask, v, d);
                    if(lane >= static_cast<uint32_t>(d))
                        v += up;
                }
                if(t < tiles)
                    row[t] = sum + v - own;
                sum += __shfl_sync(kFullMask, v, 31);
            }
            if(lane == 0)
                totals[b] = sum;
        }

        __global__ void __launch_bounds__(32 * kTileWarps) radixPlaceKernel(RadixArgs a)
        {
            __shared__ uint32_t at[kTileWarps][kBins]; // where the warp's next key of a digit goes
            __shared__ uint32_t warpSum[kTileWarps];
            uint32_t const t = threadIdx.x, warp = t / 32, lane = t % 32, bins = 1u << a.bits;
            for(uint32_t k = t; k < kTileWarps * kBins; k += 256)
                at[k / kBins][k % kBins] = 0;
            signalNext();
            waitForPrevious();
            __syncthreads();
            uint32_t const span = a.tile / kTileWarps, low = min(blockIdx.x * a.tile + warp * span, a.count),
                           high = min(low + span, a.count);
            for(uint32_t i = low + lane; i < high; i += 32)
                atomicAdd(&at[warp][a.digit(a.key(i))], 1u);
            // all keys of smaller digits: an exclusive sum of the totals, two digits a thread
            uint32_t const b0 = 2 * t, t0 = b0 < bins ? a.totals[b0] : 0u, t1 = b0 + 1 < bins ? a.totals[b0 + 1] : 0u;
            uint32_t v = t0 + t1;
#pragma unroll
            for(int d = 1; d < 32; d *= 2)
            {
                uint32_t const up = __shfl_up_sync(kFullMask, v, d);
                if(lane >= static_cast<uint32_t>(d))
                    v += up;
            }
            if(lane == 31)
                warpSum[warp] = v;
            __syncthreads();
            uint32_t start = v - t0 - t1;
            for(uint32_t w = 0; w < warp; ++w)
                start += warpSum[w];
#pragma unroll
            for(int e = 0; e < 2; ++e)
            {
                uint32_t const b = b0 + e;
                if(b < bins)
                {
                    uint32_t next = start + (e ? t0 : 0u) + a.counts[static_cast<size_t>(b) * a.tiles + blockIdx.x];
                    for(int w = 0; w < kTileWarps; ++w)
                    {
                        uint32_t const c = at[w][b];
                        at[w][b] = next;
                        next += c;
                    }
                }
            }
            __syncthreads();
            for(uint32_t first = low; first < high; first += 32)
            {
                uint32_t const i = first + lane;
                bool const live = i < high;
                unsigned const here = __ballot_sync(kFullMask, live);
                if(live)
                {
                    uint32_t const key = a.key(i), d = a.digit(key);
                    unsigned const same = __match_any_sync(here, d);
                    uint32_t const rank = __popc(same & ((1u << lane) - 1u));
                    uint32_t const to = at[warp][d] + rank;
                    __syncwarp(here);
                    if(rank == 0)
                        at[warp][d] += __popc(same);
                    a.keys[to] = key;
                    a.places[to] = a.initial ? i : a.placesIn[i];
                }
                __syncwarp();
            }
        }

        // -------------------------------------------------------------------------------------- sums by token
        // The first blocks sum: a team has a chunk of the sorted list and E columns a lane, and loads kAhead rows before it
        // adds them. The others write the rows of tokens that do not occur.
        template<typename T, typename U, int E, bool Add>
        __global__ void __launch_bounds__(kThreads) embeddingSumKernel(SumArgs a)
        {
            constexpr int kAhead = 4;
            // The kernel that joins; behind many tokens its waiting blocks take the sums' place (1 us of 39 at 16384 x 1024).
            if(a.chunks > 1 && a.count <= kRankMax)
                signalNext();
            if(a.count > 0)
                waitForPrevious(); // the sort
            if(blockIdx.x >= a.sumBlocks)
            {
                __shared__ bool present[kFillRows];
                // a block has kFillRows rows and four lots a thread of each
                uint32_t const parts = (a.n / E + 4 * kThreads - 1) / (4 * kThreads), block = blockIdx.x - a.sumBlocks;
                uint32_t const base = block / parts * kFillRows, first = block % parts * (4 * kThreads) + threadIdx.x;
                if(threadIdx.x < kFillRows)
                    present[threadIdx.x] = false;
                // Where the keys of these rows begin and end in the list: both searched by all threads together, 128 parts a
                // step (a search by halves took as long as the writing).
                uint32_t from[2] = {0, 0}, size[2] = {a.count, a.count};
                while(size[0] + size[1] > 0)
#pragma unroll
                    for(int end = 0; end < 2; ++end)
                    {
                        uint32_t const part = (size[end] + kThreads - 1) / kThreads;
                        uint64_t const at = static_cast<uint64_t>(threadIdx.x + 1) * part; // the last of a part is looked at
                        bool const below = size[end] > 0 && at <= size[end] && a.keys[from[end] + at - 1] < base + end * kFillRows;
                        uint32_t const skip = __syncthreads_count(below) * part;
                        size[end] = size[end] > 0 ? min(part - 1, size[end] - skip) : 0;
                        from[end] += skip;
                    }
                uint32_t const lead = from[0], found = from[1] - from[0];
                if(found <= kThreads)
                {
                    if(threadIdx.x < found)
                        present[a.keys[lead + threadIdx.x] - base] = true;
                }
                else if(threadIdx.x < kFillRows)
                {
                    uint32_t const row = base + threadIdx.x;
                    uint32_t low = lead, high = lead + found; // the first key that is not below row
                    while(low < high)
                    {
                        uint32_t const mid = low + (high - low) / 2;
                        if(a.keys[mid] < row)
                            low = mid + 1;
                        else
                            high = mid;
                    }
                    present[threadIdx.x] = low < lead + found && a.keys[low] == row;
                }
                __syncthreads();
                for(uint32_t r = 0; r < min(kFillRows, a.vocab - base); ++r)
                    if(!present[r])
                        fillLots<U, E, Add>(a, [&](int u, uint32_t* row, uint32_t* k)
                        {
                            *row = base + r;
                            *k = first + u * kThreads;
                            return *k < a.n / E;
                        });
                return;
            }
            uint32_t const lanes = 1u << a.shift, lane = threadIdx.x & (lanes - 1u);
            uint32_t const slice = blockIdx.x % a.slices;
            uint64_t const c64 = static_cast<uint64_t>(blockIdx.x / a.slices) * (kThreads >> a.shift) + (threadIdx.x >> a.shift);
            uint32_t const col = (slice * lanes + lane) * E;
            if(c64 >= a.chunks || col >= a.n)
                return;
            auto const c = static_cast<uint32_t>(c64);
            uint32_t const low = c * a.chunk, high = min(low + a.chunk, a.count);
            bool inward = low > 0 && a.keys[low - 1] == a.keys[low]; // the first run began in an earlier chunk
            float sum[E];
#pragma unroll
            for(int e = 0; e < E; ++e)
                sum[e] = 0.f;
            auto flush = [&](uint32_t current, bool outward, unsigned const* add)
            {
                if(inward || outward)
                {
                    if(!inward && col == 0)
                        a.runs[1 + atomicAdd(a.runs, 1u)] = c;
                    float* p = a.partial + (static_cast<size_t>(c) * 2 + (inward ? 0 : 1)) * a.n + col;
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        p[e] = sum[e];
                }
                else
                    writeRow<U, E>(a, current, col, sum, add);
            };
            // the next rows' keys and places come while these rows do
            uint32_t next[kAhead], place[kAhead];
            auto look = [&](uint32_t p)
            {
#pragma unroll
                for(int u = 0; u < kAhead; ++u)
                {
                    next[u] = p + u < high ? a.keys[p + u] : a.vocab;
                    place[u] = p + u < high ? a.places[p + u] : 0u;
                }
            };
            look(low);
            for(uint32_t p = low; p < high; p += kAhead)
            {
                uint32_t key[kAhead + 1];
                unsigned raw[kAhead][Lot<T, E>::words], add[Add ? kAhead : 1][Lot<U, E>::words];
#pragma unroll
                for(int u = 0; u < kAhead; ++u)
                {
                    key[u] = next[u];
                    if(key[u] < a.vocab)
                        Lot<T, E>::load(raw[u], static_cast<T const*>(a.g) + a.gs.at(place[u], a.inner, a.one) + col);
                }
                look(p + kAhead);
                key[kAhead] = next[0]; // `vocab` behind the chunk
                // what is added comes with a run's last row (a run that goes on into the next chunk does not need it)
                if(Add)
#pragma unroll
                    for(int u = 0; u < kAhead; ++u)
                        if(key[u] < a.vocab && key[u] != key[u + 1])
                            loadAdd<U, E>(a, key[u], col, add[u]);
#pragma unroll
                for(int u = 0; u < kAhead; ++u)
                {
                    if(key[u] >= a.vocab)
                        break; // only tokens without a row come behind
                    float v[E];
                    Lot<T, E>::unpack(v, raw[u]);
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        sum[e] += v[e];
                    if(key[u] != key[u + 1])
                    {
                        flush(key[u], p + u + 1 == high && high < a.count && a.keys[high] == key[u], Add ? add[Add ? u : 0] : nullptr);
                        inward = false;
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            sum[e] = 0.f;
                    }
                }
            }
        }

        // Joins the partial sums of the runs that cross chunks. A block takes a run and 128 columns at a time: its eight warps
        // have equal parts of the run's chunks, a lane four columns; the parts are added in their order.
        template<typename U, bool Packs>
        __global__ void __launch_bounds__(256) embeddingJoinKernel(SumArgs a)
        {
            __shared__ float4 part[8][32];
            waitForPrevious();
            uint32_t const warp = threadIdx.x / 32, lane = threadIdx.x % 32, slices = (a.n + 127) / 128, runs = a.runs[0];
            uint32_t const runStep = gridDim.x / slices, sliceStep = gridDim.x % slices; // items in steps of the grid
            for(uint32_t run = blockIdx.x / slices, slice = blockIdx.x % slices; run < runs; run += runStep, slice += sliceStep)
            {
                if(slice >= slices)
                {
                    slice -= slices;
                    if(++run >= runs)
                        break;
                }
                uint32_t const c = a.runs[1 + run], col = (slice * 32 + lane) * 4;
                uint32_t const key = a.keys[(c + 1) * a.chunk]; // it reaches out: never the last chunk
                // the chunks that begin with the run's token, 256 looked at together
                uint32_t end = c;
                for(bool more = true; more;)
                {
                    uint64_t const at = (static_cast<uint64_t>(end) + 1 + threadIdx.x) * a.chunk;
                    int const same = __syncthreads_count(at < a.count && a.keys[at] == key);
                    end += same;
                    more = same == 256;
                }
                uint32_t const parts = end - c + 1, each = (parts + 7) / 8;
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for(uint32_t q = warp * each; q < min((warp + 1) * each, parts); ++q)
                {
                    // the run reaches out of its first chunk and into the others
                    float const* p = a.partial + (static_cast<size_t>(c + q) * 2 + (q == 0 ? 1 : 0)) * a.n + col;
                    if constexpr(Packs)
                    {
                        if(col < a.n)
                        {
                            float4 const v = __ldcg(reinterpret_cast<float4 const*>(p));
                            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
                        }
                    }
                    else
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                            if(col + e < a.n)
                                s[e] += __ldcg(p + e);
                }
                part[warp][lane] = make_float4(s[0], s[1], s[2], s[3]);
                __syncthreads();
                if(warp == 0)
                {
#pragma unroll
                    for(int w = 1; w < 8; ++w)
                    {
                        float4 const v = part[w][lane];
                        s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
                    }
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        if(col + e < a.n)
                        {
                            unsigned add[1];
                            if(a.add)
                                loadAdd<U, 1>(a, key, col + e, add);
                            writeRow<U, 1>(a, key, col + e, s + e, a.add ? add : nullptr);
                        }
                }
                __syncthreads(); // `part` has been read
            }
        }

        // ------------------------------------------------------------------------------------------ workspace
        struct Plan
        {
            bool radix; // in several launches
            uint32_t chunk, chunks, tile, tiles;
            int digits, bits; // radix digits and bits of each
            size_t keys, places, keys2, places2, counts, totals, runs, partial, bytes; // offsets, and the whole
        };

        // From sizes alone (not from alignment), so that the workspace and the order of the sums are.
        Plan planFor(DeviceProps const* props, uint64_t count, uint64_t n, uint64_t vocab)
        {
            Plan p{};
            p.radix = count > kClusterMax;
            // About eight blocks of 128 threads an SM, each thread with eight columns; chunks of 16 to 256 positions (shorter ones
            // leave more runs to join: 4096 tokens of 257 in chunks of 8 take 21 us, of 16 18), but of 8 for few tokens, whose
            // chunks' latency counts (512 tokens 2 us less).
            uint64_t const perRow = std::max<uint64_t>(1, n / 8), wanted = 8ull * static_cast<unsigned>(props->smCount) * kThreads;
            uint64_t const chunk = count * perRow / wanted;
            p.chunk = static_cast<uint32_t>(std::min<uint64_t>(256, std::max<uint64_t>(count < 2048 ? 8 : 16, chunk / 4 * 4)));
            p.chunks = static_cast<uint32_t>((count + p.chunk - 1) / p.chunk);
            int bits = 1;
            while(bits < 32 && (vocab >> bits) != 0) // keys are 0 .. vocab
                ++bits;
            p.digits = (bits + 8) / 9;
            p.bits = (bits + p.digits - 1) / p.digits;
            uint32_t const whole = 32 * kTileWarps;
            uint64_t const most = 2ull * static_cast<unsigned>(props->smCount);
            uint64_t tile = ((count + most - 1) / most + whole - 1) / whole * whole;
            p.tile = static_cast<uint32_t>(std::max<uint64_t>(tile, whole));
            p.tiles = static_cast<uint32_t>((count + p.tile - 1) / p.tile);
            size_t at = 0;
            auto take = [&](size_t bytes)
            {
                size_t const here = at;
                at += (bytes + 255) / 256 * 256;
                return here;
            };
            p.keys = take(count * 4);
            p.places = take(count * 4);
            if(p.radix)
            {
                p.keys2 = take(count * 4);
                p.places2 = take(count * 4);
                p.counts = take(static_cast<size_t>(kBins) * p.tiles * 4);
                p.totals = take(kBins * 4);
            }
            p.runs = take((static_cast<size_t>(p.chunks) + 1) * 4);
            p.partial = take(static_cast<size_t>(p.chunks) * 2 * n * 4);
            p.bytes = std::max<size_t>(at, 256);
            return p;
        }

        int sortTokens(cudaStream_t stream, DeviceProps const* props, Plan const& p, Tokens const& tokens, uint32_t count, char* ws, uint32_t** keys,
                       uint32_t** places)
        {
            auto at = [&](size_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
            *keys = at(p.keys);
            *places = at(p.places);
            if(count <= kRankMax)
                return A3B_OK; // with the sums
            if(!p.radix)
            {
                static std::atomic<bool> ready[kMaxDevices];
                if(!ready[props->ordinal].load(std::memory_order_relaxed))
                {
                    A3B_CUDA(cudaFuncSetAttribute(clusterSortKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(sizeof(ClusterSort))));
                    ready[props->ordinal].store(true, std::memory_order_relaxed);
                }
                int log2Each = 0; // tokens of a thread
                while((kSortBlocks * kSortThreads << log2Each) < count)
                    ++log2Each;
                clusterSortKernel<<<kSortBlocks, kSortThreads, sizeof(ClusterSort), stream>>>(tokens, count, log2Each, p.digits, p.bits,
                                                                                            *keys, *places, at(p.runs));
                A3B_CHECK_LAUNCH("clusterSortKernel");
                return A3B_OK;
            }
            uint32_t *otherKeys = at(p.keys2), *otherPlaces = at(p.places2);
            for(int d = 0; d < p.digits; ++d)
            {
                RadixArgs a{tokens, otherKeys, otherPlaces, *keys, *places, at(p.counts), at(p.totals), at(p.runs), count, p.tile, p.tiles,
                            d * p.bits, p.bits, d == 0};
                if(d > 0) // from what the digit before wrote
                {
                    a.keysIn = *keys, a.placesIn = *places;
                    a.keys = otherKeys, a.places = otherPlaces;
                    std::swap(*keys, otherKeys);
                    std::swap(*places, otherPlaces);
                }
                int rc = A3B_OK;
                if(d > 0)
                    rc = launchNext(stream, radixCountKernel, p.tiles, 256, 0, a);
                else
                {
                    radixCountKernel<<<p.tiles, 256, 0, stream>>>(a);
                    A3B_CHECK_LAUNCH("radixCountKernel");
                }
                if(rc == A3B_OK)
                    rc = launchNext(stream, radixScanKernel, ((1u << p.bits) + 3) / 4, 128, 0, a.counts, a.totals, p.tiles, 1u << p.bits);
                if(rc == A3B_OK)
                    rc = launchNext(stream, radixPlaceKernel, p.tiles, 32 * kTileWarps, 0, a);
                if(rc != A3B_OK)
                    return rc;
            }
            return A3B_OK;
        }

        template<typename T, typename U, int E>
        int launchGradient(cudaStream_t stream, DeviceProps const* props, SumArgs a, Plan const& p, Tokens const& tokens, char* ws)
        {
            uint32_t const lots = a.n / E;
            a.shift = teamShift(lots);
            uint32_t const lanes = 1u << a.shift, teams = kThreads >> a.shift;
            a.slices = (lots + lanes - 1) / lanes;
            uint64_t const sums = static_cast<uint64_t>((a.chunks + teams - 1) / teams) * a.slices;
            uint64_t fills = a.fill ? static_cast<uint64_t>((a.vocab + kFillRows - 1) / kFillRows) * ((lots + 4 * kThreads - 1) / (4 * kThreads)) : 0;
            bool const ranked = a.count > 0 && a.count <= kRankMax;
            // at most one row in sixteen is written twice
            uint64_t const all = a.flat ? static_cast<uint64_t>(a.vocab) * a.n / PackOf<U>::E + 1 : static_cast<uint64_t>(a.vocab) * lots;
            bool const early = ranked && a.fill && a.count <= a.vocab / 16 && all <= static_cast<uint64_t>(UINT32_MAX) - kFillLots;
            if(early) // by the kernel that ranks
                fills = 0;
            if(sums + fills > static_cast<uint64_t>(INT_MAX))
            {
                setError("%u tokens of %u elements are more than one launch holds", a.count, a.n);
                return A3B_ERR_TOO_LARGE;
            }
            uint32_t *keys = nullptr, *places = nullptr;
            if(a.count > 0)
            {
                int const rs = sortTokens(stream, props, p, tokens, a.count, ws, &keys, &places);
                if(rs != A3B_OK)
                    return rs;
                a.keys = keys, a.places = places;
            }
            if(ranked)
            {
                uint32_t const ranking = (a.count + 31) / 32;
                auto kernel = early && a.add ? rankKernel<U, E, true> : rankKernel<U, E, false>;
                uint32_t const filling = early ? static_cast<uint32_t>((all + kFillLots - 1) / kFillLots) : 0;
                kernel<<<ranking + filling, 256, ranking * 32 * 4, stream>>>(tokens, a.count, keys, places, a);
                A3B_CHECK_LAUNCH("rankKernel");
            }
            a.sumBlocks = static_cast<uint32_t>(sums);
            if(sums + fills == 0)
                return A3B_OK;
            auto const grid = static_cast<unsigned>(sums + fills);
            auto kernel = a.add ? embeddingSumKernel<T, U, E, true> : embeddingSumKernel<T, U, E, false>;
            if(a.count == 0)
            {
                kernel<<<grid, kThreads, 0, stream>>>(a);
                A3B_CHECK_LAUNCH("embeddingSumKernel");
                return A3B_OK;
            }
            int const rc = launchNext(stream, kernel, grid, kThreads, 0, a);
            if(rc == A3B_OK && a.chunks > 1)
            {
                // as many blocks as SMs hold, or runs and columns there can be
                uint64_t const items = static_cast<uint64_t>(a.chunks - 1) * ((a.n + 127) / 128);
                auto const blocks = static_cast<unsigned>(std::min<uint64_t>(8ull * static_cast<unsigned>(props->smCount), items));
                return launchNext(stream, a.n % 4 == 0 ? embeddingJoinKernel<U, true> : embeddingJoinKernel<U, false>, blocks, 256, 0, a);
            }
            return rc;
        }

        // Calls f(T{}, U{}) for the two types; f32, f16 and bf16 with themselves, and f32 with the 16-bit ones.
        template<typename F>
        int withTypes(int from, int to, F&& f)
        {
            if(from == A3B_F32)
                return to == A3B_F32 ? f(float{}, float{}) : to == A3B_F16 ? f(float{}, __half{}) : f(float{}, __nv_bfloat16{});
            if(from == A3B_F16)
                return to == A3B_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
            return to == A3B_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
        }

        int checkTypes(int rowsType, int tableType, int indexType, uint64_t vocab, uint64_t outer, uint64_t inner, uint64_t n,
                       double scale)
        {
            A3B_REQUIRE(rowTypeSize(rowsType) != 0 && rowTypeSize(tableType) != 0, "rows and table must be f32, f16 or bf16");
            A3B_REQUIRE(rowsType == tableType || rowsType == A3B_F32 || tableType == A3B_F32,
                        "rows and table have one type, or one of them is f32");
            A3B_REQUIRE(indexType == A3B_I32 || indexType == A3B_I64, "tokens must be i32 or i64");
            A3B_REQUIRE(n > 0, "a row needs at least one element");
            float const f = static_cast<float>(scale);
            A3B_REQUIRE(f - f == 0.f, "scale must be finite in fp32");
            A3B_REQUIRE(outer == 0 || inner <= UINT64_MAX / outer, "rows overflow");
            if(n > static_cast<uint64_t>(INT_MAX) - 64 || outer * inner > static_cast<uint64_t>(INT_MAX) - 64
               || vocab > static_cast<uint64_t>(INT_MAX) - 64)
            {
                setError("at most 2^31 - 65 tokens, elements a row and rows of the table");
                return A3B_ERR_TOO_LARGE;
            }
            return A3B_OK;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_embedding(a3b_stream_t stream, a3b_embedding_args const* args)
    {
        A3B_REQUIRE(args, "null arguments");
        uint64_t const outer = args->outer, inner = args->inner, n = args->n, vocab = args->vocab;
        int64_t const first = args->first, table_stride = args->table_stride;
        void const *table = args->table, *tokens = args->tokens;
        a3b_rows const& out = args->out;
        double const scale = args->scale;
        int const table_dtype = args->table_dtype, index_dtype = args->index_dtype, out_dtype = args->out_dtype;
        int const rc = checkTypes(out_dtype, table_dtype, index_dtype, vocab, outer, inner, n, scale);
        if(rc != A3B_OK)
            return rc;
        uint64_t const count = outer * inner;
        if(count == 0)
            return A3B_OK;
        A3B_REQUIRE(tokens && out.data && (table || vocab == 0), "null tokens, table or output");
        int const ts = rowTypeSize(table_dtype), os = rowTypeSize(out_dtype), is = index_dtype == A3B_I64 ? 8 : 4;
        A3B_REQUIRE(alignedTo(ts, {table}) && alignedTo(os, {out.data}) && alignedTo(is, {tokens}), "an array is not aligned to its type");
        Stretch const st = Stretch::rows(vocab ? table : nullptr, 1, vocab, 0, table_stride, n, ts);
        Stretch const so = Stretch::rows(out, outer, inner, n, os);
        Stretch const si = Stretch::dense(tokens, static_cast<Wide>(count) * is);
        A3B_REQUIRE(so.separate(), "rows of the output overlap");
        A3B_REQUIRE(so.apart(st) && so.apart(si), "the output overlaps the table or the tokens");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        LookupArgs a{table, table_stride, {tokens, index_dtype == A3B_I64, first, static_cast<uint32_t>(vocab)}, out.data,
                     {out.outer_stride, out.inner_stride}, static_cast<uint32_t>(count), static_cast<uint32_t>(inner),
                     static_cast<uint32_t>(n), outer == 1, static_cast<float>(scale), 0};
        auto s = static_cast<cudaStream_t>(stream);
        return withTypes(table_dtype, out_dtype, [&](auto t, auto u)
        {
            using T = decltype(t);
            using U = decltype(u);
            constexpr int E = kLot<T, U>;
            bool const packed = n % E == 0 && rowsAligned(table, 1, vocab, 0, table_stride, ts, 16)
                                && rowsAligned(out.data, outer, inner, out.outer_stride, out.inner_stride, os, 16);
            return packed ? launchLookup<T, U, E>(s, props, a) : launchLookup<T, U, 1>(s, props, a);
        });
    }

    size_t a3b_embedding_backward_workspace(uint64_t count, uint64_t n, uint64_t vocab)
    {
        DeviceProps const* props = nullptr;
        if(currentDevice(&props) != A3B_OK)
            return 0;
        uint64_t const most = static_cast<uint64_t>(INT_MAX);
        return planFor(props, std::min(count, most), std::min(n, most), std::min(vocab, most)).bytes;
    }

    int a3b_embedding_backward(a3b_stream_t stream, a3b_embedding_backward_args const* args)
    {
        A3B_REQUIRE(args, "null arguments");
        uint64_t const outer = args->outer, inner = args->inner, n = args->n, vocab = args->vocab;
        int64_t const first = args->first, add_stride = args->add_stride, table_stride = args->table_stride;
        a3b_rows const& grad_out = args->grad_out;
        void const *tokens = args->tokens, *add = args->add;
        void *grad_table = args->grad_table, *workspace = args->workspace;
        uint64_t const workspace_bytes = args->workspace_bytes;
        double const scale = args->scale;
        int const grad_dtype = args->grad_dtype, index_dtype = args->index_dtype, table_dtype = args->table_dtype;
        int const rc = checkTypes(grad_dtype, table_dtype, index_dtype, vocab, outer, inner, n, scale);
        if(rc != A3B_OK)
            return rc;
        if(vocab == 0)
            return A3B_OK;
        uint64_t const count = outer * inner;
        A3B_REQUIRE(grad_table && (count == 0 || (grad_out.data && tokens)), "null gradient or tokens");
        int const gs = rowTypeSize(grad_dtype), ts = rowTypeSize(table_dtype), is = index_dtype == A3B_I64 ? 8 : 4;
        A3B_REQUIRE(alignedTo(gs, {grad_out.data}) && alignedTo(ts, {grad_table, add}) && alignedTo(is, {tokens}),
                    "an array is not aligned to its type");
        Stretch const sg = Stretch::rows(grad_out, outer, inner, n, gs);
        Stretch const so = Stretch::rows(grad_table, 1, vocab, 0, table_stride, n, ts);
        Stretch const sa = Stretch::rows(add, 1, vocab, 0, add_stride, n, ts);
        Stretch const si = Stretch::dense(tokens, static_cast<Wide>(count) * is);
        Stretch const sw = Stretch::dense(workspace, static_cast<Wide>(workspace_bytes));
        A3B_REQUIRE(so.separate(), "rows of the table's gradient overlap");
        bool const inPlace = !sa.empty() && so.sameAs(sa);
        A3B_REQUIRE(inPlace || so.apart(sa), "the table's gradient overlaps what is added (only the same rows in place are allowed)");
        A3B_REQUIRE(so.apart(sg) && so.apart(si) && so.apart(sw) && sw.apart(sg) && sw.apart(si) && sw.apart(sa),
                    "the table's gradient and the workspace must lie apart from the inputs and from one another");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        Plan const p = planFor(props, count, n, vocab);
        A3B_REQUIRE(count == 0 || (workspace && alignedTo(16, {workspace}) && workspace_bytes >= p.bytes),
                    "the workspace is missing, too small or not aligned to 16 bytes");
        auto s = static_cast<cudaStream_t>(stream);
        Tokens const known{tokens, index_dtype == A3B_I64, first, static_cast<uint32_t>(vocab)};
        char* const ws = static_cast<char*>(workspace);
        SumArgs a{grad_out.data, {grad_out.outer_stride, grad_out.inner_stride}, nullptr, nullptr,
                  count ? reinterpret_cast<float*>(ws + p.partial) : nullptr,
                  count ? reinterpret_cast<uint32_t*>(ws + p.runs) : nullptr, add, add_stride, grad_table,
                  table_stride, static_cast<uint32_t>(count), static_cast<uint32_t>(inner), static_cast<uint32_t>(n),
                  static_cast<uint32_t>(vocab), p.chunk, p.chunks, 0u, 0u, outer == 1, !inPlace,
                  !add && table_stride == static_cast<int64_t>(n) && alignedTo(16, {grad_table}), static_cast<float>(scale), 0};
        return withTypes(grad_dtype, table_dtype, [&](auto t, auto u)
        {
            using T = decltype(t);
            using U = decltype(u);
            constexpr int E = kLot<T, U>;
            bool const packed = n % E == 0 && rowsAligned(grad_out.data, outer, inner, grad_out.outer_stride, grad_out.inner_stride, gs, 16)
                                && rowsAligned(grad_table, 1, vocab, 0, table_stride, ts, 16)
                                && rowsAligned(add, 1, vocab, 0, add_stride, ts, 16);
            return packed ? launchGradient<T, U, E>(s, props, a, p, known, ws) : launchGradient<T, U, 1>(s, props, a, p, known, ws);
        });
    }
}
