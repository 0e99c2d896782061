// Rows of a table by tokens, and the gradient of the table: a sum by keys.
//
//   out_i = scale * W[t_i],      dW_v = add_v + scale * sum of g_i over the positions i with t_i = v
//
// Both move memory and compute next to nothing. The gradient first sorts the tokens (stably: the positions of one token
// stay in their order), then sums the sorted list in chunks of a fixed number of positions, whatever the tokens are: a token
// that fills half of a batch is as well spread over the SMs as many rare ones. A run of one token within a chunk goes
// straight to its row; one that crosses chunks leaves partial sums that a last kernel joins in order. So the bits depend on
// the sizes alone, never on which block comes first.
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
            a.shift = teamShift(lots);
            uint32_t const teams = kThreads >> a.shift, lanes = 1u << a.shift;
            uint32_t const blocks = (a.count + teams - 1) / teams;
            // four loads under way a lane, unless that leaves SMs without a block
            bool const deep = static_cast<uint64_t>(blocks) * ((lots + 4 * lanes - 1) / (4 * lanes)) >= 4u * static_cast<unsigned>(props->smCount);
            uint32_t const slices = (lots + (deep ? 4 : 1) * lanes - 1) / ((deep ? 4 : 1) * lanes);
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

        // ------------------------------------------------------------------------------------- sorting the tokens
        // Up to kRankMax tokens: the place of each is the number of those that come before it, by comparing all pairs. A
        // block ranks 32 tokens, each of its warps against an eighth of the list. Quadratic, but one launch: 8192 tokens
        // are 67 million comparisons, a few microseconds on the whole GPU.
        constexpr uint32_t kRankMax = 8192;

        __global__ void __launch_bounds__(256) rankKernel(Tokens tokens, uint32_t count, uint32_t* keys, uint32_t* places)
        {
            extern __shared__ __align__(16) uint32_t all[];
            __shared__ uint32_t part[8][32];
            uint32_t const warp = threadIdx.x / 32, lane = threadIdx.x % 32, base = blockIdx.x * 32, i = base + lane;
            uint32_t const span = ((count + 7) / 8 + 31) / 32 * 32, low = warp * span;
            uint32_t const high = min(low + span, (count + 31) / 32 * 32);
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

        // More tokens: radix sort, digits of at most nine bits from the lowest, three kernels a digit. A block counts and
        // later places one contiguous tile, its warps contiguous parts of it, so equal digits keep their order.
        constexpr int kBins = 512, kTileWarps = 8;

        struct RadixArgs
        {
            Tokens tokens; // first digit
            uint32_t const* keysIn; // later digits
            uint32_t const* placesIn;
            uint32_t* keys;
            uint32_t* places;
            uint32_t* counts; // [bin][tile]
            uint32_t* totals; // [bin]
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
        struct SumArgs
        {
            void const* g;
            RowStep gs;
            uint32_t const* keys; // sorted, `vocab` behind the last known token
            uint32_t const* places;
            float* partial; // [chunk][2][n]: the run that reaches in from the chunk before, and the one that reaches out
            void const* add; // may be null
            int64_t addStride;
            void* out;
            int64_t stride;
            uint32_t count, inner, n, vocab, chunk, chunks, slices, sumBlocks;
            bool one, fill; // fill: rows without a token are written
            float scale;
            int shift;
        };

        template<typename U, int E>
        __device__ __forceinline__ void writeRow(SumArgs const& a, uint32_t row, uint32_t k, float* v)
        {
#pragma unroll
            for(int e = 0; e < E; ++e)
                v[e] *= a.scale;
            if(a.add)
            {
                unsigned raw[Lot<U, E>::words];
                float more[E];
                Lot<U, E>::load(raw, static_cast<U const*>(a.add) + static_cast<int64_t>(row) * a.addStride + k);
                Lot<U, E>::unpack(more, raw);
#pragma unroll
                for(int e = 0; e < E; ++e)
                    v[e] += more[e];
            }
            Lot<U, E>::store(static_cast<U*>(a.out) + static_cast<int64_t>(row) * a.stride + k, v);
        }

        constexpr uint32_t kFillRows = 32;

        // The first blocks sum: a team has a chunk of the sorted list and E columns a lane, and loads kAhead rows before it
        // adds them. The others write the rows of tokens that do not occur.
        template<typename T, typename U, int E>
        __global__ void __launch_bounds__(kThreads) embeddingSumKernel(SumArgs a)
        {
            constexpr int kAhead = 8;
            if(blockIdx.x >= a.sumBlocks)
            {
                __shared__ bool absent[kFillRows];
                uint32_t const base = (blockIdx.x - a.sumBlocks) * kFillRows, lots = a.n / E;
                if(uint32_t const row = base + threadIdx.x; threadIdx.x < kFillRows)
                {
                    uint32_t low = 0, high = a.count; // the first key that is not below row
                    while(low < high)
                    {
                        uint32_t const mid = low + (high - low) / 2;
                        if(a.keys[mid] < row)
                            low = mid + 1;
                        else
                            high = mid;
                    }
                    absent[threadIdx.x] = row < a.vocab && !(low < a.count && a.keys[low] == row);
                }
                __syncthreads();
                for(uint32_t r = 0; r < kFillRows; ++r)
                    if(absent[r])
                        for(uint32_t k = threadIdx.x; k < lots; k += kThreads)
                        {
                            float v[E];
#pragma unroll
                            for(int e = 0; e < E; ++e)
                                v[e] = 0.f;
                            writeRow<U, E>(a, base + r, k * E, v);
                        }
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
            uint32_t current = a.keys[low];
            bool inward = low > 0 && a.keys[low - 1] == current; // the run began in an earlier chunk
            float sum[E];
#pragma unroll
            for(int e = 0; e < E; ++e)
                sum[e] = 0.f;
            auto flush = [&](bool outward)
            {
                if(current >= a.vocab)
                    return;
                if(inward || outward)
                {
                    float* p = a.partial + (static_cast<size_t>(c) * 2 + (inward ? 0 : 1)) * a.n + col;
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        p[e] = sum[e];
                }
                else
                    writeRow<U, E>(a, current, col, sum);
            };
            for(uint32_t p = low; p < high; p += kAhead)
            {
                uint32_t key[kAhead];
                unsigned raw[kAhead][Lot<T, E>::words];
#pragma unroll
                for(int u = 0; u < kAhead; ++u)
                {
                    key[u] = p + u < high ? a.keys[p + u] : a.vocab;
                    if(key[u] < a.vocab)
                        Lot<T, E>::load(raw[u], static_cast<T const*>(a.g) + a.gs.at(a.places[p + u], a.inner, a.one) + col);
                }
#pragma unroll
                for(int u = 0; u < kAhead; ++u)
                {
                    if(key[u] >= a.vocab)
                        break; // only tokens without a row come behind
                    if(key[u] != current)
                    {
                        flush(false);
                        current = key[u];
                        inward = false;
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            sum[e] = 0.f;
                    }
                    float v[E];
                    Lot<T, E>::unpack(v, raw[u]);
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        sum[e] += v[e];
                }
            }
            flush(high < a.count && a.keys[high] == current);
        }

        // Joins the partial sums of a run that begins in chunk blockIdx.x and ends in a later one. Eight warps take equal
        // parts of its chunks, a lane four columns; the parts are added in their order.
        template<typename U, bool Packs>
        __global__ void __launch_bounds__(256) embeddingJoinKernel(SumArgs a)
        {
            __shared__ float4 part[8][32];
            uint32_t const c = blockIdx.x, low = c * a.chunk, high = low + a.chunk; // never the last chunk
            uint32_t const key = a.keys[high - 1];
            if(key >= a.vocab || a.keys[high] != key)
                return;
            bool const whole = a.keys[low] == key; // the run fills the chunk
            if(whole && low > 0 && a.keys[low - 1] == key)
                return; // began earlier
            uint32_t first = high, last = a.count; // the first place behind the run
            while(first < last)
            {
                uint32_t const mid = first + (last - first) / 2;
                if(a.keys[mid] <= key)
                    first = mid + 1;
                else
                    last = mid;
            }
            uint32_t const end = (first - 1) / a.chunk; // the last chunk with a part of it
            uint32_t const parts = end - c + 1, each = (parts + 7) / 8;
            uint32_t const warp = threadIdx.x / 32, lane = threadIdx.x % 32;
            for(uint32_t base = blockIdx.y * 128; base < a.n; base += gridDim.y * 128)
            {
                uint32_t const col = base + lane * 4;
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
                            float4 const v = *reinterpret_cast<float4 const*>(p);
                            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
                        }
                    }
                    else
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                            if(col + e < a.n)
                                s[e] += p[e];
                }
                __syncthreads(); // the last columns' parts have been read
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
                            writeRow<U, 1>(a, key, col + e, s + e);
                }
            }
        }

        // ------------------------------------------------------------------------------------------ workspace
        struct Plan
        {
            bool radix;
            uint32_t chunk, chunks, tile, tiles;
            int digits, bits; // radix digits and bits of each
            size_t keys, places, keys2, places2, counts, totals, partial, bytes; // offsets, and the whole
        };

        // From sizes alone (not from alignment), so that the workspace and the order of the sums are.
        Plan planFor(DeviceProps const* props, uint64_t count, uint64_t n, uint64_t vocab)
        {
            Plan p{};
            p.radix = count > kRankMax;
            // About eight blocks of 128 threads an SM, each thread with eight columns; chunks of 4 to 256 positions.
            uint64_t const perRow = std::max<uint64_t>(1, n / 8), wanted = 8ull * static_cast<unsigned>(props->smCount) * kThreads;
            uint64_t const chunk = count * perRow / wanted;
            p.chunk = static_cast<uint32_t>(std::min<uint64_t>(256, std::max<uint64_t>(4, chunk / 4 * 4)));
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
            p.partial = take(static_cast<size_t>(p.chunks) * 2 * n * 4);
            p.bytes = std::max<size_t>(at, 256);
            return p;
        }

        int sortTokens(cudaStream_t stream, Plan const& p, Tokens const& tokens, uint32_t count, char* ws, uint32_t** keys,
                       uint32_t** places)
        {
            auto at = [&](size_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
            *keys = at(p.keys);
            *places = at(p.places);
            if(!p.radix)
            {
                uint32_t const blocks = (count + 31) / 32;
                rankKernel<<<blocks, 256, blocks * 32 * 4, stream>>>(tokens, count, *keys, *places);
                A3B_CHECK_LAUNCH("rankKernel");
                return A3B_OK;
            }
            uint32_t *otherKeys = at(p.keys2), *otherPlaces = at(p.places2);
            for(int d = 0; d < p.digits; ++d)
            {
                RadixArgs a{tokens, otherKeys, otherPlaces, *keys, *places, at(p.counts), at(p.totals), count, p.tile, p.tiles,
                            d * p.bits, p.bits, d == 0};
                if(d > 0) // from what the digit before wrote
                {
                    a.keysIn = *keys, a.placesIn = *places;
                    a.keys = otherKeys, a.places = otherPlaces;
                    std::swap(*keys, otherKeys);
                    std::swap(*places, otherPlaces);
                }
                radixCountKernel<<<p.tiles, 256, 0, stream>>>(a);
                A3B_CHECK_LAUNCH("radixCountKernel");
                radixScanKernel<<<((1u << p.bits) + 3) / 4, 128, 0, stream>>>(a.counts, a.totals, p.tiles, 1u << p.bits);
                A3B_CHECK_LAUNCH("radixScanKernel");
                radixPlaceKernel<<<p.tiles, 32 * kTileWarps, 0, stream>>>(a);
                A3B_CHECK_LAUNCH("radixPlaceKernel");
            }
            return A3B_OK;
        }

        template<typename T, typename U, int E>
        int launchSum(cudaStream_t stream, SumArgs a)
        {
            uint32_t const lots = a.n / E;
            a.shift = teamShift(lots);
            uint32_t const lanes = 1u << a.shift, teams = kThreads >> a.shift;
            a.slices = (lots + lanes - 1) / lanes;
            uint64_t const sums = static_cast<uint64_t>((a.chunks + teams - 1) / teams) * a.slices;
            uint64_t const fills = a.fill ? (a.vocab + kFillRows - 1) / kFillRows : 0;
            if(sums + fills > static_cast<uint64_t>(INT_MAX))
            {
                setError("%u tokens of %u elements are more than one launch holds", a.count, a.n);
                return A3B_ERR_TOO_LARGE;
            }
            a.sumBlocks = static_cast<uint32_t>(sums);
            if(sums + fills == 0)
                return A3B_OK;
            embeddingSumKernel<T, U, E><<<static_cast<unsigned>(sums + fills), kThreads, 0, stream>>>(a);
            A3B_CHECK_LAUNCH("embeddingSumKernel");
            if(a.chunks > 1)
            {
                dim3 const grid(a.chunks - 1, std::min<uint32_t>(4, (a.n + 127) / 128));
                if(a.n % 4 == 0)
                    embeddingJoinKernel<U, true><<<grid, 256, 0, stream>>>(a);
                else
                    embeddingJoinKernel<U, false><<<grid, 256, 0, stream>>>(a);
                A3B_CHECK_LAUNCH("embeddingJoinKernel");
            }
            return A3B_OK;
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
        uint32_t *keys = nullptr, *places = nullptr;
        if(count > 0)
        {
            Tokens const t{tokens, index_dtype == A3B_I64, first, static_cast<uint32_t>(vocab)};
            int const rs = sortTokens(s, p, t, static_cast<uint32_t>(count), static_cast<char*>(workspace), &keys, &places);
            if(rs != A3B_OK)
                return rs;
        }
        SumArgs a{grad_out.data, {grad_out.outer_stride, grad_out.inner_stride}, keys, places,
                  count ? reinterpret_cast<float*>(static_cast<char*>(workspace) + p.partial) : nullptr, add, add_stride, grad_table,
                  table_stride, static_cast<uint32_t>(count), static_cast<uint32_t>(inner), static_cast<uint32_t>(n),
                  static_cast<uint32_t>(vocab), p.chunk, p.chunks, 0u, 0u, outer == 1, !inPlace, static_cast<float>(scale), 0};
        return withTypes(grad_dtype, table_dtype, [&](auto t, auto u)
        {
            using T = decltype(t);
            using U = decltype(u);
            constexpr int E = kLot<T, U>;
            bool const packed = n % E == 0 && rowsAligned(grad_out.data, outer, inner, grad_out.outer_stride, grad_out.inner_stride, gs, 16)
                                && rowsAligned(grad_table, 1, vocab, 0, table_stride, ts, 16)
                                && rowsAligned(add, 1, vocab, 0, add_stride, ts, 16);
            return packed ? launchSum<T, U, E>(s, a) : launchSum<T, U, 1>(s, a);
        });
    }
}
