// Log probabilities of given tokens under rows of logits, with the entropy of each row's distribution, its log-sum-exp
// and its most likely alternatives, and their gradient. No counterpart in alpaka3, whose reductions run over a whole
// buffer (include/alpaka/onHost/algo/transformReduce.hpp:59-114); these are the same one-pass transform-reduce, one
// result per row.
//
// For a row x of V logits, z = scale * x, m = max z:
//     s = sum e^(z - m)      lse = m + ln s      logp(v) = z_v - lse = (z_v - m) - ln s
//     entropy = -sum p logp  = ln s - (sum (z - m) e^(z - m)) / s
// evaluated in one pass with a running maximum: when a larger m' arrives, the sums kept so far are rescaled by
// e^(m - m') (and the second one by what the shift of the exponents adds to it).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <initializer_list>
#include <type_traits>

#include "rows.cuh"

namespace a3b
{
    namespace
    {
        constexpr int kPacks = 8;    // 16-byte packs of a tile that one thread holds in registers
        constexpr int kMaxTop = 32;  // alternatives of a row
        constexpr float kLog2e = 1.4426950408889634f;
        constexpr float kLn2 = 0.6931471805599453f;

        // The rows of a logits-like tensor: row r starts at (r / inner) * outerStride + (r % inner) * innerStride.
        struct RowLayout
        {
            uint32_t inner;
            int64_t outerStride;
            int64_t innerStride;

            __device__ __forceinline__ int64_t at(uint32_t r) const
            {
                uint32_t const o = r / inner;
                return static_cast<int64_t>(o) * outerStride + static_cast<int64_t>(r - o * inner) * innerStride;
            }
        };

        struct LogprobArgs
        {
            void const* logits;
            RowLayout layout;
            uint64_t rows;
            uint32_t tiles; // of a row, or of its slice
            uint32_t share; // packs of a slice (the last one takes what is left)
            uint32_t vocab;
            uint32_t top;
            float scale;
            float reach; // 256 / (scale / ln 2): logits this far below the largest one do not count
            int index64; // targets and topIndex hold 64-bit (else 32-bit) integers
            void const* targets;
            float* logp;
            float* entropy;
            float* lse;
            float* topLogp;
            void* topIndex;
        };

        __device__ __forceinline__ int64_t loadIndex(void const* p, uint64_t i, int index64)
        {
            return index64 ? static_cast<int64_t const*>(p)[i] : static_cast<int64_t>(static_cast<int32_t const*>(p)[i]);
        }

        // Total order of the logits as unsigned integers: -0 equals +0, NaN comes above +infinity.
        __device__ __forceinline__ unsigned orderOf(float x)
        {
            if(isnan(x))
                return 0xffffffffu;
            unsigned const b = __float_as_uint(x + 0.0f);
            return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
        }

        __device__ __forceinline__ float valueOf(unsigned order)
        {
            return __uint_as_float((order & 0x80000000u) ? (order & 0x7fffffffu) : ~order);
        }

        // Candidate of the selection: larger is better, equal values go to the lower index.
        __device__ __forceinline__ unsigned long long keyOf(unsigned order, unsigned index)
        {
            return (static_cast<unsigned long long>(order) << 32) | static_cast<unsigned>(~index);
        }

        // Sums of one share of a row whose largest logit is `high`: s = sum 2^t and u = sum t 2^t over its logits x, with
        // t = c x + offset, one fused operation. c = scale / ln 2, and offset = -(c high) as it is rounded. The largest
        // logit's own t is what that rounding left: at most 32, as long as |c high| is at most 2^30.
        struct Stats
        {
            float high;
            float s;
            float u;
        };

        // Beyond that, fp32's steps at `high` are 64 or more in t: all logits but those equal to it together are less than
        // V 2^-64 of the sum and are left out. Then the factor is a power of two that brings `high` to 2^33 (an exact
        // product: t = 0 for what equals it, below -500 for all else), and u is 0 (and not computed: `u` holds NaN if there
        // are logits of -infinity, which no clamp separates from a maximum of fp32's lowest value).
        __device__ __forceinline__ bool isBig(float high, float c)
        {
            return !(fabsf(high * c) <= 0x1p30f);
        }

        __device__ __forceinline__ float factorOf(float high, float c)
        {
            return isBig(high, c) && high != -INFINITY
                       ? __uint_as_float(((127u + 127u + 33u) << 23) - (__float_as_uint(high) & 0x7f800000u))
                       : c;
        }

        __device__ __forceinline__ float offsetOf(float high, float c)
        {
            // rounded on its own wherever it is used: fused into a difference of offsets it would be another number
            return high == -INFINITY ? 0.0f : -__fmul_rn(high, factorOf(high, c));
        }

        // the sums of `b` moved to the maximum `high` (not below b's) and added to s, u
        __device__ __forceinline__ void addStats(float high, float c, Stats const& b, float& s, float& u)
        {
            if(b.high == -INFINITY)
                return; // nothing in that share
            bool const big = isBig(high, c) || isBig(b.high, c);
            float const d = b.high == high ? 0.0f : big ? -200.0f : fmaxf(offsetOf(high, c) - offsetOf(b.high, c), -200.0f);
            float const f = exp2Approx(d);
            s += f * b.s;
            u += big ? 0.0f : f * fmaf(d, b.s, b.u);
        }

        constexpr int kBlock = 256;
        constexpr int kMaxCluster = 8;

        // elements from p to the next 16-byte boundary
        template<typename T>
        __device__ __forceinline__ uint32_t toBoundary(T const* p)
        {
            auto const past = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u);
            return ((16u - past) & 15u) / static_cast<uint32_t>(sizeof(T));
        }

        // A row's team is S threads: a block (S = 64, 128, 256), a warp or a quarter of one in a block of kBlock.
        template<int S>
        struct Team
        {
            static constexpr int warps = S > 32 ? S / 32 : 1;
            static constexpr int perBlock = S > 32 ? 1 : kBlock / S;
            static constexpr int block = S > 32 ? S : kBlock;
            static constexpr int width = S < 32 ? S : 32; // threads of the team in one warp

            static __device__ __forceinline__ unsigned thread()
            {
                return threadIdx.x & (S - 1);
            }
            // the team's part of this warp
            static __device__ __forceinline__ unsigned mask()
            {
                return S >= 32 ? kFullMask : ((1u << (S & 31)) - 1u) << (threadIdx.x & 31u & ~(S - 1u));
            }
            static __device__ __forceinline__ void sync()
            {
                if constexpr(S > 32)
                    __syncthreads();
                else
                    __syncwarp(mask());
            }
            // the largest value of the team's part of this warp (NaN if there is one)
            static __device__ __forceinline__ float max(float v)
            {
                if constexpr(S >= 32)
                    return warpMaxNan(v);
                else
                {
#pragma unroll
                    for(int m = width / 2; m > 0; m >>= 1)
                        v = maxNan(v, __shfl_xor_sync(mask(), v, m));
                    return v;
                }
            }
            static __device__ __forceinline__ float sum(float v)
            {
#pragma unroll
                for(int m = width / 2; m > 0; m >>= 1)
                    v += __shfl_xor_sync(mask(), v, m);
                return v;
            }
        };

        // A row: `head` elements up to the first 16-byte boundary, `packs` 16-byte packs, `tail` elements behind them.
        template<typename T>
        struct Row
        {
            static constexpr uint32_t E = PackOf<T>::E;
            T const* p;
            uint32_t head, packs, tail;

            __device__ __forceinline__ Row(LogprobArgs const& a, uint64_t r)
                : p(static_cast<T const*>(a.logits) + a.layout.at(static_cast<uint32_t>(r)))
            {
                head = min(a.vocab, toBoundary(p));
                packs = (a.vocab - head) / E;
                tail = a.vocab - head - packs * E;
            }
        };

        // A tile of a row: P packs of every thread of the team, pack p of thread t being pack base + p * team + t of the
        // row.
        template<typename T, int S, int P>
        struct Tile
        {
            static constexpr int E = PackOf<T>::E;
            static constexpr uint32_t team = S;
            unsigned q[P][4];

            // packs outside [.., end) read as -infinity
            __device__ __forceinline__ void load(Row<T> const& row, uint32_t base, uint32_t end)
            {
                auto const* const from = reinterpret_cast<uint4 const*>(row.p + row.head) + base + Team<S>::thread();
                unsigned const n = PackOf<T>::negInfWord();
                if(base + P * team <= end)
                {
#pragma unroll
                    for(int p = 0; p < P; ++p)
                    {
                        uint4 const v = __ldcs(from + p * team);
                        q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    }
                }
                else
                {
#pragma unroll
                    for(int p = 0; p < P; ++p)
                    {
                        uint4 v = make_uint4(n, n, n, n);
                        if(base + p * team + Team<S>::thread() < end)
                            v = __ldcs(from + p * team);
                        q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    }
                }
            }

            // pack p from `from`, or (for the whole team) left as it is
            __device__ __forceinline__ void reload(int p, uint4 const* from, bool really)
            {
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
                             "@p ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                             : "+r"(q[p][0]), "+r"(q[p][1]), "+r"(q[p][2]), "+r"(q[p][3])
                             : "l"(from), "r"(really ? 1u : 0u)
                             : "memory");
            }

            // Keeps the compiler from carrying unpacked elements from one use of the tile to the next: unpacking again
            // is an instruction or less an element, the floats of a whole tile are 64 registers.
            __device__ __forceinline__ void fence()
            {
#pragma unroll
                for(int p = 0; p < P; ++p)
                    asm volatile("" : "+r"(q[p][0]), "+r"(q[p][1]), "+r"(q[p][2]), "+r"(q[p][3]));
            }
        };

        // ------------------------------------------------------------------------------------------ selection
        constexpr unsigned kOrderNegInf = 0x007fffffu; // orderOf(-infinity), below every other one

        // how many of m keys in shared memory are larger than `key`; independent loads, eight at a time
        __device__ __forceinline__ unsigned countAbove(unsigned long long const* keys, unsigned m, unsigned long long key)
        {
            unsigned above = 0;
            unsigned j = 0;
            for(; j + 8 <= m; j += 8)
            {
                unsigned long long k[8];
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    k[i] = keys[j + i];
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    above += k[i] > key ? 1u : 0u;
            }
            for(; j < m; ++j)
                above += keys[j] > key ? 1u : 0u;
            return above;
        }

        // Candidates for a row's `top` largest elements. Two buffers take turns: one starts with the keys kept so far, in
        // order, and collects more; ranking them writes the new kept ones to the start of the other.
        template<int S>
        struct Select
        {
            // the kept keys and one element of each thread always fit
            static constexpr unsigned room = S + 2 * kMaxTop;
            unsigned long long keys[2][room];
            unsigned long long kth; // the last of `top` kept keys
            unsigned count[2];
            unsigned bound[Team<S>::warps];

            __device__ __forceinline__ void push(unsigned buffer, unsigned order, uint32_t index)
            {
                unsigned const at = atomicAdd(&count[buffer], 1u);
                if(at < room)
                    keys[buffer][at] = keyOf(order, index);
            }

            // Ranks the first m candidates of `buffer` by counting (their order there does not matter: the keys are
            // distinct) and keeps the `top` best in the other one.
            __device__ __forceinline__ void rank(unsigned buffer, unsigned m, unsigned top)
            {
                unsigned const thread = Team<S>::thread();
                for(unsigned i = thread; i < m; i += S)
                {
                    unsigned long long const key = keys[buffer][i];
                    unsigned const above = countAbove(keys[buffer], m, key);
                    if(above < top)
                        keys[buffer ^ 1u][above] = key;
                    if(above == top - 1)
                        kth = key;
                }
                if(thread == 0)
                    count[buffer ^ 1u] = min(m, top);
            }

            // The order from which an element behind those kept can enter: it has a higher index, so an equal one cannot.
            // 0: none can (the kept ones are all NaN).
            __device__ __forceinline__ unsigned from(unsigned kept, unsigned top) const
            {
                return kept == top ? static_cast<unsigned>(kth >> 32) + 1u : kOrderNegInf + 1u;
            }

            // Every warp's need-th largest thread maximum, need = ceil(top / warps), is reached by `need` elements of that
            // warp; so at least `top` elements of the tile reach the smallest of these bounds, and no element below it
            // can be among the `top` largest. For logits in no particular order a few dozen elements of a tile pass.
            __device__ __forceinline__ unsigned boundOf(unsigned mine, unsigned top)
            {
                int const lane = threadIdx.x & 31;
                unsigned least = 0, left = mine;
                for(unsigned i = 0; i < (top + Team<S>::warps - 1) / Team<S>::warps; ++i)
                {
                    least = __reduce_max_sync(Team<S>::mask(), left);
                    if(lane == __ffs(static_cast<int>(__ballot_sync(Team<S>::mask(), left == least))) - 1)
                        left = 0u;
                }
                if(S > 32 && lane == 0)
                    bound[threadIdx.x >> 5] = least;
                Team<S>::sync();
                if constexpr(S > 32)
                {
#pragma unroll
                    for(int w = 0; w < Team<S>::warps; ++w)
                        least = min(least, bound[w]);
                }
                return max(least, kOrderNegInf + 1u);
            }

            // Collects the tile's elements with an order of `least` or more. Where a warp has any, every thread picks its
            // packs that hold one, one pack a turn, and looks at that pack's elements: mostly one turn, and code that
            // is short (a search unrolled over all packs did not fit the instruction cache).
            template<typename T, int P>
            __device__ __forceinline__ void collect(
                Tile<T, S, P> const& t, unsigned least, unsigned mine, uint32_t head, uint32_t base, unsigned buffer)
            {
                bool const has = mine >= least && least != 0u;
                if(!__any_sync(Team<S>::mask(), has))
                    return;
                float const value = valueOf(least); // NaN where `least` is: then every pack is looked at
                unsigned packs = 0;
#pragma unroll
                for(int p = 0; p < P; ++p)
                    packs |= PackOf<T>::max(t.q[p]) < value ? 0u : 1u << p;
                packs = has ? packs : 0u;
                while(packs != 0u)
                {
                    int const p = __ffs(static_cast<int>(packs)) - 1;
                    packs &= packs - 1u;
                    unsigned word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for(int i = 0; i < P; ++i)
#pragma unroll
                        for(int w = 0; w < 4; ++w)
                            word[w] = i == p ? t.q[i][w] : word[w];
                    uint32_t const index
                        = head + (base + p * Tile<T, S, P>::team + Team<S>::thread()) * Tile<T, S, P>::E;
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        float2 const v = PackOf<T>::pair(word, w);
                        auto consider = [&](float x, uint32_t i)
                        {
                            unsigned const o = orderOf(x);
                            if(o >= least)
                                push(buffer, o, i);
                        };
                        if(!(v.x < value))
                            consider(v.x, index + 2 * w);
                        if(!(v.y < value))
                            consider(v.y, index + 2 * w + 1);
                    }
                }
                __syncwarp(Team<S>::mask());
            }

            // whether any thread of the team says so (the team is synchronised)
            static __device__ __forceinline__ bool anyOf(bool b)
            {
                if constexpr(S <= 32)
                    return __any_sync(Team<S>::mask(), b);
                else
                    return __syncthreads_or(b);
            }

            // The same selection for the elements [first, last) of a row, whatever they are: where too many passed (many
            // equal ones: constant rows, masks of one low value; rows in rising order). Eight packs a thread are skipped
            // where nothing enters; else the elements are taken in steps that always fit, one of every thread. `buffer`
            // starts with `kept` keys in order, those of lower indices, and its count is `kept`.
            template<typename T>
            __device__ __noinline__ uint2 careful(
                T const* row, uint32_t first, uint32_t last, unsigned top, unsigned kept, unsigned buffer)
            {
                constexpr unsigned per = 8, E = PackOf<T>::E, stride = S * per * E;
                unsigned const thread = Team<S>::thread();
                while(first < last)
                {
                    uint32_t const edge = toBoundary(row + first);
                    uint32_t upTo = edge != 0u && edge < last - first ? first + edge : last;
                    if(edge == 0u && stride <= last - first)
                    {
                        unsigned q[per][4];
#pragma unroll
                        for(unsigned k = 0; k < per; ++k)
                        {
                            uint4 const v = __ldcs(reinterpret_cast<uint4 const*>(row + first) + k * S + thread);
                            q[k][0] = v.x, q[k][1] = v.y, q[k][2] = v.z, q[k][3] = v.w;
                        }
                        unsigned const least = from(kept, top);
                        upTo = first + stride;
                        if(!anyOf(least != 0u && orderOf(PackOf<T>::template max<per>(q)) >= least))
                        {
                            first = upTo;
                            continue;
                        }
                    }
                    for(; first < upTo; first += S * per)
                    {
                        unsigned order[per];
                        bool enters = false;
                        unsigned const least = from(kept, top);
#pragma unroll
                        for(unsigned k = 0; k < per; ++k)
                        {
                            uint32_t const i = first + k * S + thread;
                            order[k] = i < upTo ? orderOf(toFloat(row[i])) : 0u;
                            enters |= order[k] >= least && least != 0u;
                        }
                        if(!anyOf(enters))
                            continue;
                        for(unsigned k = 0; k < per; ++k)
                        {
                            unsigned o = 0;
#pragma unroll
                            for(unsigned j = 0; j < per; ++j)
                                o = j == k ? order[j] : o;
                            unsigned const now = from(kept, top);
                            if(o >= now && now != 0u)
                                push(buffer, o, first + k * S + thread);
                            Team<S>::sync();
                            unsigned const n = count[buffer];
                            if(n > kept)
                            {
                                rank(buffer, n, top);
                                kept = min(n, top);
                                buffer ^= 1u;
                            }
                            Team<S>::sync();
                        }
                    }
                    first = upTo;
                }
                return make_uint2(kept, buffer);
            }
        };

        // Fills `kept` up to `top` keys with the row's first elements of -infinity, by the team's (first) warp. All others
        // are among the kept ones, so the first 2 top elements of the row hold enough of them.
        template<int S, typename T>
        __device__ __forceinline__ void fillWithNegInf(
            T const* row, uint32_t vocab, unsigned top, unsigned kept, unsigned long long* keys)
        {
            constexpr uint32_t width = Team<S>::width;
            unsigned const lane = threadIdx.x & (width - 1u), below = (1u << (threadIdx.x & 31u)) - 1u;
            for(uint32_t i0 = 0; kept < top && i0 < vocab; i0 += width)
            {
                uint32_t const i = i0 + lane;
                bool const hit = i < vocab && toFloat(row[i]) == -INFINITY;
                unsigned const hits = __ballot_sync(Team<S>::mask(), hit);
                unsigned const at = kept + __popc(hits & below);
                if(hit && at < top)
                    keys[at] = keyOf(kOrderNegInf, i);
                kept = min(top, kept + __popc(hits));
            }
            __syncwarp(Team<S>::mask());
        }

        // What the blocks of a cluster leave in the first one's shared memory.
        template<bool TOP>
        struct Gather
        {
            Stats stats[kMaxCluster];
            unsigned long long keys[TOP ? kMaxCluster * kMaxTop : 1];
        };

        // Blocks of kBlock threads an SM that the registers are bounded to. Measured on a B200 with 3 / 4 for tiles of eight
        // packs and alternatives: 2048 x 50257 bf16 on teams of 128 threads 55 / 50 us, 300 x 131072 fp32 on 256 35 / 33;
        // on single warps, which spill at 64 registers, 16384 x 2048 bf16 31 / 34 us.
        template<int S, int P, bool TOP>
        constexpr int residentBlocks()
        {
            return P == 2 ? (TOP ? 4 : 6) : P == 8 && TOP && S <= 32 ? 3 : 4;
        }

        // One row a team. In a launch with clusters, slice b of a row is the tiles of the cluster's block b, and the first
        // block joins the slices. Every logit is read once and kept in registers for the maximum, the candidates and the
        // exponents: no second read and no shared memory for the tile, short blocks that overlap one another's loads.
        // Measured on a B200: 8192 x 131072 bf16 320 us, 6.7 TB/s (HBM, exponent pipe 77% busy); 2048 x 50257 bf16 with 4
        // alternatives 50 us, without 39; 64 x 131072 fp32 with 5 15 us (latency).
        template<typename T, int S, int P, bool TOP, bool ENT>
        __global__ void __launch_bounds__(Team<S>::block, kBlock / Team<S>::block * residentBlocks<S, P, TOP>())
            logprobKernel(LogprobArgs a)
        {
            constexpr int teams = Team<S>::perBlock;
            __shared__ Stats stats[Team<S>::warps];
            __shared__ Select<S> select[TOP ? teams : 1];
            __shared__ Gather<TOP> gather;
            Select<S>& sel = select[TOP && S <= 32 ? threadIdx.x / S : 0];
            unsigned const thread = Team<S>::thread();
            unsigned slice = 0, slices = 1;
            uint64_t r = S <= 32 ? static_cast<uint64_t>(blockIdx.x) * teams + threadIdx.x / S : blockIdx.x;
            if constexpr(S > 32)
            {
                slices = clusterBlocks();
                if(slices > 1)
                {
                    clusterArrive(); // waited for before the first block's shared memory is written
                    slice = clusterRank();
                    r = blockIdx.x / slices;
                }
            }
            else if(r >= a.rows)
                return;
            Row<T> const row(a, r);
            float const c = a.scale * kLog2e;
            uint32_t const span = P * S; // packs of a tile
            uint32_t const begin = min(row.packs, slice * a.share);
            uint32_t const end = slice == slices - 1 ? row.packs : min(row.packs, begin + a.share);
            int64_t const target = a.logp ? loadIndex(a.targets, r, a.index64) : -1;
            // What lies outside the packs, one element each of the first eight threads: the head is taken with the first
            // tile, in front of it, the tail with the last one.
            float const inHead = thread < row.head && slice == 0 ? toFloat(row.p[thread]) : -INFINITY;
            uint32_t const tailIndex = a.vocab - row.tail + thread;
            float const inTail = thread < row.tail && slice == slices - 1 ? toFloat(row.p[tailIndex]) : -INFINITY;
            float xt = 0.0f;

            float high = -INFINITY, factor = c, offset = 0.0f;
            unsigned low = PackOf<T>::negInfWord();
            float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
            unsigned kept = 0, buffer = 0;
            uint32_t ranked = 0, rankAfter = 1; // tiles whose candidates have been ranked, or will be next
            // The first of the tiles whose candidates were too many: from there the row is selected again at the end (a call
            // in the loop would keep the tile's registers from being all there is).
            constexpr uint32_t kNever = UINT32_MAX;
            uint32_t again = kNever;
            if(TOP && thread == 0)
                sel.count[0] = 0u;
            Tile<T, S, P> t;
            t.load(row, begin, end);
            if(target >= 0 && target < static_cast<int64_t>(a.vocab))
                xt = toFloat(row.p[target]);
            for(uint32_t tile = 0; tile < a.tiles; ++tile)
            {
                uint32_t const base = begin + tile * span;
                bool const last = tile + 1 == a.tiles;
                float const front = tile == 0 ? inHead : -INFINITY, behind = last ? inTail : -INFINITY;
                float const threadMax = maxNan(maxNan(front, behind), PackOf<T>::template max<P>(t.q));
                t.fence();
                // the warp's running maximum, and its sums moved there
                float const to = maxNan(high, Team<S>::max(threadMax));
                if(tile == 0 || to != high)
                {
                    if(tile > 0)
                    {
                        Stats const before{high, s2.x + s2.y, u2.x + u2.y};
                        s2 = u2 = make_float2(0.0f, 0.0f);
                        addStats(to, c, before, s2.x, u2.x);
                    }
                    high = to;
                    factor = factorOf(high, c);
                    offset = offsetOf(high, c);
                    // far below what counts (t < -200), for logits of -infinity: see below
                    low = PackOf<T>::twice(high - fmaf(fabsf(high), 0x1p-6f, a.reach));
                }
                if constexpr(TOP)
                {
                    // The first tile's candidates are ranked at once, later ones are collected without a barrier,
                    // against what was kept when they were last ranked.
                    unsigned const mine = orderOf(threadMax);
                    unsigned const least
                        = tile == 0 ? sel.boundOf(mine, a.top) : again == kNever ? sel.from(kept, a.top) : 0u;
                    sel.collect(t, least, mine, row.head, base, buffer);
                    if((tile == 0 || last) && least != 0u)
                    {
                        if(orderOf(front) >= least)
                            sel.push(buffer, orderOf(front), thread);
                        if(orderOf(behind) >= least)
                            sel.push(buffer, orderOf(behind), tailIndex);
                    }
                    t.fence();
                }
                float2 const offset2 = make_float2(offset, offset), factor2 = make_float2(factor, factor);
                auto add = [&](float2 x)
                {
                    float2 d = fma2(x, factor2, offset2);
                    if constexpr(ENT && !std::is_same_v<T, __nv_bfloat16>)
                    {
                        // -infinity times the zero that it gives would be NaN; 2^-200 is zero in fp32
                        d.x = maxNan(d.x, -200.0f);
                        d.y = maxNan(d.y, -200.0f);
                    }
                    float2 const e = make_float2(exp2Approx(d.x), exp2Approx(d.y));
                    s2 = add2(s2, e);
                    if constexpr(ENT)
                        u2 = fma2(d, e, u2);
                };
                // The registers of a pack that is done take the same pack of the next tile, if that is a full one: its
                // loads run under the rest of this tile.
                bool const nextFull = !last && base + 2 * span <= end;
                auto const* const next = reinterpret_cast<uint4 const*>(row.p + row.head) + base + span + thread;
#pragma unroll
                for(int p = 0; p < P; ++p)
                {
                    // a short tile's packs in the second half: none, for the whole team
                    if(p == P / 2 && base + p * S >= end)
                        break;
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        // bf16: the same bound in front of the conversion, for two elements at once
                        unsigned word[4] = {t.q[p][0], t.q[p][1], t.q[p][2], t.q[p][3]};
                        if constexpr(ENT && std::is_same_v<T, __nv_bfloat16>)
                            word[w] = PackOf<T>::maxWord(word[w], low);
                        add(PackOf<T>::pair(word, w));
                    }
                    t.reload(p, next + p * S, nextFull);
                }
                if((tile == 0 || last) && (S <= 32 || threadIdx.x < 32))
                {
                    float const least = high - fmaf(fabsf(high), 0x1p-6f, a.reach);
                    add(make_float2(maxNan(front, least), maxNan(behind, least)));
                }
                if(!last && !nextFull)
                    t.load(row, base + span, end);
                if constexpr(TOP)
                {
                    if((last || tile + 1 == rankAfter) && again == kNever)
                    {
                        Team<S>::sync();
                        unsigned const n = sel.count[buffer];
                        if(n > sel.room)
                            again = ranked;
                        else if(n > kept)
                        {
                            sel.rank(buffer, n, a.top);
                            kept = min(n, a.top);
                            buffer ^= 1u;
                        }
                        Team<S>::sync(); // ranked, and every thread has read the count before anyone collects more
                        ranked = tile + 1;
                        // Between ranking at n tiles and at k n about (k - 1) top elements pass: k = 4 as long as they fit
                        // with room to spare.
                        rankAfter = ranked * (8u * a.top <= sel.room ? 4u : 2u);
                    }
                }
            }
            if constexpr(TOP)
                if(again != kNever)
                {
                    if(thread == 0)
                        sel.count[buffer] = kept;
                    Team<S>::sync();
                    uint64_t const body = begin + uint64_t{again} * span;
                    uint64_t const from = again == 0 && slice == 0 ? 0 : row.head + min(uint64_t{end}, body) * PackOf<T>::E;
                    uint64_t const to = slice == slices - 1 ? a.vocab : row.head + uint64_t{end} * PackOf<T>::E;
                    uint2 const got = sel.careful(
                        row.p, static_cast<uint32_t>(from), static_cast<uint32_t>(to), a.top, kept, buffer);
                    kept = got.x;
                    buffer = got.y;
                }
            float s = Team<S>::sum(s2.x + s2.y), u = ENT ? Team<S>::sum(u2.x + u2.y) : 0.0f;
            unsigned long long* const best = sel.keys[buffer];
            if constexpr(S > 32)
            {
                if((threadIdx.x & 31) == 0)
                    stats[threadIdx.x >> 5] = Stats{high, s, u};
                __syncthreads();
                if(slices == 1 && threadIdx.x >= 32)
                    return;
                // one share a lane, for every warp that is still here alike
                auto join = [&](Stats const* all, unsigned n)
                {
                    unsigned const lane = threadIdx.x & 31u;
                    Stats const mine = lane < n ? all[lane] : Stats{-INFINITY, 0.0f, 0.0f};
                    high = warpMaxNan(mine.high);
                    s = u = 0.0f;
                    addStats(high, c, mine, s, u);
#pragma unroll
                    for(int m = 4; m > 0; m >>= 1)
                    {
                        s += __shfl_xor_sync(kFullMask, s, m);
                        u += __shfl_xor_sync(kFullMask, u, m);
                    }
                    s = __shfl_sync(kFullMask, s, 0);
                    u = __shfl_sync(kFullMask, u, 0);
                };
                static_assert(Team<S>::warps <= 8 && kMaxCluster <= 8, "join() sums eight lanes");
                join(stats, Team<S>::warps);
                if(slices > 1)
                {
                    clusterWait();
                    if(threadIdx.x == 0)
                        *inBlock(&gather.stats[slice], 0u) = Stats{high, s, u};
                    if constexpr(TOP)
                        if(threadIdx.x < a.top)
                            *inBlock(&gather.keys[slice * a.top + threadIdx.x], 0u)
                                = threadIdx.x < kept ? best[threadIdx.x] : 0ull;
                    clusterArrive();
                    clusterWait();
                    if(slice != 0)
                        return;
                    join(gather.stats, slices);
                    if constexpr(TOP)
                    {
                        unsigned const n = slices * a.top;
                        unsigned long long const key = threadIdx.x < n ? gather.keys[threadIdx.x] : 0ull;
                        if(key != 0ull)
                        {
                            unsigned const above = countAbove(gather.keys, n, key);
                            if(above < a.top)
                                best[above] = key;
                        }
                        kept = min(a.top, static_cast<unsigned>(__syncthreads_count(key != 0ull)));
                    }
                    if(threadIdx.x >= 32)
                        return;
                }
            }

            // The largest logit's own t is what the rounding of the offset left (not quite 0): s over its 2^t is the sum
            // of e^(z - m), 1 in a row with one logit left.
            bool const nothing = high == -INFINITY, big = isBig(high, c);
            float const rest = big ? 0.0f : fmaf(high, c, offsetOf(high, c));
            float const lnS = high == INFINITY ? 0.0f : logf(s / exp2Approx(rest));
            auto logpOf = [&](float x) { return nothing ? -INFINITY : fmaf(x - high, a.scale, -lnS); };
            if(thread == 0)
            {
                if(a.logp)
                    a.logp[r] = target >= 0 && target < static_cast<int64_t>(a.vocab) ? logpOf(xt) : 0.0f;
                if(a.lse)
                    a.lse[r] = nothing ? -INFINITY : fmaf(high, a.scale, lnS);
                if constexpr(ENT)
                {
                    float const h = lnS - (big ? 0.0f : kLn2 * (u / s - rest));
                    a.entropy[r] = nothing ? 0.0f : !(high < INFINITY) ? NAN : (h < 0.0f ? 0.0f : h);
                }
            }
            if constexpr(TOP)
            {
                fillWithNegInf<S>(row.p, a.vocab, a.top, kept, best);
                if(thread < a.top)
                {
                    unsigned long long const key = best[thread];
                    uint64_t const at = r * a.top + thread;
                    unsigned const index = ~static_cast<unsigned>(key);
                    a.topLogp[at] = logpOf(valueOf(static_cast<unsigned>(key >> 32)));
                    if(a.index64)
                        static_cast<int64_t*>(a.topIndex)[at] = index;
                    else
                        static_cast<int32_t*>(a.topIndex)[at] = static_cast<int32_t>(index);
                }
            }
        }

        template<typename T, int S, int P, bool TOP, bool ENT>
        int launchRows(cudaStream_t stream, unsigned cluster, LogprobArgs const& a)
        {
            uint64_t const teams = Team<S>::perBlock;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = cluster;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(static_cast<unsigned>((a.rows + teams - 1) / teams) * cluster);
            cfg.blockDim = dim3(Team<S>::block);
            cfg.stream = stream;
            cfg.attrs = attr;
            cfg.numAttrs = cluster > 1 ? 1 : 0;
            A3B_CUDA(cudaLaunchKernelEx(&cfg, logprobKernel<T, S, P, TOP, ENT>, a));
            return A3B_OK;
        }

        // The team of a row. Warps that need no barrier are best as long as there are enough of them: it has the fewest
        // warps that make kEnoughWarps of all rows, but not more than a row fills with one tile. Measured on a B200,
        // bf16, 1 / 2 / 4 / 8 warps, in microseconds: 8192 rows of 8192 logits 26 / 28 / 30 / 42; 4096 x 16384
        // 28 / 27 / 28 / 30; 2048 x 50257 46 / 40 / 40 / 43, with 20 alternatives 87 / 77 / 72 / 80. With alternatives a
        // single warp takes rows of one tile only (8192 x 8192 with 5: 52 on one warp, 44 on two; 32768 x 4096 98 / 96).
        // Short rows in great number take a quarter or half of a warp, which spreads what a row costs besides its logits
        // over four or two rows (32768 rows of 257 fp16 with 2 alternatives 18 us, one warp each 31; 500 fp16 24 / 33;
        // 1000 bf16 with 3 38 / 49; but 100 rows of 500 6.9 / 4.2). More alternatives than half the team's threads are
        // badly bounded by its thread maxima. Other rows of up to 64 packs take tiles of two packs a thread, whose kernel
        // has fewer registers (16 / 18 us for 32768 x 257).
        // Few long rows are cut into slices over a cluster, as many as keep three blocks an SM or less (a fourth fits, but more
        // and shorter slices cost more in joining than they gain): 1 / 2 / 4 / 8 slices of 16 rows of 131072 bf16 with 20
        // alternatives 20 / 15 / 11 / 10, of 64 fp32 rows with 5 19 / 15 / 12 / 12, of 100 of them 20 / 17 / 14 / 18, of 64 rows
        // of 50257 bf16 11 / 10 / 8 / 10, of one row of 32000 with 20 8.5 / 7.7 / 7.6 / 8.0 (logits in L2).
        constexpr uint64_t kEnoughWarps = 8192;

        template<typename T>
        int launchLogprob(cudaStream_t stream, DeviceProps const* props, LogprobArgs a)
        {
            uint64_t const packs = a.vocab / PackOf<T>::E;
            auto go = [&](auto size, auto p, unsigned cluster)
            {
                constexpr int S = decltype(size)::value, P = decltype(p)::value;
                // Whole tiles, if the last slice keeps a quarter of one; else equal shares: a slice of a few packs leaves
                // warps without a maximum, and the bound of its alternatives with it (8 rows of 50257 bf16 with 20
                // alternatives 14 us with 138 packs in the last of four slices, 9 with equal ones).
                uint64_t const tile = uint64_t{S} * P, whole = ((packs + cluster - 1) / cluster + tile - 1) / tile * tile;
                uint64_t const share = (cluster - 1) * whole + tile / 4 <= packs ? whole : (packs + cluster - 1) / cluster;
                a.share = static_cast<uint32_t>(share);
                a.tiles = static_cast<uint32_t>(std::max<uint64_t>((share + tile - 1) / tile, 1));
                if(a.top > 0)
                    return a.entropy ? launchRows<T, S, P, true, true>(stream, cluster, a)
                                     : launchRows<T, S, P, true, false>(stream, cluster, a);
                return a.entropy ? launchRows<T, S, P, false, true>(stream, cluster, a)
                                 : launchRows<T, S, P, false, false>(stream, cluster, a);
            };
            using std::integral_constant;
            constexpr integral_constant<int, kPacks> full;
            uint64_t const oneTile = 32 * kPacks; // packs of a warp's tile
            if(a.rows >= kEnoughWarps && packs <= 128 && a.top <= (packs <= 64 ? 4u : 8u))
            {
                if(packs <= 32)
                    return go(integral_constant<int, 8>{}, integral_constant<int, 4>{}, 1u);
                return packs <= 64 ? go(integral_constant<int, 8>{}, full, 1u) : go(integral_constant<int, 16>{}, full, 1u);
            }
            if(packs <= 64)
                return go(integral_constant<int, 32>{}, integral_constant<int, 2>{}, 1u);
            if((a.rows >= kEnoughWarps && a.top == 0) || packs <= oneTile)
                return go(integral_constant<int, 32>{}, full, 1u);
            if(a.rows >= kEnoughWarps / 2 || packs <= 2 * oneTile)
                return go(integral_constant<int, 64>{}, full, 1u);
            if(a.rows >= kEnoughWarps / 4 || packs <= 4 * oneTile)
                return go(integral_constant<int, 128>{}, full, 1u);
            uint64_t const held = static_cast<uint64_t>(props->smCount) * 3; // blocks
            unsigned cluster = 1;
            while(cluster < kMaxCluster && a.rows * cluster * 2 <= held && packs > cluster * 8 * oneTile)
                cluster *= 2;
            return go(integral_constant<int, 256>{}, full, cluster);
        }

        // ------------------------------------------------------------------------------------------- gradient
        struct BackwardArgs
        {
            void const* logits;
            void* grad;
            RowLayout layout;
            RowLayout gradLayout;
            uint32_t total; // chunks of all rows
            uint32_t chunks; // of a row
            uint32_t vocab;
            float scale;
            float factor;     // scale / ln 2, rounded, and what that leaves
            float factorRest;
            int index64;
            void const* targets;
            float const* lse;
            float const* entropy;
            float const* gradLogp;
            float const* gradEntropy;
            float const* gradLse;
        };

        // grad_v = scale (g [v == t] + p_v ((g_lse - g) - g_H (ln p_v + H))). With t = ln p / ln 2 = c x - lse / ln 2, one
        // fused operation, it is 2^t (a + b t), a = scale (g_lse - g - g_H H), b = -scale g_H ln 2. What the roundings of c
        // and lse / ln 2 leave is one number for a row (where p counts, x is near lse / scale): 2^ of it goes into a and b.
        // It grows with lse, and from some 2^30 would leave fp32's range. A row whose |lse| is above 2^24 (a step of it is 2
        // or more: rows at a large mask value and nothing else) has its difference formed from lse itself: scale x rounded to
        // fp32 before lse is taken off, as it was when lse was rounded, so that z <= lse stays true and p <= 1.
        //
        // L threads take a chunk of kBackPacks packs each and need no others: chunks are handed out in the order of
        // memory. Measured on a B200: 4096 x 131072 fp32 624 us, 2048 x 50257 bf16 63 us, HBM-bound. The bound of 40
        // registers (6 blocks of 8 warps an SM) is what took the second one from 148 to 78, the fused exponents the rest.
        constexpr int kBackPacks = 4;

        __device__ __forceinline__ bool isFar(float lse)
        {
            return !(fabsf(lse) <= 0x1p24f);
        }

        template<typename T, int L>
        __global__ void __launch_bounds__(kBlock, 6) logprobBackwardKernel(BackwardArgs a)
        {
            constexpr int E = PackOf<T>::E;
            constexpr uint32_t span = L * kBackPacks;
            uint32_t const id = blockIdx.x * (kBlock / L) + threadIdx.x / L, lane = threadIdx.x & (L - 1u);
            if(id >= a.total)
                return;
            uint32_t const r = id / a.chunks, base = (id - r * a.chunks) * span;
            T const* const row = static_cast<T const*>(a.logits) + a.layout.at(r);
            T* const out = static_cast<T*>(a.grad) + a.gradLayout.at(r);
            // packs on the 16-byte boundaries of the output row, as in the forward pass; the input row may lie differently
            uint32_t const head = min(a.vocab, toBoundary(out));
            uint32_t const packs = (a.vocab - head) / E, tail = a.vocab - head - packs * E;
            bool const alike = (reinterpret_cast<uintptr_t>(row) & 15u) == (reinterpret_cast<uintptr_t>(out) & 15u);

            float const lse = a.lse[r];
            int64_t const target = a.gradLogp ? loadIndex(a.targets, r, a.index64) : -1;
            bool const counts = target >= 0 && target < static_cast<int64_t>(a.vocab);
            bool const nothing = lse == -INFINITY; // every logit is -infinity: a gradient of zeros
            float const g = counts && !nothing ? a.gradLogp[r] : 0.0f;
            float const gl = a.gradLse && !nothing ? a.gradLse[r] : 0.0f;
            float const gh = a.gradEntropy && !nothing ? a.gradEntropy[r] : 0.0f;
            float const h = a.gradEntropy ? a.entropy[r] : 0.0f;
            if(isFar(lse) && !nothing)
            {
                // A branch of its own: sharing the other rows' loads and stores cost those 2 to 4%. Whatever has one writer
                // there has the same one here. With infinite lse the entropy is NaN, but what has no probability has no
                // gradient: it counts as 0, and the infinite logits' own t is NaN.
                float const b = -a.scale * gh, a0 = fmaf(b, lse == INFINITY ? 0.0f : h, a.scale * (gl - g)), own = a.scale * g;
                uint32_t const at = static_cast<uint32_t>(target); // without a token `own` is 0
                auto one = [&](float x, uint32_t v)
                {
                    float const t = maxNan(__fmul_rn(x, a.scale) - lse, -200.0f);
                    float const d = exp2Approx(t * kLog2e) * fmaf(t, b, a0);
                    return v == at ? d + own : d;
                };
                auto gradOf = [&](float2 x, uint32_t v) { return make_float2(one(x.x, v), one(x.y, v + 1)); };
                constexpr int ahead = E == 4 ? 2 : kBackPacks; // loads in flight; 4 cost the other rows of fp32 10%
#pragma unroll 1
                for(int p0 = 0; p0 < kBackPacks; p0 += ahead)
                {
                    unsigned q[ahead][4];
#pragma unroll
                    for(int p = 0; p < ahead; ++p)
                    {
                        uint32_t const k = base + (p0 + p) * L + lane;
                        uint4 v = make_uint4(0u, 0u, 0u, 0u);
                        if(k < packs && alike)
                            v = __ldcs(reinterpret_cast<uint4 const*>(row + head) + k);
                        q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    }
#pragma unroll
                    for(int p = 0; p < ahead; ++p)
                    {
                        uint32_t const k = base + (p0 + p) * L + lane, first = head + k * E;
                        if(k >= packs)
                            break;
                        if(!alike)
                        {
#pragma unroll
                            for(int e = 0; e < E; ++e)
                                PackOf<T>::setRaw(q[p], e, row + first + e);
                        }
#pragma unroll
                        for(int w = 0; w < PackOf<T>::pairs; ++w)
                            PackOf<T>::setPair(q[p], w, gradOf(PackOf<T>::pair(q[p], w), first + 2 * w));
                        __stcs(reinterpret_cast<uint4*>(out + head) + k, make_uint4(q[p][0], q[p][1], q[p][2], q[p][3]));
                    }
                }
                // the elements in front of and behind the packs, by the threads of the row's first chunk
                for(uint32_t j = lane; base == 0 && j < head + tail; j += L)
                {
                    uint32_t const v = j < head ? j : a.vocab - tail + j - head;
                    out[v] = fromFloat<T>(gradOf(make_float2(toFloat(row[v]), 0.0f), v).x);
                }
                return;
            }
            unsigned q[kBackPacks][4];
            if(alike && base + span <= packs)
            {
                auto const* const from = reinterpret_cast<uint4 const*>(row + head) + base + lane;
#pragma unroll
                for(int p = 0; p < kBackPacks; ++p)
                {
                    uint4 const v = __ldcs(from + p * L);
                    q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                }
            }
            else
            {
#pragma unroll
                for(int p = 0; p < kBackPacks; ++p)
                {
                    uint32_t const k = base + p * L + lane;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    T const* const from = row + head + static_cast<uint64_t>(k) * E;
                    if(k < packs && alike)
                        v = __ldcs(reinterpret_cast<uint4 const*>(from));
                    q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    if(k < packs && !alike)
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            PackOf<T>::setRaw(q[p], e, from + e);
                }
            }
            // the elements in front of and behind the packs, up to eight each, by the threads of the row's first chunk
            constexpr int asides = L < 16 ? 16 / L : 1;
            uint32_t aside[asides];
            bool isAside[asides];
            float asideValue[asides];
#pragma unroll
            for(int i = 0; i < asides; ++i)
            {
                uint32_t const j = lane + i * L;
                aside[i] = j < 8 ? j : a.vocab - tail + j - 8;
                isAside[i] = base == 0 && (j < 8 ? j < head : j < 8 + tail);
                asideValue[i] = isAside[i] ? toFloat(row[aside[i]]) : 0.0f;
            }

            // where the target is in this chunk's packs
            uint32_t const place = static_cast<uint32_t>(target) - head, hitPack = place / E - base;
            bool const hit = counts && static_cast<uint32_t>(target) >= head && hitPack < span && place / E < packs
                             && hitPack % L == lane;
            float const hitValue = hit ? toFloat(row[target]) : 0.0f;

            constexpr float log2eRest = 1.92596299e-8f; // 1 / ln 2 - kLog2e
            float const offset = nothing ? 0.0f : -__fmul_rn(lse, kLog2e);
            float const rest
                = nothing ? 0.0f : (-fmaf(lse, kLog2e, offset) - lse * log2eRest) + lse / a.scale * a.factorRest;
            float const up = exp2Approx(rest);
            float const b = -a.scale * gh * kLn2;
            float const a0 = fmaf(b, rest, a.scale * ((gl - g) - gh * h));
            float const ca = a0 * up, cb = b * up;
            float2 const offset2 = make_float2(offset, offset), factor2 = make_float2(a.factor, a.factor);
            float2 const ca2 = make_float2(ca, ca), cb2 = make_float2(cb, cb);
            auto gradOf = [&](float2 x)
            {
                float2 t = fma2(x, factor2, offset2);
                t.x = maxNan(t.x, -200.0f); // 2^-inf times the -inf in the second factor would be NaN
                t.y = maxNan(t.y, -200.0f);
                return mul2(make_float2(exp2Approx(t.x), exp2Approx(t.y)), fma2(t, cb2, ca2));
            };
#pragma unroll
            for(int p = 0; p < kBackPacks; ++p)
            {
                uint32_t const k = base + p * L + lane;
                unsigned o[4];
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                    PackOf<T>::setPair(o, w, gradOf(PackOf<T>::pair(q[p], w)));
                if(k < packs)
                    __stcs(reinterpret_cast<uint4*>(out + head) + k, make_uint4(o[0], o[1], o[2], o[3]));
            }
            if(hit)
                out[target] = fromFloat<T>(gradOf(make_float2(hitValue, 0.0f)).x + a.scale * g);
#pragma unroll
            for(int i = 0; i < asides; ++i)
                if(isAside[i])
                {
                    float const d = gradOf(make_float2(asideValue[i], 0.0f)).x;
                    bool const isTarget = counts && target == static_cast<int64_t>(aside[i]);
                    out[aside[i]] = fromFloat<T>(isTarget ? d + a.scale * g : d);
                }
        }

        template<typename T>
        int launchBackward(cudaStream_t stream, uint64_t rows, BackwardArgs a)
        {
            // Short rows in great number take a quarter of a warp each, as in the forward pass (a whole one / a quarter on
            // a B200: 32768 x 257 fp16 22 / 12 us, 65536 x 64 fp32 31 / 12, 100 x 257 3.4 / 4.0).
            uint64_t const packs = a.vocab / PackOf<T>::E;
            bool const quarter = rows >= kEnoughWarps / 4 && packs <= 8 * kBackPacks;
            uint64_t const span = (quarter ? 8 : 32) * kBackPacks, perBlock = kBlock / (quarter ? 8 : 32);
            uint64_t const chunks = std::max<uint64_t>((packs + span - 1) / span, 1);
            if(rows * chunks > static_cast<uint64_t>(UINT32_MAX) - perBlock)
            {
                setError("%llu rows of %u logits are more than one launch holds",
                         static_cast<unsigned long long>(rows), a.vocab);
                return A3B_ERR_TOO_LARGE;
            }
            a.total = static_cast<uint32_t>(rows * chunks);
            a.chunks = static_cast<uint32_t>(chunks);
            auto const grid = static_cast<unsigned>((a.total + perBlock - 1) / perBlock);
            if(quarter)
                logprobBackwardKernel<T, 8><<<grid, kBlock, 0, stream>>>(a);
            else
                logprobBackwardKernel<T, 32><<<grid, kBlock, 0, stream>>>(a);
            A3B_CHECK_LAUNCH("logprobBackwardKernel");
            return A3B_OK;
        }

        // ------------------------------------------------------------------------------------------ arguments
        int checkRows(
            int dtype,
            void const* logits,
            uint64_t outer,
            uint64_t inner,
            uint64_t vocab,
            double scale,
            int indexDtype)
        {
            A3B_REQUIRE(dtype == A3B_F32 || dtype == A3B_F16 || dtype == A3B_BF16, "logits must be f32, f16 or bf16");
            A3B_REQUIRE(indexDtype == A3B_I32 || indexDtype == A3B_I64, "token indices must be i32 or i64");
            A3B_REQUIRE(vocab > 0, "a row needs at least one logit");
            A3B_REQUIRE(scale >= 0x1p-20 && scale <= 0x1p20, "scale must lie between 2^-20 and 2^20");
            A3B_REQUIRE(outer == 0 || inner <= UINT64_MAX / outer, "rows overflow");
            if(vocab > static_cast<uint64_t>(INT_MAX) - 64 || outer * inner > static_cast<uint64_t>(INT_MAX))
            {
                setError("at most 2^31 - 1 rows and 2^31 - 65 logits a row");
                return A3B_ERR_TOO_LARGE;
            }
            A3B_REQUIRE(logits || outer * inner == 0, "null logits");
            uintptr_t const es = dtype == A3B_F32 ? 4 : 2;
            A3B_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (es - 1)) == 0, "logits are not aligned to their type");
            return A3B_OK;
        }

        bool alignedTo(uintptr_t size, std::initializer_list<void const*> pointers)
        {
            for(void const* p : pointers)
                if(reinterpret_cast<uintptr_t>(p) % size != 0u)
                    return false;
            return true;
        }

        // In 128 bits: strides come from the caller and may be anything.
        using Wide = __int128;

        Wide magnitude(int64_t v)
        {
            return v < 0 ? -static_cast<Wide>(v) : static_cast<Wide>(v);
        }

        // the addresses [lo, hi) that a layout's rows reach
        void extent(void const* base, uint64_t outer, uint64_t inner, uint64_t vocab, int64_t so, int64_t si, int es,
                    Wide* lo, Wide* hi)
        {
            Wide const a = static_cast<Wide>(outer - 1) * so, b = static_cast<Wide>(inner - 1) * si;
            auto const at = static_cast<Wide>(reinterpret_cast<uintptr_t>(base));
            *lo = at + ((a < 0 ? a : 0) + (b < 0 ? b : 0)) * es;
            *hi = at + ((a > 0 ? a : 0) + (b > 0 ? b : 0) + static_cast<Wide>(vocab)) * es;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_token_logprobs(
        a3b_stream_t stream,
        int dtype,
        void const* logits,
        uint64_t outer,
        uint64_t inner,
        uint64_t vocab,
        int64_t outer_stride,
        int64_t inner_stride,
        double scale,
        int index_dtype,
        void const* targets,
        float* logp,
        float* entropy,
        float* lse,
        uint32_t top,
        float* top_logp,
        void* top_index)
    {
        int const rc = checkRows(dtype, logits, outer, inner, vocab, scale, index_dtype);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(top <= static_cast<uint32_t>(kMaxTop), "at most 32 alternatives");
        A3B_REQUIRE(top <= vocab, "more alternatives than logits in a row");
        uint64_t const rows = outer * inner;
        if(rows == 0)
            return A3B_OK;
        A3B_REQUIRE(logp || entropy || lse || top > 0, "nothing to compute: no output is given");
        A3B_REQUIRE(!logp || targets, "log probabilities need targets");
        A3B_REQUIRE(top == 0 || (top_logp && top_index), "null output for the alternatives");
        A3B_REQUIRE(alignedTo(4, {logp, entropy, lse, top_logp})
                        && alignedTo(index_dtype == A3B_I64 ? 8 : 4, {targets, top_index}),
                    "an array is not aligned to its type");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        LogprobArgs a{logits, {static_cast<uint32_t>(inner), outer_stride, inner_stride}, rows, 1u, 0u,
                      static_cast<uint32_t>(vocab), top, static_cast<float>(scale),
                      static_cast<float>(256.0 / (scale * 1.4426950408889634074)), index_dtype == A3B_I64, targets, logp,
                      entropy, lse, top_logp, top_index};
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchLogprob<float>(s, props, a);
        if(dtype == A3B_F16)
            return launchLogprob<__half>(s, props, a);
        return launchLogprob<__nv_bfloat16>(s, props, a);
    }

    int a3b_token_logprobs_backward(
        a3b_stream_t stream,
        int dtype,
        void const* logits,
        uint64_t outer,
        uint64_t inner,
        uint64_t vocab,
        int64_t outer_stride,
        int64_t inner_stride,
        double scale,
        int index_dtype,
        void const* targets,
        float const* lse,
        float const* entropy,
        float const* grad_logp,
        float const* grad_entropy,
        float const* grad_lse,
        void* grad_logits,
        int64_t grad_outer_stride,
        int64_t grad_inner_stride)
    {
        int const rc = checkRows(dtype, logits, outer, inner, vocab, scale, index_dtype);
        if(rc != A3B_OK)
            return rc;
        uint64_t const rows = outer * inner;
        if(rows == 0)
            return A3B_OK;
        A3B_REQUIRE(lse && grad_logits, "null lse or grad_logits");
        A3B_REQUIRE(!grad_logp || targets, "a gradient of the log probabilities needs targets");
        A3B_REQUIRE(!grad_entropy || entropy, "a gradient of the entropy needs the entropy");
        A3B_REQUIRE(alignedTo(4, {lse, entropy, grad_logp, grad_entropy, grad_lse})
                        && alignedTo(index_dtype == A3B_I64 ? 8 : 4, {targets}),
                    "an array is not aligned to its type");
        int const es = dtype == A3B_F32 ? 4 : 2;
        A3B_REQUIRE((reinterpret_cast<uintptr_t>(grad_logits) & static_cast<uintptr_t>(es - 1)) == 0,
                    "grad_logits is not aligned to its type");
        // rows of the gradient may not overlap one another
        Wide const v = static_cast<Wide>(vocab), so = magnitude(grad_outer_stride), si = magnitude(grad_inner_stride);
        A3B_REQUIRE(inner == 1 || si >= v, "rows of grad_logits overlap");
        A3B_REQUIRE(outer == 1 || so >= v, "rows of grad_logits overlap");
        A3B_REQUIRE(outer == 1 || inner == 1 || so >= v + static_cast<Wide>(inner - 1) * si
                        || si >= v + static_cast<Wide>(outer - 1) * so,
                    "rows of grad_logits overlap");
        // in place, or apart from the logits
        if(!(grad_logits == logits && (outer == 1 || grad_outer_stride == outer_stride)
             && (inner == 1 || grad_inner_stride == inner_stride)))
        {
            Wide lo, hi, glo, ghi;
            extent(logits, outer, inner, vocab, outer_stride, inner_stride, es, &lo, &hi);
            extent(grad_logits, outer, inner, vocab, grad_outer_stride, grad_inner_stride, es, &glo, &ghi);
            A3B_REQUIRE(hi <= glo || ghi <= lo,
                        "grad_logits overlaps the logits (only the same rows in place are allowed)");
        }
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        double const factor = scale * 1.4426950408889634074;
        BackwardArgs a{logits, grad_logits, {static_cast<uint32_t>(inner), outer_stride, inner_stride},
                       {static_cast<uint32_t>(inner), grad_outer_stride, grad_inner_stride}, 0u, 1u,
                       static_cast<uint32_t>(vocab), static_cast<float>(scale), static_cast<float>(factor),
                       static_cast<float>(factor - static_cast<float>(factor)), index_dtype == A3B_I64, targets, lse,
                       entropy, grad_logp, grad_entropy, grad_lse};
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchBackward<float>(s, rows, a);
        if(dtype == A3B_F16)
            return launchBackward<__half>(s, rows, a);
        return launchBackward<__nv_bfloat16>(s, rows, a);
    }
}
