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
#include <cfloat>
#include <climits>

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
            uint64_t inner;
            int64_t outerStride;
            int64_t innerStride;

            __device__ __forceinline__ int64_t at(uint64_t r) const
            {
                uint64_t const o = r / inner;
                return static_cast<int64_t>(o) * outerStride + static_cast<int64_t>(r - o * inner) * innerStride;
            }
        };

        struct LogprobArgs
        {
            void const* logits;
            RowLayout layout;
            uint32_t vocab;
            uint32_t top;
            float scale;
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

        // Sums of one share of a row: e^(z - m) and (z - m) / ln 2 * e^(z - m), m = scale * high.
        struct Stats
        {
            float high;
            float s;
            float u;
        };

        __device__ __forceinline__ float finiteOrZero(float high)
        {
            return high == -INFINITY ? 0.0f : high;
        }

        // the sums of `b` moved to the maximum `high` (not below b's) and added to s, u; c = scale / ln 2
        __device__ __forceinline__ void addStats(float high, float c, Stats const& b, float& s, float& u)
        {
            if(b.high == -INFINITY)
                return; // nothing in that share
            float const d = (b.high - finiteOrZero(high)) * c;
            float const f = exp2Approx(d);
            s += f * b.s;
            u += f * fmaf(fmaxf(d, -200.0f), b.s, b.u);
        }

        constexpr int kBlock = 256;
        constexpr int kWarps = kBlock / 32;
        constexpr int kCandidates = kBlock + kMaxTop;

        struct SelectSmem
        {
            unsigned long long keys[kCandidates];
            unsigned long long kept[kMaxTop]; // the best so far, in order
            unsigned bound[kWarps];
            unsigned count;
            unsigned floor; // an element below this order cannot enter `kept`
            unsigned tally[3];
        };

        // One tile of a row in the registers of a block: pack p of thread t is pack base + p * kBlock + t of the row,
        // counted from the 16-byte boundary at or below the row's first element (`lead` elements before it).
        template<typename T>
        struct Tile
        {
            static constexpr int E = PackOf<T>::E;
            unsigned q[kPacks][4];

            // Packs outside [.., end) and the elements outside the row read as -infinity; a pack that the row fills
            // only partly is read element by element.
            __device__ __forceinline__ void load(T const* row, uint32_t vocab, int lead, uint32_t base, uint32_t end)
            {
                T const* const origin = row - lead;
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                {
                    uint32_t const k = base + p * kBlock + threadIdx.x;
                    int64_t const first = static_cast<int64_t>(k) * E - lead;
                    if(k < end && first >= 0 && first + E <= static_cast<int64_t>(vocab))
                    {
                        uint4 const v = __ldcs(reinterpret_cast<uint4 const*>(origin) + k);
                        q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    }
                    else
                    {
                        q[p][0] = q[p][1] = q[p][2] = q[p][3] = PackOf<T>::negInfWord();
                        if(k < end)
                        {
#pragma unroll
                            for(int e = 0; e < E; ++e)
                                if(first + e >= 0 && first + e < static_cast<int64_t>(vocab))
                                    PackOf<T>::setRaw(q[p], e, row + first + e);
                        }
                    }
                }
            }

            // Keeps the compiler from carrying unpacked elements from one use of the tile to the next: unpacking again
            // is an instruction or less an element, the floats of a whole tile are 64 registers.
            __device__ __forceinline__ void fence()
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                    asm volatile("" : "+r"(q[p][0]), "+r"(q[p][1]), "+r"(q[p][2]), "+r"(q[p][3]));
            }

            // f(value, index) for every element of the row that this thread holds
            template<typename F>
            __device__ __forceinline__ void each(uint32_t vocab, int lead, uint32_t base, uint32_t end, F&& f) const
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                {
                    uint32_t const k = base + p * kBlock + threadIdx.x;
                    if(k >= end)
                        continue;
                    int64_t const first = static_cast<int64_t>(k) * E - lead;
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        float2 const v = PackOf<T>::pair(q[p], w);
                        int64_t const i = first + 2 * w;
                        if(i >= 0 && i < static_cast<int64_t>(vocab))
                            f(v.x, static_cast<uint32_t>(i));
                        if(i + 1 >= 0 && i + 1 < static_cast<int64_t>(vocab))
                            f(v.y, static_cast<uint32_t>(i + 1));
                    }
                }
            }
        };

        // how many elements of the tile satisfy `f`, over the block; `turn` counts the calls of one selection
        template<typename T, typename F>
        __device__ __forceinline__ unsigned countIf(
            Tile<T>& t, uint32_t vocab, int lead, uint32_t base, uint32_t end, SelectSmem& s, int& turn, F&& f)
        {
            unsigned n = 0;
            t.fence();
            t.each(vocab, lead, base, end, [&](float x, uint32_t i) { n += f(orderOf(x), i) ? 1u : 0u; });
            n = __reduce_add_sync(kFullMask, n);
            if((threadIdx.x & 31) == 0)
                atomicAdd(&s.tally[turn % 3], n);
            if(threadIdx.x == 0)
                s.tally[(turn + 1) % 3] = 0u; // nobody reads it any more: the last reads were two calls ago
            __syncthreads();
            unsigned const total = s.tally[turn % 3];
            ++turn;
            return total;
        }

        // Adds the tile to the selection of the row's `top` largest elements (ties to the lower index). s.kept holds
        // `kept` keys in order before and the returned number after; the block is synchronised on return.
        //
        // Every warp's need-th largest thread maximum, need = ceil(top / warps), is reached by `need` elements of that
        // warp; so at least `top` elements of the tile reach the smallest of these bounds, and no element below it can
        // be among the `top` largest. For logits in no particular order a few dozen elements of a tile pass. They are
        // collected in shared memory (their order there does not matter: the keys are distinct) and ranked by
        // counting. Where more pass than there is room for (many equal values), the tile's `top` are found by
        // bisection over the values, then over the index among equal ones.
        template<typename T>
        __device__ __forceinline__ unsigned selectTile(
            Tile<T>& t,
            float threadMax,
            uint32_t vocab,
            int lead,
            uint32_t base,
            uint32_t end,
            unsigned top,
            unsigned kept,
            SelectSmem& s)
        {
            int const lane = threadIdx.x & 31;
            unsigned const mine = orderOf(threadMax);
            unsigned bound = 0, left = mine;
            for(unsigned i = 0; i < (top + kWarps - 1) / kWarps; ++i)
            {
                bound = __reduce_max_sync(kFullMask, left);
                if(lane == __ffs(static_cast<int>(__ballot_sync(kFullMask, left == bound))) - 1)
                    left = 0u;
            }
            if(lane == 0)
                s.bound[threadIdx.x >> 5] = bound;
            if(threadIdx.x < kept)
                s.keys[threadIdx.x] = s.kept[threadIdx.x];
            if(threadIdx.x == 0)
                s.count = kept;
            __syncthreads();
#pragma unroll
            for(int w = 0; w < kWarps; ++w)
                bound = min(bound, s.bound[w]);
            if(kept == top)
                bound = max(bound, s.floor);

            auto push = [&](float x, uint32_t i)
            {
                unsigned const at = atomicAdd(&s.count, 1u);
                if(at < kCandidates)
                    s.keys[at] = keyOf(orderOf(x), i);
            };
            if(mine >= bound)
                t.each(vocab, lead, base, end, [&](float x, uint32_t i) {
                    if(orderOf(x) >= bound)
                        push(x, i);
                });
            __syncthreads();
            t.fence();
            unsigned n = s.count;
            if(n > kCandidates)
            {
                // more than `top` elements reach `bound`: the largest value that `top` of them reach
                __syncthreads(); // every thread has read the count
                if(threadIdx.x == 0)
                {
                    s.count = kept;
                    s.tally[0] = 0u;
                }
                __syncthreads();
                int turn = 0;
                auto count = [&](auto&& f) { return countIf(t, vocab, lead, base, end, s, turn, f); };
                unsigned long long lo = bound, hi = 0x100000000ull; // reached by `top` elements / by fewer
                if(count([&](unsigned o, uint32_t) { return o > bound; }) < top)
                    hi = lo + 1;
                while(hi - lo > 1)
                {
                    unsigned long long const mid = lo + (hi - lo) / 2;
                    if(count([&](unsigned o, uint32_t) { return o >= mid; }) >= top)
                        lo = mid;
                    else
                        hi = mid;
                }
                // of the elements with that value, the first ones, up to the index that makes `top` in all
                unsigned const value = static_cast<unsigned>(lo);
                unsigned const above = count([&](unsigned o, uint32_t) { return o > value; });
                uint32_t a = 0, b = vocab - 1;
                while(a < b)
                {
                    uint32_t const mid = a + (b - a) / 2;
                    if(above + count([&](unsigned o, uint32_t i) { return o == value && i <= mid; }) >= top)
                        b = mid;
                    else
                        a = mid + 1;
                }
                t.each(vocab, lead, base, end, [&](float x, uint32_t i) {
                    unsigned const o = orderOf(x);
                    if(o > value || (o == value && i <= a))
                        push(x, i);
                });
                __syncthreads();
                n = s.count;
            }
            if(n == kept)
                return kept; // nothing new (a thread already in the next tile stores this same number in s.count)
            for(unsigned i = threadIdx.x; i < n; i += kBlock)
            {
                unsigned long long const key = s.keys[i];
                unsigned rank = 0;
                for(unsigned j = 0; j < n; ++j)
                    rank += s.keys[j] > key ? 1u : 0u;
                if(rank < top)
                    s.kept[rank] = key;
                if(rank == top - 1)
                {
                    unsigned const o = static_cast<unsigned>(key >> 32);
                    s.floor = o == 0xffffffffu ? o : o + 1u; // later tiles have higher indices: equal is not enough
                }
            }
            __syncthreads();
            return min(n, top);
        }

        template<typename T, bool TOP, bool ENT>
        __global__ void __launch_bounds__(kBlock) logprobKernel(LogprobArgs a)
        {
            __shared__ Stats stats[kWarps];
            __shared__ SelectSmem sel;
            uint64_t const r = blockIdx.x;
            T const* const row = static_cast<T const*>(a.logits) + a.layout.at(r);
            int const lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
            uint32_t const packs
                = static_cast<uint32_t>((static_cast<uint64_t>(lead) + a.vocab + Tile<T>::E - 1) / Tile<T>::E);
            float const c = a.scale * kLog2e;
            int64_t const target = a.logp ? loadIndex(a.targets, r, a.index64) : -1;
            bool const counts = target >= 0 && target < static_cast<int64_t>(a.vocab);
            float const xt = counts ? toFloat(row[target]) : 0.0f;

            float high = -INFINITY;
            float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
            unsigned kept = 0;
            for(uint32_t base = 0; base < packs; base += kBlock * kPacks)
            {
                Tile<T> t;
                t.load(row, a.vocab, lead, base, packs);
                float threadMax = -INFINITY;
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        float2 const v = PackOf<T>::pair(t.q[p], w);
                        threadMax = maxNan(threadMax, maxNan(v.x, v.y));
                    }
                t.fence();
                // the warp's running maximum, and its sums moved there
                float const to = maxNan(high, warpMaxNan(threadMax));
                if(to != high)
                {
                    Stats const x{high, s2.x, u2.x}, y{high, s2.y, u2.y};
                    s2 = u2 = make_float2(0.0f, 0.0f);
                    addStats(to, c, x, s2.x, u2.x);
                    addStats(to, c, y, s2.y, u2.y);
                    high = to;
                }
                float const off = -finiteOrZero(high);
                float2 const off2 = make_float2(off, off), c2 = make_float2(c, c);
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        float2 d = mul2(add2(PackOf<T>::pair(t.q[p], w), off2), c2);
                        if constexpr(ENT)
                        {
                            // -infinity times the zero that it gives would be NaN; 2^-200 is zero in fp32
                            d.x = maxNan(d.x, -200.0f);
                            d.y = maxNan(d.y, -200.0f);
                        }
                        float2 const e = make_float2(exp2Approx(d.x), exp2Approx(d.y));
                        s2 = add2(s2, e);
                        if constexpr(ENT)
                            u2 = fma2(d, e, u2);
                    }
                t.fence();
                if constexpr(TOP)
                    kept = selectTile(t, threadMax, a.vocab, lead, base, packs, a.top, kept, sel);
            }
            float s = s2.x + s2.y, u = u2.x + u2.y;
#pragma unroll
            for(int m = 16; m > 0; m >>= 1)
            {
                s += __shfl_xor_sync(kFullMask, s, m);
                u += __shfl_xor_sync(kFullMask, u, m);
            }
            if((threadIdx.x & 31) == 0)
                stats[threadIdx.x >> 5] = Stats{high, s, u};
            __syncthreads();
            if(threadIdx.x >= 32)
                return;
            high = stats[0].high;
#pragma unroll
            for(int w = 1; w < kWarps; ++w)
                high = maxNan(high, stats[w].high);
            s = u = 0.0f;
#pragma unroll
            for(int w = 0; w < kWarps; ++w)
                addStats(high, c, stats[w], s, u);

            bool const nothing = high == -INFINITY;
            float const lnS = high == INFINITY ? 0.0f : logf(s);
            auto logpOf = [&](float x) { return nothing ? -INFINITY : fmaf(x - high, a.scale, -lnS); };
            if(threadIdx.x == 0)
            {
                if(a.logp)
                    a.logp[r] = counts ? logpOf(xt) : 0.0f;
                if(a.lse)
                    a.lse[r] = nothing ? -INFINITY : fmaf(high, a.scale, lnS);
                if constexpr(ENT)
                {
                    float const h = lnS - kLn2 * (u / s);
                    a.entropy[r] = nothing ? 0.0f : (high == INFINITY ? NAN : (h < 0.0f ? 0.0f : h));
                }
            }
            if constexpr(TOP)
                if(threadIdx.x < a.top)
                {
                    unsigned long long const key = sel.kept[threadIdx.x];
                    uint64_t const at = r * a.top + threadIdx.x;
                    unsigned const index = ~static_cast<unsigned>(key);
                    a.topLogp[at] = logpOf(valueOf(static_cast<unsigned>(key >> 32)));
                    if(a.index64)
                        static_cast<int64_t*>(a.topIndex)[at] = index;
                    else
                        static_cast<int32_t*>(a.topIndex)[at] = static_cast<int32_t>(index);
                }
        }

        template<typename T>
        int launchLogprob(cudaStream_t stream, uint64_t rows, LogprobArgs const& a)
        {
            auto const grid = static_cast<unsigned>(rows);
            if(a.top > 0)
            {
                if(a.entropy)
                    logprobKernel<T, true, true><<<grid, kBlock, 0, stream>>>(a);
                else
                    logprobKernel<T, true, false><<<grid, kBlock, 0, stream>>>(a);
            }
            else if(a.entropy)
                logprobKernel<T, false, true><<<grid, kBlock, 0, stream>>>(a);
            else
                logprobKernel<T, false, false><<<grid, kBlock, 0, stream>>>(a);
            A3B_CHECK_LAUNCH("logprobKernel");
            return A3B_OK;
        }

        // ------------------------------------------------------------------------------------------- gradient
        struct BackwardArgs
        {
            void const* logits;
            void* grad;
            RowLayout layout;
            RowLayout gradLayout;
            uint32_t vocab;
            uint32_t chunks; // blocks per row
            float scale;
            int index64;
            void const* targets;
            float const* lse;
            float const* entropy;
            float const* gradLogp;
            float const* gradEntropy;
            float const* gradLse;
        };

        // dx_v = scale (g [v == t] + p_v ((g_lse - g) - g_H (logp_v + H))), p_v = e^(logp_v): with t = logp / ln 2,
        // p (a + b t), a = scale (g_lse - g - g_H H), b = -scale g_H ln 2.
        constexpr int kBackPacks = 4;

        template<typename T>
        __global__ void __launch_bounds__(kBlock) logprobBackwardKernel(BackwardArgs a)
        {
            constexpr int E = PackOf<T>::E;
            uint64_t const r = blockIdx.x / a.chunks;
            uint32_t const chunk = blockIdx.x - static_cast<uint32_t>(r * a.chunks);
            T const* const row = static_cast<T const*>(a.logits) + a.layout.at(r);
            T* const out = static_cast<T*>(a.grad) + a.gradLayout.at(r);
            // packs on the 16-byte boundaries of the output row; the input row may lie differently
            int const lead = static_cast<int>((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T));
            bool const alike = (reinterpret_cast<uintptr_t>(row) & 15u) == (reinterpret_cast<uintptr_t>(out) & 15u);

            float const lse = a.lse[r];
            int64_t const target = a.gradLogp ? loadIndex(a.targets, r, a.index64) : -1;
            bool const counts = target >= 0 && target < static_cast<int64_t>(a.vocab);
            bool const nothing = lse == -INFINITY; // every logit is -infinity: a gradient of zeros
            float const g = counts && !nothing ? a.gradLogp[r] : 0.0f;
            float const gl = a.gradLse && !nothing ? a.gradLse[r] : 0.0f;
            float const gh = a.gradEntropy && !nothing ? a.gradEntropy[r] : 0.0f;
            float const h = a.gradEntropy ? a.entropy[r] : 0.0f;
            float const ca = a.scale * ((gl - g) - gh * h), cb = -a.scale * gh * kLn2;
            float const atTarget = a.scale * g;
            float const off = nothing ? 0.0f : -lse;
            float2 const off2 = make_float2(off, off), sc2 = make_float2(a.scale, a.scale);
            float2 const l2 = make_float2(kLog2e, kLog2e), ca2 = make_float2(ca, ca), cb2 = make_float2(cb, cb);

            uint32_t const first = chunk * (kBlock * kBackPacks) + threadIdx.x;
            unsigned q[kBackPacks][4];
            auto bounds = [&](int p, int64_t& i) -> bool
            {
                i = static_cast<int64_t>(first + p * kBlock) * E - lead;
                return i >= 0 && i + E <= static_cast<int64_t>(a.vocab);
            };
#pragma unroll
            for(int p = 0; p < kBackPacks; ++p)
            {
                int64_t i;
                if(bounds(p, i) && alike)
                {
                    uint4 const v = __ldcs(reinterpret_cast<uint4 const*>(row + i));
                    q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                }
                else
                {
                    q[p][0] = q[p][1] = q[p][2] = q[p][3] = PackOf<T>::negInfWord();
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        if(i + e >= 0 && i + e < static_cast<int64_t>(a.vocab))
                            PackOf<T>::setRaw(q[p], e, row + i + e);
                }
            }
#pragma unroll
            for(int p = 0; p < kBackPacks; ++p)
            {
                int64_t i;
                bool const whole = bounds(p, i);
                unsigned o[4];
                bool const hit = counts && target >= i && target < i + E;
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                {
                    float2 t = mul2(fma2(PackOf<T>::pair(q[p], w), sc2, off2), l2);
                    t.x = maxNan(t.x, -200.0f); // e^-inf times the -inf in the second factor would be NaN
                    t.y = maxNan(t.y, -200.0f);
                    float2 const e = make_float2(exp2Approx(t.x), exp2Approx(t.y));
                    float2 d = mul2(e, fma2(t, cb2, ca2));
                    if(hit)
                    {
                        d.x += target == i + 2 * w ? atTarget : 0.0f;
                        d.y += target == i + 2 * w + 1 ? atTarget : 0.0f;
                    }
                    PackOf<T>::setPair(o, w, d);
                }
                if(whole)
                    __stcs(reinterpret_cast<uint4*>(out + i), make_uint4(o[0], o[1], o[2], o[3]));
                else
                {
#pragma unroll
                    for(int e = 0; e < E; ++e)
                        if(i + e >= 0 && i + e < static_cast<int64_t>(a.vocab))
                            PackOf<T>::storeRaw(o, e, out + i + e);
                }
            }
        }

        template<typename T>
        int launchBackward(cudaStream_t stream, uint64_t rows, BackwardArgs a)
        {
            constexpr uint64_t E = PackOf<T>::E;
            // room for a row that starts just below a 16-byte boundary
            uint64_t const packs = (a.vocab + E - 1 + E - 1) / E;
            a.chunks = static_cast<uint32_t>((packs + kBlock * kBackPacks - 1) / (kBlock * kBackPacks));
            uint64_t const grid = rows * a.chunks;
            if(grid > static_cast<uint64_t>(INT_MAX))
            {
                setError("%llu rows of %u logits are more than one launch holds",
                         static_cast<unsigned long long>(rows), a.vocab);
                return A3B_ERR_TOO_LARGE;
            }
            logprobBackwardKernel<T><<<static_cast<unsigned>(grid), kBlock, 0, stream>>>(a);
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
            A3B_REQUIRE(scale > 0.0 && scale <= static_cast<double>(FLT_MAX), "scale must be positive and finite");
            A3B_REQUIRE(static_cast<float>(scale) > 0.0f, "scale is too small for fp32");
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
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        LogprobArgs a{logits, {inner, outer_stride, inner_stride}, static_cast<uint32_t>(vocab), top,
                      static_cast<float>(scale), index_dtype == A3B_I64, targets, logp, entropy, lse, top_logp,
                      top_index};
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchLogprob<float>(s, rows, a);
        if(dtype == A3B_F16)
            return launchLogprob<__half>(s, rows, a);
        return launchLogprob<__nv_bfloat16>(s, rows, a);
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
        BackwardArgs a{logits, grad_logits, {inner, outer_stride, inner_stride},
                       {inner, grad_outer_stride, grad_inner_stride}, static_cast<uint32_t>(vocab), 1u,
                       static_cast<float>(scale), index_dtype == A3B_I64, targets, lse, entropy, grad_logp,
                       grad_entropy, grad_lse};
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchBackward<float>(s, rows, a);
        if(dtype == A3B_F16)
            return launchBackward<__half>(s, rows, a);
        return launchBackward<__nv_bfloat16>(s, rows, a);
    }
}
