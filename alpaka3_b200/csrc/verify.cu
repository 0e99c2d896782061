// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   p_v = e^(scale z_v - lse),  q_v = e^(draft_scale z'_v - lse')   (or q = 1 at the drafted token alone)
//   draft i stands while u_i q(t_i) < p(t_i);  at the first that does not, the token is drawn from (p - q)+, and behind
//   drafts that all stand from p: the first of exponential clocks with these rates, argmax of rate_v / noise_v.
//
// Every token that comes out is what the formula gives in 64 bits for these inputs, at the cost of 32: in fp32 every
// probability and quotient has an interval that holds its true value, and only what intervals cannot tell apart (drafts next
// to the border, quotients next to the largest) is computed again in fp64; mostly that is nothing.
//
// As (p - q)+ <= p, a token can only win if p_v / noise_v reaches the best lower end known so far. So the draw reads one row
// of the target and one of the noise, tests p_v against a product, without a division, and reads of the draft's row only what
// stands where that test passes (a few dozen tokens). It is bound by memory where sequences are many, by latency where they
// are few: a cluster of blocks shares one sequence.
#include <algorithm>

#include "layout.cuh"
#include "rows.cuh"

namespace a3b
{
    namespace
    {
        constexpr int kThreads = 512;

        struct VerifyArgs
        {
            void const* logits; // null: only greedy sequences
            RowStep ls;
            float const* lse;
            void const* draft; // null: the drafts were certain
            RowStep ds;
            float const* draftLse;
            void const* drafts;
            void const* top; // null: no greedy sequences
            float const* uniform;
            float const* noise;
            int64_t noiseStride;
            void* tokens;
            void* accepted;
            uint32_t batch, length, vocab; // length: drafts a sequence
            bool wide; // int64 tokens
            double scale, draftScale;

            __device__ __forceinline__ int64_t index(void const* p, size_t i) const
            {
                return wide ? static_cast<int64_t const*>(p)[i] : static_cast<int32_t const*>(p)[i];
            }
            __device__ __forceinline__ void put(void* p, size_t i, int64_t v) const
            {
                if(wide)
                    static_cast<int64_t*>(p)[i] = v;
                else
                    static_cast<int32_t*>(p)[i] = static_cast<int32_t>(v);
            }
            __device__ __forceinline__ bool known(int64_t t) const
            {
                return t >= 0 && t < static_cast<int64_t>(vocab);
            }
        };

        constexpr double kLog2e = 1.4426950408889634074;

        // What the fp32 pass keeps: the largest lower end and the largest upper end.
        struct Ends
        {
            float low, high;
        };

        // One row's probability in fp32: 2^(c z - l). The factor and l are rounded and the sum is: with |c z| <= |l| + 160
        // wherever the result is a normal number, the exponent is off by at most 2^-24 (2 |l| + 320), so the result by
        // 2^-23 (|l| + 160) of itself, beside two units of ex2.approx. `off` is four times that: it also holds
        // the reciprocal's and the last roundings. Beyond |l| = 2^20 the error is no longer small (`far`).
        struct Rough
        {
            float c, l, off;

            __device__ __forceinline__ Rough(double scale, float lse)
                : c(static_cast<float>(scale * kLog2e))
                , l(static_cast<float>(lse * kLog2e))
                , off(0x1p-21f * (fabsf(l) + 160.f) + 0x1p-20f)
            {
            }
            __device__ __forceinline__ float operator()(float z) const
            {
                return exp2Approx(fmaf(c, z, -l));
            }
            __device__ __forceinline__ bool far() const
            {
                return fabsf(l) > 0x1p20f;
            }
            // the interval of (this row's probability - b) / noise
            __device__ __forceinline__ void widen(float z, float b, float noise, float off, Ends* ends) const
            {
                float const a = (*this)(z);
                float r;
                asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(noise));
                r = noise < 0.f ? NAN : r; // no part: two negative factors would make an end that nothing reaches
                // what flushed to zero counts as up to fp32's least normal numbers
                float const rate = a - b, wide = fmaf(off, a + b, 0x1p-125f);
                // fmax drops NaN: an element with one takes no part
                ends->low = fmaxf(ends->low, (rate - wide) * r);
                ends->high = fmaxf(ends->high, (rate + wide) * r);
            }
        };

        __device__ __noinline__ double exactly(double scale, float z, float lse)
        {
            // Not fused: the product has the rounding of a formula in 64-bit steps, so that far masked logits, whose product is off by
            // more than lse is small, give its probabilities, and equal exponents are equal.
            return exp(__dsub_rn(__dmul_rn(scale, static_cast<double>(z)), static_cast<double>(lse)));
        }

        // The scores of a row without a rate, and of one with rates but no noise they could be divided by; what can be drawn has
        // a score of 0 or more.
        constexpr double kNoRate = -1., kNoClock = -0.5;

        struct Best
        {
            double score;
            uint32_t index;

            static __device__ __forceinline__ Best none()
            {
                return {kNoRate, UINT32_MAX};
            }

            // larger, or as large and further left
            __device__ __forceinline__ void take(double s, uint32_t i)
            {
                if(s > score || (s == score && i < index))
                {
                    score = s;
                    index = i;
                }
            }
        };

        __device__ __forceinline__ Best warpBest(Best b)
        {
#pragma unroll
            for(int d = 16; d > 0; d /= 2)
            {
                double const s = __shfl_xor_sync(kFullMask, b.score, d);
                uint32_t const i = __shfl_xor_sync(kFullMask, b.index, d);
                b.take(s, i);
            }
            return b;
        }

        // Whether a draft stands, u q < p: by intervals in fp32 where they lie apart, else in 64 bits.
        __device__ __forceinline__ bool stands(VerifyArgs const& a, float z, float lse, bool other, float y, float draftLse, float u)
        {
            Rough const p(a.scale, lse), q(a.draftScale, draftLse);
            float const have = p(z), need = u * (other ? q(y) : 1.f);
            float const wide = fmaf(other ? fmaxf(p.off, q.off) : p.off, have + need, 0x1p-125f);
            if(!p.far() && !(other && q.far()))
            {
                if(need + wide < have)
                    return true;
                if(need > have + wide)
                    return false;
            }
            return static_cast<double>(u) * (other ? exactly(a.draftScale, y, draftLse) : 1.) < exactly(a.scale, z, lse);
        }

        // How many drafts stand; every thread of the block gets the same answer.
        template<typename T>
        __device__ __forceinline__ uint32_t accepted(VerifyArgs const& a, uint32_t b, bool* refused)
        {
            // each warp on its own: 32 drafts at a time
            uint32_t const lane = threadIdx.x % 32;
            size_t const at = static_cast<size_t>(b) * a.length;
            for(uint32_t first = 0; first < a.length; first += 32)
            {
                uint32_t const i = first + lane;
                int64_t const t = i < a.length ? a.index(a.drafts, at + i) : -1;
                bool const known = a.known(t);
                bool yes = false;
                if(known)
                {
                    T const* row = static_cast<T const*>(a.logits) + static_cast<int64_t>(b) * a.ls.outer
                                   + static_cast<int64_t>(i) * a.ls.step;
                    float const z = toFloat(row[t]), lse = a.lse[at + b + i], u = a.uniform[at + i];
                    float y = 0.f, draftLse = 0.f;
                    if(a.draft)
                    {
                        T const* other = static_cast<T const*>(a.draft) + static_cast<int64_t>(b) * a.ds.outer
                                         + static_cast<int64_t>(i) * a.ds.step;
                        y = toFloat(other[t]);
                        draftLse = a.draftLse[at + i];
                    }
                    yes = stands(a, z, lse, a.draft != nullptr, y, draftLse, u);
                }
                unsigned const all = __ballot_sync(kFullMask, yes), some = __ballot_sync(kFullMask, known);
                if(all != kFullMask)
                {
                    uint32_t const n = __ffs(~all) - 1;
                    *refused = (some >> n) & 1u;
                    return first + n;
                }
            }
            *refused = false;
            return a.length;
        }

        // E neighbouring logits, or single ones
        template<typename T, int E>
        struct Lot
        {
            static constexpr int words = E == 1 ? 1 : 4;
            unsigned w[words];

            __device__ __forceinline__ void load(T const* row, uint32_t k)
            {
                if constexpr(E > 1)
                {
                    uint4 const v = *reinterpret_cast<uint4 const*>(row + static_cast<size_t>(k) * E);
                    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                }
                else if constexpr(sizeof(T) == 4)
                    w[0] = *reinterpret_cast<unsigned const*>(row + k);
                else
                    w[0] = *reinterpret_cast<unsigned short const*>(row + k);
            }
            __device__ __forceinline__ void unpack(float* v) const
            {
                if constexpr(E == 1 && std::is_same_v<T, float>)
                    v[0] = __uint_as_float(w[0]);
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
        };

        template<int E>
        __device__ __forceinline__ void loadNoise(float* noise, float const* clock, uint32_t k)
        {
            if constexpr(E == 1)
                noise[0] = clock[k];
            else
#pragma unroll
                for(int e = 0; e < E; e += 4)
                {
                    float4 const f = *reinterpret_cast<float4 const*>(clock + static_cast<size_t>(k) * E + e);
                    noise[e] = f.x, noise[e + 1] = f.y, noise[e + 2] = f.z, noise[e + 3] = f.w;
                }
        }

        constexpr uint32_t kList = 1024;

        // This thread's lots first, first + kThreads, ...: tokens with p / noise >= least go to the list. U lots are loaded
        // together, without conditions between the loads: 64 x 131072 bf16 takes 16.3 us with two packs together, 17.1 with
        // one (in blocks of 256 threads 17.5, 18.8, and 18.4 with three); 256 x 50257 fp32, single tokens, with eight, four
        // and twelve 31.6, 35.9 and 39 (spills). Stages in shared memory filled by bulk copies took 26 and 39 (a barrier a
        // stage), noise brought into L2 while the drafts are tested 5% more.
        template<typename T, int E, int U>
        __device__ __forceinline__ void scan(T const* row, float const* clock, uint32_t first, uint32_t end, Rough const& p, float least,
                                             uint32_t* list, unsigned* listed)
        {
            float const more = 1.f + p.off;
            auto test = [&](Lot<T, E> const& t, float const* noise, uint32_t k)
            {
                float z[E];
                t.unpack(z);
                unsigned pass = 0;
#pragma unroll
                for(int e = 0; e < E; ++e)
                    pass |= fmaf(p(z[e]), more, 0x1p-125f) >= least * noise[e] ? 1u << e : 0u; // not where either is NaN
                while(pass)
                {
                    unsigned const e = __ffs(pass) - 1, at = atomicAdd(listed, 1u);
                    pass &= pass - 1;
                    if(at < kList)
                        list[at] = k * E + e;
                }
            };
            uint32_t k = first;
            if constexpr(U > 1)
            {
#pragma unroll 1
                for(; k + (U - 1) * kThreads < end; k += U * kThreads)
                {
                    Lot<T, E> t[U];
                    float noise[U][E];
#pragma unroll
                    for(int u = 0; u < U; ++u)
                    {
                        t[u].load(row, k + u * kThreads);
                        loadNoise<E>(noise[u], clock, k + u * kThreads);
                    }
#pragma unroll
                    for(int u = 0; u < U; ++u)
                        test(t[u], noise[u], k + u * kThreads);
                }
            }
#pragma unroll 1
            for(; k < end; k += kThreads)
            {
                Lot<T, E> t;
                float noise[E];
                t.load(row, k);
                loadNoise<E>(noise, clock, k);
                test(t, noise, k);
            }
        }

        // token i in 64 bits
        template<typename T>
        __device__ __forceinline__ void again(VerifyArgs const& a, T const* row, T const* other, float const* clock, uint32_t certain,
                                              float lse, float draftLse, uint32_t i, Best* best)
        {
            double rate = exactly(a.scale, toFloat(row[i]), lse);
            if(other)
                rate -= exactly(a.draftScale, toFloat(other[i]), draftLse);
            else if(i == certain)
                rate -= 1.;
            if(rate > 0.)
            {
                double const score = rate / static_cast<double>(clock[i]);
                if(score >= 0.)
                    best->take(score, i);
                else // negative noise or NaN
                    best->take(kNoClock, UINT32_MAX);
            }
        }

        constexpr uint32_t kReach = 64;

        // Packed: every row of logits, draft and noise begins at 16 bytes.
        template<typename T, bool Packed>
        __global__ void __launch_bounds__(kThreads, 2) verifyKernel(VerifyArgs a)
        {
            constexpr int E = PackOf<T>::E, kWarps = kThreads / 32;
            __shared__ float lows[kWarps];
            __shared__ float blockLow;
            __shared__ Best bests[kWarps];
            __shared__ Best blockBest;
            __shared__ uint32_t list[kList];
            __shared__ unsigned listed;
            __shared__ bool blockFull;
            __shared__ uint32_t found[kReach]; // of the cluster's first block: tokens whose interval reaches the best lower end
            __shared__ unsigned founds;
            unsigned const rank = clusterRank(), blocks = clusterBlocks();
            uint32_t const b = blockIdx.x / blocks, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
            size_t const at = static_cast<size_t>(b) * a.length, to = at + b;

            if(a.top && (!a.logits || a.known(a.index(a.top, to))))
            {
                // a greedy sequence: no random numbers; the whole cluster takes this way
                if(rank == 0 && warp == 0)
                {
                    uint32_t n = a.length;
                    for(uint32_t first = 0; first < a.length; first += 32)
                    {
                        uint32_t const i = first + lane;
                        int64_t const t = i < a.length ? a.index(a.drafts, at + i) : -1;
                        unsigned const yes = __ballot_sync(kFullMask, a.known(t) && t == a.index(a.top, to + min(i, a.length)));
                        if(yes != kFullMask)
                        {
                            n = first + __ffs(~yes) - 1;
                            break;
                        }
                    }
                    for(uint32_t i = lane; i <= a.length; i += 32)
                    {
                        int64_t const top = a.index(a.top, to + i);
                        a.put(a.tokens, to + i, i > n ? -1 : i == n ? (a.known(top) ? top : -1) : a.index(a.drafts, at + i));
                    }
                    if(lane == 0)
                        a.put(a.accepted, b, n);
                }
                return;
            }

            // The block's share of the vocabulary: lots [low, high) of E tokens, and behind the last lot single ones.
            uint32_t const lots = Packed ? a.vocab / E : 0, per = (lots + blocks - 1) / blocks;
            uint32_t const low = min(rank * per, lots), high = min(low + per, lots);
            uint32_t const ones = a.vocab - lots * E, onesPer = (ones + blocks - 1) / blocks;
            uint32_t const oneLow = lots * E + min(rank * onesPer, ones), oneHigh = min(oneLow + onesPer, a.vocab);
            float const* clock = a.noise + static_cast<int64_t>(b) * a.noiseStride;
            if(tid == 0)
                founds = 0;

            bool refused = false;
            uint32_t const n = accepted<T>(a, b, &refused);
            T const* row = static_cast<T const*>(a.logits) + static_cast<int64_t>(b) * a.ls.outer + static_cast<int64_t>(n) * a.ls.step;
            float const lse = a.lse[to + n];
            Rough const p(a.scale, lse);
            uint32_t drawn = UINT32_MAX;
            bool certainly = false;
            // once with what the draft took away; if that leaves nothing, once more without
            for(int turn = refused ? 0 : 1; turn < 2; ++turn)
            {
                T const* other = nullptr;
                uint32_t certain = UINT32_MAX;
                float draftLse = 0.f;
                if(turn == 0)
                {
                    if(a.draft)
                    {
                        other = static_cast<T const*>(a.draft) + static_cast<int64_t>(b) * a.ds.outer
                                + static_cast<int64_t>(n) * a.ds.step;
                        draftLse = a.draftLse[at + n];
                    }
                    else
                        certain = static_cast<uint32_t>(a.index(a.drafts, at + n));
                }
                Rough const q(a.draftScale, draftLse);
                bool const far = p.far() || q.far(); // then every token is computed in 64 bits
                float const off = other ? fmaxf(p.off, q.off) : p.off;
                auto interval = [&](uint32_t i)
                {
                    Ends one{-INFINITY, -INFINITY};
                    p.widen(toFloat(row[i]), other ? q(toFloat(other[i])) : i == certain ? 1.f : 0.f, clock[i], off, &one);
                    return one;
                };
                auto blockMax = [&](float v)
                {
#pragma unroll
                    for(int d = 16; d > 0; d /= 2)
                        v = fmaxf(v, __shfl_xor_sync(kFullMask, v, d));
                    if(lane == 0)
                        lows[warp] = v;
                    __syncthreads();
#pragma unroll
                    for(int w = 0; w < kWarps; ++w)
                        v = fmaxf(v, lows[w]);
                    __syncthreads(); // `lows` may be written again
                    return v;
                };
                float least = 0.f, upper[kList / kThreads];
                bool full = far;
                if(!far)
                {
                    // a first bound from the first lot of each thread, or its first four tokens
                    Ends ends{-INFINITY, -INFINITY};
                    if(Packed && low + tid < high)
                    {
                        Lot<T, E> t, s;
                        float z[E], y[E], noise[E];
                        t.load(row, low + tid);
                        if(other)
                            s.load(other, low + tid);
                        loadNoise<E>(noise, clock, low + tid);
                        t.unpack(z);
                        if(other)
                            s.unpack(y);
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            p.widen(z[e], other ? q(y[e]) : (low + tid) * E + e == certain ? 1.f : 0.f, noise[e], off, &ends);
                    }
                    else if(!Packed)
#pragma unroll
                        for(int u = 0; u < 4; ++u)
                            if(uint32_t const i = oneLow + u * kThreads + tid; i < oneHigh)
                                ends.low = fmaxf(ends.low, interval(i).low);
                    // Then what can reach the bound; more than the list holds give a better bound and another try.
                    full = true;
                    for(int round = 0; full && round < 4; ++round)
                    {
                        if(tid == 0)
                            listed = 0;
                        float const better = blockMax(ends.low);
                        if(round > 0 && !(better > least))
                            break;
                        least = fmaxf(least, better);
                        if constexpr(Packed)
                            scan<T, E, 2>(row, clock, low + tid, high, p, least, list, &listed);
                        scan<T, 1, 8>(row, clock, oneLow + tid, oneHigh, p, least, list, &listed);
                        __syncthreads();
                        full = listed > kList;
#pragma unroll
                        for(int u = 0; u < static_cast<int>(kList) / kThreads; ++u)
                        {
                            uint32_t const k = u * kThreads + tid;
                            Ends one{-INFINITY, -INFINITY};
                            if(k < min(listed, kList))
                                one = interval(list[k]);
                            upper[u] = one.high;
                            ends.low = fmaxf(ends.low, one.low);
                        }
                        __syncthreads(); // `listed` has been read
                    }
                    least = fmaxf(least, blockMax(ends.low));
                }
                if(tid == 0)
                {
                    blockLow = least;
                    blockFull = full;
                }
                clusterArrive();
                clusterWait();
                // the best lower end of the sequence
                float bar = 0.f;
                bool useless = false;
                for(unsigned r = 0; r < blocks; ++r)
                {
                    bar = fmaxf(bar, *inBlock(&blockLow, r));
                    useless |= *inBlock(&blockFull, r);
                }
                // Below fp32's normal numbers (large noise) a rounding is more than an interval allows for.
                if(bar >= 0x1p-126f && bar < INFINITY && !useless)
                {
                    // The token with this lower end has a positive rate. If no other one reaches it, it is the token, and
                    // nothing is computed again.
#pragma unroll
                    for(int u = 0; u < static_cast<int>(kList) / kThreads; ++u)
                        if(upper[u] >= bar)
                        {
                            unsigned const k = atomicAdd(inBlock(&founds, 0), 1u);
                            if(k < kReach)
                                *inBlock(found + k, 0) = list[u * kThreads + tid];
                        }
                    __syncwarp();
                    clusterArrive();
                    clusterWait();
                    unsigned const all = *inBlock(&founds, 0);
                    certainly = all > 0 && all <= kReach;
                    if(certainly)
                    {
                        clusterArrive(); // the first block may leave when all have read its count
                        if(rank != 0)
                        {
                            clusterWait();
                            return;
                        }
                        if(all == 1)
                            drawn = found[0];
                        else if(warp == 0)
                        {
                            Best best = Best::none();
                            for(uint32_t k = lane; k < all; k += 32)
                                again<T>(a, row, other, clock, certain, lse, draftLse, found[k], &best);
                            drawn = warpBest(best).index;
                        }
                    }
                }
                if(!certainly)
                {
                    // Intervals say nothing (rows with nothing left, far logits, many equal quotients, noise at 0 or so large that
                    // quotients are subnormal): all tokens in 64 bits.
                    Best best = Best::none();
                    for(uint32_t i = low * E + tid; i < high * E; i += kThreads)
                        again<T>(a, row, other, clock, certain, lse, draftLse, i, &best);
                    for(uint32_t i = oneLow + tid; i < oneHigh; i += kThreads)
                        again<T>(a, row, other, clock, certain, lse, draftLse, i, &best);
                    best = warpBest(best);
                    if(lane == 0)
                        bests[warp] = best;
                    __syncthreads();
                    if(tid == 0)
                    {
#pragma unroll
                        for(int w = 1; w < kWarps; ++w)
                            best.take(bests[w].score, bests[w].index);
                        blockBest = best;
                    }
                    clusterArrive();
                    clusterWait();
                    Best result = Best::none();
                    for(unsigned r = 0; r < blocks; ++r)
                    {
                        Best const* there = inBlock(&blockBest, r);
                        result.take(there->score, there->index);
                    }
                    drawn = result.index;
                    if(result.score > kNoRate)
                        break; // the same in every thread of the cluster
                }
                if(certainly)
                    break;
            }
            if(rank == 0 && warp == 0)
            {
                for(uint32_t i = lane; i <= a.length; i += 32)
                    a.put(a.tokens, to + i,
                          i > n ? -1 : i < n ? a.index(a.drafts, at + i) : drawn == UINT32_MAX ? -1 : static_cast<int64_t>(drawn));
                if(lane == 0)
                    a.put(a.accepted, b, n);
            }
            // no block leaves while another may still read its shared memory
            __syncwarp();
            if(!certainly)
                clusterArrive();
            clusterWait();
        }

        template<typename T>
        int launchVerify(cudaStream_t stream, DeviceProps const* props, VerifyArgs const& a, bool packed)
        {
            // A cluster of up to eight blocks a sequence: as many as leave each thread a pack or more, and fewer when the
            // sequences alone fill the GPU (two blocks an SM; 256 x 50256 fp32 24.6 us with one block a sequence, 30.2 with
            // two of half the threads; 64 x 131072 bf16 with four 16.3, with eight of half the threads 16.6).
            constexpr uint32_t E = PackOf<T>::E;
            uint32_t blocks = 1;
            uint64_t const room = 2ull * static_cast<unsigned>(props->smCount);
            if(a.logits)
                while(blocks < 8 && a.vocab > blocks * kThreads * E && static_cast<uint64_t>(a.batch) * blocks * 2 <= room)
                    blocks *= 2;
            if(static_cast<uint64_t>(a.batch) * blocks > static_cast<uint64_t>(INT_MAX))
                blocks = 1;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(a.batch * blocks);
            config.blockDim = dim3(kThreads);
            config.stream = stream;
            cudaLaunchAttribute attribute{};
            attribute.id = cudaLaunchAttributeClusterDimension;
            attribute.val.clusterDim.x = blocks;
            attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
            config.attrs = &attribute;
            config.numAttrs = 1;
            A3B_CUDA(cudaLaunchKernelEx(&config, packed ? verifyKernel<T, true> : verifyKernel<T, false>, a));
            return A3B_OK;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_verify_drafts(a3b_stream_t stream, a3b_verify_drafts_args const* args)
    {
        A3B_REQUIRE(args, "null arguments");
        uint64_t const batch = args->batch, length = args->length, vocab = args->vocab;
        int const dtype = args->dtype, index_dtype = args->index_dtype;
        a3b_rows const &rows = args->logits, &draftRows = args->draft_logits;
        void const *logits = rows.data, *draft_logits = draftRows.data, *drafts = args->drafts, *top_index = args->top_index;
        float const *lse = args->lse, *draft_lse = args->draft_lse, *uniform = args->uniform, *noise = args->noise;
        double const scale = args->scale, draft_scale = args->draft_scale;
        int64_t const noise_stride = args->noise_stride;
        void *tokens = args->tokens, *accepted = args->accepted;
        A3B_REQUIRE(rowTypeSize(dtype) != 0, "logits must be f32, f16 or bf16");
        A3B_REQUIRE(index_dtype == A3B_I32 || index_dtype == A3B_I64, "token indices must be i32 or i64");
        A3B_REQUIRE(vocab > 0, "a row needs at least one logit");
        A3B_REQUIRE(length == UINT64_MAX || batch <= UINT64_MAX / (length + 1), "rows overflow");
        if(vocab > static_cast<uint64_t>(INT_MAX) - 64 || length >= static_cast<uint64_t>(INT_MAX)
           || batch * (length + 1) > static_cast<uint64_t>(INT_MAX))
        {
            setError("at most 2^31 - 1 rows of 2^31 - 65 logits");
            return A3B_ERR_TOO_LARGE;
        }
        if(batch == 0)
            return A3B_OK;
        int const es = rowTypeSize(dtype), is = index_dtype == A3B_I64 ? 8 : 4;
        A3B_REQUIRE(tokens && accepted && (drafts || length == 0), "null drafts or output");
        A3B_REQUIRE(logits || top_index, "neither logits nor a greedy choice is given");
        A3B_REQUIRE(!logits || (lse && noise && (uniform || length == 0)), "logits need lse, uniform and noise");
        A3B_REQUIRE(!draft_logits || (logits && draft_lse), "the draft's logits need their lse and the target's logits");
        A3B_REQUIRE(!logits || (scale >= 0x1p-20 && scale <= 0x1p20), "scale must lie between 2^-20 and 2^20");
        A3B_REQUIRE(!draft_logits || (draft_scale >= 0x1p-20 && draft_scale <= 0x1p20), "scale must lie between 2^-20 and 2^20");
        A3B_REQUIRE(alignedTo(es, {logits, draft_logits}) && alignedTo(4, {lse, draft_lse, uniform, noise})
                        && alignedTo(is, {drafts, top_index, tokens, accepted}),
                    "an array is not aligned to its type");
        Wide const b = static_cast<Wide>(batch), k = static_cast<Wide>(length);
        Stretch const out = Stretch::dense(tokens, b * (k + 1) * is), count = Stretch::dense(accepted, b * is);
        Stretch const ins[] = {Stretch::rows(rows, batch, length + 1, vocab, es),
                               Stretch::rows(draftRows, batch, length, vocab, es),
                               Stretch::rows(noise, 1, batch, 0, noise_stride, vocab, 4),
                               Stretch::dense(lse, b * (k + 1) * 4),
                               Stretch::dense(draft_lse, b * k * 4),
                               Stretch::dense(uniform, b * k * 4),
                               Stretch::dense(drafts, b * k * is),
                               Stretch::dense(top_index, b * (k + 1) * is)};
        A3B_REQUIRE(out.apart(count), "the outputs overlap");
        for(Stretch const& in : ins)
            A3B_REQUIRE(out.apart(in) && count.apart(in), "an output overlaps its inputs");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        VerifyArgs a{logits, {rows.outer_stride, rows.inner_stride}, lse, length ? draft_logits : nullptr,
                     {draftRows.outer_stride, draftRows.inner_stride}, draft_lse, drafts, top_index, uniform, noise, noise_stride, tokens, accepted,
                     static_cast<uint32_t>(batch), static_cast<uint32_t>(length), static_cast<uint32_t>(vocab),
                     index_dtype == A3B_I64, scale, draft_scale};
        bool const packed = rowsAligned(logits, batch, length + 1, rows.outer_stride, rows.inner_stride, es, 16)
                            && (!a.draft || rowsAligned(draft_logits, batch, length, draftRows.outer_stride, draftRows.inner_stride, es, 16))
                            && rowsAligned(noise, 1, batch, 0, noise_stride, 4, 16);
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchVerify<float>(s, props, a, packed);
        if(dtype == A3B_F16)
            return launchVerify<__half>(s, props, a, packed);
        return launchVerify<__nv_bfloat16>(s, props, a, packed);
    }
}
