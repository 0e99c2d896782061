// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   p_v = e^(scale z_v - lse),  q_v = e^(draft_scale z'_v - lse')   (or q = 1 at the drafted token alone)
//   draft i stands while u_i q(t_i) < p(t_i);  at the first that does not, the token is drawn from (p - q)+, and behind
//   drafts that all stand from p: the first of exponential clocks with these rates, argmax of rate_v / noise_v.
//
// Every token that comes out is what the formula gives in 64 bits for these inputs, at the cost of 32: the tests take a few
// exponentials and are done in fp64; of the draw, a pass in fp32 gives every quotient an interval that holds its true value,
// and only the tokens whose interval reaches the best lower end (mostly one) are computed again in fp64. The pass reads one
// row of the target, one of the noise and, after a refusal, one of the draft, and is bound by memory where sequences are
// many, by latency where they are few: a cluster of blocks shares one sequence.
#include <algorithm>

#include "layout.cuh"
#include "rows.cuh"

namespace a3b
{
    namespace
    {
        constexpr int kThreads = 256;

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
                // what flushed to zero counts as up to fp32's least normal numbers
                float const rate = a - b, wide = fmaf(off, a + b, 0x1p-125f);
                // fmax drops NaN: an element with one takes no part
                ends->low = fmaxf(ends->low, (rate - wide) * r);
                ends->high = fmaxf(ends->high, (rate + wide) * r);
            }
        };

        __device__ __forceinline__ double exactly(double scale, float z, float lse)
        {
            return exp(scale * static_cast<double>(z) - static_cast<double>(lse));
        }

        struct Best
        {
            double score;
            uint32_t index;

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

        // How many drafts stand; every thread of the block gets the same answer. Also reads the drafts' ends.
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
                bool stands = false;
                if(known)
                {
                    T const* row = static_cast<T const*>(a.logits) + static_cast<int64_t>(b) * a.ls.outer
                                   + static_cast<int64_t>(i) * a.ls.step;
                    double const p = exactly(a.scale, toFloat(row[t]), a.lse[at + b + i]);
                    double q = 1.;
                    if(a.draft)
                    {
                        T const* other = static_cast<T const*>(a.draft) + static_cast<int64_t>(b) * a.ds.outer
                                         + static_cast<int64_t>(i) * a.ds.step;
                        q = exactly(a.draftScale, toFloat(other[t]), a.draftLse[at + i]);
                    }
                    stands = static_cast<double>(a.uniform[at + i]) * q < p;
                }
                unsigned const yes = __ballot_sync(kFullMask, stands), some = __ballot_sync(kFullMask, known);
                if(yes != kFullMask)
                {
                    uint32_t const n = __ffs(~yes) - 1;
                    *refused = (some >> n) & 1u;
                    return first + n;
                }
            }
            *refused = false;
            return a.length;
        }

        // E neighbouring elements of the three rows
        template<typename T, int E>
        struct Terms
        {
            static constexpr int words = E == 1 ? 1 : 4;
            unsigned z[words], y[words];
            float noise[E];

            __device__ __forceinline__ void load(T const* row, T const* other, float const* clock, uint32_t k)
            {
                if constexpr(E == 1)
                {
                    z[0] = raw(row + k);
                    if(other)
                        y[0] = raw(other + k);
                    noise[0] = clock[k];
                }
                else
                {
                    uint4 v = *reinterpret_cast<uint4 const*>(row + static_cast<size_t>(k) * E);
                    z[0] = v.x, z[1] = v.y, z[2] = v.z, z[3] = v.w;
                    if(other)
                    {
                        v = *reinterpret_cast<uint4 const*>(other + static_cast<size_t>(k) * E);
                        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
                    }
#pragma unroll
                    for(int e = 0; e < E; e += 4)
                    {
                        float4 const f = *reinterpret_cast<float4 const*>(clock + static_cast<size_t>(k) * E + e);
                        noise[e] = f.x, noise[e + 1] = f.y, noise[e + 2] = f.z, noise[e + 3] = f.w;
                    }
                }
            }
            static __device__ __forceinline__ unsigned raw(T const* p)
            {
                if constexpr(sizeof(T) == 4)
                    return *reinterpret_cast<unsigned const*>(p);
                else
                    return *reinterpret_cast<unsigned short const*>(p);
            }
            static __device__ __forceinline__ void unpack(float* v, unsigned const* w)
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

        template<typename T, int E>
        __device__ __forceinline__ void roughly(Terms<T, E> const& t, bool other, uint32_t certain, uint32_t first, Rough const& p,
                                                Rough const& q, Ends* ends)
        {
            float z[E], y[E];
            Terms<T, E>::unpack(z, t.z);
            if(other)
                Terms<T, E>::unpack(y, t.y);
            float const off = other ? fmaxf(p.off, q.off) : p.off;
#pragma unroll
            for(int e = 0; e < E; ++e)
                p.widen(z[e], other ? q(y[e]) : first + e == certain ? 1.f : 0.f, t.noise[e], off, ends);
        }

        // Token i in 64 bits, if its interval reaches `bar` (or intervals say nothing: `far`).
        template<typename T>
        __device__ __noinline__ void again(VerifyArgs const& a, T const* row, T const* other, float const* clock, uint32_t certain,
                                           float lse, float draftLse, float bar, bool far, uint32_t i, Best* best)
        {
            float const z = toFloat(row[i]), y = other ? toFloat(other[i]) : 0.f, noise = clock[i];
            if(!far)
            {
                Rough const p(a.scale, lse), q(a.draftScale, draftLse);
                Ends ends{-INFINITY, -INFINITY};
                p.widen(z, other ? q(y) : i == certain ? 1.f : 0.f, noise, other ? fmaxf(p.off, q.off) : p.off, &ends);
                if(!(ends.high >= bar))
                    return;
            }
            double rate = exactly(a.scale, z, lse);
            if(other)
                rate -= exactly(a.draftScale, y, draftLse);
            else if(i == certain)
                rate -= 1.;
            if(rate > 0.)
                best->take(rate / static_cast<double>(noise), i);
        }

        template<typename T>
        __global__ void __launch_bounds__(kThreads) verifyKernel(VerifyArgs a)
        {
            constexpr int E = PackOf<T>::E, kWarps = kThreads / 32;
            __shared__ float lows[kWarps];
            __shared__ float blockLow;
            __shared__ Best bests[kWarps];
            __shared__ Best blockBest;
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

            bool refused = false;
            uint32_t const n = accepted<T>(a, b, &refused);
            T const* row = static_cast<T const*>(a.logits) + static_cast<int64_t>(b) * a.ls.outer + static_cast<int64_t>(n) * a.ls.step;
            float const lse = a.lse[to + n];
            float const* clock = a.noise + static_cast<int64_t>(b) * a.noiseStride;
            Rough const p(a.scale, lse);
            Best result{0., UINT32_MAX};
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
                bool const packed = ((reinterpret_cast<uintptr_t>(row) | reinterpret_cast<uintptr_t>(other)
                                      | reinterpret_cast<uintptr_t>(clock)) & 15u) == 0u;
                uint32_t const packs = packed ? a.vocab / E : 0, step = blocks * kThreads, mine = rank * kThreads + tid;
                bool const far = p.far() || q.far(); // then every token is computed in 64 bits
                Ends ends{-INFINITY, far ? INFINITY : -INFINITY};
                if(!far)
                {
#pragma unroll 2
                    for(uint32_t k = mine; k < packs; k += step)
                    {
                        Terms<T, E> t;
                        t.load(row, other, clock, k);
                        roughly<T, E>(t, other, certain, k * E, p, q, &ends);
                    }
#pragma unroll 4
                    for(uint32_t k = packs * E + mine; k < a.vocab; k += step)
                    {
                        Terms<T, 1> t;
                        t.load(row, other, clock, k);
                        roughly<T, 1>(t, other, certain, k, p, q, &ends);
                    }
                }
                // the best lower end of the sequence
                float low = ends.low;
#pragma unroll
                for(int d = 16; d > 0; d /= 2)
                    low = fmaxf(low, __shfl_xor_sync(kFullMask, low, d));
                if(lane == 0)
                    lows[warp] = low;
                __syncthreads();
                if(tid == 0)
                {
#pragma unroll
                    for(int w = 1; w < kWarps; ++w)
                        low = fmaxf(low, lows[w]);
                    blockLow = low;
                }
                clusterArrive();
                clusterWait();
                float bar = -INFINITY;
                for(unsigned r = 0; r < blocks; ++r)
                    bar = fmaxf(bar, *inBlock(&blockLow, r));
                // the few tokens that reach it, in 64 bits
                Best best{0., UINT32_MAX};
                if(ends.high >= bar)
                {
                    for(uint32_t k = mine; k < packs; k += step)
                        for(uint32_t e = 0; e < E; ++e)
                            again<T>(a, row, other, clock, certain, lse, draftLse, bar, far, k * E + e, &best);
                    for(uint32_t k = packs * E + mine; k < a.vocab; k += step)
                        again<T>(a, row, other, clock, certain, lse, draftLse, bar, far, k, &best);
                }
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
                for(unsigned r = 0; r < blocks; ++r)
                {
                    Best const* far = inBlock(&blockBest, r);
                    result.take(far->score, far->index);
                }
                if(result.index != UINT32_MAX)
                    break; // the same in every thread of the cluster
            }
            if(rank == 0 && warp == 0)
            {
                for(uint32_t i = lane; i <= a.length; i += 32)
                    a.put(a.tokens, to + i,
                          i > n ? -1 : i < n ? a.index(a.drafts, at + i) : result.index == UINT32_MAX ? -1 : static_cast<int64_t>(result.index));
                if(lane == 0)
                    a.put(a.accepted, b, n);
            }
            // no block leaves while another may still read its shared memory
            clusterArrive();
            clusterWait();
        }

        template<typename T>
        int launchVerify(cudaStream_t stream, DeviceProps const* props, VerifyArgs const& a)
        {
            // A cluster of up to eight blocks a sequence: as many as leave each thread about two packs, and fewer when the
            // sequences alone fill the GPU.
            constexpr uint32_t E = PackOf<T>::E;
            uint32_t blocks = 1;
            uint64_t const room = 8ull * static_cast<unsigned>(props->smCount);
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
            A3B_CUDA(cudaLaunchKernelEx(&config, verifyKernel<T>, a));
            return A3B_OK;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_verify_drafts(
        a3b_stream_t stream,
        int dtype,
        uint64_t batch,
        uint64_t length,
        uint64_t vocab,
        void const* logits,
        int64_t logits_batch_stride,
        int64_t logits_stride,
        float const* lse,
        double scale,
        void const* draft_logits,
        int64_t draft_batch_stride,
        int64_t draft_stride,
        float const* draft_lse,
        double draft_scale,
        int index_dtype,
        void const* drafts,
        void const* top_index,
        float const* uniform,
        float const* noise,
        int64_t noise_stride,
        void* tokens,
        void* accepted)
    {
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
        Stretch const ins[] = {Stretch::rows(logits, batch, length + 1, logits_batch_stride, logits_stride, vocab, es),
                               Stretch::rows(draft_logits, batch, length, draft_batch_stride, draft_stride, vocab, es),
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
        VerifyArgs a{logits, {logits_batch_stride, logits_stride}, lse, length ? draft_logits : nullptr,
                     {draft_batch_stride, draft_stride}, draft_lse, drafts, top_index, uniform, noise, noise_stride, tokens, accepted,
                     static_cast<uint32_t>(batch), static_cast<uint32_t>(length), static_cast<uint32_t>(vocab),
                     index_dtype == A3B_I64, scale, draft_scale};
        auto s = static_cast<cudaStream_t>(stream);
        if(dtype == A3B_F32)
            return launchVerify<float>(s, props, a);
        if(dtype == A3B_F16)
            return launchVerify<__half>(s, props, a);
        return launchVerify<__nv_bfloat16>(s, props, a);
    }
}
