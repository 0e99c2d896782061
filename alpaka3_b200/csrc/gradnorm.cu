// Norm over a list of gradient tensors, and the tensors scaled down to a largest norm. No counterpart in alpaka3, whose
// transformReduce and transform take one buffer (include/alpaka/onHost/algo/transformReduce.hpp:59-114,
// transform.hpp:50-88): a training step has hundreds of them, most of them small.
//
// The list travels in the kernels' parameters (addresses and sizes by value, up to kEntries tensors a launch), so a call
// copies nothing to the device and can be captured in a graph. The tensors are cut into chunks of kChunkPacks 16-byte
// packs, numbered through the list; a block finds the tensor of a chunk by bisection over the chunks' running count.
//   * normKernel: resident blocks, each folds a run of consecutive chunks into one fp64 partial in the workspace
//     (7.1 TB/s on a B200 over 2.1 GB);
//   * finishKernel: one block folds the partials in their order;
//   * clipKernel: a block for every chunk, handed out in order (6.8 TB/s read and written; resident blocks reached 5.9).
//     It and finishKernel are launched while the kernel before drains (programmatic dependent launch);
//   * clipSmallKernel: both for a short list, one launch of one cluster.
// The workspace holds nothing between calls (no tickets), and no block waits for another one's progress in memory:
// captured graphs and streams only need a workspace each.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <exception>
#include <new>
#include <type_traits>
#include <vector>

#include "rows.cuh"

namespace a3b
{
    namespace
    {
        constexpr int kBlock = 256;
        constexpr int kWarps = kBlock / 32;
        constexpr int kPacks = 4;                                // packs of a chunk per thread
        constexpr uint64_t kChunkPacks = uint64_t{kBlock} * kPacks; // 16 KB
        constexpr int kEntries = 960;     // tensors a launch: 32 bytes each, of 32764
        constexpr int kFewEntries = 120;  // parameters under 4 KB: 30 KB cost the host 2 us a launch
        constexpr int kBlocksPerSm = 6;
        constexpr uint32_t kSmallChunks = 32; // up to here one cluster does it all
        constexpr unsigned kSmallCluster = 8;

        struct Entry
        {
            void const* in;
            void* out;
            uint64_t n;
            uint32_t firstChunk;
            int32_t dtype;
        };

        template<int N>
        struct BatchOf
        {
            uint32_t count;
            uint32_t chunks;
            Entry e[N];
        };
        using Batch = BatchOf<kEntries>;
        static_assert(sizeof(Batch) <= 32000, "kernel parameters hold 32764 bytes");

        int sizeOf(int dtype)
        {
            return dtype == A3B_F64 ? 8 : dtype == A3B_F32 ? 4 : 2;
        }

        // ----------------------------------------------------------------------------------------- device side
        template<int KIND>
        __device__ __forceinline__ double fold(double a, double b)
        {
            if constexpr(KIND == A3B_NORM_MAX)
                return a != a || b != b ? a + b : (a > b ? a : b);
            else
                return a + b;
        }

        // |x| or x^2 of one element in fp64
        template<int KIND>
        __device__ __forceinline__ double term(double x)
        {
            return KIND == A3B_NORM_L2 ? x * x : fabs(x);
        }

        // one pack's share of the norm
        template<int KIND, typename T>
        __device__ __forceinline__ double packNorm(unsigned const* q)
        {
            if constexpr(std::is_same_v<T, double>)
            {
                double d[2];
                memcpy(d, q, 16);
                return fold<KIND>(term<KIND>(d[0]), term<KIND>(d[1]));
            }
            else if constexpr(KIND == A3B_NORM_MAX)
            {
                float m = 0.0f;
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                {
                    float2 const v = PackOf<T>::pair(q, w);
                    m = maxNan(m, maxNan(fabsf(v.x), fabsf(v.y)));
                }
                return static_cast<double>(m);
            }
            else
            {
                // the pack's sum in fp32 (at most 8 terms), the sum over packs in fp64
                float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                {
                    float2 const v = PackOf<T>::pair(q, w);
                    if constexpr(KIND == A3B_NORM_L2)
                        s = fma2(v, v, s);
                    else
                        s = add2(s, make_float2(fabsf(v.x), fabsf(v.y)));
                }
                float const f = s.x + s.y;
                // Squares of values below 2^-63 or above 2^63 may leave fp32's range: such a pack (seen by its sum)
                // is formed again in fp64. A pack of zeros is not. fp32 loses at most 8 * 2^-150 of a sum of 2^-96.
                if(!(f >= 0x1p-96f && f <= FLT_MAX))
                {
                    unsigned any = 0;
#pragma unroll
                    for(int w = 0; w < 4; ++w)
                        any |= q[w];
                    if((any & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0u)
                        return 0.0;
                    double d = 0.0;
#pragma unroll
                    for(int w = 0; w < PackOf<T>::pairs; ++w)
                    {
                        float2 const v = PackOf<T>::pair(q, w);
                        d += term<KIND>(static_cast<double>(v.x)) + term<KIND>(static_cast<double>(v.y));
                    }
                    return d;
                }
                return static_cast<double>(f);
            }
        }

        // the product in fp32, or, where the factor is an fp64 number, in fp64 and rounded to fp32 before T
        template<typename T, typename F>
        __device__ __forceinline__ void scalePack(unsigned* q, F factor)
        {
            if constexpr(std::is_same_v<T, double>)
            {
                double d[2];
                memcpy(d, q, 16);
                d[0] *= factor, d[1] *= factor;
                memcpy(q, d, 16);
            }
            else
            {
                auto scaled = [&](float2 v)
                {
                    if constexpr(std::is_same_v<F, double>)
                        return make_float2(static_cast<float>(v.x * factor), static_cast<float>(v.y * factor));
                    else
                        return mul2(v, make_float2(factor, factor));
                };
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                    PackOf<T>::setPair(q, w, scaled(PackOf<T>::pair(q, w)));
            }
        }

        template<typename T>
        __device__ __forceinline__ void putElement(unsigned* q, int e, T const* p)
        {
            if constexpr(std::is_same_v<T, double>)
                memcpy(q + 2 * e, p, 8);
            else
                PackOf<T>::setRaw(q, e, p);
        }

        template<typename T>
        __device__ __forceinline__ void takeElement(unsigned const* q, int e, T* p)
        {
            if constexpr(std::is_same_v<T, double>)
                memcpy(p, q + 2 * e, 8);
            else
                PackOf<T>::storeRaw(q, e, p);
        }

        // The packs of chunk `c` of a tensor in one thread's registers. Packs lie on the 16-byte boundaries of `base`
        // (`lead` elements of the first one before the tensor); what is outside the tensor reads as zero.
        template<typename T>
        struct Chunk
        {
            static constexpr int E = 16 / static_cast<int>(sizeof(T));
            unsigned q[kPacks][4];

            __device__ __forceinline__ static bool whole(uint64_t n, int lead, uint64_t c, int p, int64_t& i)
            {
                i = static_cast<int64_t>((c * kChunkPacks + p * kBlock + threadIdx.x) * E) - lead;
                return i >= 0 && i + E <= static_cast<int64_t>(n);
            }

            __device__ __forceinline__ void load(T const* in, uint64_t n, int lead, uint64_t c, bool aligned)
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                {
                    int64_t i;
                    if(whole(n, lead, c, p, i) && aligned)
                    {
                        uint4 const v = __ldcs(reinterpret_cast<uint4 const*>(in + i));
                        q[p][0] = v.x, q[p][1] = v.y, q[p][2] = v.z, q[p][3] = v.w;
                    }
                    else
                    {
                        q[p][0] = q[p][1] = q[p][2] = q[p][3] = 0u;
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            if(i + e >= 0 && i + e < static_cast<int64_t>(n))
                                putElement<T>(q[p], e, in + i + e);
                    }
                }
            }

            __device__ __forceinline__ void store(T* out, uint64_t n, int lead, uint64_t c) const
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                {
                    int64_t i;
                    if(whole(n, lead, c, p, i))
                        __stcs(reinterpret_cast<uint4*>(out + i), make_uint4(q[p][0], q[p][1], q[p][2], q[p][3]));
                    else
                    {
#pragma unroll
                        for(int e = 0; e < E; ++e)
                            if(i + e >= 0 && i + e < static_cast<int64_t>(n))
                                takeElement<T>(q[p], e, out + i + e);
                    }
                }
            }
        };

        // index of the tensor that chunk `chunk` of the list belongs to
        template<int N>
        __device__ __forceinline__ uint32_t entryOf(BatchOf<N> const& b, uint32_t chunk)
        {
            uint32_t lo = 0, hi = b.count; // e[lo].firstChunk <= chunk < e[hi].firstChunk
            while(hi - lo > 1)
            {
                uint32_t const mid = (lo + hi) / 2;
                if(b.e[mid].firstChunk <= chunk)
                    lo = mid;
                else
                    hi = mid;
            }
            return lo;
        }

        // the run of chunks that block `block` of `blocks` takes
        __device__ __forceinline__ uint2 runOf(uint32_t chunks, uint32_t block, uint32_t blocks)
        {
            return make_uint2(static_cast<uint32_t>(uint64_t{chunks} * block / blocks),
                              static_cast<uint32_t>(uint64_t{chunks} * (block + 1u) / blocks));
        }

        __device__ __forceinline__ int leadOf(void const* p, int size)
        {
            return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / static_cast<unsigned>(size));
        }

        template<int KIND, typename T>
        __device__ __forceinline__ double chunkNorm(Entry const& e, uint64_t c)
        {
            Chunk<T> x;
            x.load(static_cast<T const*>(e.in), e.n, leadOf(e.in, sizeof(T)), c, true);
            double r = 0.0;
#pragma unroll
            for(int p = 0; p < kPacks; ++p)
                r = fold<KIND>(r, packNorm<KIND, T>(x.q[p]));
            return r;
        }

        // the block's fold of every thread's `v`, in thread 0 .. 31 alike
        template<int KIND>
        __device__ __forceinline__ double blockFold(double v, double* smem)
        {
#pragma unroll
            for(int m = 16; m > 0; m >>= 1)
                v = fold<KIND>(v, __shfl_xor_sync(kFullMask, v, m));
            if((threadIdx.x & 31) == 0)
                smem[threadIdx.x >> 5] = v;
            __syncthreads();
            double r = smem[0];
#pragma unroll
            for(int w = 1; w < kWarps; ++w)
                r = fold<KIND>(r, smem[w]);
            return r;
        }

        // this block's share of the norm: the chunks [run.x, run.y), in order
        template<int KIND, int N>
        __device__ __forceinline__ double runNorm(BatchOf<N> const& b, uint2 run)
        {
            double r = 0.0;
            uint32_t k = run.x < run.y ? entryOf(b, run.x) : 0;
            for(uint32_t c = run.x; c < run.y; ++c)
            {
                while(k + 1 < b.count && b.e[k + 1].firstChunk <= c)
                    ++k;
                Entry const& e = b.e[k];
                uint64_t const at = c - e.firstChunk;
                switch(e.dtype)
                {
                case A3B_F32:
                    r = fold<KIND>(r, chunkNorm<KIND, float>(e, at));
                    break;
                case A3B_F64:
                    r = fold<KIND>(r, chunkNorm<KIND, double>(e, at));
                    break;
                case A3B_F16:
                    r = fold<KIND>(r, chunkNorm<KIND, __half>(e, at));
                    break;
                default:
                    r = fold<KIND>(r, chunkNorm<KIND, __nv_bfloat16>(e, at));
                }
            }
            return r;
        }

        template<int KIND, int N>
        __global__ void __launch_bounds__(kBlock, kBlocksPerSm)
            normKernel(__grid_constant__ BatchOf<N> const b, double* partials)
        {
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // they wait before they read `partials`
            __shared__ double smem[kWarps];
            double const r = blockFold<KIND>(runNorm<KIND>(b, runOf(b.chunks, blockIdx.x, gridDim.x)), smem);
            if(threadIdx.x == 0)
                partials[blockIdx.x] = r;
        }

        // fold of all partials, the same in every thread of every block that calls it
        template<int KIND>
        __device__ __forceinline__ double total(double const* partials, uint32_t count, double* smem)
        {
            double r = 0.0;
            for(uint32_t k = threadIdx.x; k < count; k += kBlock)
                r = fold<KIND>(r, __ldcg(partials + k));
            return blockFold<KIND>(r, smem);
        }

        template<int KIND>
        __device__ __forceinline__ double normOf(double t)
        {
            return KIND == A3B_NORM_L2 ? sqrt(t) : t;
        }

        __device__ __forceinline__ void writeNorm(double v, int dtype, void* out)
        {
            if(!out)
                return;
            if(dtype == A3B_F64)
                *static_cast<double*>(out) = v;
            else
                *static_cast<float*>(out) = static_cast<float>(v);
        }

        template<int KIND>
        __global__ void __launch_bounds__(kBlock)
            finishKernel(double const* partials, uint32_t count, double* partial, int dtype, void* norm, bool clips)
        {
            __shared__ double smem[kWarps];
            // clipKernel waits before it reads the result; whatever else comes next on the stream may not
            if(clips)
                asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            asm volatile("griddepcontrol.wait;" ::: "memory");
            double const t = total<KIND>(partials, count, smem);
            if(threadIdx.x == 0)
            {
                if(partial)
                    *partial = t;
                writeNorm(normOf<KIND>(t), dtype, norm);
            }
        }

        // min(1, maxNorm / (norm + 1e-6)), NaN stays
        __device__ __forceinline__ double factorOf(double norm, double maxNorm)
        {
            double const ratio = maxNorm / (norm + 1e-6);
            return ratio > 1.0 ? 1.0 : ratio;
        }

        template<typename T>
        __device__ __forceinline__ void clipChunk(Entry const& e, uint64_t c, double factor)
        {
            // packs on the output's boundaries; the input is read by elements where it lies differently
            Chunk<T> x;
            int const lead = leadOf(e.out, sizeof(T));
            x.load(static_cast<T const*>(e.in), e.n, lead, c, lead == leadOf(e.in, sizeof(T)));
            if constexpr(std::is_same_v<T, double>)
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                    scalePack<T>(x.q[p], factor);
            }
            else if(factor >= static_cast<double>(FLT_MIN) || !(factor > 0.0))
            {
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                    scalePack<T>(x.q[p], static_cast<float>(factor));
            }
            else
            {
                // below fp32's normal numbers (norms of 1e38 and more, from elements near FLT_MAX) the factor would lose bits
#pragma unroll
                for(int p = 0; p < kPacks; ++p)
                    scalePack<T>(x.q[p], factor);
            }
            x.store(static_cast<T*>(e.out), e.n, lead, c);
        }

        template<int N>
        __device__ __forceinline__ void clipOne(BatchOf<N> const& b, uint32_t c, double factor)
        {
            Entry const& e = b.e[entryOf(b, c)];
            uint64_t const at = c - e.firstChunk;
            if(factor == 1.0 && e.in == e.out)
                return;
            switch(e.dtype)
            {
            case A3B_F32:
                clipChunk<float>(e, at, factor);
                break;
            case A3B_F64:
                clipChunk<double>(e, at, factor);
                break;
            case A3B_F16:
                clipChunk<__half>(e, at, factor);
                break;
            default:
                clipChunk<__nv_bfloat16>(e, at, factor);
            }
        }

        // Block b scales chunk b. `partials`: those of normKernel, or (count = 1) their fold.
        template<int KIND, int N>
        __global__ void __launch_bounds__(kBlock, kBlocksPerSm) clipKernel(
            __grid_constant__ BatchOf<N> const b,
            double const* partials,
            uint32_t count,
            double maxNorm,
            int dtype,
            void* normOut)
        {
            __shared__ double smem[kWarps];
            asm volatile("griddepcontrol.wait;" ::: "memory");
            double const norm
                = normOf<KIND>(count == 1u ? __ldcg(partials) : total<KIND>(partials, count, smem));
            if(blockIdx.x == 0 && threadIdx.x == 0)
                writeNorm(norm, dtype, normOut);
            clipOne(b, blockIdx.x, factorOf(norm, maxNorm));
        }

        // Norm and clipping of a list of up to kSmallChunks chunks by one cluster: the blocks leave their partials in one
        // another's shared memory. One launch instead of two, and nothing in the workspace.
        template<int KIND, int N>
        __global__ void __launch_bounds__(kBlock) __cluster_dims__(kSmallCluster, 1, 1)
            clipSmallKernel(__grid_constant__ BatchOf<N> const b, double maxNorm, int dtype, void* normOut)
        {
            __shared__ double smem[kWarps];
            __shared__ double all[kSmallCluster];
            clusterArrive();
            uint2 const run = runOf(b.chunks, blockIdx.x, kSmallCluster);
            double const r = blockFold<KIND>(runNorm<KIND>(b, run), smem);
            clusterWait(); // every block has started
            if(threadIdx.x < kSmallCluster)
                *inBlock(all + blockIdx.x, threadIdx.x) = r;
            clusterArrive();
            clusterWait();
            double t = all[0];
#pragma unroll
            for(unsigned k = 1; k < kSmallCluster; ++k)
                t = fold<KIND>(t, all[k]);
            double const norm = normOf<KIND>(t);
            if(blockIdx.x == 0 && threadIdx.x == 0)
                writeNorm(norm, dtype, normOut);
            for(uint32_t c = run.x; c < run.y; ++c)
                clipOne(b, c, factorOf(norm, maxNorm));
        }
    } // namespace
} // namespace a3b

// the list cut into launches
struct a3b_tensor_list
{
    std::vector<a3b::Batch> batches;
    char const* notClippable = nullptr; // why the list cannot be scaled, or null
};

namespace a3b
{
    namespace
    {
        struct Range
        {
            uintptr_t lo, hi;
            size_t index;
            bool output;
        };

        // Outputs disjoint from one another, and from every input but their own.
        char const* overlapOf(std::vector<Range>& all)
        {
            std::sort(all.begin(), all.end(), [](Range const& a, Range const& b) { return a.lo < b.lo; });
            // of the ranges so far: the output and the input that reach furthest, and the input of another tensor that
            // reaches furthest beside it
            Range const* out = nullptr;
            Range const* in = nullptr;
            Range const* second = nullptr;
            for(Range const& r : all)
            {
                auto foreign = [&](Range const* other)
                { return other && other->hi > r.lo && (other->index != r.index || other->lo != r.lo); };
                if(r.output)
                {
                    if(out && out->hi > r.lo)
                        return "outputs of the list overlap one another";
                    if(foreign(in) || foreign(second))
                        return "an output of the list overlaps an input that is not its own";
                    out = &r; // the outputs so far are disjoint: the last one reaches furthest
                }
                else
                {
                    if(foreign(out))
                        return "an output of the list overlaps an input that is not its own";
                    if(!in || r.hi > in->hi)
                    {
                        second = in;
                        in = &r;
                    }
                    else if(!second || r.hi > second->hi)
                        second = &r;
                }
            }
            return nullptr;
        }

        // blocks of normKernel for one batch: a function of the batch and the device
        uint32_t gridOf(Batch const& b, DeviceProps const* props)
        {
            return std::min<uint32_t>(b.chunks, static_cast<uint32_t>(props->smCount) * kBlocksPerSm);
        }

        // whether two stretches of memory share a byte; a null one shares none
        bool overlap(void const* a, size_t an, void const* b, size_t bn)
        {
            auto const x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
            return a && b && (x < y ? y - x < an : x - y < bn);
        }

        // A block that has the norm writes it while others still read what it comes from: the two lie apart.
        int checkCall(a3b_tensor_list const* list, int kind, double const* partial, int normDtype, void const* norm)
        {
            A3B_REQUIRE(list, "null tensor list");
            A3B_REQUIRE(kind == A3B_NORM_L2 || kind == A3B_NORM_L1 || kind == A3B_NORM_MAX, "unknown norm kind");
            A3B_REQUIRE(normDtype == A3B_F32 || normDtype == A3B_F64, "the norm is f32 or f64");
            A3B_REQUIRE(reinterpret_cast<uintptr_t>(norm) % (normDtype == A3B_F64 ? 8u : 4u) == 0u
                            && reinterpret_cast<uintptr_t>(partial) % 8u == 0u,
                        "norm or partial is not aligned to its type");
            A3B_REQUIRE(!overlap(norm, normDtype == A3B_F64 ? 8u : 4u, partial, 8u), "norm and partial overlap");
            return A3B_OK;
        }

        size_t workspaceOf(a3b_tensor_list const* list, DeviceProps const* props)
        {
            size_t n = 1;
            for(Batch const& b : list->batches)
                n += gridOf(b, props);
            return n * sizeof(double);
        }

        // f(the batch as kernel parameters): few tensors as the short form
        template<typename F>
        int withBatch(Batch const& b, F&& f)
        {
            if(b.count > static_cast<uint32_t>(kFewEntries))
                return f(b);
            BatchOf<kFewEntries> few;
            few.count = b.count;
            few.chunks = b.chunks;
            std::copy(b.e, b.e + b.count, few.e);
            return f(few);
        }

        // Launches `kernel` so that it may start while the kernel before it drains; it waits by itself.
        template<typename... P, typename... A>
        int launchAfter(cudaStream_t s, uint32_t grid, void (*kernel)(P...), A const&... args)
        {
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(grid);
            cfg.blockDim = dim3(kBlock);
            cfg.stream = s;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            A3B_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
            return A3B_OK;
        }

        template<int KIND>
        int launchNorm(
            cudaStream_t s, a3b_tensor_list const* list, DeviceProps const* props, double* partials, uint32_t* count)
        {
            *count = 0;
            for(Batch const& b : list->batches)
            {
                uint32_t const grid = gridOf(b, props);
                withBatch(b, [&](auto const& p) {
                    normKernel<KIND><<<grid, kBlock, 0, s>>>(p, partials + *count);
                    return A3B_OK;
                });
                A3B_CHECK_LAUNCH("normKernel");
                *count += grid;
            }
            return A3B_OK;
        }

        template<int KIND>
        int launchFinish(
            cudaStream_t s, double const* partials, uint32_t count, double* partial, int dtype, void* norm, bool clips)
        {
            return launchAfter(s, 1, finishKernel<KIND>, partials, count, partial, dtype, norm, clips);
        }

        // `early`: the kernel right before on the stream is normKernel or finishKernel
        template<int KIND>
        int launchClip(
            cudaStream_t s,
            a3b_tensor_list const* list,
            double const* partials,
            uint32_t count,
            double maxNorm,
            int dtype,
            void* norm,
            bool early)
        {
            for(Batch const& b : list->batches)
            {
                int const rc = withBatch(b, [&](auto const& p) {
                    constexpr int N = sizeof(p.e) / sizeof(Entry);
                    if(early)
                        return launchAfter(s, b.chunks, clipKernel<KIND, N>, p, partials, count, maxNorm, dtype, norm);
                    clipKernel<KIND, N><<<b.chunks, kBlock, 0, s>>>(p, partials, count, maxNorm, dtype, norm);
                    A3B_CHECK_LAUNCH("clipKernel");
                    return static_cast<int>(A3B_OK);
                });
                if(rc != A3B_OK)
                    return rc;
                norm = nullptr;
                early = false;
            }
            return A3B_OK;
        }

        // Norm, then clipping. Lists of one wave of blocks: every block folds the partials. Longer ones: one block does, in
        // a launch of its own, and a block for every chunk reads the result (162 tensors, 2.1 GB of bf16 on a B200:
        // 938 us; resident blocks that walk runs of chunks 1042).
        template<int KIND>
        int launchBoth(
            cudaStream_t s,
            a3b_tensor_list const* list,
            DeviceProps const* props,
            double maxNorm,
            double* workspace,
            int dtype,
            void* norm)
        {
            if(list->batches.empty())
                return norm ? launchFinish<KIND>(s, workspace, 0u, nullptr, dtype, norm, false) : A3B_OK;
            Batch const& first = list->batches[0];
            if(list->batches.size() == 1 && first.chunks <= kSmallChunks)
                return withBatch(first, [&](auto const& p) {
                    clipSmallKernel<KIND><<<kSmallCluster, kBlock, 0, s>>>(p, maxNorm, dtype, norm);
                    A3B_CHECK_LAUNCH("clipSmallKernel");
                    return static_cast<int>(A3B_OK);
                });
            double* const partials = workspace + 1;
            uint32_t count = 0;
            int const rc = launchNorm<KIND>(s, list, props, partials, &count);
            if(rc != A3B_OK)
                return rc;
            if(list->batches.size() == 1 && first.chunks <= gridOf(first, props))
                return launchClip<KIND>(s, list, partials, count, maxNorm, dtype, norm, true);
            int const rf = launchFinish<KIND>(s, partials, count, workspace, dtype, norm, true);
            return rf != A3B_OK ? rf : launchClip<KIND>(s, list, workspace, 1u, maxNorm, dtype, nullptr, true);
        }

        // f(std::integral_constant<int, kind>)
        template<typename F>
        int withKind(int kind, F&& f)
        {
            if(kind == A3B_NORM_L1)
                return f(std::integral_constant<int, A3B_NORM_L1>{});
            if(kind == A3B_NORM_MAX)
                return f(std::integral_constant<int, A3B_NORM_MAX>{});
            return f(std::integral_constant<int, A3B_NORM_L2>{});
        }

        int buildList(void const* const* in, void* const* out, uint64_t const* n, int const* dtype, uint64_t count,
                      a3b_tensor_list* list)
        {
            std::vector<Range> ranges;
            ranges.reserve(2 * count);
            uint64_t chunks = 0;
            for(uint64_t k = 0; k < count; ++k)
            {
                int const d = dtype[k];
                A3B_REQUIRE(d == A3B_F32 || d == A3B_F64 || d == A3B_F16 || d == A3B_BF16,
                            "tensors must be f32, f64, f16 or bf16");
                if(n[k] == 0)
                    continue;
                A3B_REQUIRE(in[k], "null tensor in the list");
                auto const size = static_cast<uintptr_t>(sizeOf(d));
                Entry e{in[k], out && out[k] ? out[k] : const_cast<void*>(in[k]), n[k], 0u, d};
                auto const from = reinterpret_cast<uintptr_t>(e.in), to = reinterpret_cast<uintptr_t>(e.out);
                A3B_REQUIRE(from % size == 0 && to % size == 0, "a tensor is not aligned to its type");
                A3B_REQUIRE(n[k] <= (uint64_t{1} << 46), "a tensor is larger than any device");
                ranges.push_back({from, from + n[k] * size, k, false});
                ranges.push_back({to, to + n[k] * size, k, true});
                // chunks on the boundaries of the input (norm) or the output (clip): room for either
                uint64_t const most = std::max(from & 15u, to & 15u) / size;
                uint64_t const perPack = 16 / size;
                uint64_t const own = ((n[k] + most + perPack - 1) / perPack + kChunkPacks - 1) / kChunkPacks;
                if(list->batches.empty() || list->batches.back().count == static_cast<uint32_t>(kEntries)
                   || chunks + own > static_cast<uint64_t>(INT_MAX))
                {
                    A3B_REQUIRE(own <= static_cast<uint64_t>(INT_MAX), "a tensor is larger than any device");
                    list->batches.emplace_back();
                    list->batches.back().count = 0;
                    chunks = 0;
                }
                Batch& b = list->batches.back();
                e.firstChunk = static_cast<uint32_t>(chunks);
                b.e[b.count++] = e;
                chunks += own;
                b.chunks = static_cast<uint32_t>(chunks);
            }
            list->notClippable = overlapOf(ranges);
            return A3B_OK;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_tensor_list_create(
        void const* const* in,
        void* const* out,
        uint64_t const* n,
        int const* dtype,
        uint64_t count,
        a3b_tensor_list** list)
    {
        A3B_REQUIRE(list, "list is null");
        *list = nullptr;
        A3B_REQUIRE(count == 0 || (in && n && dtype), "null array");
        a3b_tensor_list* made = nullptr;
        try
        {
            made = new a3b_tensor_list();
            int const rc = buildList(in, out, n, dtype, count, made);
            if(rc != A3B_OK)
            {
                delete made;
                return rc;
            }
        }
        catch(std::exception const&) // std::bad_alloc, std::length_error
        {
            delete made;
            setError("no host memory for a list of %llu tensors", static_cast<unsigned long long>(count));
            return A3B_ERR_NOMEM;
        }
        *list = made;
        return A3B_OK;
    }

    int a3b_tensor_list_destroy(a3b_tensor_list* list)
    {
        delete list;
        return A3B_OK;
    }

    size_t a3b_grad_norm_workspace(a3b_tensor_list const* list)
    {
        DeviceProps const* props = nullptr;
        if(!list || currentDevice(&props) != A3B_OK)
            return 0;
        return workspaceOf(list, props);
    }

    int a3b_grad_norm(
        a3b_stream_t stream,
        a3b_tensor_list const* list,
        int kind,
        void* workspace,
        size_t workspace_bytes,
        double* partial,
        int norm_dtype,
        void* norm)
    {
        int const rc = checkCall(list, kind, partial, norm_dtype, norm);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(partial || norm, "nothing to compute: no output is given");
        A3B_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "workspace is null or unaligned");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        size_t const used = workspaceOf(list, props);
        A3B_REQUIRE(workspace_bytes >= used, "workspace is too small");
        A3B_REQUIRE(!overlap(workspace, used, norm, norm_dtype == A3B_F64 ? 8u : 4u) && !overlap(workspace, used, partial, 8u),
                    "norm or partial lies in the workspace");
        auto s = static_cast<cudaStream_t>(stream);
        return withKind(kind, [&](auto k) {
            auto* const partials = static_cast<double*>(workspace);
            uint32_t count = 0;
            int const e = launchNorm<k()>(s, list, props, partials, &count);
            return e != A3B_OK ? e : launchFinish<k()>(s, partials, count, partial, norm_dtype, norm, false);
        });
    }

    int a3b_clip_grads(
        a3b_stream_t stream,
        a3b_tensor_list const* list,
        int kind,
        double const* partial,
        double max_norm,
        int norm_dtype,
        void* norm)
    {
        int const rc = checkCall(list, kind, partial, norm_dtype, norm);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(partial, "null partial");
        A3B_REQUIRE(!list->notClippable, list->notClippable);
        A3B_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        auto s = static_cast<cudaStream_t>(stream);
        return withKind(kind, [&](auto k) {
            if(list->batches.empty())
                return norm ? launchFinish<k()>(s, partial, 1u, nullptr, norm_dtype, norm, false) : static_cast<int>(A3B_OK);
            return launchClip<k()>(s, list, partial, 1u, max_norm, norm_dtype, norm, false);
        });
    }

    int a3b_clip_grad_norm(
        a3b_stream_t stream,
        a3b_tensor_list const* list,
        int kind,
        double max_norm,
        void* workspace,
        size_t workspace_bytes,
        int norm_dtype,
        void* norm)
    {
        int const rc = checkCall(list, kind, nullptr, norm_dtype, norm);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(!list->notClippable, list->notClippable);
        A3B_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
        A3B_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "workspace is null or unaligned");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        size_t const used = workspaceOf(list, props);
        A3B_REQUIRE(workspace_bytes >= used, "workspace is too small");
        A3B_REQUIRE(!overlap(workspace, used, norm, norm_dtype == A3B_F64 ? 8u : 4u), "norm lies in the workspace");
        auto s = static_cast<cudaStream_t>(stream);
        return withKind(kind, [&](auto k) {
            return launchBoth<k()>(s, list, props, max_norm, static_cast<double*>(workspace), norm_dtype, norm);
        });
    }
}
