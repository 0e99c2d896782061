// Norm over a list of gradient tensors, and the tensors scaled down to a largest norm. No counterpart in alpaka3, whose
// transformReduce and transform take one buffer (include/alpaka/onHost/algo/transformReduce.hpp:59-114,
// transform.hpp:50-88): a training step has hundreds of them, most of them small.
//
// The list travels in the kernels' parameters (addresses and sizes by value, up to kEntries tensors a launch), so a call
// copies nothing to the device and can be captured in a graph. The tensors are cut into chunks of kChunkPacks 16-byte
// packs; a block finds the tensor of a chunk by bisection over the chunks' running count.
//   * normKernel: every block folds its chunks into one fp64 partial in the workspace;
//   * clipKernel: every block folds all partials in the same order, then scales its chunks.
// The workspace holds nothing between calls (no tickets), and no block waits for another: captured graphs and streams
// only need a workspace each.
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
        constexpr int kEntries = 960;                            // tensors a launch: 32 bytes each, of 32764
        constexpr int kBlocksPerSm = 4;

        struct Entry
        {
            void const* in;
            void* out;
            uint64_t n;
            uint32_t firstChunk;
            int32_t dtype;
        };

        struct Batch
        {
            uint32_t count;
            uint32_t chunks;
            Entry e[kEntries];
        };
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
                float2 const f2 = make_float2(factor, factor);
#pragma unroll
                for(int w = 0; w < PackOf<T>::pairs; ++w)
                    PackOf<T>::setPair(q, w, mul2(PackOf<T>::pair(q, w), f2));
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
                        uint4 const v = __ldg(reinterpret_cast<uint4 const*>(in + i));
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

        __device__ __forceinline__ Entry const& entryOf(Batch const& b, uint32_t chunk)
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
            return b.e[lo];
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

        template<int KIND>
        __global__ void __launch_bounds__(kBlock) normKernel(__grid_constant__ Batch const b, double* partials)
        {
            __shared__ double smem[kWarps];
            double r = 0.0;
            for(uint32_t c = blockIdx.x; c < b.chunks; c += gridDim.x)
            {
                Entry const& e = entryOf(b, c);
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
            r = blockFold<KIND>(r, smem);
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
            finishKernel(double const* partials, uint32_t count, double* partial, int dtype, void* norm)
        {
            __shared__ double smem[kWarps];
            double const t = total<KIND>(partials, count, smem);
            if(threadIdx.x == 0)
            {
                if(partial)
                    *partial = t;
                writeNorm(normOf<KIND>(t), dtype, norm);
            }
        }

        template<typename T, typename F>
        __device__ __forceinline__ void clipChunk(Entry const& e, uint64_t c, F factor)
        {
            // packs on the output's boundaries; the input is read by elements where it lies differently
            Chunk<T> x;
            int const lead = leadOf(e.out, sizeof(T));
            x.load(static_cast<T const*>(e.in), e.n, lead, c, lead == leadOf(e.in, sizeof(T)));
#pragma unroll
            for(int p = 0; p < kPacks; ++p)
                scalePack<T>(x.q[p], factor);
            x.store(static_cast<T*>(e.out), e.n, lead, c);
        }

        template<int KIND>
        __global__ void __launch_bounds__(kBlock) clipKernel(
            __grid_constant__ Batch const b,
            double const* partials,
            uint32_t count,
            double maxNorm,
            int dtype,
            void* normOut)
        {
            __shared__ double smem[kWarps];
            double const norm = normOf<KIND>(total<KIND>(partials, count, smem));
            if(blockIdx.x == 0 && threadIdx.x == 0)
                writeNorm(norm, dtype, normOut);
            double const ratio = maxNorm / (norm + 1e-6);
            double const factor = ratio > 1.0 ? 1.0 : ratio; // NaN stays
            for(uint32_t c = blockIdx.x; c < b.chunks; c += gridDim.x)
            {
                Entry const& e = entryOf(b, c);
                uint64_t const at = c - e.firstChunk;
                if(factor == 1.0 && e.in == e.out)
                    continue;
                switch(e.dtype)
                {
                case A3B_F32:
                    clipChunk<float>(e, at, static_cast<float>(factor));
                    break;
                case A3B_F64:
                    clipChunk<double>(e, at, factor);
                    break;
                case A3B_F16:
                    clipChunk<__half>(e, at, static_cast<float>(factor));
                    break;
                default:
                    clipChunk<__nv_bfloat16>(e, at, static_cast<float>(factor));
                }
            }
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

        int checkCall(a3b_tensor_list const* list, int kind, int normDtype)
        {
            A3B_REQUIRE(list, "null tensor list");
            A3B_REQUIRE(kind == A3B_NORM_L2 || kind == A3B_NORM_L1 || kind == A3B_NORM_MAX, "unknown norm kind");
            A3B_REQUIRE(normDtype == A3B_F32 || normDtype == A3B_F64, "the norm is f32 or f64");
            return A3B_OK;
        }

        size_t workspaceOf(a3b_tensor_list const* list, DeviceProps const* props)
        {
            size_t n = 1;
            for(Batch const& b : list->batches)
                n += gridOf(b, props);
            return n * sizeof(double);
        }

        template<int KIND>
        int launchNorm(cudaStream_t s, a3b_tensor_list const* list, DeviceProps const* props, double* partials, uint32_t* count)
        {
            *count = 0;
            for(Batch const& b : list->batches)
            {
                uint32_t const grid = gridOf(b, props);
                normKernel<KIND><<<grid, kBlock, 0, s>>>(b, partials + *count);
                A3B_CHECK_LAUNCH("normKernel");
                *count += grid;
            }
            return A3B_OK;
        }

        template<int KIND>
        int launchFinish(cudaStream_t s, double const* partials, uint32_t count, double* partial, int dtype, void* norm)
        {
            finishKernel<KIND><<<1, kBlock, 0, s>>>(partials, count, partial, dtype, norm);
            A3B_CHECK_LAUNCH("finishKernel");
            return A3B_OK;
        }

        template<int KIND>
        int launchClip(
            cudaStream_t s,
            a3b_tensor_list const* list,
            DeviceProps const* props,
            double const* partials,
            uint32_t count,
            double maxNorm,
            int dtype,
            void* norm)
        {
            if(list->batches.empty())
                return norm ? launchFinish<KIND>(s, partials, count, nullptr, dtype, norm) : A3B_OK;
            for(Batch const& b : list->batches)
            {
                clipKernel<KIND><<<gridOf(b, props), kBlock, 0, s>>>(b, partials, count, maxNorm, dtype, norm);
                A3B_CHECK_LAUNCH("clipKernel");
                norm = nullptr;
            }
            return A3B_OK;
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
                   || chunks + own > static_cast<uint64_t>(UINT32_MAX))
                {
                    A3B_REQUIRE(own <= static_cast<uint64_t>(UINT32_MAX), "a tensor is larger than any device");
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
        int const rc = checkCall(list, kind, norm_dtype);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(partial || norm, "nothing to compute: no output is given");
        A3B_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "workspace is null or unaligned");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        A3B_REQUIRE(workspace_bytes >= workspaceOf(list, props), "workspace is too small");
        auto s = static_cast<cudaStream_t>(stream);
        return withKind(kind, [&](auto k) {
            auto* const partials = static_cast<double*>(workspace);
            uint32_t count = 0;
            int const e = launchNorm<k()>(s, list, props, partials, &count);
            return e != A3B_OK ? e : launchFinish<k()>(s, partials, count, partial, norm_dtype, norm);
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
        int const rc = checkCall(list, kind, norm_dtype);
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
            return launchClip<k()>(s, list, props, partial, 1u, max_norm, norm_dtype, norm);
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
        int const rc = checkCall(list, kind, norm_dtype);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(!list->notClippable, list->notClippable);
        A3B_REQUIRE(max_norm >= 0.0, "max_norm must not be negative or NaN");
        A3B_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "workspace is null or unaligned");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        A3B_REQUIRE(workspace_bytes >= workspaceOf(list, props), "workspace is too small");
        auto s = static_cast<cudaStream_t>(stream);
        return withKind(kind, [&](auto k) {
            auto* const partials = static_cast<double*>(workspace);
            uint32_t count = 0;
            int const e = launchNorm<k()>(s, list, props, partials, &count);
            return e != A3B_OK ? e : launchClip<k()>(s, list, props, partials, count, max_norm, norm_dtype, norm);
        });
    }
}
