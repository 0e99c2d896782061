// Rows in memory: the steps between them, and the host's checks that what a call writes lies apart from what it reads.
// Shared by the operators around a model's layers (norm.cu, embedding.cu, verify.cu).
#pragma once

#include <climits>
#include <initializer_list>

#include "common.cuh"

namespace a3b
{
    // Row r = o * inner + i starts at element o * outer + i * step.
    struct RowStep
    {
        int64_t outer;
        int64_t step;

        __device__ __forceinline__ int64_t at(uint32_t row, uint32_t inner, bool one) const
        {
            if(one) // all rows in one level: no division
                return static_cast<int64_t>(row) * step;
            uint32_t const o = row / inner;
            return static_cast<int64_t>(o) * outer + static_cast<int64_t>(row - o * inner) * step;
        }
    };

    // ------------------------------------------------------------------------------------------ host checks
    // In 128 bits: strides come from the caller and may be anything.
    using Wide = __int128;

    inline Wide wideAbs(Wide v)
    {
        return v < 0 ? -v : v;
    }

    inline Wide wideGcd(Wide a, Wide b)
    {
        while(b != 0)
        {
            Wide const r = a % b;
            a = b;
            b = r;
        }
        return a;
    }

    // The bytes that one array of rows occupies (a dense array is one row).
    struct Stretch
    {
        uintptr_t base = 0;
        Wide outer = 1, inner = 1, outerStep = 0, step = 0, bytes = 0; // steps and a row's length in bytes

        static Stretch rows(void const* p, uint64_t outer, uint64_t inner, int64_t outerStep, int64_t step, uint64_t n, int size)
        {
            Stretch s;
            s.base = reinterpret_cast<uintptr_t>(p);
            s.outer = outer;
            s.inner = inner;
            s.outerStep = outer > 1 ? static_cast<Wide>(outerStep) * size : 0;
            s.step = inner > 1 ? static_cast<Wide>(step) * size : 0;
            s.bytes = static_cast<Wide>(n) * size;
            return s;
        }
        static Stretch rows(a3b_rows const& r, uint64_t outer, uint64_t inner, uint64_t n, int size)
        {
            return rows(r.data, outer, inner, r.outer_stride, r.inner_stride, n, size);
        }
        static Stretch dense(void const* p, Wide bytes)
        {
            Stretch s;
            s.base = reinterpret_cast<uintptr_t>(p);
            s.bytes = bytes;
            return s;
        }

        Wide low() const
        {
            Wide const a = (outer - 1) * outerStep, b = (inner - 1) * step;
            return static_cast<Wide>(base) + (a < 0 ? a : 0) + (b < 0 ? b : 0);
        }
        Wide high() const
        {
            Wide const a = (outer - 1) * outerStep, b = (inner - 1) * step;
            return static_cast<Wide>(base) + (a > 0 ? a : 0) + (b > 0 ? b : 0) + bytes;
        }
        bool empty() const
        {
            return base == 0 || bytes == 0 || outer == 0 || inner == 0;
        }

        // no two of its own rows share a byte
        bool separate() const
        {
            Wide const so = wideAbs(outerStep), si = wideAbs(step);
            if(inner > 1 && si < bytes)
                return false;
            if(outer > 1 && so < bytes)
                return false;
            return outer == 1 || inner == 1 || so >= bytes + (inner - 1) * si || si >= bytes + (outer - 1) * so;
        }
        bool sameAs(Stretch const& b) const
        {
            return base == b.base && outerStep == b.outerStep && step == b.step && bytes == b.bytes;
        }
        // Certain to share no byte with b: one ends before the other begins, or the rows of both lie in columns of
        // one grid (all steps are multiples of one length) that do not meet. Other arrangements count as overlapping.
        bool apart(Stretch const& b) const
        {
            if(empty() || b.empty() || high() <= b.low() || b.high() <= low())
                return true;
            Wide const grid = wideGcd(wideGcd(wideAbs(outerStep), wideAbs(step)), wideGcd(wideAbs(b.outerStep), wideAbs(b.step)));
            if(grid == 0)
                return false;
            Wide off = (static_cast<Wide>(b.base) - static_cast<Wide>(base)) % grid;
            if(off < 0)
                off += grid;
            return off >= bytes && off + b.bytes <= grid;
        }
    };

    inline bool alignedTo(uintptr_t size, std::initializer_list<void const*> pointers)
    {
        for(void const* p : pointers)
            if(reinterpret_cast<uintptr_t>(p) % size != 0u)
                return false;
        return true;
    }

    // Launches a kernel that begins with waitForPrevious() right behind one that calls signalNext(): its blocks may start while
    // the other's last ones run. Only for kernels of one call: the first of a call is launched in full order, and the last
    // signals nothing, so that nothing of another call starts early.
    template<typename... Parameters, typename... Args>
    int launchNext(cudaStream_t stream, void (*kernel)(Parameters...), dim3 grid, unsigned threads, size_t shared, Args const&... args)
    {
        cudaLaunchAttribute attribute{};
        attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = grid;
        config.blockDim = dim3(threads);
        config.dynamicSmemBytes = shared;
        config.stream = stream;
        config.attrs = &attribute;
        config.numAttrs = 1;
        A3B_CUDA(cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(args)...));
        return A3B_OK;
    }

    __device__ __forceinline__ void waitForPrevious()
    {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    __device__ __forceinline__ void signalNext()
    {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }

    // bytes of an element of a floating-point type that rows may have; 0 for every other type
    inline int rowTypeSize(int dtype)
    {
        return dtype == A3B_F32 ? 4 : dtype == A3B_F16 || dtype == A3B_BF16 ? 2 : 0;
    }

    // every row of an array begins at a multiple of `size` bytes
    inline bool rowsAligned(void const* p, uint64_t outer, uint64_t inner, int64_t outerStep, int64_t step, int es, int size)
    {
        return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(size) == 0 && (outer == 1 || outerStep * es % size == 0)
               && (inner == 1 || step * es % size == 0);
    }
} // namespace a3b
