// 16-byte packs of 16- and 32-bit floating-point elements, shared by the kernels over rows of logits (logprob.cu) and
// over lists of gradients (gradnorm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace a3b
{
    constexpr unsigned kFullMask = 0xffffffffu;

    // max with NaN winning over every number
    __device__ __forceinline__ float maxNan(float a, float b)
    {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
        return r;
    }

    __device__ __forceinline__ float exp2Approx(float x)
    {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
        return r;
    }

    // the largest lane's value (NaN if any lane has one)
    __device__ __forceinline__ float warpMaxNan(float v)
    {
        float r;
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    }

    // ------------------------------------------------------------------------------------- thread-block clusters
    __device__ __forceinline__ unsigned clusterRank()
    {
        unsigned r;
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
        return r;
    }

    __device__ __forceinline__ unsigned clusterBlocks()
    {
        unsigned r;
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
        return r;
    }

    __device__ __forceinline__ void clusterArrive()
    {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }

    __device__ __forceinline__ void clusterWait()
    {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }

    // the address of the same shared variable in block `rank` of the cluster
    template<typename V>
    __device__ __forceinline__ V* inBlock(V* p, unsigned rank)
    {
        V* r;
        asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
        return r;
    }

    // Elements of one 16-byte pack (E of them, W = 4 words) as 32-bit floats, two at a time: element 2w and 2w + 1 of
    // a 16-bit type come from word w, of a 32-bit type from words 2w and 2w + 1.
    template<typename T>
    struct PackOf
    {
        static constexpr int E = 16 / static_cast<int>(sizeof(T));
        static constexpr int pairs = E / 2;

        static __device__ __forceinline__ float2 pair(unsigned const* word, int w)
        {
            if constexpr(std::is_same_v<T, float>)
                return make_float2(__uint_as_float(word[2 * w]), __uint_as_float(word[2 * w + 1]));
            else if constexpr(std::is_same_v<T, __nv_bfloat16>)
                return make_float2(__uint_as_float(word[w] << 16), __uint_as_float(word[w] & 0xffff0000u));
            else
            {
                __half2 h;
                memcpy(&h, word + w, 4);
                return __half22float2(h);
            }
        }

        // each element rounded to the nearest value of T (the one rounding of a stored result)
        static __device__ __forceinline__ void setPair(unsigned* word, int w, float2 v)
        {
            if constexpr(std::is_same_v<T, float>)
            {
                word[2 * w] = __float_as_uint(v.x);
                word[2 * w + 1] = __float_as_uint(v.y);
            }
            else if constexpr(std::is_same_v<T, __nv_bfloat16>)
            {
                __nv_bfloat162 const h = __float22bfloat162_rn(v);
                memcpy(word + w, &h, 4);
            }
            else
            {
                __half2 const h = __float22half2_rn(v);
                memcpy(word + w, &h, 4);
            }
        }

        // largest element of one pack, or of N packs (NaN if any is one); 16-bit types two at a time
        template<int N>
        static __device__ __forceinline__ float max(unsigned const (&word)[N][4])
        {
            if constexpr(std::is_same_v<T, float>)
            {
                float m = -INFINITY;
#pragma unroll
                for(int p = 0; p < N; ++p)
                    m = maxNan(m, max(word[p]));
                return m;
            }
            else
            {
                unsigned m = word[0][0];
#pragma unroll
                for(int p = 0; p < N; ++p)
#pragma unroll
                    for(int w = 0; w < 4; ++w)
                        m = maxWord(m, word[p][w]);
                return halves(m);
            }
        }

        static __device__ __forceinline__ float max(unsigned const* word)
        {
            if constexpr(std::is_same_v<T, float>)
                return maxNan(maxNan(__uint_as_float(word[0]), __uint_as_float(word[1])),
                              maxNan(__uint_as_float(word[2]), __uint_as_float(word[3])));
            else
                return halves(maxWord(maxWord(word[0], word[1]), maxWord(word[2], word[3])));
        }

        // of two elements in one word each
        static __device__ __forceinline__ unsigned maxWord(unsigned a, unsigned b)
        {
            unsigned r;
            if constexpr(std::is_same_v<T, __nv_bfloat16>)
                asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
            else
                asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
            return r;
        }

        // a word of `v` rounded to T, twice for 16-bit types
        static __device__ __forceinline__ unsigned twice(float v)
        {
            unsigned word[4] = {__float_as_uint(v), 0u, 0u, 0u};
            if constexpr(!std::is_same_v<T, float>)
                setPair(word, 0, make_float2(v, v));
            return word[0];
        }

        static __device__ __forceinline__ float halves(unsigned w)
        {
            float2 const v = pair(&w, 0);
            return maxNan(v.x, v.y);
        }

        static __device__ __forceinline__ unsigned negInfWord()
        {
            if constexpr(std::is_same_v<T, float>)
                return 0xff800000u;
            else if constexpr(std::is_same_v<T, __nv_bfloat16>)
                return 0xff80ff80u;
            else
                return 0xfc00fc00u;
        }

        // element e (a compile-time constant after unrolling) of a pack set from / taken as its raw bits
        static __device__ __forceinline__ void setRaw(unsigned* word, int e, T const* p)
        {
            if constexpr(std::is_same_v<T, float>)
                word[e] = *reinterpret_cast<unsigned const*>(p);
            else
            {
                unsigned const b = *reinterpret_cast<unsigned short const*>(p);
                word[e / 2] = (e & 1) ? ((word[e / 2] & 0xffffu) | (b << 16)) : ((word[e / 2] & 0xffff0000u) | b);
            }
        }

        static __device__ __forceinline__ void storeRaw(unsigned const* word, int e, T* p)
        {
            if constexpr(std::is_same_v<T, float>)
                *reinterpret_cast<unsigned*>(p) = word[e];
            else
                *reinterpret_cast<unsigned short*>(p)
                    = static_cast<unsigned short>((e & 1) ? word[e / 2] >> 16 : word[e / 2] & 0xffffu);
        }
    };

    template<typename T>
    __device__ __forceinline__ float toFloat(T v)
    {
        if constexpr(std::is_same_v<T, float>)
            return v;
        else if constexpr(std::is_same_v<T, __nv_bfloat16>)
            return __bfloat162float(v);
        else
            return __half2float(v);
    }

    // rounded to the nearest value of T
    template<typename T>
    __device__ __forceinline__ T fromFloat(float v)
    {
        if constexpr(std::is_same_v<T, float>)
            return v;
        else if constexpr(std::is_same_v<T, __nv_bfloat16>)
            return __float2bfloat16_rn(v);
        else
            return __float2half_rn(v);
    }

    // Two fp32 operations in one instruction (sm_100's packed fp32 pipe), each rounded on its own.
    __device__ __forceinline__ float2 add2(float2 a, float2 b)
    {
        return __fadd2_rn(a, b);
    }
    __device__ __forceinline__ float2 mul2(float2 a, float2 b)
    {
        return __fmul2_rn(a, b);
    }
    __device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
    {
        return __ffma2_rn(a, b, c);
    }
} // namespace a3b
