// Root-mean-square norm of rows, with the residual's addition in front and an output in 8 bits behind it, and its gradient.
//
//   h = x + residual,  r = (mean h^2 + eps)^(-1/2),  y = h r w,  q = y / s with s = max|y| / (largest 8-bit value)
//   dy = g w,  c = mean(dy h r),  dh = r (dy - h r c) + dtotal,  dw = sum over rows of g h r
//
// Both are bound by memory: about 5 and 9 operations an element against 4 to 16 bytes. So every row is read once and stays
// in registers between its sum and its output; a row is one team's (part of a warp, a warp or a block, by its length), and
// teams are many, so that while one waits in its reduction others load.
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>

#include "layout.cuh"
#include "rows.cuh"

namespace a3b
{
    namespace
    {
        // E elements of T (one 16-byte pack, or a single element where rows do not allow packs) as raw words.
        template<typename T, int E>
        struct Access
        {
            static constexpr int words = E == 1 ? 1 : 4, pairs = E == 1 ? 1 : E / 2;

            // a single element is a pair with 0
            static __device__ __forceinline__ float2 pair(unsigned const* w, int k)
            {
                if constexpr(E > 1)
                    return PackOf<T>::pair(w, k);
                else if constexpr(sizeof(T) == 4)
                    return make_float2(__uint_as_float(w[0]), 0.f);
                else
                    return make_float2(PackOf<T>::pair(w, 0).x, 0.f);
            }
            // rounded to the nearest values of T
            static __device__ __forceinline__ void setPair(unsigned* w, int k, float2 v)
            {
                if constexpr(E > 1)
                    PackOf<T>::setPair(w, k, v);
                else
                {
                    unsigned two[2];
                    PackOf<T>::setPair(two, 0, v);
                    w[0] = two[0];
                }
            }
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
                {
                    uint4 const v = *reinterpret_cast<uint4 const*>(p);
                    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                }
            }
            static __device__ __forceinline__ void store(T* p, unsigned const* w)
            {
                if constexpr(E == 1)
                {
                    if constexpr(sizeof(T) == 4)
                        *reinterpret_cast<unsigned*>(p) = w[0];
                    else
                        *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
                }
                else
                    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        };

        // E weights, of T or fp32, in the 16-byte words they come in
        template<typename WT, int E>
        struct Weights
        {
            static constexpr int words = E == 1 ? 1 : E * static_cast<int>(sizeof(WT)) / 4;

            // without a weight: ones, so that the loops over elements have no branch
            static __device__ __forceinline__ void load(unsigned* w, WT const* weight, uint32_t k)
            {
                if(weight)
                    return read(w, weight + static_cast<size_t>(k) * E);
#pragma unroll
                for(int i = 0; i < words; ++i)
                    w[i] = PackOf<WT>::twice(1.f);
            }
            static __device__ __forceinline__ void read(unsigned* w, WT const* p)
            {
                if constexpr(E == 1)
                    Access<WT, 1>::load(w, p);
                else
#pragma unroll
                    for(int k = 0; k < words / 4; ++k)
                    {
                        uint4 const v = __ldg(reinterpret_cast<uint4 const*>(p) + k);
                        w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
                    }
            }
            static __device__ __forceinline__ float2 pair(unsigned const* w, int k)
            {
                if constexpr(E == 1)
                    return Access<WT, 1>::pair(w, 0);
                else if constexpr(std::is_same_v<WT, float>)
                    return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
                else
                    return PackOf<WT>::pair(w, k);
            }
        };

        // ------------------------------------------------------------------------------------- sums over a team
        // Butterflies: every lane ends with the same bits.
        template<int L, typename V>
        __device__ __forceinline__ V lanesSum(V v)
        {
#pragma unroll
            for(int d = L / 2; d > 0; d /= 2)
                v += __shfl_xor_sync(kFullMask, v, d);
            return v;
        }

        // the largest of 1 << log2 neighbouring lanes (the same for the whole warp)
        __device__ __forceinline__ float lanesMax(float v, int log2)
        {
#pragma unroll
            for(int d = 0; d < 5; ++d)
                if(d < log2)
                    v = maxNan(v, __shfl_xor_sync(kFullMask, v, 1 << d));
            return v;
        }

        // Sum over the team: L lanes, or the block (L = 0) by way of `room` (one value a warp), which the next sum may
        // not use before another barrier.
        template<int L, typename V>
        __device__ __forceinline__ V teamSum(V v, V* room)
        {
            if constexpr(L > 0)
                return lanesSum<L>(v);
            else
            {
                v = lanesSum<32>(v);
                unsigned const warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
                if(lane == 0)
                    room[warp] = v;
                __syncthreads();
                return lanesSum<32>(lane < warps ? room[lane] : V(0));
            }
        }

        template<int L>
        __device__ __forceinline__ float teamMax(float v, float* room)
        {
            if constexpr(L > 0)
                return lanesMax(v, L == 32 ? 5 : L == 16 ? 4 : 3);
            else
            {
                v = lanesMax(v, 5);
                unsigned const warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
                if(lane == 0)
                    room[warp] = v;
                __syncthreads();
                return lanesMax(lane < warps ? room[lane] : 0.f, 5);
            }
        }

        // ---------------------------------------------------------------------------------------------- forward
        struct NormArgs
        {
            void const* x;
            void const* residual; // may be null
            void* total; // may be null
            void* out;
            RowStep xs, rs, ts, os;
            uint32_t rows, inner, n;
            bool one;
            void const* weight; // may be null
            float* rstd; // may be null
            float* scales; // 8-bit outputs
            uint32_t group, groups; // elements that share a scale (0: the row), and groups a row
            bool e5m2;
            double eps;
            float eps32, inverse; // inverse: 1 / n
            bool tiny; // eps gives nothing to sums below fp32's range
        };

        // fp32 squares are exact enough unless their sum leaves fp32's range: above it, or below it with nothing from eps.
        __device__ __forceinline__ bool sumLost(float sum, bool tiny)
        {
            return !(sum < INFINITY) || (tiny && sum < 0x1p-100f);
        }

        // rsqrtf is off by two units at most: with the product's and the sum's roundings 2^-21, where a row's own sum may lose
        // more; the division and square root it replaces cost short rows a fifth of their time
        __device__ __forceinline__ float rootOf(float sum, float inverse, float eps)
        {
            return rsqrtf(fmaf(sum, inverse, eps));
        }
        __device__ __forceinline__ float rootOf(double sum, uint32_t n, double eps)
        {
            return static_cast<float>(1. / sqrt(sum / n + eps));
        }

        __device__ __noinline__ float2 quotient(float2 v, float by)
        {
            return make_float2(__fdiv_rn(v.x, by), __fdiv_rn(v.y, by));
        }

        // The scale of a group whose largest magnitude is `high`: a product with the rounded 1 / largest, and the values are
        // multiplied by its reciprocal. That is the nearest fp32 value: rcp.approx, off by up to a unit (of one scale in eight), and
        // one step of Newton's iteration, which was compared with __frcp_rn at every scale from 2^-126 to 2^121. So values in the
        // middle between two of 8 bits (4 in 10000 of bf16 rows) fall to the side that elementary operations give; without the
        // step one in 25 of them did not (8192 x 8192 to e4m3 77.3 us, with it 77.6, with __frcp_rn 79.2). A scale below fp32's
        // normal numbers has no reciprocal there: its values are divided.
        template<int N>
        __device__ __forceinline__ float scaled(float high, bool e5m2, float2 (&y)[N])
        {
            float const scale = high * (e5m2 ? 1.f / 57344.f : 1.f / 448.f);
            if(scale > 0.f && scale < 0x1p-126f)
            {
#pragma unroll
                for(int k = 0; k < N; ++k)
                    y[k] = quotient(y[k], scale);
            }
            else
            {
                float inverse;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
                inverse = scale == 0.f ? 0.f : inverse;
                inverse = fmaf(inverse, fmaf(-fminf(scale, FLT_MAX), inverse, 1.f), inverse);
#pragma unroll
                for(int k = 0; k < N; ++k)
                    y[k] = mul2(y[k], make_float2(inverse, inverse));
            }
            return scale;
        }

        // two values rounded to 8 bits, beyond the largest to the largest
        __device__ __forceinline__ unsigned eight(float2 v, bool e5m2)
        {
            return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, e5m2 ? __NV_E5M2 : __NV_E4M3);
        }

        // A row stays in registers as the words it is stored in (half the registers of its fp32 values, so twice the blocks an
        // SM; unpacking it again costs less than the spills of holding it did) and is computed on in pairs.

        // Adds the residual's words to a lane's, stores the sum, and returns the lane's sum of squares.
        template<typename T, int E, int P>
        __device__ __forceinline__ float addRow(NormArgs const& a, uint32_t row, bool live, uint32_t lanes, uint32_t t,
                                                unsigned (&raw)[P][Access<T, E>::words],
                                                unsigned const (&add)[P][Access<T, E>::words])
        {
            using A = Access<T, E>;
            uint32_t const packs = a.n / E;
            T* total = a.total && live ? static_cast<T*>(a.total) + a.ts.at(row, a.inner, a.one) : nullptr;
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(uint32_t const k = p * lanes + t; k < packs)
                {
                    if(a.residual)
                    {
                        // The sum is rounded to the rows' type, stored or not: the norm is that of the row which the next
                        // layer and the gradient read.
#pragma unroll
                        for(int e = 0; e < A::pairs; ++e)
                            A::setPair(raw[p], e, add2(A::pair(raw[p], e), A::pair(add[p], e)));
                        if(total)
                            A::store(total + static_cast<size_t>(k) * E, raw[p]);
                    }
#pragma unroll
                    for(int e = 0; e < A::pairs; ++e)
                    {
                        float2 const h = A::pair(raw[p], e);
                        sum = fma2(h, h, sum);
                    }
                }
            return sum.x + sum.y;
        }

        // 1 / sqrt(mean h^2 + eps) from the team's sum of squares, or in fp64 from h itself where that is lost
        template<typename T, int E, int P, int L>
        __device__ __forceinline__ float rootRow(NormArgs const& a, uint32_t lanes, uint32_t t, float sum,
                                                 unsigned const (&raw)[P][Access<T, E>::words], double* roomD)
        {
            using A = Access<T, E>;
            bool const lost = sumLost(sum, a.tiny);
            if(!(L == 0 ? lost : __any_sync(kFullMask, lost)))
                return rootOf(sum, a.inverse, a.eps32);
            double wide = 0.;
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(p * lanes + t < a.n / E)
#pragma unroll
                    for(int e = 0; e < A::pairs; ++e)
                    {
                        float2 const h = A::pair(raw[p], e);
                        wide = fma(static_cast<double>(h.x), static_cast<double>(h.x), wide);
                        wide = fma(static_cast<double>(h.y), static_cast<double>(h.y), wide);
                    }
            wide = teamSum<L>(wide, roomD);
            return lost ? rootOf(wide, a.n, a.eps) : rootOf(sum, a.inverse, a.eps32);
        }

        // One row a team of L lanes (0: a block), P accesses of E elements a lane; the whole row is in registers.
        template<typename T, typename WT, int E, int P, int L, bool F8>
        __global__ void __launch_bounds__(L > 0 ? 128 : P == 2 ? 512 : 1024, L > 0 || P != 2 ? 1 : 3) rmsNormKernel(NormArgs a)
        {
            using A = Access<T, E>;
            using W = Weights<WT, E>;
            __shared__ float roomF[32], roomM[32];
            __shared__ double roomD[32];
            uint32_t const lanes = L == 0 ? blockDim.x : L, t = L == 0 ? threadIdx.x : threadIdx.x % (L == 0 ? 1 : L);
            uint32_t const team = L == 0 ? blockIdx.x : blockIdx.x * (128u / (L == 0 ? 1 : L)) + threadIdx.x / (L == 0 ? 1 : L);
            bool const live = team < a.rows;
            uint32_t const row = live ? team : a.rows - 1u, packs = a.n / E;
            T const* x = static_cast<T const*>(a.x) + a.xs.at(row, a.inner, a.one);
            WT const* weight = static_cast<WT const*>(a.weight);

            unsigned raw[P][A::words], add[P][A::words];
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(uint32_t const k = p * lanes + t; k < packs)
                    A::load(raw[p], x + static_cast<size_t>(k) * E);
            if(a.residual)
            {
                T const* r = static_cast<T const*>(a.residual) + a.rs.at(row, a.inner, a.one);
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs)
                        A::load(add[p], r + static_cast<size_t>(k) * E);
            }
            // with the row's loads under way; more than two packs' weights would cost blocks an SM
            constexpr bool early = P * W::words <= 8;
            unsigned wraw[early ? P : 1][W::words];
            if(early)
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs)
                        W::load(wraw[early ? p : 0], weight, k);

            float const sum = teamSum<L>(addRow<T, E, P>(a, row, live, lanes, t, raw, add), roomF);
            float const r = rootRow<T, E, P, L>(a, lanes, t, sum, raw, roomD);
            if(a.rstd && t == 0 && live)
                a.rstd[row] = r;

            // y of access p, in pairs
            auto scaledRow = [&](int p, float2 (&y)[A::pairs])
            {
                uint32_t const k = p * lanes + t;
                if constexpr(!early)
                    W::load(wraw[0], weight, k);
#pragma unroll
                for(int e = 0; e < A::pairs; ++e)
                    y[e] = mul2(mul2(A::pair(raw[p], e), make_float2(r, r)), W::pair(wraw[early ? p : 0], e));
            };
            auto largest = [&](float2 const (&y)[A::pairs])
            {
                float high = 0.f;
#pragma unroll
                for(int e = 0; e < A::pairs; ++e)
                    high = maxNan(high, maxNan(fabsf(y[e].x), fabsf(y[e].y)));
                return high;
            };
            if constexpr(!F8)
            {
                T* out = static_cast<T*>(a.out) + a.os.at(row, a.inner, a.one);
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs && live)
                    {
                        float2 y[A::pairs];
                        scaledRow(p, y);
                        unsigned words[A::words];
#pragma unroll
                        for(int e = 0; e < A::pairs; ++e)
                            A::setPair(words, e, y[e]);
                        A::store(out + static_cast<size_t>(k) * E, words);
                    }
            }
            else
            {
                static_assert(E > 1 && (L == 0 || L == 32), "groups lie on neighbouring lanes");
                auto* out = static_cast<unsigned char*>(a.out) + a.os.at(row, a.inner, a.one);
                float* scales = a.scales + static_cast<size_t>(row) * a.groups;
                int const near = 31 - __clz(static_cast<int>(a.group) / E); // log2 of the lanes of one group
                float high = 0.f;
                if(a.group == 0)
                {
#pragma unroll
                    for(int p = 0; p < P; ++p)
                        if(p * lanes + t < packs)
                        {
                            float2 y[A::pairs];
                            scaledRow(p, y);
                            high = maxNan(high, largest(y));
                        }
                    high = teamMax<L>(high, roomM);
                }
#pragma unroll
                for(int p = 0; p < P; ++p)
                {
                    uint32_t const k = p * lanes + t;
                    float2 y[A::pairs];
#pragma unroll
                    for(int e = 0; e < A::pairs; ++e)
                        y[e] = make_float2(0.f, 0.f);
                    if(k < packs)
                        scaledRow(p, y);
                    if(a.group != 0)
                        high = lanesMax(largest(y), near);
                    float const scale = scaled<A::pairs>(high, a.e5m2, y);
                    if(k < packs && live)
                    {
                        if(a.group == 0)
                        {
                            if(k == 0)
                                scales[0] = scale;
                        }
                        else if((k & ((1u << near) - 1u)) == 0)
                            scales[k >> near] = scale;
                        unsigned w[E / 4];
#pragma unroll
                        for(int e = 0; e < E / 4; ++e)
                            w[e] = eight(y[2 * e], a.e5m2) | (eight(y[2 * e + 1], a.e5m2) << 16);
                        if constexpr(E == 8)
                            *reinterpret_cast<uint2*>(out + static_cast<size_t>(k) * E) = make_uint2(w[0], w[1]);
                        else
                            *reinterpret_cast<unsigned*>(out + static_cast<size_t>(k) * E) = w[0];
                    }
                }
            }
        }

        // Short rows in great number: a team of L lanes has R of them at once, one access a lane each, so that R rows' loads
        // are under way (with one, a block waits for 2 KB).
        template<typename T, typename WT, int E, int L, int R>
        __global__ void __launch_bounds__(128) rmsNormShortKernel(NormArgs a)
        {
            using A = Access<T, E>;
            using W = Weights<WT, E>;
            constexpr uint32_t teams = 128 / L;
            uint32_t const t = threadIdx.x % L, first = blockIdx.x * (teams * R) + threadIdx.x / L;
            bool const in = t < a.n / E;
            WT const* weight = static_cast<WT const*>(a.weight);
            unsigned raw[R][1][A::words], add[R][1][A::words], wraw[W::words];
#pragma unroll
            for(int q = 0; q < R; ++q)
            {
                uint32_t const row = min(first + q * teams, a.rows - 1u);
                if(in)
                    A::load(raw[q][0], static_cast<T const*>(a.x) + a.xs.at(row, a.inner, a.one) + t * E);
                if(in && a.residual)
                    A::load(add[q][0], static_cast<T const*>(a.residual) + a.rs.at(row, a.inner, a.one) + t * E);
            }
            if(in)
                W::load(wraw, weight, t);
            float sum[R];
#pragma unroll
            for(int q = 0; q < R; ++q)
            {
                uint32_t const row = first + q * teams;
                sum[q] = addRow<T, E, 1>(a, min(row, a.rows - 1u), row < a.rows, L, t, raw[q], add[q]);
            }
#pragma unroll
            for(int q = 0; q < R; ++q)
                sum[q] = lanesSum<L>(sum[q]);
#pragma unroll
            for(int q = 0; q < R; ++q)
            {
                uint32_t const row = first + q * teams;
                float const r = rootRow<T, E, 1, L>(a, L, t, sum[q], raw[q], nullptr);
                if(row >= a.rows)
                    continue;
                if(a.rstd && t == 0)
                    a.rstd[row] = r;
                if(in)
                {
                    unsigned words[A::words];
#pragma unroll
                    for(int e = 0; e < A::pairs; ++e)
                        A::setPair(words, e, mul2(mul2(A::pair(raw[q][0], e), make_float2(r, r)), W::pair(wraw, e)));
                    A::store(static_cast<T*>(a.out) + a.os.at(row, a.inner, a.one) + t * E, words);
                }
            }
        }

        // 8-bit outputs of rows without 16-byte packs: one block a row, in registers by single elements. A warp has Q stretches of
        // 128 neighbouring elements, four a lane and each 32 apart, so every group of 32, 64 or 128 is one warp's. (By the long
        // kernel below, a group at a time, 9769 x 2587 bf16 with residual took 290 us; now 92, bound by issue: 76% of the slots, DRAM
        // at 18%.) Eight stretches (8193 to 32768 elements) do not fit 64 registers: 56 to 112 bytes a thread are in local memory.
        template<typename T, typename WT, int Q>
        __global__ void __launch_bounds__(1024, Q == 1 ? 2 : 1) rmsNormOddKernel(NormArgs a)
        {
            __shared__ float roomF[32], roomM[32];
            __shared__ double roomD[32];
            uint32_t const row = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
            T const* x = static_cast<T const*>(a.x) + a.xs.at(row, a.inner, a.one);
            T const* add = a.residual ? static_cast<T const*>(a.residual) + a.rs.at(row, a.inner, a.one) : nullptr;
            T* total = add && a.total ? static_cast<T*>(a.total) + a.ts.at(row, a.inner, a.one) : nullptr;
            WT const* weight = static_cast<WT const*>(a.weight);
            auto at = [&](int q, int e) { return (static_cast<uint32_t>(q) * warps + warp) * 128u + static_cast<uint32_t>(e) * 32u + lane; };
            float v[Q][4];
#pragma unroll
            for(int q = 0; q < Q; ++q)
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    uint32_t const k = at(q, e);
                    v[q][e] = k < a.n ? toFloat(x[k]) : 0.f;
                }
            if(add)
#pragma unroll
                for(int q = 0; q < Q; ++q)
                {
                    float other[4];
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        uint32_t const k = at(q, e);
                        other[e] = k < a.n ? toFloat(add[k]) : 0.f;
                    }
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        T const h = fromFloat<T>(v[q][e] + other[e]);
                        if(uint32_t const k = at(q, e); total && k < a.n)
                            total[k] = h;
                        v[q][e] = toFloat(h);
                    }
                }
            float sum = 0.f;
#pragma unroll
            for(int q = 0; q < Q; ++q)
#pragma unroll
                for(int e = 0; e < 4; ++e)
                    sum = fmaf(v[q][e], v[q][e], sum);
            sum = teamSum<0>(sum, roomF);
            float r;
            if(sumLost(sum, a.tiny))
            {
                double wide = 0.;
#pragma unroll
                for(int q = 0; q < Q; ++q)
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        wide = fma(static_cast<double>(v[q][e]), static_cast<double>(v[q][e]), wide);
                r = rootOf(teamSum<0>(wide, roomD), a.n, a.eps);
            }
            else
                r = rootOf(sum, a.inverse, a.eps32);
            if(a.rstd && threadIdx.x == 0)
                a.rstd[row] = r;
            float high = 0.f;
#pragma unroll
            for(int q = 0; q < Q; ++q)
            {
                float w[4];
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    uint32_t const k = at(q, e);
                    w[e] = weight && k < a.n ? toFloat(weight[k]) : 1.f;
                }
#pragma unroll
                for(int e = 0; e < 4; ++e)
                {
                    // beyond the row zero, even where r is infinite or NaN
                    v[q][e] = at(q, e) < a.n ? v[q][e] * r * w[e] : 0.f;
                    high = maxNan(high, fabsf(v[q][e]));
                }
            }
            auto* out = static_cast<unsigned char*>(a.out) + a.os.at(row, a.inner, a.one);
            float* scales = a.scales + static_cast<size_t>(row) * a.groups;
            if(a.group == 0)
                high = teamMax<0>(high, roomM);
#pragma unroll
            for(int q = 0; q < Q; ++q)
            {
                if(at(q, 0) - lane >= a.n) // the same for the warp
                    continue;
                float top[4];
                if(a.group == 0)
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        top[e] = high;
                else
                {
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        // magnitudes order as their bits do, and NaN is above infinity
                        top[e] = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(fabsf(v[q][e]))));
                    if(a.group >= 64)
                        top[0] = top[1] = maxNan(top[0], top[1]), top[2] = top[3] = maxNan(top[2], top[3]);
                    if(a.group == 128)
                        top[0] = top[1] = top[2] = top[3] = maxNan(top[0], top[2]);
                }
                float scale[4];
                float2 y[4];
#pragma unroll
                for(int e = 0; e < 4; ++e)
                    y[e] = make_float2(v[q][e], 0.f);
                if(a.group == 32)
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        scale[e] = scaled(top[e], a.e5m2, reinterpret_cast<float2(&)[1]>(y[e]));
                else
#pragma unroll
                    for(int e = 0; e < 4; e += 2)
                        scale[e] = scale[e + 1] = scaled(top[e], a.e5m2, reinterpret_cast<float2(&)[2]>(y[e]));
#pragma unroll
                for(int e = 0; e < 4; ++e)
                    if(uint32_t const k = at(q, e); k < a.n)
                    {
                        if(a.group == 0)
                        {
                            if(k == 0)
                                scales[0] = scale[e];
                        }
                        else if((k & (a.group - 1u)) == 0)
                            scales[k / 32 >> (a.group / 64)] = scale[e]; // k / group: 32, 64 or 128
                        out[k] = static_cast<unsigned char>(eight(y[e], a.e5m2));
                    }
            }
        }

        // Rows that no team holds (longer than 32768 16-bit or 16384 32-bit elements; without 16-byte packs than 16384, with 8-bit
        // outputs than 32768): one block a row, which goes over it two to four times, element by element; the later passes
        // find it in L2. The gradient's limits are half of that, below.
        constexpr uint32_t kLongThreads = 1024;

        template<typename T, typename WT>
        __global__ void __launch_bounds__(kLongThreads) rmsNormLongKernel(NormArgs a, int kind) // kind: 0 T, 1 8 bits
        {
            __shared__ float roomF[32], roomM[32];
            __shared__ double roomD[32];
            uint32_t const row = blockIdx.x, t = threadIdx.x, threads = blockDim.x;
            T const* x = static_cast<T const*>(a.x) + a.xs.at(row, a.inner, a.one);
            T const* add = a.residual ? static_cast<T const*>(a.residual) + a.rs.at(row, a.inner, a.one) : nullptr;
            T* total = a.total ? static_cast<T*>(a.total) + a.ts.at(row, a.inner, a.one) : nullptr;
            WT const* weight = static_cast<WT const*>(a.weight);
            // a sum that was stored is read back: x and residual may have given it their place
            auto value = [&](uint32_t k)
            {
                if(total && add)
                    return toFloat(total[k]);
                float const v = toFloat(x[k]);
                return add ? toFloat(fromFloat<T>(v + toFloat(add[k]))) : v;
            };
            float sum = 0.f;
#pragma unroll 8
            for(uint32_t k = t; k < a.n; k += threads)
            {
                float v = toFloat(x[k]);
                if(add)
                {
                    T const s = fromFloat<T>(v + toFloat(add[k]));
                    if(total)
                        total[k] = s;
                    v = toFloat(s);
                }
                sum = fmaf(v, v, sum);
            }
            sum = teamSum<0>(sum, roomF); // also orders the stores of `total` before the reads below
            float r;
            if(sumLost(sum, a.tiny))
            {
                double wide = 0.;
                for(uint32_t k = t; k < a.n; k += threads)
                {
                    double const v = value(k);
                    wide = fma(v, v, wide);
                }
                r = rootOf(teamSum<0>(wide, roomD), a.n, a.eps);
            }
            else
                r = rootOf(sum, a.inverse, a.eps32);
            if(a.rstd && t == 0)
                a.rstd[row] = r;
            auto y = [&](uint32_t k)
            {
                float const v = value(k) * r;
                return weight ? v * toFloat(weight[k]) : v;
            };
            if(kind == 0)
            {
                T* out = static_cast<T*>(a.out) + a.os.at(row, a.inner, a.one);
#pragma unroll 4
                for(uint32_t k = t; k < a.n; k += threads)
                    out[k] = fromFloat<T>(y(k));
                return;
            }
            auto* out = static_cast<unsigned char*>(a.out) + a.os.at(row, a.inner, a.one);
            float* scales = a.scales + static_cast<size_t>(row) * a.groups;
            if(a.group == 0)
            {
                float high = 0.f;
#pragma unroll 4
                for(uint32_t k = t; k < a.n; k += threads)
                    high = maxNan(high, fabsf(y(k)));
                high = teamMax<0>(high, roomM);
#pragma unroll 4
                for(uint32_t k = t; k < a.n; k += threads)
                {
                    float2 v[1] = {make_float2(y(k), 0.f)};
                    float const scale = scaled(high, a.e5m2, v);
                    if(k == 0)
                        scales[0] = scale;
                    out[k] = static_cast<unsigned char>(eight(v[0], a.e5m2));
                }
                return;
            }
            // a warp takes a group of 32, 64 or 128 elements
            uint32_t const warp = t / 32, lane = t % 32;
            for(uint32_t g = warp; g < a.groups; g += threads / 32)
            {
                float2 v[4];
                float high = 0.f;
#pragma unroll
                for(uint32_t e = 0; e < 4; ++e)
                {
                    uint32_t const in = e * 32 + lane, k = g * a.group + in;
                    v[e] = make_float2(in < a.group && k < a.n ? y(k) : 0.f, 0.f);
                    high = maxNan(high, fabsf(v[e].x));
                }
                float const scale = scaled(lanesMax(high, 5), a.e5m2, v);
                if(lane == 0)
                    scales[g] = scale;
#pragma unroll
                for(uint32_t e = 0; e < 4; ++e)
                    if(uint32_t const in = e * 32 + lane, k = g * a.group + in; in < a.group && k < a.n)
                        out[k] = static_cast<unsigned char>(eight(v[e], a.e5m2));
            }
        }

        uint32_t roundUp(uint32_t v, uint32_t to)
        {
            return (v + to - 1) / to * to;
        }

        template<typename T, typename WT, bool F8>
        int launchNorm(cudaStream_t stream, DeviceProps const* props, NormArgs const& a, bool packed)
        {
            constexpr int E = PackOf<T>::E;
            auto teams = [&](uint32_t lanes) { return (a.rows + 128 / lanes - 1) / (128 / lanes); };
            if(packed)
            {
                uint32_t const packs = a.n / E;
                bool const many = a.rows >= 4u * static_cast<uint32_t>(props->smCount);
                // Two rows a team where that leaves eight blocks an SM (65536 x 128 bf16 8.2 us, 9.2 with one, 8.8 with four; but
                // 4096 x 128 2.5, 2.1 with one).
                uint32_t const part = packs <= 8 ? 8 : packs <= 16 ? 16 : 32, pairBlocks = (a.rows + 256 / part - 1) / (256 / part);
                if(!F8 && packs <= 32 && pairBlocks >= 8u * static_cast<uint32_t>(props->smCount))
                {
                    if(part == 8)
                        rmsNormShortKernel<T, WT, E, 8, 2><<<pairBlocks, 128, 0, stream>>>(a);
                    else if(part == 16)
                        rmsNormShortKernel<T, WT, E, 16, 2><<<pairBlocks, 128, 0, stream>>>(a);
                    else
                        rmsNormShortKernel<T, WT, E, 32, 2><<<pairBlocks, 128, 0, stream>>>(a);
                }
                else if(!F8 && packs <= 8 && many)
                    rmsNormKernel<T, WT, E, 1, F8 ? 32 : 8, F8><<<teams(8), 128, 0, stream>>>(a);
                else if(!F8 && packs <= 16 && many)
                    rmsNormKernel<T, WT, E, 1, F8 ? 32 : 16, F8><<<teams(16), 128, 0, stream>>>(a);
                else if(packs <= 32)
                    rmsNormKernel<T, WT, E, 1, 32, F8><<<teams(32), 128, 0, stream>>>(a);
                else if(packs <= 64 && many)
                    rmsNormKernel<T, WT, E, 2, 32, F8><<<teams(32), 128, 0, stream>>>(a);
                else if(packs <= 128 && many)
                    rmsNormKernel<T, WT, E, 4, 32, F8><<<teams(32), 128, 0, stream>>>(a);
                else if(packs <= 1024 && !many)
                    rmsNormKernel<T, WT, E, 1, 0, F8><<<a.rows, roundUp(packs, 32), 0, stream>>>(a);
                else if(packs <= 1024)
                    rmsNormKernel<T, WT, E, 2, 0, F8><<<a.rows, roundUp((packs + 1) / 2, 32), 0, stream>>>(a);
                else if(packs <= 4096)
                    rmsNormKernel<T, WT, E, 4, 0, F8><<<a.rows, roundUp((packs + 3) / 4, 32), 0, stream>>>(a);
                else
                    rmsNormLongKernel<T, WT><<<a.rows, kLongThreads, 0, stream>>>(a, F8);
            }
            else if constexpr(!F8)
            {
                if(a.n <= 2048)
                    rmsNormKernel<T, WT, 1, 4, 0, false><<<a.rows, roundUp((a.n + 3) / 4, 32), 0, stream>>>(a);
                else if(a.n <= 16384)
                    rmsNormKernel<T, WT, 1, 16, 0, false><<<a.rows, roundUp((a.n + 15) / 16, 32), 0, stream>>>(a);
                else
                    rmsNormLongKernel<T, WT><<<a.rows, kLongThreads, 0, stream>>>(a, 0);
            }
            else
            {
                auto threads = [&](uint32_t stretches) { return (a.n + 128 * stretches - 1) / (128 * stretches) * 32; };
                // One stretch a warp, 32 registers: with a residual 4000 x 4001 fp32 58 us, with two stretches 61, 9769 x 2587 bf16 92 and
                // 100; without one 50 and 44, 73 and 69.
                if(a.n <= 4096)
                    rmsNormOddKernel<T, WT, 1><<<a.rows, threads(1), 0, stream>>>(a);
                else if(a.n <= 8192)
                    rmsNormOddKernel<T, WT, 2><<<a.rows, threads(2), 0, stream>>>(a);
                else if(a.n <= 32768)
                    rmsNormOddKernel<T, WT, 8><<<a.rows, threads(8), 0, stream>>>(a);
                else
                    rmsNormLongKernel<T, WT><<<a.rows, kLongThreads, 0, stream>>>(a, 1);
            }
            A3B_CHECK_LAUNCH("rmsNormKernel");
            return A3B_OK;
        }

        // --------------------------------------------------------------------------------------------- backward
        struct NormBackArgs
        {
            void const* g;
            void const* x;
            void const* gtotal; // may be null
            void* gx;
            RowStep gs, xs, ts, os;
            uint32_t rows, inner, n;
            bool one;
            void const* weight; // may be null
            float const* rstd;
            float* partial; // one row of n sums a block; null: no gradient of the weight
            float inverse; // 1 / n
            uint32_t team; // threads of a team
            void* gw; // a single block writes the weight's gradient itself; else null
        };

        // The block's row of partial sums (or the weight's gradient, if it is the only block) from its teams', added in the
        // teams' order: the same bits every time.
        template<typename WT, int E, int P>
        __device__ __forceinline__ void addTeams(NormBackArgs const& a, float2 const (&dw)[P][E == 1 ? 1 : E / 2], float* sums,
                                                 uint32_t teams, uint32_t mine, uint32_t lanes, uint32_t t)
        {
            float* partial = a.partial + static_cast<size_t>(blockIdx.x) * a.n;
            auto put = [&](uint32_t k, float v)
            {
                if(a.gw)
                    static_cast<WT*>(a.gw)[k] = fromFloat<WT>(v);
                else
                    partial[k] = v;
            };
#pragma unroll
            for(int p = 0; p < P; ++p)
                if(uint32_t const k = p * lanes + t; k < a.n / E)
#pragma unroll
                    for(int e = 0; e < E; ++e)
                    {
                        float const v = e % 2 ? dw[p][e / 2].y : dw[p][e / 2].x;
                        if(teams == 1)
                            put(k * E + e, v);
                        else
                            sums[mine * a.n + k * E + e] = v;
                    }
            if(teams == 1)
                return;
            __syncthreads();
            for(uint32_t k = threadIdx.x; k < a.n; k += blockDim.x)
            {
                float v = sums[k];
#pragma unroll 4
                for(uint32_t of = 1; of < teams; ++of)
                    v += sums[of * a.n + k];
                put(k, v);
            }
        }

        // Teams go from row to row, a lane always at the same columns, so that the weight's gradient gathers in registers. A
        // team is L lanes of a warp, or (L = 0) a.team threads, several in a block of up to 512, which adds up theirs and writes
        // one row of partial sums. As in the forward pass a row is held as the words it is stored in: with 64 registers a
        // thread two blocks of 512 share an SM, and one team's loads run under the others' sums.
        template<typename T, typename WT, int E, int P, int L>
        __global__ void __launch_bounds__(512, P <= 2 ? 2 : 1) rmsNormBackwardKernel(NormBackArgs a)
        {
            using A = Access<T, E>;
            using W = Weights<WT, E>;
            constexpr bool held = P * W::words < 8; // weights in registers; more of them spill: then from L1 row by row
            __shared__ float room[2][16];
            extern __shared__ float sums[];
            uint32_t const lanes = L > 0 ? L : a.team, mine = threadIdx.x / lanes, t = threadIdx.x - mine * lanes;
            uint32_t const teams = blockDim.x / lanes, packs = a.n / E, step = gridDim.x * teams;
            WT const* weight = static_cast<WT const*>(a.weight);
            unsigned wraw[held ? P : 1][W::words];
            float2 dw[P][A::pairs];
#pragma unroll
            for(int p = 0; p < P; ++p)
            {
                if(uint32_t const k = p * lanes + t; held && k < packs)
                    W::load(wraw[held ? p : 0], weight, k);
#pragma unroll
                for(int e = 0; e < A::pairs; ++e)
                    dw[p][e] = make_float2(0.f, 0.f);
            }
            uint32_t row = blockIdx.x * teams + mine, turn = 0;
            // lanes of one warp that belong to two teams make the same number of steps
            for(uint32_t first = L > 0 ? blockIdx.x * teams : row; first < a.rows; first += step, row += step, ++turn)
            {
                bool const live = L == 0 || row < a.rows;
                uint32_t const here = live ? row : a.rows - 1u;
                T const* g = static_cast<T const*>(a.g) + a.gs.at(here, a.inner, a.one);
                T const* x = static_cast<T const*>(a.x) + a.xs.at(here, a.inner, a.one);
                T const* gt = a.gtotal ? static_cast<T const*>(a.gtotal) + a.ts.at(here, a.inner, a.one) : nullptr;
                float const r = live ? a.rstd[here] : 0.f;
                unsigned graw[P][A::words], xraw[P][A::words], traw[P][A::words];
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs && live)
                    {
                        A::load(graw[p], g + static_cast<size_t>(k) * E);
                        A::load(xraw[p], x + static_cast<size_t>(k) * E);
                    }
                if(gt)
#pragma unroll
                    for(int p = 0; p < P; ++p)
                        if(uint32_t const k = p * lanes + t; k < packs && live)
                            A::load(traw[p], gt + static_cast<size_t>(k) * E);
                auto weighted = [&](int p, int e) { return mul2(A::pair(graw[p], e), W::pair(wraw[held ? p : 0], e)); }; // d = g w
                float2 c2 = make_float2(0.f, 0.f);
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs && live)
                    {
                        if(!held)
                            W::load(wraw[0], weight, k);
#pragma unroll
                        for(int e = 0; e < A::pairs; ++e)
                        {
                            float2 const hat = mul2(A::pair(xraw[p], e), make_float2(r, r));
                            dw[p][e] = fma2(A::pair(graw[p], e), hat, dw[p][e]);
                            c2 = fma2(weighted(p, e), hat, c2);
                        }
                    }
                float c = c2.x + c2.y;
                if constexpr(L > 0)
                    c = lanesSum<L>(c);
                else
                {
                    c = lanesSum<32>(c);
                    uint32_t const warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = lanes / 32;
                    if(lane == 0)
                        room[turn & 1][warp] = c;
                    // A barrier for each team, 1 to 8, since one has two warps or more (there are 16 barriers, the block's is 0).
                    asm volatile("bar.sync %0, %1;" ::"r"(mine + 1u), "r"(lanes) : "memory");
                    c = lanesSum<32>(lane < warps ? room[turn & 1][mine * warps + lane] : 0.f);
                }
                c *= a.inverse;
                if(!live)
                    continue;
                T* gx = static_cast<T*>(a.gx) + a.os.at(here, a.inner, a.one);
#pragma unroll
                for(int p = 0; p < P; ++p)
                    if(uint32_t const k = p * lanes + t; k < packs)
                    {
                        if(!held)
                            W::load(wraw[0], weight, k);
                        unsigned raw[A::words];
                        float2 d[A::pairs];
#pragma unroll
                        for(int e = 0; e < A::pairs; ++e)
                        {
                            float2 const hat = mul2(A::pair(xraw[p], e), make_float2(-r, -r));
                            d[e] = mul2(fma2(hat, make_float2(c, c), weighted(p, e)), make_float2(r, r));
                        }
                        if(gt)
#pragma unroll
                            for(int e = 0; e < A::pairs; ++e)
                                d[e] = add2(d[e], A::pair(traw[p], e));
#pragma unroll
                        for(int e = 0; e < A::pairs; ++e)
                            A::setPair(raw, e, d[e]);
                        A::store(gx + static_cast<size_t>(k) * E, raw);
                    }
            }
            if(a.partial)
            {
                if(!a.gw)
                    signalNext(); // the fold
                addTeams<WT, E, P>(a, dw, sums, teams, mine, lanes, t);
            }
        }

        // Rows that no team holds (longer than 16384 16-bit or 8192 32-bit elements; without 16-byte packs than 8192): two passes over
        // the row for its gradient ...
        template<typename T, typename WT>
        __global__ void __launch_bounds__(kLongThreads) rmsNormBackwardLongKernel(NormBackArgs a)
        {
            __shared__ float roomF[32];
            uint32_t const row = blockIdx.x, t = threadIdx.x, threads = blockDim.x;
            T const* g = static_cast<T const*>(a.g) + a.gs.at(row, a.inner, a.one);
            T const* x = static_cast<T const*>(a.x) + a.xs.at(row, a.inner, a.one);
            T const* gt = a.gtotal ? static_cast<T const*>(a.gtotal) + a.ts.at(row, a.inner, a.one) : nullptr;
            T* gx = static_cast<T*>(a.gx) + a.os.at(row, a.inner, a.one);
            WT const* weight = static_cast<WT const*>(a.weight);
            float const r = a.rstd[row];
            float c = 0.f;
#pragma unroll 8
            for(uint32_t k = t; k < a.n; k += threads)
                c = fmaf(toFloat(g[k]) * (weight ? toFloat(weight[k]) : 1.f), toFloat(x[k]) * r, c);
            c = teamSum<0>(c, roomF) * a.inverse;
#pragma unroll 8
            for(uint32_t k = t; k < a.n; k += threads)
            {
                float const d = r * fmaf(-toFloat(x[k]) * r, c, toFloat(g[k]) * (weight ? toFloat(weight[k]) : 1.f));
                gx[k] = fromFloat<T>(gt ? d + toFloat(gt[k]) : d);
            }
        }

        // ... and, in front of it (gx may be g or x), the weight's: a block sums 32 columns over a share of the rows.
        template<typename T>
        __global__ void __launch_bounds__(256) rmsNormWeightKernel(NormBackArgs a)
        {
            __shared__ float part[8][32];
            uint32_t const lane = threadIdx.x % 32, warp = threadIdx.x / 32, k = blockIdx.x * 32 + lane;
            float s = 0.f;
            if(k < a.n)
#pragma unroll 4
                for(uint32_t row = blockIdx.y * 8 + warp; row < a.rows; row += gridDim.y * 8)
                {
                    float const g = toFloat(static_cast<T const*>(a.g)[a.gs.at(row, a.inner, a.one) + k]);
                    float const x = toFloat(static_cast<T const*>(a.x)[a.xs.at(row, a.inner, a.one) + k]);
                    s = fmaf(g, x * a.rstd[row], s);
                }
            part[warp][lane] = s;
            __syncthreads();
            if(warp == 0 && k < a.n)
            {
#pragma unroll
                for(int w = 1; w < 8; ++w)
                    s += part[w][lane];
                a.partial[static_cast<size_t>(blockIdx.y) * a.n + k] = s;
            }
        }

        // dw = the sum of the partial rows, in their order within and over the warps: a block has 32 columns, its warps
        // every 32nd row.
        template<typename WT>
        __global__ void __launch_bounds__(1024) rmsNormFoldKernel(float const* partial, uint32_t count, uint32_t n, WT* out)
        {
            __shared__ float part[32][33];
            uint32_t const lane = threadIdx.x % 32, warp = threadIdx.x / 32, k = blockIdx.x * 32 + lane;
            waitForPrevious();
            float s = 0.f;
            if(k < n)
#pragma unroll 10
                for(uint32_t row = warp; row < count; row += 32)
                    s += __ldcg(partial + static_cast<size_t>(row) * n + k);
            part[warp][lane] = s;
            __syncthreads();
            s = lanesSum<32>(part[lane][warp]); // now the warp has one column
            if(lane == 0 && blockIdx.x * 32 + warp < n)
                out[blockIdx.x * 32 + warp] = fromFloat<WT>(s);
        }

        // rows of partial sums at most, whatever a call's alignment: four blocks an SM
        uint32_t partialRows(DeviceProps const* props, uint64_t rows)
        {
            return static_cast<uint32_t>(std::min<uint64_t>(rows, 4ull * static_cast<unsigned>(props->smCount)));
        }

        // How many rows of partial sums the fold has to add; none when a single block wrote the weight's gradient.
        template<typename T, typename WT, int E, int P, int L>
        uint32_t launchBackwardTeams(cudaStream_t stream, DeviceProps const* props, NormBackArgs a, WT* gw)
        {
            auto const sms = static_cast<uint32_t>(props->smCount);
            a.team = L > 0 ? L : std::max(64u, roundUp((a.n / E + P - 1) / P, 32)); // several warps: a barrier each
            // Teams side by side in a block, unless SMs would go without. Rows that one block takes in one turn are left to it: it
            // needs no fold (1 x 4096 bf16 3.9 us, with two launches 5.6; with a second turn 6.7 against 5.7).
            uint32_t const most = 512 / a.team;
            bool const single = gw && a.rows <= most;
            uint32_t const teams = std::max(1u, std::min(most, L > 0 ? most : single ? a.rows : a.rows / sms));
            uint32_t const threads = teams * a.team, resident = std::max(1u, (P <= 2 ? 1024u : 512u) / threads);
            uint32_t const blocks
                = single ? 1 : std::min({(a.rows + teams - 1) / teams, sms * resident, partialRows(props, a.rows)});
            a.gw = single ? gw : nullptr;
            // a row of sums for each team: at most threads * P * E values, 32 KB
            size_t const sums = a.partial && teams > 1 ? teams * a.n * sizeof(float) : 0;
            rmsNormBackwardKernel<T, WT, E, P, L><<<blocks, threads, sums, stream>>>(a);
            return single ? 0 : blocks;
        }

        template<typename T, typename WT>
        int launchNormBackward(cudaStream_t stream, DeviceProps const* props, NormBackArgs const& a, bool packed, WT* gw)
        {
            constexpr int E = PackOf<T>::E;
            uint32_t const packs = packed ? a.n / E : a.n;
            uint32_t blocks = 0;
            if(packed && packs <= 16)
                blocks = launchBackwardTeams<T, WT, E, 2, 8>(stream, props, a, gw);
            else if(packed && packs <= 32)
                blocks = launchBackwardTeams<T, WT, E, 2, 16>(stream, props, a, gw);
            else if(packed && packs <= 64)
                blocks = launchBackwardTeams<T, WT, E, 2, 32>(stream, props, a, gw);
            else if(packed && packs <= 1024)
                blocks = launchBackwardTeams<T, WT, E, 2, 0>(stream, props, a, gw);
            else if(packed && packs <= 2048)
                blocks = launchBackwardTeams<T, WT, E, 4, 0>(stream, props, a, gw);
            else if(!packed && packs <= 128) // a warp, without a barrier (29861 x 101 bf16 16.2 us; asking for it in the loop: 17.9)
                blocks = launchBackwardTeams<T, WT, 1, 4, 32>(stream, props, a, gw);
            else if(!packed && packs <= 2048)
                blocks = launchBackwardTeams<T, WT, 1, 4, 0>(stream, props, a, gw);
            else if(!packed && packs <= 8192)
                blocks = launchBackwardTeams<T, WT, 1, 16, 0>(stream, props, a, gw);
            else
            {
                blocks = std::min(64u, std::max(1u, a.rows / 64)); // eight rows a warp and more
                if(a.partial)
                    rmsNormWeightKernel<T><<<dim3((a.n + 31) / 32, blocks), 256, 0, stream>>>(a);
                rmsNormBackwardLongKernel<T, WT><<<a.rows, kLongThreads, 0, stream>>>(a);
            }
            A3B_CHECK_LAUNCH("rmsNormBackwardKernel");
            if(a.partial && blocks > 0)
            {
                return launchNext(stream, rmsNormFoldKernel<WT>, dim3((a.n + 31) / 32), 1024, 0, a.partial, blocks, a.n, gw);
            }
            return A3B_OK;
        }

        // ------------------------------------------------------------------------------------------ arguments
        int checkShape(int dtype, uint64_t outer, uint64_t inner, uint64_t n, double eps)
        {
            A3B_REQUIRE(rowTypeSize(dtype) != 0, "rows must be f32, f16 or bf16");
            A3B_REQUIRE(n > 0, "a row needs at least one element");
            A3B_REQUIRE(eps >= 0 && eps <= 0x1p100, "eps must lie between 0 and 2^100");
            A3B_REQUIRE(outer == 0 || inner <= UINT64_MAX / outer, "rows overflow");
            if(n > static_cast<uint64_t>(INT_MAX) - 64 || outer * inner > static_cast<uint64_t>(INT_MAX))
            {
                setError("at most 2^31 - 1 rows of 2^31 - 65 elements");
                return A3B_ERR_TOO_LARGE;
            }
            return A3B_OK;
        }
    } // namespace
} // namespace a3b

using namespace a3b;

extern "C"
{
    int a3b_rms_norm(a3b_stream_t stream, a3b_rms_norm_args const* args)
    {
        A3B_REQUIRE(args, "null arguments");
        uint64_t const outer = args->outer, inner = args->inner, n = args->n;
        int const dtype = args->dtype, out_dtype = args->out_dtype, weight_dtype = args->weight_dtype;
        a3b_rows const &x = args->x, &residual = args->residual, &total = args->total, &out = args->out;
        void const* weight = args->weight;
        float *rstd = args->rstd, *scales = args->scales;
        double const eps = args->eps;
        uint32_t const group = args->group;
        int const rc = checkShape(dtype, outer, inner, n, eps);
        if(rc != A3B_OK)
            return rc;
        bool const eightBits = out_dtype == A3B_E4M3 || out_dtype == A3B_E5M2;
        A3B_REQUIRE(out_dtype == dtype || eightBits, "the output has the rows' type, e4m3 or e5m2");
        A3B_REQUIRE(!weight || weight_dtype == dtype || weight_dtype == A3B_F32, "the weight has the rows' type or f32");
        A3B_REQUIRE(group == 0 || (eightBits && (group == 32 || group == 64 || group == 128)),
                    "groups of 8-bit outputs have 32, 64 or 128 elements");
        if(outer * inner == 0)
            return A3B_OK;
        A3B_REQUIRE(x.data && out.data, "null rows or output");
        A3B_REQUIRE(!total.data || residual.data, "a sum needs a residual");
        A3B_REQUIRE(eightBits == (scales != nullptr), "scales belong to 8-bit outputs");
        int const es = rowTypeSize(dtype), os = eightBits ? 1 : es, ws = weight_dtype == A3B_F32 ? 4 : 2;
        A3B_REQUIRE(alignedTo(es, {x.data, residual.data, total.data}) && alignedTo(os, {out.data}) && alignedTo(ws, {weight})
                        && alignedTo(4, {rstd, scales}),
                    "an array is not aligned to its type");
        uint64_t const rows = outer * inner, groups = group ? (n + group - 1) / group : 1;
        Stretch const sx = Stretch::rows(x, outer, inner, n, es);
        Stretch const sr = Stretch::rows(residual, outer, inner, n, es);
        Stretch const st = Stretch::rows(total, outer, inner, n, es);
        Stretch const so = Stretch::rows(out, outer, inner, n, os);
        Stretch const sw = Stretch::dense(weight, static_cast<Wide>(n) * ws);
        Stretch const s1 = Stretch::dense(rstd, static_cast<Wide>(rows) * 4);
        Stretch const s8 = Stretch::dense(scales, static_cast<Wide>(rows) * groups * 4);
        A3B_REQUIRE(so.separate() && (!total.data || st.separate()), "rows of an output overlap");
        for(Stretch const* w : {&so, &st})
            for(Stretch const* r : {&sx, &sr})
                A3B_REQUIRE(w->empty() || w->sameAs(*r) || w->apart(*r),
                            "an output overlaps its inputs (only the same rows in place are allowed)");
        A3B_REQUIRE(so.apart(st), "the outputs overlap");
        for(Stretch const* w : {&so, &st, &s1, &s8})
            A3B_REQUIRE(w->apart(sw), "an output overlaps the weight");
        for(Stretch const* w : {&sx, &sr, &st, &so})
            A3B_REQUIRE(w->apart(s1) && w->apart(s8), "rows overlap rstd or the scales");
        A3B_REQUIRE(s1.apart(s8), "the outputs overlap");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        int const E = 16 / es;
        auto fits = [&](a3b_rows const& r, int size, int to)
        { return !r.data || rowsAligned(r.data, outer, inner, r.outer_stride, r.inner_stride, size, to); };
        bool const packed = n % E == 0 && fits(x, es, 16)
                            && fits(residual, es, 16)
                            && fits(total, es, 16)
                            && fits(out, os, eightBits ? E : 16) && alignedTo(16, {weight});
        bool const one = outer == 1;
        NormArgs a{x.data, residual.data, total.data, out.data, {x.outer_stride, x.inner_stride}, {residual.outer_stride, residual.inner_stride},
                   {total.outer_stride, total.inner_stride}, {out.outer_stride, out.inner_stride},
                   static_cast<uint32_t>(rows), static_cast<uint32_t>(inner), static_cast<uint32_t>(n), one, weight, rstd,
                   scales, group, static_cast<uint32_t>(groups), out_dtype == A3B_E5M2, eps, static_cast<float>(eps),
                   1.f / static_cast<float>(n), eps < 0x1p-60};
        auto s = static_cast<cudaStream_t>(stream);
        bool const wide = weight && weight_dtype == A3B_F32;
        if(dtype == A3B_F32)
            return eightBits ? launchNorm<float, float, true>(s, props, a, packed)
                             : launchNorm<float, float, false>(s, props, a, packed);
        if(dtype == A3B_F16)
        {
            if(wide)
                return eightBits ? launchNorm<__half, float, true>(s, props, a, packed)
                                 : launchNorm<__half, float, false>(s, props, a, packed);
            return eightBits ? launchNorm<__half, __half, true>(s, props, a, packed)
                             : launchNorm<__half, __half, false>(s, props, a, packed);
        }
        if(wide)
            return eightBits ? launchNorm<__nv_bfloat16, float, true>(s, props, a, packed)
                             : launchNorm<__nv_bfloat16, float, false>(s, props, a, packed);
        return eightBits ? launchNorm<__nv_bfloat16, __nv_bfloat16, true>(s, props, a, packed)
                         : launchNorm<__nv_bfloat16, __nv_bfloat16, false>(s, props, a, packed);
    }

    size_t a3b_rms_norm_backward_workspace(uint64_t rows, uint64_t n)
    {
        DeviceProps const* props = nullptr;
        if(currentDevice(&props) != A3B_OK)
            return 0;
        if(rows == 0 || n == 0 || n > static_cast<uint64_t>(INT_MAX) || rows > static_cast<uint64_t>(INT_MAX))
            return 16;
        return std::max<size_t>(16, static_cast<size_t>(partialRows(props, rows)) * n * sizeof(float));
    }

    int a3b_rms_norm_backward(a3b_stream_t stream, a3b_rms_norm_backward_args const* args)
    {
        A3B_REQUIRE(args, "null arguments");
        uint64_t const outer = args->outer, inner = args->inner, n = args->n;
        int const dtype = args->dtype, weight_dtype = args->weight_dtype, grad_weight_dtype = args->grad_weight_dtype;
        a3b_rows const &grad_out = args->grad_out, &x = args->x, &grad_total = args->grad_total, &grad_x = args->grad_x;
        void const* weight = args->weight;
        float const* rstd = args->rstd;
        void *grad_weight = args->grad_weight, *workspace = args->workspace;
        uint64_t const workspace_bytes = args->workspace_bytes;
        int const rc = checkShape(dtype, outer, inner, n, 0.);
        if(rc != A3B_OK)
            return rc;
        A3B_REQUIRE(!weight || weight_dtype == dtype || weight_dtype == A3B_F32, "the weight has the rows' type or f32");
        A3B_REQUIRE(!grad_weight || grad_weight_dtype == dtype || grad_weight_dtype == A3B_F32,
                    "the weight's gradient has the rows' type or f32");
        A3B_REQUIRE(!grad_weight || !weight || grad_weight_dtype == weight_dtype, "the weight's gradient has the weight's type");
        auto s = static_cast<cudaStream_t>(stream);
        int const es = rowTypeSize(dtype), ws = (weight ? weight_dtype : grad_weight_dtype) == A3B_F32 ? 4 : 2;
        A3B_REQUIRE(alignedTo(ws, {weight, grad_weight}), "an array is not aligned to its type");
        if(outer * inner == 0)
        {
            if(grad_weight) // the sum over no rows
                A3B_CUDA(cudaMemsetAsync(grad_weight, 0, n * static_cast<size_t>(ws), s));
            return A3B_OK;
        }
        A3B_REQUIRE(grad_out.data && x.data && grad_x.data && rstd, "null rows, rstd or output");
        A3B_REQUIRE(alignedTo(es, {grad_out.data, x.data, grad_total.data, grad_x.data}) && alignedTo(4, {rstd}), "an array is not aligned to its type");
        uint64_t const rows = outer * inner;
        Stretch const sg = Stretch::rows(grad_out, outer, inner, n, es);
        Stretch const sx = Stretch::rows(x, outer, inner, n, es);
        Stretch const st = Stretch::rows(grad_total, outer, inner, n, es);
        Stretch const so = Stretch::rows(grad_x, outer, inner, n, es);
        Stretch const sw = Stretch::dense(weight, static_cast<Wide>(n) * ws);
        Stretch const sd = Stretch::dense(grad_weight, static_cast<Wide>(n) * ws);
        Stretch const s1 = Stretch::dense(rstd, static_cast<Wide>(rows) * 4);
        Stretch const s2 = Stretch::dense(grad_weight ? workspace : nullptr, static_cast<Wide>(workspace_bytes));
        A3B_REQUIRE(so.separate(), "rows of grad_x overlap");
        for(Stretch const* r : {&sg, &sx, &st})
        {
            A3B_REQUIRE(r->empty() || so.sameAs(*r) || so.apart(*r),
                        "grad_x overlaps its inputs (only the same rows in place are allowed)");
            A3B_REQUIRE(r->apart(sd) && r->apart(s2), "the weight's gradient or the workspace overlaps the rows");
        }
        A3B_REQUIRE(so.apart(sd) && so.apart(s2) && so.apart(sw) && so.apart(s1) && sd.apart(sw) && sd.apart(s1) && sd.apart(s2)
                        && s2.apart(sw) && s2.apart(s1),
                    "outputs and workspace must lie apart from one another, the weight and rstd");
        DeviceProps const* props = nullptr;
        int const rd = currentDevice(&props);
        if(rd != A3B_OK)
            return rd;
        A3B_REQUIRE(!grad_weight || (workspace && alignedTo(16, {workspace})
                                     && workspace_bytes >= a3b_rms_norm_backward_workspace(rows, n)),
                    "the workspace is missing, too small or not aligned to 16 bytes");
        int const E = 16 / es;
        auto fits = [&](a3b_rows const& r)
        { return !r.data || rowsAligned(r.data, outer, inner, r.outer_stride, r.inner_stride, es, 16); };
        bool const packed = n % E == 0 && fits(grad_out)
                            && fits(x)
                            && fits(grad_total)
                            && fits(grad_x) && alignedTo(16, {weight});
        NormBackArgs a{grad_out.data, x.data, grad_total.data, grad_x.data, {grad_out.outer_stride, grad_out.inner_stride},
                       {x.outer_stride, x.inner_stride}, {grad_total.outer_stride, grad_total.inner_stride},
                       {grad_x.outer_stride, grad_x.inner_stride}, static_cast<uint32_t>(rows), static_cast<uint32_t>(inner),
                       static_cast<uint32_t>(n), outer == 1, weight, rstd,
                       grad_weight ? static_cast<float*>(workspace) : nullptr, 1.f / static_cast<float>(n), 0u, nullptr};
        bool const wide = ws == 4;
        if(dtype == A3B_F32)
            return launchNormBackward<float, float>(s, props, a, packed, static_cast<float*>(grad_weight));
        if(dtype == A3B_F16)
            return wide ? launchNormBackward<__half, float>(s, props, a, packed, static_cast<float*>(grad_weight))
                        : launchNormBackward<__half, __half>(s, props, a, packed, static_cast<__half*>(grad_weight));
        return wide ? launchNormBackward<__nv_bfloat16, float>(s, props, a, packed, static_cast<float*>(grad_weight))
                    : launchNormBackward<__nv_bfloat16, __nv_bfloat16>(s, props, a, packed, static_cast<__nv_bfloat16*>(grad_weight));
    }
}
