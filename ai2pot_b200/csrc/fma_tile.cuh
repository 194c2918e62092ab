// A 64 x 64 tile of a matrix product on the FMA pipes, for operands of any type and any strides.
#pragma once
#include "fitnet.cuh"

namespace ai2b {

// C[i][j] = sum_k A[i][k] B[j][k] for a 64 x 64 tile of C, 256 threads with 4 x 4 sums each. Any strides: what the tensor-core
// kernels do not take comes here.
constexpr int FT = 64, FK = 32;

template <typename T>
struct Operand {
    const T *p;
    long long si, sk;         // strides of the tile's index and of the summed index
    long long ni, nk;         // their extents
};

// This thread's eight elements of a 64 x 32 piece: neighbouring threads along the direction that is contiguous in memory
template <typename T>
__device__ __forceinline__ void fma_fetch(float (&v)[FT * FK / 256], const Operand<T> &o, long long i0, long long k0)
{
#pragma unroll
    for (int u = 0; u < FT * FK / 256; u++) {
        const int e = threadIdx.x + 256 * u, i = o.sk == 1 ? e / FK : e % FT, k = o.sk == 1 ? e % FK : e / FT;
        v[u] = i0 + i < o.ni && k0 + k < o.nk ? to_float(o.p[(i0 + i) * o.si + (k0 + k) * o.sk]) : 0.f;
    }
}
__device__ __forceinline__ void fma_put(float (*s)[FT + 4], const float (&v)[FT * FK / 256], bool k_contiguous)
{
#pragma unroll
    for (int u = 0; u < FT * FK / 256; u++) {
        const int e = threadIdx.x + 256 * u;
        s[k_contiguous ? e % FK : e / FT][k_contiguous ? e / FK : e % FT] = v[u];
    }
}

// The next piece is on its way from memory while this one is multiplied.
template <typename TA, typename TB>
__device__ __forceinline__ void fma_tile(float (&acc)[4][4], const Operand<TA> &A, const Operand<TB> &B, long long i0, long long j0, float (*As)[FT + 4], float (*Bs)[FT + 4])
{
    const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    float a_next[FT * FK / 256], b_next[FT * FK / 256];
    if (A.nk > 0) {
        fma_fetch(a_next, A, i0, 0);
        fma_fetch(b_next, B, j0, 0);
    }
    for (long long k0 = 0; k0 < A.nk; k0 += FK) {
        fma_put(As, a_next, A.sk == 1);
        fma_put(Bs, b_next, B.sk == 1);
        __syncthreads();
        if (k0 + FK < A.nk) {
            fma_fetch(a_next, A, i0, k0 + FK);
            fma_fetch(b_next, B, j0, k0 + FK);
        }
#pragma unroll 8
        for (int k = 0; k < FK; k++) {
            const float4 a = *reinterpret_cast<const float4 *>(&As[k][4 * ti]), b = *reinterpret_cast<const float4 *>(&Bs[k][4 * tj]);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
}

}  // namespace ai2b
