// A 64 x 64 tile of a matrix product on the FMA pipes, for operands of any type and any strides.
#pragma once
#include "fitnet.cuh"

namespace ai2b {

// C[i][j] = sum_k A[i][k] B[j][k] for a 64 x 64 tile of C, 256 threads with 4 x 4 sums each. Any strides: what the tensor-core
// kernels do not take comes here.
constexpr int FT = 64, FK = 16;

template <typename T>
struct Operand {
    const T *p;
    long long si, sk;         // strides of the tile's index and of the summed index
    long long ni, nk;         // their extents
};

template <typename TA, typename TB>
__device__ __forceinline__ void fma_tile(float (&acc)[4][4], const Operand<TA> &A, const Operand<TB> &B, long long i0, long long j0, float (*As)[FT + 4], float (*Bs)[FT + 4])
{
    const int tid = threadIdx.x, ti = tid / 16, tj = tid % 16;
    for (long long k0 = 0; k0 < A.nk; k0 += FK) {
#pragma unroll
        for (int u = 0; u < FT * FK / 256; u++) {
            const int e = tid + 256 * u;
            // neighbouring threads along the direction that is contiguous in memory
            const int ia = A.sk == 1 ? e / FK : e % FT, ka = A.sk == 1 ? e % FK : e / FT;
            const int jb = B.sk == 1 ? e / FK : e % FT, kb = B.sk == 1 ? e % FK : e / FT;
            As[ka][ia] = i0 + ia < A.ni && k0 + ka < A.nk ? to_float(A.p[(i0 + ia) * A.si + (k0 + ka) * A.sk]) : 0.f;
            Bs[kb][jb] = j0 + jb < B.ni && k0 + kb < B.nk ? to_float(B.p[(j0 + jb) * B.si + (k0 + kb) * B.sk]) : 0.f;
        }
        __syncthreads();
#pragma unroll
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
