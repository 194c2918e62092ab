// Newton-Schulz orthogonalisation of a batch of matrices G[b][m][n]:
//
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  X = a X + (b A + c A A) X      (m <= n; else A = X^T X and X = a X + X (b A + c A A))
//
// The iteration acts on each singular value alone, sigma -> a sigma + b sigma^3 + c sigma^5, so X is carried in float: what a rounding
// of X adds to directions of small singular values is multiplied by up to a^steps.
#include "fitnet.cuh"
#include "fma_tile.cuh"

namespace ai2b {

constexpr int NORM_BLOCKS = 64;           // partial sums of squares per matrix

// Squares are added in double: G may hold any float
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(const T *__restrict__ g, long long size, double *__restrict__ part)
{
    __shared__ double sums[8];
    chain_wait();
    chain_release();
    const T *mine = g + blockIdx.y * size;
    double sum = 0.0;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < size; i += (long long)gridDim.x * blockDim.x) {
        const double v = to_float(mine[i]);
        sum += v * v;
    }
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) sum += sums[w];
        part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = sum;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) normalise_kernel(float *__restrict__ x, const T *__restrict__ g, long long size, int parts, const double *__restrict__ part, double eps)
{
    chain_wait();
    chain_release();
    double sum = 0.0;
    for (int i = 0; i < parts; i++) sum += part[blockIdx.y * NORM_BLOCKS + i];
    const double scale = 1.0 / (sqrt(sum) + eps);
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < size; i += (long long)gridDim.x * blockDim.x)
        x[blockIdx.y * size + i] = (float)((double)to_float(g[blockIdx.y * size + i]) * scale);
}

// out[b] = alpha D[b] + beta A[b] B[b]^T for a batch of row-major results [ni][nj]
template <typename T>
__global__ void __launch_bounds__(256) product_fma_kernel(T *__restrict__ out, float alpha, const float *__restrict__ d, float beta, Operand<float> A, Operand<float> B,
                                                          long long a_size, long long b_size)
{
    __shared__ float As[FK][FT + 4], Bs[FK][FT + 4];
    chain_wait();
    chain_release();
    const int i0 = blockIdx.y * FT, j0 = blockIdx.x * FT, ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    A.p += blockIdx.z * a_size;
    B.p += blockIdx.z * b_size;
    float acc[4][4] = {};
    fma_tile(acc, A, B, i0, j0, As, Bs);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = i0 + 4 * ti + i, col = j0 + 4 * tj + j;
            if (row >= A.ni || col >= B.ni) continue;
            const long long at = (blockIdx.z * A.ni + row) * B.ni + col;
            float v = beta * acc[i][j];
            if (d) v = fmaf(alpha, d[at], v);
            out[at] = from_float<T>(v);
        }
}

struct OrthogonalizePlan {
    size_t norm, x[2], gram, poly, total;
};
static OrthogonalizePlan plan_orthogonalize(int batch, int m, int n)
{
    OrthogonalizePlan p{};
    const size_t s = m < n ? m : n;
    size_t at = 0;
    p.norm = at;
    at += round256(sizeof(double) * (size_t)batch * NORM_BLOCKS);
    for (int i = 0; i < 2; i++) {
        p.x[i] = at;
        at += round256(sizeof(float) * (size_t)batch * m * n);
    }
    p.gram = at;
    at += round256(sizeof(float) * (size_t)batch * s * s);
    p.poly = at;
    at += round256(sizeof(float) * (size_t)batch * s * s);
    p.total = at;
    return p;
}

template <typename T>
static int product(T *out, float alpha, const float *d, float beta, Operand<float> A, Operand<float> B, long long a_size, long long b_size, int batch, cudaStream_t st)
{
    const dim3 grid((unsigned)((B.ni + FT - 1) / FT), (unsigned)((A.ni + FT - 1) / FT), batch);
    AI2B_CUDA(launch_chained(product_fma_kernel<T>, grid, dim3(256), 0, st, out, alpha, d, beta, A, B, a_size, b_size));
    return AI2B_OK;
}

}  // namespace ai2b

using namespace ai2b;

extern "C" size_t ai2b_orthogonalize_workspace_bytes(int dtype, int batch, int m, int n)
{
    if (!known_dtype(dtype) || batch < 1 || m < 1 || n < 1) return 256;
    return plan_orthogonalize(batch, m, n).total + 256;
}

extern "C" int ai2b_orthogonalize(int dtype, void *d_out, const void *d_g, int batch, int m, int n, int steps, double a, double b, double c, double eps, void *d_workspace,
                                  size_t workspace_bytes, void *stream)
{
    AI2B_REQUIRE(known_dtype(dtype), AI2B_ERR_INVALID, "ai2b_orthogonalize: unknown element type %d", dtype);
    AI2B_REQUIRE(batch >= 0 && m >= 1 && n >= 1 && steps >= 0, AI2B_ERR_INVALID, "ai2b_orthogonalize: batch %d, m %d, n %d, steps %d", batch, m, n, steps);
    AI2B_REQUIRE(eps >= 0.0, AI2B_ERR_INVALID, "ai2b_orthogonalize: eps must not be negative");
    AI2B_REQUIRE(batch <= 65535 && m <= (1 << 20) && n <= (1 << 20), AI2B_ERR_UNSUPPORTED, "ai2b_orthogonalize: at most 65535 matrices of 2^20 rows and columns");
    if (batch == 0) return AI2B_OK;
    AI2B_REQUIRE(d_out && d_g, AI2B_ERR_INVALID, "ai2b_orthogonalize: NULL pointer");
    const OrthogonalizePlan p = plan_orthogonalize(batch, m, n);
    AI2B_REQUIRE(d_workspace && workspace_bytes >= p.total, AI2B_ERR_WORKSPACE, "ai2b_orthogonalize: workspace of %zu bytes, %zu needed", workspace_bytes, p.total);
    cudaStream_t st = (cudaStream_t)stream;
    unsigned char *ws = (unsigned char *)d_workspace;
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const long long size = (long long)m * n;
        const int s = m < n ? m : n, parts = (int)(size < NORM_BLOCKS * 1024LL ? (size + 1023) / 1024 : NORM_BLOCKS);
        double *norm = (double *)(ws + p.norm);
        float *x = (float *)(ws + p.x[0]), *next = (float *)(ws + p.x[1]), *gram = (float *)(ws + p.gram), *poly = (float *)(ws + p.poly);
        AI2B_CUDA(launch_chained(norm_kernel<T>, dim3(parts, batch), dim3(256), 0, st, (const T *)d_g, size, norm));
        const int blocks = (int)(size < 512 * 256LL ? (size + 255) / 256 : 512);
        AI2B_CUDA(launch_chained(normalise_kernel<T>, dim3(blocks, batch), dim3(256), 0, st, x, (const T *)d_g, size, parts, (const double *)norm, eps));
        const long long ss = (long long)s * s;
        for (int i = 0; i < steps; i++) {
            const Operand<float> rows{x, n, 1, m, n}, cols{x, 1, n, n, m}, g{gram, s, 1, s, s}, q{poly, s, 1, s, s};      // rows: X as [m][n], cols: its transpose
            const Operand<float> side = m <= n ? rows : cols;
            int rc = product(gram, 0.f, (const float *)nullptr, 1.f, side, side, size, size, batch, st);
            if (rc == AI2B_OK) rc = product(poly, (float)b, (const float *)gram, (float)c, g, g, ss, ss, batch, st);
            // (poly is symmetric: X poly = X poly^T)
            const Operand<float> left = m <= n ? q : rows, right = m <= n ? cols : q;
            const long long left_size = m <= n ? ss : size, right_size = m <= n ? size : ss;
            if (rc == AI2B_OK) {
                if (i + 1 < steps) rc = product(next, (float)a, (const float *)x, 1.f, left, right, left_size, right_size, batch, st);
                else rc = product((T *)d_out, (float)a, (const float *)x, 1.f, left, right, left_size, right_size, batch, st);
            }
            if (rc != AI2B_OK) return rc;
            float *was = x;
            x = next;
            next = was;
        }
        if (steps == 0) {
            // the normalised matrix itself, rounded to its type
            AI2B_CUDA(launch_chained(product_fma_kernel<T>, dim3((n + FT - 1) / FT, (m + FT - 1) / FT, batch), dim3(256), 0, st, (T *)d_out, 1.f, (const float *)x, 0.f,
                                     Operand<float>{x, n, 1, m, 0}, Operand<float>{x, 1, n, n, 0}, size, size));
        }
        return (int)AI2B_OK;
    });
}
