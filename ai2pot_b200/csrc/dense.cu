// One layer of all networks: y = residual + act(x W_e^T + b_e) for the rows of each group e, and its gradient.
//
//   z = x W_e^T + b_e,  y = residual + act(z),  s = act'(z) (kept for the gradient)
//   gz = gy * s;  gx = gz W_e;  gW_e = sum over the rows of e of gz^T x;  gb_e = sum of gz;  gresidual = gy
//   rows after the last group belong to no network: y, gx and gresidual are zero there
//
// Products are accumulated in float. gz is rounded to the element type of x where it becomes a factor of the products (their other factor
// has that type already); gb adds it unrounded. s lies between -0.13 and 1.13, so that 16-bit layers of either type keep it as a half, which
// has the more digits: rounding it costs nothing next to gz in bfloat16 (errors of gx against 64 bits: 0.0030 with s in bfloat16, 0.0024).
// The sums over rows (gW, gb) are cut into slabs of rows whose partial sums are added in a fixed order: no atomics.
#include "fitnet.cuh"
#include "fma_tile.cuh"

namespace ai2b {

constexpr int MAX_GROUPS = 1024;

// ---- activations ----------------------------------------------------------------------------------------------------------

struct Activated {
    float value, slope;
};
template <int ACT>
__device__ __forceinline__ Activated activate(float z)
{
    if constexpr (ACT == AI2B_ACT_TANH) {
        const float t = tanhf(z);
        return {t, 1.f - t * t};
    } else if constexpr (ACT == AI2B_ACT_SILU) {
        const float p = 1.f / (1.f + expf(-z));
        return {z * p, p * (1.f + z * (1.f - p))};
    } else if constexpr (ACT == AI2B_ACT_GELU) {
        const float p = 0.5f * erfcf(-0.70710678118654752f * z);
        return {z * p, fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), p)};
    } else {
        return {z, 1.f};
    }
}

// ---- tiles of rows --------------------------------------------------------------------------------------------------------

// Rows are cut into tiles of `height` rows that do not cross groups; the rows after the last group make up pseudo-group `groups`.
struct RowTile {
    int group;                // -1: there are fewer tiles
    long long begin, end;
};
__device__ __forceinline__ long long tiles_of(long long n, int height) { return (n + height - 1) / height; }

// Executed by whole warps; every lane returns the same tile.
__device__ __forceinline__ RowTile find_tile(const int *offsets, int groups, long long rows, int height, long long tile)
{
    const int lane = threadIdx.x & 31;
    long long base = 0;
    for (int e0 = 0; e0 < groups; e0 += 32) {
        const int e = e0 + lane;
        RowRange r{0, 0};
        if (e < groups) r = group_rows(offsets, e, rows);
        const long long mine = tiles_of(r.end - r.begin, height);
        long long scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(FULL_MASK, scan, o);
            if (lane >= o) scan += up;
        }
        const unsigned hit = __ballot_sync(FULL_MASK, base + scan > tile);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const long long begin = __shfl_sync(FULL_MASK, r.begin, src), end = __shfl_sync(FULL_MASK, r.end, src);
            const long long first = base + __shfl_sync(FULL_MASK, scan - mine, src);
            const long long row = begin + (tile - first) * height;
            return RowTile{e0 + src, row, min(row + height, end)};
        }
        base += __shfl_sync(FULL_MASK, scan, 31);
    }
    if (!offsets) return RowTile{-1, 0, 0};
    const long long row = group_rows(offsets, groups - 1, rows).end + (tile - base) * height;
    if (row >= rows) return RowTile{-1, 0, 0};
    return RowTile{groups, row, min(row + height, rows)};
}

// Tiles before group e (whole warps)
__device__ __forceinline__ long long tiles_before(const int *offsets, int e, long long rows, int height)
{
    long long n = 0;
    for (int i = threadIdx.x & 31; i < e; i += 32) {
        const RowRange r = group_rows(offsets, i, rows);
        n += tiles_of(r.end - r.begin, height);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) n += __shfl_xor_sync(FULL_MASK, n, o);
    return n;
}

// ---- products on the FMA pipes --------------------------------------------------------------------------------------------

// What happens to a sum before it is stored: bias, activation, slope, residual
template <typename T> using Slope = std::conditional_t<std::is_same<T, float>::value, float, f16>;

template <typename T>
struct RowOutput {
    T *out;                   // [rows][columns]
    Slope<T> *slope;
    const T *bias;            // [groups][columns]
    const T *residual;
    long long residual_stride;
    int activation;
};
template <typename T>
__device__ __forceinline__ void store_row_element(const RowOutput<T> &o, long long row, int col, int columns, int group, float z)
{
    if (o.bias) z += to_float(o.bias[(long long)group * columns + col]);
    Activated a;
    switch (o.activation) {
    case AI2B_ACT_TANH: a = activate<AI2B_ACT_TANH>(z); break;
    case AI2B_ACT_SILU: a = activate<AI2B_ACT_SILU>(z); break;
    case AI2B_ACT_GELU: a = activate<AI2B_ACT_GELU>(z); break;
    default: a = activate<AI2B_ACT_NONE>(z);
    }
    if (o.slope) o.slope[row * columns + col] = from_float<Slope<T>>(a.slope);
    if (o.residual) a.value += to_float(o.residual[row * o.residual_stride + col]);
    o.out[row * columns + col] = from_float<T>(a.value);
}

// Rows of every group times the group's matrix: w[group][.][.] has strides sj (column of the output) and sk (summed index).
template <typename T>
__global__ void __launch_bounds__(256) rows_fma_kernel(const T *__restrict__ x, long long x_stride, const T *__restrict__ w, long long w_size, long long w_sj, long long w_sk,
                                                       const int *__restrict__ offsets, int groups, long long rows, int inner, int columns, RowOutput<T> o)
{
    __shared__ float As[FK][FT + 4], Bs[FK][FT + 4];
    chain_wait();
    chain_release();
    const RowTile tile = find_tile(offsets, groups, rows, FT, blockIdx.x);
    if (tile.group < 0) return;
    const int j0 = blockIdx.y * FT, ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    float acc[4][4] = {};
    if (tile.group < groups)
        fma_tile(acc, Operand<T>{x, x_stride, 1, tile.end, inner}, Operand<T>{w + tile.group * w_size, w_sj, w_sk, columns, inner}, tile.begin, j0, As, Bs);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long row = tile.begin + 4 * ti + i;
            const int col = j0 + 4 * tj + j;
            if (row >= tile.end || col >= columns) continue;
            if (tile.group < groups) store_row_element(o, row, col, columns, tile.group, acc[i][j]);
            else o.out[row * columns + col] = from_float<T>(0.f);
        }
}

// Partial sums of gz^T x over slabs of rows: part[slab][outer][inner]
template <typename T>
__global__ void __launch_bounds__(256) weight_fma_kernel(const T *__restrict__ gz, long long gz_stride, const T *__restrict__ x, long long x_stride, const int *__restrict__ offsets,
                                                         int groups, long long rows, int height, int outer, int inner, float *__restrict__ part)
{
    __shared__ float As[FK][FT + 4], Bs[FK][FT + 4];
    chain_wait();
    chain_release();
    const RowTile tile = find_tile(offsets, groups, rows, height, blockIdx.x);
    if (tile.group < 0 || tile.group >= groups) return;
    const int i0 = blockIdx.y * FT, j0 = blockIdx.z * FT, ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    float acc[4][4] = {};
    const long long n = tile.end - tile.begin;
    fma_tile(acc, Operand<T>{gz + tile.begin * gz_stride, 1, gz_stride, outer, n}, Operand<T>{x + tile.begin * x_stride, 1, x_stride, inner, n}, i0, j0, As, Bs);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = i0 + 4 * ti + i, col = j0 + 4 * tj + j;
            if (row < outer && col < inner) part[((long long)blockIdx.x * outer + row) * inner + col] = acc[i][j];
        }
}

// gz = gy * slope, gresidual = gy (zero after the last group), and the column sums of gz over each slab: part[slab][outer]
template <typename T>
__global__ void __launch_bounds__(256) slope_kernel(T *__restrict__ gz, T *__restrict__ gresidual, float *__restrict__ part, const T *__restrict__ gy, long long gy_stride,
                                                    const Slope<T> *__restrict__ slope, const int *__restrict__ offsets, int groups, long long rows, int height, int outer)
{
    __shared__ float sums[8][32];
    chain_wait();
    chain_release();
    const RowTile tile = find_tile(offsets, groups, rows, height, blockIdx.x);
    if (tile.group < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * 32 + lane;
    const bool kept = tile.group < groups;
    float sum = 0.f;
    if (col < outer) {
        for (long long r = tile.begin + warp; r < tile.end; r += 8) {
            float g = 0.f;
            if (kept) g = to_float(gy[r * gy_stride + col]);
            if (gresidual) gresidual[r * outer + col] = from_float<T>(g);
            if (slope && kept) {
                g *= to_float(slope[r * outer + col]);
                gz[r * outer + col] = from_float<T>(g);
            }
            sum += g;
        }
    }
    if (!part || !kept) return;
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && col < outer) {
#pragma unroll
        for (int w = 1; w < 8; w++) sum += sums[w][lane];
        part[(long long)blockIdx.x * outer + col] = sum;
    }
}

// out[e][i] = sum of part[slab][i] over the slabs of group e, in ascending order
template <typename T>
__global__ void __launch_bounds__(256) sum_slabs_kernel(T *__restrict__ out, const float *__restrict__ part, const int *__restrict__ offsets, long long rows, int height,
                                                        long long size, long long slabs)
{
    chain_wait();
    chain_release();
    const int e = blockIdx.y;
    const long long first = tiles_before(offsets, e, rows, height);
    const RowRange r = group_rows(offsets, e, rows);
    const long long n = min(tiles_of(r.end - r.begin, height), slabs - first);       // (`slabs` are there, whatever the offsets say)
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < size; i += (long long)gridDim.x * blockDim.x) {
        float sum = 0.f;
        for (long long s = 0; s < n; s++) sum += part[(first + s) * size + i];
        out[e * size + i] = from_float<T>(sum);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------

// Rows of a slab: enough slabs that the products of a slab keep all SMs busy, none shorter than 256 rows
static int slab_height(long long rows, long long tiles_per_slab)
{
    long long slabs = (2LL * sm_count() + tiles_per_slab - 1) / tiles_per_slab;
    if (slabs > (rows + 255) / 256) slabs = (rows + 255) / 256;
    if (slabs < 1) slabs = 1;
    const long long height = ((rows + slabs - 1) / slabs + 63) / 64 * 64;
    return (int)(height < 64 ? 64 : height > (1 << 30) ? (1 << 30) : height);
}
static long long slab_bound(long long rows, int height, int groups) { return (rows + height - 1) / height + groups; }

struct BackwardPlan {
    int weight_height, bias_height;
    size_t gz, weight_part, bias_part, total;
};
static BackwardPlan plan_backward(const ai2b_dense *d)
{
    BackwardPlan p{};
    const long long tiles = (long long)((d->outer + FT - 1) / FT) * ((d->inner + FT - 1) / FT);
    p.weight_height = slab_height(d->rows, tiles);
    p.bias_height = slab_height(d->rows, (d->outer + 31) / 32);
    size_t at = 0;
    p.gz = at;
    if (d->activation != AI2B_ACT_NONE) at += round256(element_bytes(d->dtype) * (size_t)d->rows * d->outer);
    p.weight_part = at;
    at += round256(sizeof(float) * (size_t)slab_bound(d->rows, p.weight_height, d->groups) * d->outer * d->inner);
    p.bias_part = at;
    at += round256(sizeof(float) * (size_t)slab_bound(d->rows, p.bias_height, d->groups) * d->outer);
    p.total = at;
    return p;
}

static int check_dense(const ai2b_dense *d, const char *what)
{
    AI2B_REQUIRE(d, AI2B_ERR_INVALID, "%s: NULL description", what);
    AI2B_REQUIRE(known_dtype(d->dtype), AI2B_ERR_INVALID, "%s: unknown element type %d", what, d->dtype);
    AI2B_REQUIRE(d->activation >= AI2B_ACT_NONE && d->activation <= AI2B_ACT_GELU, AI2B_ERR_INVALID, "%s: unknown activation %d", what, d->activation);
    AI2B_REQUIRE(d->rows >= 0 && d->inner >= 1 && d->outer >= 1 && d->groups >= 1, AI2B_ERR_INVALID, "%s: rows %lld, inner %d, outer %d, groups %d", what, d->rows, d->inner,
                 d->outer, d->groups);
    AI2B_REQUIRE(d->rows <= 0x7fffffffLL && d->inner <= (1 << 20) && d->outer <= (1 << 20), AI2B_ERR_UNSUPPORTED,
                 "%s: at most 2^31 - 1 rows and layers of 2^20 (got rows %lld, inner %d, outer %d)", what, d->rows, d->inner, d->outer);
    AI2B_REQUIRE(d->groups <= MAX_GROUPS, AI2B_ERR_UNSUPPORTED, "%s: at most %d groups (got %d)", what, MAX_GROUPS, d->groups);
    AI2B_REQUIRE(d->d_offsets || d->groups == 1, AI2B_ERR_INVALID, "%s: several groups need offsets", what);
    AI2B_REQUIRE(d->rows == 0 || (d->d_x && (d->x_stride >= d->inner || d->rows == 1)), AI2B_ERR_INVALID, "%s: x is NULL or its row stride %lld is below %d", what, d->x_stride,
                 d->inner);
    AI2B_REQUIRE(d->d_weight, AI2B_ERR_INVALID, "%s: weight is NULL", what);
    return AI2B_OK;
}

}  // namespace ai2b

using namespace ai2b;

extern "C" size_t ai2b_dense_workspace_bytes(const ai2b_dense *d, int backward)
{
    if (!d || check_dense(d, "ai2b_dense_workspace_bytes") != AI2B_OK || !backward) return 256;
    return plan_backward(d).total + 256;
}

extern "C" int ai2b_dense_forward(const ai2b_dense *d, void *stream)
{
    int rc = check_dense(d, "ai2b_dense_forward");
    if (rc != AI2B_OK || d->rows == 0) return rc;
    AI2B_REQUIRE(d->d_y, AI2B_ERR_INVALID, "ai2b_dense_forward: y is NULL");
    AI2B_REQUIRE(!d->d_residual || d->residual_stride >= d->outer || d->rows == 1, AI2B_ERR_INVALID, "ai2b_dense_forward: row stride %lld of the residual is below %d",
                 d->residual_stride, d->outer);
    cudaStream_t st = (cudaStream_t)stream;
    return with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        const RowOutput<T> o{(T *)d->d_y, d->activation != AI2B_ACT_NONE ? (Slope<T> *)d->d_slope : nullptr, (const T *)d->d_bias, (const T *)d->d_residual, d->residual_stride,
                             d->activation};
        const dim3 grid((unsigned)((d->rows + FT - 1) / FT + d->groups), (d->outer + FT - 1) / FT);
        AI2B_CUDA(launch_chained(rows_fma_kernel<T>, grid, dim3(256), 0, st, (const T *)d->d_x, d->x_stride, (const T *)d->d_weight, (long long)d->outer * d->inner,
                                 (long long)d->inner, 1LL, d->d_offsets, d->groups, d->rows, d->inner, d->outer, o));
        return (int)AI2B_OK;
    });
}

extern "C" int ai2b_dense_backward(const ai2b_dense *d, void *stream)
{
    int rc = check_dense(d, "ai2b_dense_backward");
    if (rc != AI2B_OK) return rc;
    const bool slopes = d->activation != AI2B_ACT_NONE;
    AI2B_REQUIRE(d->rows == 0 || d->d_gy, AI2B_ERR_INVALID, "ai2b_dense_backward: gy is NULL");
    AI2B_REQUIRE(d->gy_stride >= d->outer || d->rows <= 1, AI2B_ERR_INVALID, "ai2b_dense_backward: row stride %lld of gy is below %d", d->gy_stride, d->outer);
    AI2B_REQUIRE(!slopes || d->rows == 0 || d->d_slope, AI2B_ERR_INVALID, "ai2b_dense_backward: the slopes that the forward call kept are NULL");
    const BackwardPlan p = plan_backward(d);
    AI2B_REQUIRE(d->d_workspace && d->workspace_bytes >= p.total, AI2B_ERR_WORKSPACE, "ai2b_dense_backward: workspace of %zu bytes, %zu needed", d->workspace_bytes, p.total);
    cudaStream_t st = (cudaStream_t)stream;
    unsigned char *ws = (unsigned char *)d->d_workspace;
    return with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        T *made = (T *)(ws + p.gz);
        const T *gz = slopes ? made : (const T *)d->d_gy;
        const long long gz_stride = slopes ? d->outer : d->gy_stride;
        float *wpart = (float *)(ws + p.weight_part), *bpart = (float *)(ws + p.bias_part);
        const bool products = d->d_gx || d->d_gweight;
        if (d->rows > 0 && ((slopes && products) || d->d_gresidual || d->d_gbias)) {
            const dim3 grid((unsigned)(slab_bound(d->rows, p.bias_height, d->groups) + 1), (d->outer + 31) / 32);
            AI2B_CUDA(launch_chained(slope_kernel<T>, grid, dim3(256), 0, st, made, (T *)d->d_gresidual, d->d_gbias ? bpart : (float *)nullptr, (const T *)d->d_gy,
                                     d->gy_stride, slopes ? (const Slope<T> *)d->d_slope : (const Slope<T> *)nullptr, d->d_offsets, d->groups, d->rows, p.bias_height, d->outer));
        }
        if (d->d_gbias) {
            const dim3 grid((d->outer + 255) / 256, d->groups);
            AI2B_CUDA(launch_chained(sum_slabs_kernel<T>, grid, dim3(256), 0, st, (T *)d->d_gbias, (const float *)bpart, d->d_offsets, d->rows, p.bias_height,
                                     (long long)d->outer, slab_bound(d->rows, p.bias_height, d->groups)));
        }
        if (d->d_gx && d->rows > 0) {
            const RowOutput<T> o{(T *)d->d_gx, nullptr, nullptr, nullptr, 0, AI2B_ACT_NONE};
            const dim3 grid((unsigned)((d->rows + FT - 1) / FT + d->groups), (d->inner + FT - 1) / FT);
            AI2B_CUDA(launch_chained(rows_fma_kernel<T>, grid, dim3(256), 0, st, gz, gz_stride, (const T *)d->d_weight, (long long)d->outer * d->inner, 1LL,
                                     (long long)d->inner, d->d_offsets, d->groups, d->rows, d->outer, d->inner, o));
        }
        if (d->d_gweight) {
            if (d->rows > 0) {
                const dim3 grid((unsigned)slab_bound(d->rows, p.weight_height, d->groups), (d->outer + FT - 1) / FT, (d->inner + FT - 1) / FT);
                AI2B_CUDA(launch_chained(weight_fma_kernel<T>, grid, dim3(256), 0, st, gz, gz_stride, (const T *)d->d_x, d->x_stride, d->d_offsets, d->groups, d->rows,
                                         p.weight_height, d->outer, d->inner, wpart));
            }
            const long long size = (long long)d->outer * d->inner;
            const dim3 grid((unsigned)((size + 255) / 256 < 4096 ? (size + 255) / 256 : 4096), d->groups);
            AI2B_CUDA(launch_chained(sum_slabs_kernel<T>, grid, dim3(256), 0, st, (T *)d->d_gweight, (const float *)wpart, d->d_offsets, d->rows, p.weight_height, size,
                                     slab_bound(d->rows, p.weight_height, d->groups)));
        }
        return (int)AI2B_OK;
    });
}
