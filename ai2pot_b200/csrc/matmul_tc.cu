// Host side of the tensor-core products: tensor maps, and the report of waits that ran out.
#include "matmul_tc.cuh"

namespace ai2b {
namespace tc {

static __device__ int gave_up = 0;

int flag_address(int **flag)
{
    static std::mutex mu;
    static int *known[MAX_DEVICES] = {};
    int dev = 0;
    AI2B_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> guard(mu);
    if (dev < MAX_DEVICES && known[dev]) {
        *flag = known[dev];
        return AI2B_OK;
    }
    void *p = nullptr;
    AI2B_CUDA(cudaGetSymbolAddress(&p, gave_up));
    *flag = (int *)p;
    if (dev < MAX_DEVICES) known[dev] = *flag;
    return AI2B_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int encoder(EncodeTiled *out)
{
    static EncodeTiled encode = nullptr;
    static std::mutex mu;
    std::lock_guard<std::mutex> guard(mu);
    if (!encode) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        AI2B_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
        AI2B_REQUIRE(f && found == cudaDriverEntryPointSuccess, AI2B_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        encode = (EncodeTiled)f;
    }
    *out = encode;
    return AI2B_OK;
}

static int make_map(CUtensorMap *map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void *p, int size, long long columns, long long rows, long long batch,
                    long long row_stride, long long batch_stride, int box_columns, int box_rows)
{
    EncodeTiled encode;
    const int rc0 = encoder(&encode);
    if (rc0 != AI2B_OK) return rc0;
    const cuuint64_t dims[3] = {(cuuint64_t)columns, (cuuint64_t)(rows > 0 ? rows : 1), (cuuint64_t)batch};
    const cuuint64_t strides[2] = {(cuuint64_t)row_stride * size, (cuuint64_t)batch_stride * size};
    const cuuint32_t box[3] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows, 1}, steps[3] = {1, 1, 1};
    const CUresult rc = encode(map, type, 3, const_cast<void *>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    AI2B_REQUIRE(rc == CUDA_SUCCESS, AI2B_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): %lld x %lld x %lld, strides %lld and %lld", (int)rc, columns, rows, batch, row_stride,
                 batch_stride);
    return AI2B_OK;
}

int make_map(CUtensorMap *map, const void *p, bool is_bf16, long long columns, long long rows, long long batch, long long row_stride, long long batch_stride, int box_rows)
{
    return make_map(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, p, 2, columns, rows, batch, row_stride,
                    batch_stride, 64, box_rows);
}

int make_prefetch_map(CUtensorMap *map, const void *p, int dtype, long long columns, long long rows, long long row_stride)
{
    const CUtensorMapDataType type = dtype == AI2B_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == AI2B_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int size = (int)element_bytes(dtype);
    return make_map(map, type, CU_TENSOR_MAP_SWIZZLE_NONE, p, size, columns, rows, 1, row_stride, rows * row_stride, 128 / size, BM);
}

}  // namespace tc
}  // namespace ai2b

using namespace ai2b;

extern "C" int ai2b_fitnet_check(void *stream)
{
    int flag = 0, *where = nullptr;
    const int rc = tc::flag_address(&where);
    if (rc != AI2B_OK) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    AI2B_CUDA(cudaMemcpyAsync(&flag, where, sizeof(flag), cudaMemcpyDeviceToHost, st));
    AI2B_CUDA(cudaStreamSynchronize(st));
    if (flag) {
        AI2B_CUDA(cudaMemsetAsync(where, 0, sizeof(flag), st));
        set_error("a product's wait on its own copies or accumulators ran out: results since the last check are not valid");
        return AI2B_ERR_TIMEOUT;
    }
    return AI2B_OK;
}
