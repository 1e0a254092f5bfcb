// Scratch context, paged cache and argument checks of the decoder's serving step.
#include "lm.h"

#include <new>

namespace gpx {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The codes of a cache as rows of `dim` bytes.  A box is what a block of 64 keys takes from one page; the swizzle
// spreads the rows of a box over the banks of shared memory.
static int make_page_map(CUtensorMap *map, void *base, const gpx_kv_cache &c) {
    EncodeTiledFn encode = reinterpret_cast<EncodeTiledFn>(driver_entry("cuTensorMapEncodeTiled"));
    GPX_REQUIRE(encode, GPX_FAIL, "driver has no cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)c.dim, (cuuint64_t)c.pages * c.kv_heads * c.page_tokens};
    cuuint64_t strides[1] = {(cuuint64_t)c.dim};
    cuuint32_t box[2] = {(cuuint32_t)c.dim, (cuuint32_t)(c.page_tokens < 64 ? c.page_tokens : 64)};
    cuuint32_t estr[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    GPX_REQUIRE(rc == CUDA_SUCCESS, GPX_FAIL, "cuTensorMapEncodeTiled failed with %d", (int)rc);
    return GPX_SUCC;
}

int lm_check_batch(const gpx_kv_batch *b, LmBatch *out) {
    GPX_REQUIRE(b && b->table && b->context && b->first, GPX_FAIL, "the batch's table, context or first is NULL");
    GPX_REQUIRE((uintptr_t)b->table % 4 == 0 && (uintptr_t)b->context % 4 == 0 && (uintptr_t)b->first % 4 == 0, GPX_FAIL,
                "table, context and first must be 4-byte aligned");
    GPX_REQUIRE(b->seqs > 0 && b->seqs <= kLmMaxSeqs, GPX_OUT_OF_RANGE, "a batch has 1 to %d sequences, not %d", kLmMaxSeqs, b->seqs);
    GPX_REQUIRE(b->table_ld > 0, GPX_OUT_OF_RANGE, "table_ld is %d", b->table_ld);
    GPX_REQUIRE(b->most_new >= 0 && b->tokens >= b->most_new, GPX_OUT_OF_RANGE, "%d new tokens of a sequence, %d in all", b->most_new,
                b->tokens);
    *out = LmBatch{(const int *)b->table, (const int *)b->context, (const int *)b->first, b->table_ld, b->seqs, b->tokens, b->most_new};
    return GPX_SUCC;
}

int lm_check_blp(const gpx_blp *blp, BlpArgs *out) {
    BlpArgs b{};
    if (blp) {
        b.preempted = (const int *)blp->preempted;
        b.stop_index = (int *)blp->stop_index;
        b.executed = (int *)blp->executed;
        b.kernel_id = blp->kernel_id;
        b.trace = (unsigned long long *)blp->trace;
        GPX_REQUIRE(!b.preempted || (b.stop_index && b.executed), GPX_FAIL, "preemptible launch needs stop_index and executed");
    }
    *out = b;
    return GPX_SUCC;
}

int lm_elem(const char *dtype, bool f32_too, int *elem) {
    GPX_REQUIRE(dtype, GPX_FAIL, "dtype is NULL");
    if (!strcmp(dtype, "bfloat16")) *elem = LM_BF16;
    else if (!strcmp(dtype, "float16")) *elem = LM_F16;
    else if (f32_too && !strcmp(dtype, "float32")) *elem = LM_F32;
    else {
        set_error("dtype \"%s\" is none of %s\"bfloat16\", \"float16\"", dtype, f32_too ? "\"float32\", " : "");
        return GPX_OUT_OF_RANGE;
    }
    return GPX_SUCC;
}

cudaError_t lm_resident(const void *kernel, int threads, size_t smem, size_t most, int device, int *per_sm) {
    struct Known {
        const void *kernel;
        size_t kib;
        int device, per_sm;
    };
    static thread_local Known table[64] = {};
    const size_t kib = (smem + 1023) / 1024;
    Known &k = table[(reinterpret_cast<uintptr_t>(kernel) >> 4 ^ (uintptr_t)device ^ kib) % 64];
    if (k.kernel != kernel || k.kib != kib || k.device != device) {
        cudaError_t e = cudaSuccess;
        if (most > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        int n = 0;
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, kib * 1024);
        if (e != cudaSuccess) return e;
        k = Known{kernel, kib, device, n > 1 ? n : 1};
    }
    *per_sm = k.per_sm;
    return cudaSuccess;
}

}  // namespace gpx

using namespace gpx;

extern "C" {

int gpx_lm_ctx_bytes(size_t *bytes) {
    GPX_REQUIRE(bytes, GPX_FAIL, "bytes is NULL");
    *bytes = kLmCtxBytes;
    return GPX_SUCC;
}

int gpx_lm_ctx_reset(void *ctx, gpx_event *ready) {
    GPX_REQUIRE(ctx, GPX_FAIL, "ctx is NULL");
    GPX_CUDA(cudaMemsetAsync(ctx, 0, kLmResetBytes, nullptr));
    return record_ready(ready);
}

int gpx_lm_status(const void *ctx, int *error, int *where) {
    GPX_REQUIRE(ctx && error, GPX_FAIL, "NULL argument");
    int h[2];
    GPX_CUDA(cudaMemcpy(h, ctx, sizeof(h), cudaMemcpyDeviceToHost));
    *error = h[0];
    if (where) *where = h[1];
    return GPX_SUCC;
}

int gpx_kv_cache_create(void *k, void *v, void *k_scale, void *v_scale, int pages, int page_tokens, int kv_heads, int head_dim,
                        gpx_kv_cache **cache) {
    GPX_REQUIRE(cache, GPX_FAIL, "cache is NULL");
    *cache = nullptr;
    GPX_REQUIRE(k && v && k_scale && v_scale, GPX_FAIL, "k, v, k_scale or v_scale is NULL");
    GPX_REQUIRE(page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128, GPX_OUT_OF_RANGE,
                "page_tokens is 16, 32, 64 or 128, not %d", page_tokens);
    GPX_REQUIRE(head_dim == 64 || head_dim == 128, GPX_OUT_OF_RANGE, "head_dim is 64 or 128, not %d", head_dim);
    GPX_REQUIRE(pages > 0 && kv_heads > 0 && (long long)pages * kv_heads <= 0x7fffffffll / page_tokens, GPX_OUT_OF_RANGE,
                "%d pages of %d heads and %d tokens are not 1 to 2^31 - 1 rows", pages, kv_heads, page_tokens);
    GPX_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)k_scale % 4 == 0 && (uintptr_t)v_scale % 4 == 0,
                GPX_FAIL, "k and v must be 16-byte aligned, the scales 4-byte aligned");
    gpx_kv_cache c{(unsigned char *)k, (unsigned char *)v, (float *)k_scale, (float *)v_scale, pages, page_tokens, kv_heads, head_dim, {}, {}};
    GPX_TRY(make_page_map(&c.map_k, k, c));
    GPX_TRY(make_page_map(&c.map_v, v, c));
    gpx_kv_cache *made = new (std::nothrow) gpx_kv_cache(c);
    GPX_REQUIRE(made, GPX_FAIL, "out of host memory");
    *cache = made;
    return GPX_SUCC;
}

int gpx_kv_cache_destroy(gpx_kv_cache *cache) {
    delete cache;
    return GPX_SUCC;
}

}  // extern "C"
