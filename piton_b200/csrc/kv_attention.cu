// Attention of a few query tokens per sequence over the paged 8-bit cache (kv_append.cu's layout).
//
// A CTA takes one query row (token, head); its warps walk the keys in turn, each with its own
// running maximum and sum of the softmax in fp32, and join at the end.
#include "decode.cuh"

namespace piton {
namespace decode {

__device__ int g_cached_status = 0;

namespace {

constexpr int THREADS = 128, WARPS = THREADS / 32;

struct CachedParams {
    const void *q;
    void *out;
    float *lse;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *lengths, *cu;
    int64_t batch, tokens, q_heads, kv_heads, page_size, num_pages, table_width, table_stride;
    int64_t sqt, sqh, sot, soh;
    int64_t window, uniform, max_new;
    float scale;
};

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_cached_status, 0, code); }

template <typename T, int D>
__global__ void __launch_bounds__(THREADS) kv_attention_kernel(const CachedParams p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.z, i = blockIdx.y, h = blockIdx.x, kvh = h / (p.q_heads / p.kv_heads);
    const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
    if (i >= sp.n) return;
    const int64_t pos = (int64_t)p.lengths[b] - sp.n + i;
    const int64_t first = p.window ? max(pos - p.window + 1, (int64_t)0) : 0;
    const T *q = reinterpret_cast<const T *>(p.q) + (sp.t0 + i) * p.sqt + h * p.sqh;
    float qv[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) qv[e] = to_float(q[lane * E + e]) * p.scale;
    for (int64_t j = first + warp; j <= pos; j += WARPS) {
        const int64_t place = j / p.page_size;
        if (place >= p.table_width) {
            if (lane == 0) record_status(STATUS_BAD_POSITION);
            break;
        }
        const int64_t page = p.table[b * p.table_stride + place];
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) record_status(STATUS_BAD_PAGE);
            continue;
        }
        const int64_t block = page * p.kv_heads + kvh, at = (block * p.page_size + j % p.page_size) * D + lane * E;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += qv[e] * e4m3_to_float(p.kc[at + e]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.ks[block];
        const float m2 = fmaxf(m, s), f = m2 == -INFINITY ? 1.0f : expf(m - m2);
        const float w = s == -INFINITY ? 0.0f : expf(s - m2), vw = w * p.vs[block];
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + vw * e4m3_to_float(p.vc[at + e]);
        m = m2;
    }
    __shared__ float so[WARPS][D], sm[WARPS], sl[WARPS];
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    __syncthreads();
    float top = -INFINITY, total = 0.0f;
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm[w]);
    float f[WARPS];
    for (int w = 0; w < WARPS; ++w) {
        f[w] = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - top);
        total += f[w] * sl[w];
    }
    T *out = reinterpret_cast<T *>(p.out) + (sp.t0 + i) * p.sot + h * p.soh;
    for (int d = threadIdx.x; d < D; d += THREADS) {
        float acc = 0.0f;
        for (int w = 0; w < WARPS; ++w) acc += f[w] == 0.0f ? 0.0f : f[w] * so[w][d];
        out[d] = from_float<T>(total == 0.0f ? 0.0f : acc / total);
    }
    if (p.lse && threadIdx.x == 0) p.lse[(sp.t0 + i) * p.q_heads + h] = total == 0.0f ? -INFINITY : top + logf(total);
}

}  // namespace

int kv_attention_status_read_and_clear(int *status) {
    int zero = 0;
    PITON_CUDA(cudaMemcpyFromSymbol(status, g_cached_status, sizeof(int)));
    PITON_CUDA(cudaMemcpyToSymbol(g_cached_status, &zero, sizeof(int)));
    return PITON_B200_OK;
}

}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

namespace {

int check_attention(const piton_kv_attention_args *a) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->kv_heads > 0 && a->q_heads > 0 && a->num_pages >= 0 &&
                      a->table_width >= 0 && a->window >= 0 && a->max_length >= 0 && a->max_new >= 0,
                  "bad shape");
    PITON_REQUIRE(a->q_heads % a->kv_heads == 0, "%lld query heads over %lld key heads", (long long)a->q_heads,
                  (long long)a->kv_heads);
    PITON_REQUIRE(a->batch <= 65535 && a->tokens < (1ll << 31) && a->q_heads <= (1 << 16) && a->num_pages < (1ll << 31),
                  "batch, tokens, heads or pages too large");
    if ((a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) ||
        (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128))
        return set_error(PITON_B200_ENOTSUP, "head_dim %lld (32, 64, 128) or page_size %lld (16, 32, 64, 128)",
                         (long long)a->head_dim, (long long)a->page_size);
    PITON_REQUIRE(a->batch == 0 || a->cu || a->tokens % a->batch == 0, "%lld tokens are not the same number for %lld sequences",
                  (long long)a->tokens, (long long)a->batch);
    return PITON_B200_OK;
}

}  // namespace

extern "C" size_t piton_b200_kv_attention_workspace_size(const piton_kv_attention_args *) { return 0; }

extern "C" int piton_b200_kv_attention(const piton_kv_attention_args *a, void *stream) {
    if (int rc = check_attention(a)) return rc;
    if (a->batch == 0 || a->tokens == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->q && a->out && a->k_codes && a->v_codes && a->k_scale && a->v_scale && a->table && a->lengths,
                  "NULL pointer");
    PITON_REQUIRE(a->k_codes % 16 == 0 && a->v_codes % 16 == 0, "codes are not 16-byte aligned");
    CachedParams p;
    p.q = reinterpret_cast<const void *>(a->q);
    p.out = reinterpret_cast<void *>(a->out);
    p.lse = reinterpret_cast<float *>(a->lse);
    p.kc = reinterpret_cast<const uint8_t *>(a->k_codes);
    p.vc = reinterpret_cast<const uint8_t *>(a->v_codes);
    p.ks = reinterpret_cast<const float *>(a->k_scale);
    p.vs = reinterpret_cast<const float *>(a->v_scale);
    p.table = reinterpret_cast<const int32_t *>(a->table);
    p.lengths = reinterpret_cast<const int32_t *>(a->lengths);
    p.cu = reinterpret_cast<const int32_t *>(a->cu);
    p.batch = a->batch; p.tokens = a->tokens; p.q_heads = a->q_heads; p.kv_heads = a->kv_heads;
    p.page_size = a->page_size; p.num_pages = a->num_pages; p.table_width = a->table_width; p.table_stride = a->table_stride;
    p.sqt = a->stride_qt; p.sqh = a->stride_qh; p.sot = a->stride_ot; p.soh = a->stride_oh;
    p.window = a->window;
    p.uniform = a->cu ? 0 : a->tokens / a->batch;
    p.max_new = a->cu ? (a->max_new ? a->max_new : a->tokens) : p.uniform;
    p.scale = (float)a->sm_scale;
    PITON_REQUIRE(p.max_new <= 65535, "%lld query tokens a sequence", (long long)p.max_new);
    const dim3 grid((unsigned)a->q_heads, (unsigned)p.max_new, (unsigned)a->batch);
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        cudaStream_t s = as_stream(stream);
        if (a->head_dim == 32) kv_attention_kernel<T, 32><<<grid, THREADS, 0, s>>>(p);
        else if (a->head_dim == 64) kv_attention_kernel<T, 64><<<grid, THREADS, 0, s>>>(p);
        else kv_attention_kernel<T, 128><<<grid, THREADS, 0, s>>>(p);
        return check_launch("kv_attention");
    });
}
