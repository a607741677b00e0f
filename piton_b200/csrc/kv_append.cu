// Appending to a paged 8-bit cache: keys rotated by position, keys and values quantised to e4m3
// with a power-of-two scale per (page, head), queries rotated in the same launch.
//
// A unit is one page that one sequence's new tokens touch; a CTA takes one (unit, head, key or
// value): the block's largest finite magnitude, its scale, the older tokens requantised where the
// scale grows, the new tokens' codes.  The scale is a power of two, so dividing by it is exact and a
// growing scale moves old codes without a second rounding until they reach e4m3's subnormals; the
// format's relative precision does not depend on where in a binade the scale sits.
#include "decode.cuh"

namespace piton {
namespace decode {

__device__ int g_append_status = 0;

namespace {

constexpr int THREADS = 128;

struct AppendParams {
    const void *k, *v, *q;
    void *q_out;
    uint8_t *codes[2];
    float *scale[2];
    const int32_t *table, *starts, *cu;
    int32_t *lengths;
    const float *cos_table, *sin_table;
    int64_t batch, tokens, kv_heads, q_heads, page_size, num_pages, table_width, table_stride;
    int64_t st[2], sh[2], sqt, sqh, sot, soh;   // strides of k and v, q, q_out
    int64_t rope_len, units, uniform, unit_blocks;
    int32_t dim, rot, interleaved;
};

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_append_status, 0, code); }

// The least power of two s in [2^-120, 2^120] with a <= 448 s (a >= 0): 448 = 1.75 * 2^8, so the
// exponent is a's less 8, one more when its significand exceeds 1.75.
__device__ __forceinline__ float block_scale(float a) {
    const uint32_t u = __float_as_uint(a);
    int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    if ((u >> 23) == 0) e = 7;                                       // zero and denormals: the least scale
    e = min(max(e, 7), 247);
    return __uint_as_float((uint32_t)e << 23);
}

__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.0f; }

// Element d of the row x rotated by the row (c, s): every product and sum rounded by itself, so the
// result does not depend on how a compiler contracts them.
template <typename T>
__device__ __forceinline__ float rotated(const T *x, int d, const float *c, const float *s, int rot, bool interleaved) {
    const float a = to_float(x[d]);
    if (d >= rot) return a;
    const int half = rot >> 1;
    const bool second = interleaved ? (d & 1) : d >= half;
    const int i = interleaved ? d >> 1 : (second ? d - half : d);
    const float b = to_float(x[interleaved ? d ^ 1 : (second ? d - half : d + half)]);
    return second ? __fadd_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i])) : __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
}

// The sequence of new token t (ragged): the last b with cu[b] <= t.
__device__ __forceinline__ int64_t sequence_of_token(const AppendParams &p, int64_t t) {
    if (!p.cu) return t / p.uniform;
    int64_t lo = 0, hi = p.batch - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Units are numbered sequence by sequence.  Uniform: a fixed number each.  Ragged: sequence b's
// start at cu[b] / page_size + 2 b, which leaves it at least the n / page_size + 2 pages that n
// tokens can touch.
__device__ __forceinline__ int64_t first_unit(const AppendParams &p, int64_t b) {
    return (p.cu ? max((int64_t)p.cu[b], (int64_t)0) / p.page_size : 0) + 2 * b;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(const AppendParams p) {
    const int tid = threadIdx.x;
    if (blockIdx.x >= p.unit_blocks) {                               // queries: a warp per (token, head)
        const int64_t row = ((int64_t)blockIdx.x - p.unit_blocks) * (THREADS / 32) + (tid >> 5);
        if (row >= p.tokens * p.q_heads) return;
        const int64_t t = row / p.q_heads, h = row % p.q_heads, b = sequence_of_token(p, t);
        const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
        const int64_t pos = (int64_t)p.starts[b] + t - sp.t0;
        const bool ok = p.rot == 0 || (pos >= 0 && pos < p.rope_len && t >= sp.t0 && t < sp.t0 + sp.n);
        if (!ok) {
            if ((tid & 31) == 0) record_status(STATUS_BAD_POSITION);
            return;
        }
        const T *x = reinterpret_cast<const T *>(p.q) + t * p.sqt + h * p.sqh;
        T *y = reinterpret_cast<T *>(p.q_out) + t * p.sot + h * p.soh;
        const float *c = p.cos_table + pos * (p.rot >> 1), *s = p.sin_table + pos * (p.rot >> 1);
        for (int d = tid & 31; d < p.dim; d += 32) y[d] = from_float<T>(rotated(x, d, c, s, p.rot, p.interleaved));
        return;
    }
    const int64_t per_unit = 2 * p.kv_heads;
    const int64_t unit = blockIdx.x / per_unit;
    const int64_t h = (blockIdx.x % per_unit) >> 1;
    const int which = blockIdx.x & 1;
    int64_t b, j;
    if (!p.cu) {
        const int64_t each = p.units / p.batch;
        b = unit / each;
        j = unit % each;
    } else {
        int64_t lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (first_unit(p, mid) <= unit) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        j = unit - first_unit(p, b);
    }
    const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
    const int64_t start = p.starts[b], end = start + sp.n;
    if (j == 0 && h == 0 && which == 0 && tid == 0 && p.lengths) p.lengths[b] = (int32_t)end;
    if (start < 0) {
        if (tid == 0) record_status(STATUS_BAD_POSITION);
        return;
    }
    const int64_t place = start / p.page_size + j;                   // this unit's page of the sequence
    const int64_t page0 = place * p.page_size;
    const int64_t lo = max(start, page0), hi = min(end, page0 + p.page_size);
    if (lo >= hi) return;
    if (place >= p.table_width || (which == 0 && p.rot && hi > p.rope_len)) {
        if (tid == 0) record_status(STATUS_BAD_POSITION);
        return;
    }
    const int64_t page = p.table[b * p.table_stride + place];
    if (page < 0 || page >= p.num_pages) {
        if (tid == 0) record_status(STATUS_BAD_PAGE);
        return;
    }
    const int rot = which == 0 ? p.rot : 0;
    const T *x = reinterpret_cast<const T *>(which == 0 ? p.k : p.v) + (sp.t0 + lo - start) * p.st[which] + h * p.sh[which];
    uint8_t *codes = p.codes[which] + (page * p.kv_heads + h) * p.page_size * p.dim;
    float *scale = p.scale[which] + page * p.kv_heads + h;
    const int count = (int)(hi - lo) * p.dim, held = (int)(lo - page0);
    auto value = [&](int i) {
        const int t = i / p.dim, d = i % p.dim;
        const int64_t row = (lo + t) * (rot >> 1);
        return rotated(x + t * p.st[which], d, p.cos_table + row, p.sin_table + row, rot, p.interleaved);
    };
    float a = 0.0f;
    for (int i = tid; i < count; i += THREADS) a = fmaxf(a, finite_abs(value(i)));
    __shared__ float red[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((tid & 31) == 0) red[tid >> 5] = a;
    const float before = held ? *scale : 0.0f;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) a = fmaxf(a, red[w]);
    const float s = fmaxf(block_scale(a), before);
    const float inv = 1.0f / s;                                      // a power of two: exact
    if (held && s > before) {
        const float ratio = before * inv;
        for (int i = tid; i < held * p.dim; i += THREADS) codes[i] = float_to_e4m3(e4m3_to_float(codes[i]) * ratio);
    }
    for (int i = tid; i < count; i += THREADS) {
        const float y = value(i);
        codes[held * p.dim + i] = float_to_e4m3(isfinite(y) ? y * inv : __int_as_float(0x7FC00000));
    }
    if (tid == 0) *scale = s;
}

}  // namespace

int kv_append_status_read_and_clear(int *status) {
    int zero = 0;
    PITON_CUDA(cudaMemcpyFromSymbol(status, g_append_status, sizeof(int)));
    PITON_CUDA(cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int)));
    return PITON_B200_OK;
}

}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

extern "C" int piton_b200_kv_append(const piton_kv_append_args *a, void *stream) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->kv_heads > 0 && a->q_heads >= 0 && a->num_pages >= 0 &&
                      a->table_width >= 0 && a->rope_len >= 0,
                  "bad shape");
    PITON_REQUIRE(a->batch < (1 << 24) && a->tokens < (1ll << 31) && a->kv_heads <= (1 << 16) && a->q_heads <= (1 << 16) &&
                      a->num_pages < (1ll << 31),
                  "batch, tokens, heads or pages beyond the 32-bit offsets");
    if ((a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) ||
        (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128))
        return set_error(PITON_B200_ENOTSUP, "head_dim %lld (32, 64, 128) or page_size %lld (16, 32, 64, 128)",
                         (long long)a->head_dim, (long long)a->page_size);
    PITON_REQUIRE(a->rot_dim >= 0 && a->rot_dim <= a->head_dim && a->rot_dim % 2 == 0, "rot_dim %lld", (long long)a->rot_dim);
    if (a->batch == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->cu || a->tokens % a->batch == 0, "%lld tokens are not the same number for %lld sequences",
                  (long long)a->tokens, (long long)a->batch);
    PITON_REQUIRE(a->starts && a->lengths != a->starts, "starts is NULL or the same as lengths");
    PITON_REQUIRE(a->tokens == 0 || (a->k && a->v && a->k_codes && a->v_codes && a->k_scale && a->v_scale && a->table),
                  "NULL pointer");
    PITON_REQUIRE(a->k_codes % 16 == 0 && a->v_codes % 16 == 0, "codes are not 16-byte aligned");
    PITON_REQUIRE(a->tokens == 0 || a->rot_dim == 0 || (a->cos_table && a->sin_table), "rotation tables are NULL");
    PITON_REQUIRE(a->tokens == 0 || a->q_heads == 0 || (a->q && a->q_out), "q or q_out is NULL");
    AppendParams p;
    p.k = reinterpret_cast<const void *>(a->k);
    p.v = reinterpret_cast<const void *>(a->v);
    p.q = reinterpret_cast<const void *>(a->q);
    p.q_out = reinterpret_cast<void *>(a->q_out);
    p.codes[0] = reinterpret_cast<uint8_t *>(a->k_codes);
    p.codes[1] = reinterpret_cast<uint8_t *>(a->v_codes);
    p.scale[0] = reinterpret_cast<float *>(a->k_scale);
    p.scale[1] = reinterpret_cast<float *>(a->v_scale);
    p.table = reinterpret_cast<const int32_t *>(a->table);
    p.starts = reinterpret_cast<const int32_t *>(a->starts);
    p.cu = reinterpret_cast<const int32_t *>(a->cu);
    p.lengths = reinterpret_cast<int32_t *>(a->lengths);
    p.cos_table = reinterpret_cast<const float *>(a->cos_table);
    p.sin_table = reinterpret_cast<const float *>(a->sin_table);
    p.batch = a->batch; p.tokens = a->tokens; p.kv_heads = a->kv_heads; p.q_heads = a->q_heads;
    p.page_size = a->page_size; p.num_pages = a->num_pages; p.table_width = a->table_width; p.table_stride = a->table_stride;
    p.st[0] = a->stride_kt; p.sh[0] = a->stride_kh; p.st[1] = a->stride_vt; p.sh[1] = a->stride_vh;
    p.sqt = a->stride_qt; p.sqh = a->stride_qh; p.sot = a->stride_ot; p.soh = a->stride_oh;
    p.rope_len = a->rope_len;
    p.dim = (int32_t)a->head_dim; p.rot = (int32_t)a->rot_dim; p.interleaved = a->interleaved;
    p.uniform = a->cu ? 0 : a->tokens / a->batch;
    // a run of n tokens touches at most ceil((n - 1) / page_size) + 1 pages
    p.units = a->cu ? a->tokens / a->page_size + 2 * a->batch
                    : a->batch * (p.uniform ? cdiv(p.uniform - 1, a->page_size) + 1 : 1);
    p.unit_blocks = p.units * 2 * a->kv_heads;
    const int64_t blocks = p.unit_blocks + cdiv(a->tokens * a->q_heads, THREADS / 32);
    PITON_REQUIRE(blocks < (1ll << 31), "too many blocks: %lld", (long long)blocks);
    return with_type(a->type, [&](auto t) {
        kv_append_kernel<decltype(t)><<<(unsigned)blocks, THREADS, 0, as_stream(stream)>>>(p);
        return check_launch("kv_append");
    });
}
