// GQA decode attention over the 4-bit KV cache (format: kv_int4.cuh).
//
// One CTA per (sequence, q head); warp w takes positions w, w + 4, ...; lanes stride over the units of a row.  Online
// softmax per warp in fp32, merged across the warps at the end.
#include "kv_int4.cuh"

namespace b200k {

struct Attn4Args {
    const void *q;                // [B, Hq, D]
    void *out;                    // [B, Hq, D]
    const int32_t *lens;
    Kv4Cache C;
    int hq;
    float scale;
    int *status;
};

template <typename T>
__global__ void __launch_bounds__(128)
attn4_kernel(Attn4Args A) {
    __shared__ float sm_acc[4][256], sm_m[4], sm_l[4];
    const Kv4Cache &C = A.C;
    const int h = blockIdx.x, b = blockIdx.y, kvh = h / (A.hq / C.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = C.d / 4, nb = C.d / 32, groups = C.d / C.g;
    pdl_wait();
    pdl_launch_dependents();
    int len = A.lens[b];
    if (len > C.capacity) {
        len = C.capacity;
        if (threadIdx.x == 0 && h == 0) atomicOr(A.status, KV4_BAD_POSITION);
    }
    const T *q = (const T *)A.q + ((long)b * A.hq + h) * C.d;
    float qr[2][4], acc[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int place = lane + 32 * i, u = (place % nb) * 8 + place / nb;
#pragma unroll
        for (int e = 0; e < 4; ++e) qr[i][e] = acc[i][e] = 0.f;
        if (place < units) Kv4Elem<T>::load(q + 4 * u, qr[i]);
    }
    float m = -INFINITY, l = 0.f;
    for (int pos = warp; pos < len; pos += 4) {
        const long row = kv4_row(C, b, kvh, pos);
        if (row < 0) {      // a block that the pool does not have: its positions are left out
            if (lane == 0) atomicOr(A.status, KV4_BAD_BLOCK);
            continue;
        }
        float dot = 0.f, v[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int place = lane + 32 * i, gi = 4 * ((place % nb) * 8 + place / nb) / C.g;
            if (place >= units) continue;
            const uint32_t kb = reinterpret_cast<const uint16_t *>(C.k_codes)[row * units + place];
            const uint32_t vb = reinterpret_cast<const uint16_t *>(C.v_codes)[row * units + place];
            const float2 kp = __half22float2(reinterpret_cast<const __half2 *>(C.k_params)[row * groups + gi]);
            const float2 vp = __half22float2(reinterpret_cast<const __half2 *>(C.v_params)[row * groups + gi]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dot += qr[i][e] * fmaf((float)((kb >> (4 * e)) & 15u), kp.x, kp.y);
                v[i][e] = fmaf((float)((vb >> (4 * e)) & 15u), vp.x, vp.y);
            }
        }
        const float s = warp_sum(dot) * A.scale;
        const float mn = fmaxf(m, s), alpha = expf(m - mn), p = expf(s - mn);
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 32 * i < units) acc[i][e] = acc[i][e] * alpha + p * v[i][e];
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int place = lane + 32 * i, u = (place % nb) * 8 + place / nb;
        if (place < units)
#pragma unroll
            for (int e = 0; e < 4; ++e) sm_acc[warp][4 * u + e] = acc[i][e];
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    float w[4], L = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] = sm_l[j] == 0.f ? 0.f : expf(sm_m[j] - M);
        L += sm_l[j] * w[j];
    }
    for (int i = 2 * threadIdx.x; i < C.d; i += 256) {
        float o[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[0] += sm_acc[j][i] * w[j];
            o[1] += sm_acc[j][i + 1] * w[j];
        }
        // no keys: a zero output row
        reinterpret_cast<uint32_t *>((T *)A.out + ((long)b * A.hq + h) * C.d)[i / 2] = L == 0.f ? 0u : Kv4Elem<T>::pack(o[0] / L, o[1] / L);
    }
}

constexpr size_t ATTN4_WS_BYTES = 128 * 1024;

template <typename T>
static int attn4_launch(const char *name, const void *q, const Kv4Cache &C, bool paged, const int32_t *lens, void *out, int batch, int hq,
                        float scale, void *ws, size_t ws_bytes, bool own_ws, b200k_stream stream) {
    B200K_REQUIRE(q && lens && out, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, paged);
    if (rc) return rc;
    B200K_REQUIRE(hq > 0 && hq % C.heads == 0, B200K_E_SHAPE, "%s: num_q_heads %d, num_kv_heads %d", name, hq, C.heads);
    B200K_REQUIRE(aligned16(q) && aligned16(out), B200K_E_ALIGN, "%s: q and output must be 16-byte aligned", name);
    if (batch == 0) return 0;
    if (own_ws) {
        rc = default_workspace(&ws, &ws_bytes);
        if (rc) return rc;
    }
    B200K_REQUIRE(ws && aligned16(ws) && ws_bytes >= ATTN4_WS_BYTES, B200K_E_WORKSPACE, "%s: workspace %zu bytes, need %zu", name, ws_bytes, ATTN4_WS_BYTES);
    Attn4Args A = {};
    A.q = q; A.out = out; A.lens = lens; A.C = C; A.hq = hq; A.scale = scale; A.status = (int *)ws;
    launch_kernel(attn4_kernel<T>, dim3(hq, batch), dim3(128), 0, to_stream(stream), A);
    return launch_status(name);
}

}  // namespace b200k

using namespace b200k;

extern "C" size_t b200k_attention_int4_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int head_dim) {
    if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0) return 0;
    return ATTN4_WS_BYTES;
}

#define ATTN4_ENTRIES(SUF, ABI, T)                                                                                                          \
    extern "C" int batched_decode_attention_hm_int4_##SUF##_ws(const ABI *q, const int32_t *k_codes, const b200k_half *k_params,             \
                                                               const int32_t *v_codes, const b200k_half *v_params,                          \
                                                               const int32_t *context_lens, ABI *output, int batch_size, int num_q_heads,   \
                                                               int num_kv_heads, int head_dim, int group_size, int max_len, float scale,    \
                                                               void *workspace, size_t workspace_bytes, b200k_stream stream) {              \
        return attn4_launch<T>("batched_decode_attention_hm_int4_" #SUF, q,                                                                 \
                               kv4_cache(k_codes, k_params, v_codes, v_params, num_kv_heads, head_dim, group_size, max_len), false,         \
                               context_lens, output, batch_size, num_q_heads, scale, workspace, workspace_bytes, workspace == nullptr, stream); \
    }                                                                                                                                       \
    extern "C" int batched_decode_attention_hm_int4_##SUF(const ABI *q, const int32_t *k_codes, const b200k_half *k_params,                  \
                                                          const int32_t *v_codes, const b200k_half *v_params, const int32_t *context_lens,  \
                                                          ABI *output, int batch_size, int num_q_heads, int num_kv_heads, int head_dim,     \
                                                          int group_size, int max_len, float scale, b200k_stream stream) {                  \
        return batched_decode_attention_hm_int4_##SUF##_ws(q, k_codes, k_params, v_codes, v_params, context_lens, output, batch_size,       \
                                                           num_q_heads, num_kv_heads, head_dim, group_size, max_len, scale, nullptr, 0, stream); \
    }                                                                                                                                       \
    extern "C" int batched_decode_attention_paged_int4_##SUF##_ws(                                                                          \
        const ABI *q, const int32_t *k_codes, const b200k_half *k_params, const int32_t *v_codes, const b200k_half *v_params,               \
        const int32_t *block_table, const int32_t *context_lens, ABI *output, int batch_size, int num_q_heads, int num_kv_heads,            \
        int head_dim, int group_size, int block_size, int num_blocks, int max_blocks_per_seq, float scale, void *workspace,                 \
        size_t workspace_bytes, b200k_stream stream) {                                                                                      \
        return attn4_launch<T>("batched_decode_attention_paged_int4_" #SUF, q,                                                              \
                               kv4_pool(k_codes, k_params, v_codes, v_params, block_table, num_kv_heads, head_dim, group_size, block_size,  \
                                        num_blocks, max_blocks_per_seq), true, context_lens, output, batch_size, num_q_heads, scale,        \
                               workspace, workspace_bytes, workspace == nullptr, stream);                                                   \
    }                                                                                                                                       \
    extern "C" int batched_decode_attention_paged_int4_##SUF(                                                                               \
        const ABI *q, const int32_t *k_codes, const b200k_half *k_params, const int32_t *v_codes, const b200k_half *v_params,               \
        const int32_t *block_table, const int32_t *context_lens, ABI *output, int batch_size, int num_q_heads, int num_kv_heads,            \
        int head_dim, int group_size, int block_size, int num_blocks, int max_blocks_per_seq, float scale, b200k_stream stream) {           \
        return batched_decode_attention_paged_int4_##SUF##_ws(q, k_codes, k_params, v_codes, v_params, block_table, context_lens, output,   \
                                                              batch_size, num_q_heads, num_kv_heads, head_dim, group_size, block_size,      \
                                                              num_blocks, max_blocks_per_seq, scale, nullptr, 0, stream);                   \
    }

ATTN4_ENTRIES(f16, b200k_half, __half)
ATTN4_ENTRIES(bf16, b200k_bf16, __nv_bfloat16)
