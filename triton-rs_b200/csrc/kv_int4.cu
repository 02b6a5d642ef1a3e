// Writing the 4-bit KV cache and reading it back (format: kv_int4.cuh).
//
// All three kernels are one pass over their rows and bound by memory: an append reads 2 D bytes a row and writes
// D/2 + 4 D/G, the read-back the other way round.
#include "kv_int4.cuh"

namespace b200k {

// min / max that keep a NaN (fminf and fmaxf drop it)
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One unit (four dims) of a row per thread; the G/4 threads of a group are neighbours in a warp and agree on its range by
// shuffles.  Every thread of the warp calls this; `row` < 0 stores nothing.
__device__ __forceinline__ void kv4_store_unit(float (&x)[4], long row, int u, int d, int g, int32_t *codes, __half *params) {
    float lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = max_nan(min_nan(x[i], KV4_LIMIT), -KV4_LIMIT);
        lo = i ? min_nan(lo, x[i]) : x[0];
        hi = i ? max_nan(hi, x[i]) : x[0];
    }
    for (int o = 1; o < g / 4; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (row < 0) return;
    const __half base_h = __float2half_rn(lo);
    const float base = __half2float(base_h);
    const __half scale_h = __float2half_rn((hi - base) / 15.f);
    const float scale = __half2float(scale_h);
    uint32_t bits = 0;
    if (scale > 0.f) {   // false for a NaN too: its codes are 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // a division, not a product with the reciprocal: a quotient on the border of two codes is common in 16-bit
            // data and has to be met exactly to go to the even one
            const int c = __float2int_rn((x[i] - base) / scale);
            bits |= (uint32_t)min(max(c, 0), 15) << (4 * i);
        }
    }
    const int place = (u & 7) * (d / 32) + (u >> 3);
    reinterpret_cast<uint16_t *>(codes)[row * (d / 4) + place] = (uint16_t)bits;
    if (u % (g / 4) == 0) reinterpret_cast<__half2 *>(params)[row * (d / g) + u / (g / 4)] = __halves2half2(scale_h, base_h);
}

// New rows [batch, tokens, heads, D] (token pitch stride_t elements) -> cache rows first[b] + t.  Threads are numbered
// (b, t, h, unit), units fastest, and walk the grid in strides of whole warps, so a group never straddles a warp.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const T *__restrict__ nk, const T *__restrict__ nv, Kv4Cache C, const int32_t *__restrict__ first,
                  const int32_t *__restrict__ new_lens, int tokens, long stride_kt, long stride_vt, long total, int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int units = C.d / 4;
    for (long i0 = ((long)blockIdx.x * blockDim.x + threadIdx.x) & ~31l; i0 < total; i0 += (long)gridDim.x * blockDim.x) {
        const long i = i0 + (threadIdx.x & 31);
        const bool live = i < total;
        const long rh = (live ? i : total - 1) / units;
        const int u = (int)((live ? i : total - 1) - rh * units);
        const long bt = rh / C.heads;
        const int h = (int)(rh - bt * C.heads), b = (int)(bt / tokens), t = (int)(bt - (long)b * tokens);
        int n = tokens;
        if (new_lens) {
            n = new_lens[b];
            if (n > tokens) {
                n = tokens;
                if (t == 0 && h == 0 && u == 0) atomicOr(status, KV4_BAD_POSITION);
            }
        }
        long row = -1;
        if (live && t < n) {
            const long pos = (long)first[b] + t;
            if ((unsigned long)pos < (unsigned long)C.capacity) {
                row = kv4_row(C, b, h, (int)pos);
                if (row < 0 && u == 0) atomicOr(status, KV4_BAD_BLOCK);
            } else if (u == 0) {
                atomicOr(status, KV4_BAD_POSITION);
            }
        }
        float x[4], y[4];
        Kv4Elem<T>::load(nk + bt * stride_kt + (long)h * C.d + 4 * u, x);
        Kv4Elem<T>::load(nv + bt * stride_vt + (long)h * C.d + 4 * u, y);
        kv4_store_unit(x, row, u, C.d, C.g, C.k_codes, C.k_params);
        kv4_store_unit(y, row, u, C.d, C.g, C.v_codes, C.v_params);
    }
}

// A fused QKV row a sequence [q heads | k heads | v heads] -> q_out rotated, k rotated and quantised, v quantised.
// Rotation of the pairs (i, i + D/2) as in rope_full; the products and their sum are each rounded on their own, so that
// the key that is quantised does not depend on which of them a compiler contracts, and the key is rounded to its type
// first, as in the unfused sequence.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_rope_append_kernel(const T *__restrict__ qkv, const float *__restrict__ cos_t, const float *__restrict__ sin_t,
                       const int32_t *__restrict__ positions, T *__restrict__ q_out, Kv4Cache C, int32_t *__restrict__ lens_out, int hq,
                       int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, units = C.d / 4, heads = hq + 2 * C.heads, total = heads * units;
    int pos = positions[b];
    // A position outside the cache: as in rope_kv_append_hm, nothing is stored, q is rotated with the nearest valid table
    // row, the length handed on stays within the cache and the status word says so.
    const bool in_range = (unsigned)pos < (unsigned)C.capacity;
    if (!in_range) {
        pos = pos < 0 ? 0 : C.capacity - 1;
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(status, KV4_BAD_POSITION);
    }
    if (lens_out && threadIdx.x == 0 && blockIdx.x == 0) lens_out[b] = pos + 1;
    const int half = C.d / 2;
    const T *row = qkv + (size_t)b * heads * C.d;
    for (int i0 = (blockIdx.x * blockDim.x + threadIdx.x) & ~31; i0 < total; i0 += gridDim.x * blockDim.x) {
        const bool live = i0 + (int)(threadIdx.x & 31) < total;
        const int i = live ? i0 + (threadIdx.x & 31) : total - 1;
        const int h = i / units, u = i - h * units;
        float x[4];
        Kv4Elem<T>::load(row + (size_t)h * C.d + 4 * u, x);
        if (h < hq + C.heads) {
            const bool upper = 4 * u >= half;
            const int p = 4 * u - (upper ? half : 0);
            float y[4];
            Kv4Elem<T>::load(row + (size_t)h * C.d + (upper ? p : p + half), y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c = cos_t[(size_t)pos * half + p + e], s = sin_t[(size_t)pos * half + p + e];
                const float a = __fmul_rn(x[e], c), z = __fmul_rn(y[e], s);
                x[e] = Kv4Elem<T>::round(upper ? __fadd_rn(a, z) : __fsub_rn(a, z));
            }
            if (h < hq && live)
                *reinterpret_cast<uint2 *>(q_out + ((size_t)b * hq + h) * C.d + 4 * u) =
                    make_uint2(Kv4Elem<T>::pack(x[0], x[1]), Kv4Elem<T>::pack(x[2], x[3]));
        }
        const int kvh = h < hq + C.heads ? h - hq : h - hq - C.heads;
        const long r = live && in_range && h >= hq ? kv4_row(C, b, kvh, pos) : -1;
        const bool is_v = h >= hq + C.heads;
        kv4_store_unit(x, r, u, C.d, C.g, is_v ? C.v_codes : C.k_codes, is_v ? C.v_params : C.k_params);
    }
}

// Rows first[b] + i of the cache, i < out_len and below context_lens[b] -> out [batch, heads, out_len, D]; rows behind
// them are left as they were.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Cache C, const int32_t *__restrict__ first, const int32_t *__restrict__ lens, T *__restrict__ k_out, T *__restrict__ v_out,
                int out_len, long total, int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int units = C.d / 4;
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long)gridDim.x * blockDim.x) {
        const long r = i / units;                 // row of the output
        const int place = (int)(i - r * units);
        const long bh = r / out_len;
        const int b = (int)(bh / C.heads), h = (int)(bh - (long)b * C.heads);
        const long pos = (first ? (long)first[b] : 0) + (r - bh * out_len);
        int len = lens[b];
        if (len > C.capacity) {
            len = C.capacity;
            if (place == 0) atomicOr(status, KV4_BAD_POSITION);
        }
        if (pos >= len) continue;
        if (pos < 0) {
            if (place == 0) atomicOr(status, KV4_BAD_POSITION);
            continue;
        }
        const long row = kv4_row(C, b, h, (int)pos);
        if (row < 0) {
            if (place == 0) atomicOr(status, KV4_BAD_BLOCK);
            continue;
        }
        const int nb = C.d / 32, u = (place % nb) * 8 + place / nb;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint32_t bits = reinterpret_cast<const uint16_t *>(kv ? C.v_codes : C.k_codes)[row * units + place];
            const float2 p = __half22float2(reinterpret_cast<const __half2 *>(kv ? C.v_params : C.k_params)[row * (C.d / C.g) + 4 * u / C.g]);
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = fmaf((float)((bits >> (4 * e)) & 15u), p.x, p.y);
            *reinterpret_cast<uint2 *>((kv ? v_out : k_out) + r * C.d + 4 * u) =
                make_uint2(Kv4Elem<T>::pack(f[0], f[1]), Kv4Elem<T>::pack(f[2], f[3]));
        }
    }
}

static int kv4_grid(long threads) {
    const long blocks = (threads + 255) / 256, cap = (long)sm_count() * 32;
    return (int)(blocks < cap ? blocks : cap);
}

template <typename T>
static int kv4_append_launch(const char *name, const T *nk, const T *nv, const Kv4Cache &C, bool paged, const int32_t *first, const int32_t *new_lens,
                             int batch, int tokens, int stride_kt, int stride_vt, b200k_stream stream) {
    B200K_REQUIRE(nk && nv && first, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, paged);
    if (rc) return rc;
    B200K_REQUIRE(tokens >= 0 && stride_kt >= C.heads * C.d && stride_vt >= C.heads * C.d, B200K_E_SHAPE,
                  "%s: tokens %d, strides %d and %d (at least heads * head_dim = %d)", name, tokens, stride_kt, stride_vt, C.heads * C.d);
    B200K_REQUIRE(aligned16(nk) && aligned16(nv) && stride_kt % 8 == 0 && stride_vt % 8 == 0, B200K_E_ALIGN,
                  "%s: new_keys and new_values must be 16-byte aligned, their token strides multiples of 8", name);
    const long total = (long)batch * tokens * C.heads * (C.d / 4);
    if (total == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    launch_kernel(kv4_append_kernel<T>, dim3(kv4_grid(total)), dim3(256), 0, to_stream(stream), nk, nv, C, first, new_lens, tokens, (long)stride_kt,
                  (long)stride_vt, total, status);
    return launch_status(name);
}

template <typename T>
static int kv4_rope_append_launch(const char *name, const T *qkv, const float *cos_t, const float *sin_t, const int32_t *positions, T *q_out,
                                  const Kv4Cache &C, int32_t *lens_out, int hq, int batch, b200k_stream stream) {
    B200K_REQUIRE(qkv && cos_t && sin_t && positions && q_out, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, false);
    if (rc) return rc;
    B200K_REQUIRE(hq > 0, B200K_E_SHAPE, "%s: num_q_heads %d", name, hq);
    B200K_REQUIRE(aligned16(qkv) && aligned16(q_out), B200K_E_ALIGN, "%s: qkv and q_out must be 16-byte aligned", name);
    if (batch == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    const int total = (hq + 2 * C.heads) * (C.d / 4);
    launch_kernel(kv4_rope_append_kernel<T>, dim3(ceil_div(total, 256), batch), dim3(256), 0, to_stream(stream), qkv, cos_t, sin_t, positions, q_out, C,
                  lens_out, hq, status);
    return launch_status(name);
}

template <typename T>
static int kv4_read_launch(const char *name, const Kv4Cache &C, bool paged, const int32_t *first, const int32_t *lens, T *k_out, T *v_out, int batch,
                           int out_len, b200k_stream stream) {
    B200K_REQUIRE(lens && k_out && v_out, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, paged);
    if (rc) return rc;
    B200K_REQUIRE(out_len >= 0, B200K_E_SHAPE, "%s: out_len %d", name, out_len);
    B200K_REQUIRE(aligned16(k_out) && aligned16(v_out), B200K_E_ALIGN, "%s: k_out and v_out must be 16-byte aligned", name);
    const long total = (long)batch * C.heads * out_len * (C.d / 4);
    if (total == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    launch_kernel(kv4_read_kernel<T>, dim3(kv4_grid(total)), dim3(256), 0, to_stream(stream), C, first, lens, k_out, v_out, out_len, total, status);
    return launch_status(name);
}

int rope_kv_append_int4_lens_launch(const __half *qkv, const float *cos_t, const float *sin_t, const int32_t *positions, __half *q_out, int32_t *kc,
                                    __half *kp, int32_t *vc, __half *vp, int32_t *lens_out, int hq, int hkv, int d, int g, int max_len, int batch,
                                    cudaStream_t st) {
    return kv4_rope_append_launch<__half>("rope_kv_append_hm_int4_f16", qkv, cos_t, sin_t, positions, q_out,
                                          kv4_cache(kc, (const b200k_half *)kp, vc, (const b200k_half *)vp, hkv, d, g, max_len), lens_out, hq, batch,
                                          (b200k_stream)st);
}

}  // namespace b200k

using namespace b200k;

// ---------------------------------------------------------------------------
// C ABI: each entry point in an fp16 and a bf16 edition
// ---------------------------------------------------------------------------
#define KV4_ENTRIES(SUF, ABI, T)                                                                                                          \
    extern "C" int kv_cache_append_hm_int4_##SUF(const ABI *new_keys, const ABI *new_values, int32_t *k_codes, b200k_half *k_params,       \
                                                 int32_t *v_codes, b200k_half *v_params, const int32_t *cache_idx, const int32_t *new_lens, \
                                                 int num_heads, int head_dim, int group_size, int max_len, int batch, int tokens,          \
                                                 int stride_kt, int stride_vt, b200k_stream stream) {                                      \
        return kv4_append_launch<T>("kv_cache_append_hm_int4_" #SUF, (const T *)new_keys, (const T *)new_values,                           \
                                    kv4_cache(k_codes, k_params, v_codes, v_params, num_heads, head_dim, group_size, max_len), false,      \
                                    cache_idx, new_lens, batch, tokens, stride_kt, stride_vt, stream);                                     \
    }                                                                                                                                      \
    extern "C" int kv_cache_append_paged_int4_##SUF(const ABI *new_keys, const ABI *new_values, int32_t *k_codes, b200k_half *k_params,    \
                                                    int32_t *v_codes, b200k_half *v_params, const int32_t *block_table,                    \
                                                    const int32_t *cache_idx, const int32_t *new_lens, int num_heads, int head_dim,        \
                                                    int group_size, int block_size, int num_blocks, int max_blocks_per_seq, int batch,     \
                                                    int tokens, int stride_kt, int stride_vt, b200k_stream stream) {                       \
        return kv4_append_launch<T>("kv_cache_append_paged_int4_" #SUF, (const T *)new_keys, (const T *)new_values,                        \
                                    kv4_pool(k_codes, k_params, v_codes, v_params, block_table, num_heads, head_dim, group_size,           \
                                             block_size, num_blocks, max_blocks_per_seq), true, cache_idx, new_lens, batch, tokens,        \
                                    stride_kt, stride_vt, stream);                                                                         \
    }                                                                                                                                      \
    extern "C" int rope_kv_append_hm_int4_##SUF(const ABI *qkv, const float *cos_table, const float *sin_table, const int32_t *positions,  \
                                                ABI *q_out, int32_t *k_codes, b200k_half *k_params, int32_t *v_codes,                      \
                                                b200k_half *v_params, int num_q_heads, int num_kv_heads, int head_dim, int group_size,     \
                                                int max_len, int batch, b200k_stream stream) {                                             \
        return kv4_rope_append_launch<T>("rope_kv_append_hm_int4_" #SUF, (const T *)qkv, cos_table, sin_table, positions, (T *)q_out,      \
                                         kv4_cache(k_codes, k_params, v_codes, v_params, num_kv_heads, head_dim, group_size, max_len),     \
                                         nullptr, num_q_heads, batch, stream);                                                             \
    }                                                                                                                                      \
    extern "C" int kv_cache_read_hm_int4_##SUF(const int32_t *k_codes, const b200k_half *k_params, const int32_t *v_codes,                 \
                                               const b200k_half *v_params, const int32_t *first, const int32_t *context_lens, ABI *k_out,  \
                                               ABI *v_out, int num_heads, int head_dim, int group_size, int max_len, int batch,            \
                                               int out_len, b200k_stream stream) {                                                         \
        return kv4_read_launch<T>("kv_cache_read_hm_int4_" #SUF,                                                                           \
                                  kv4_cache(k_codes, k_params, v_codes, v_params, num_heads, head_dim, group_size, max_len), false, first, \
                                  context_lens, (T *)k_out, (T *)v_out, batch, out_len, stream);                                           \
    }                                                                                                                                      \
    extern "C" int kv_cache_read_paged_int4_##SUF(const int32_t *k_codes, const b200k_half *k_params, const int32_t *v_codes,              \
                                                  const b200k_half *v_params, const int32_t *block_table, const int32_t *first,            \
                                                  const int32_t *context_lens, ABI *k_out, ABI *v_out, int num_heads, int head_dim,        \
                                                  int group_size, int block_size, int num_blocks, int max_blocks_per_seq, int batch,       \
                                                  int out_len, b200k_stream stream) {                                                      \
        return kv4_read_launch<T>("kv_cache_read_paged_int4_" #SUF,                                                                        \
                                  kv4_pool(k_codes, k_params, v_codes, v_params, block_table, num_heads, head_dim, group_size, block_size, \
                                           num_blocks, max_blocks_per_seq), true, first, context_lens, (T *)k_out, (T *)v_out, batch,      \
                                  out_len, stream);                                                                                        \
    }

KV4_ENTRIES(f16, b200k_half, __half)
KV4_ENTRIES(bf16, b200k_bf16, __nv_bfloat16)
