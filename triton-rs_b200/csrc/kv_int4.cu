// Writing the 4-bit KV cache and reading it back (format: kv_int4.cuh).
//
// All three kernels are one pass over their rows and bound by memory: an append reads 2 D bytes a row and writes
// D/2 + 4 D/G, the read-back the other way round.
#include <type_traits>

#include "kv_int4.cuh"

namespace b200k {

// ---- 16-bit pairs ---------------------------------------------------------------------------------------------------
template <typename T> struct Kv4Pair;
template <> struct Kv4Pair<__half> {
    using type = __half2;
    __device__ static float2 wide(uint32_t w) { return h2_to_f2(w); }
    __device__ static uint32_t pack(float a, float b) { return f2_to_h2(a, b); }
};
template <> struct Kv4Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    __device__ static float2 wide(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    __device__ static uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
// minimum and maximum of both halves; a NaN stays
template <typename T> __device__ __forceinline__ uint32_t pair_min(uint32_t a, uint32_t b) {
    using P = typename Kv4Pair<T>::type;
    const P m = __hmin2_nan(*reinterpret_cast<P *>(&a), *reinterpret_cast<P *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}
template <typename T> __device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
    using P = typename Kv4Pair<T>::type;
    const P m = __hmax2_nan(*reinterpret_cast<P *>(&a), *reinterpret_cast<P *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}

// a / b for normal a, b and y = 1 / b to 2^-23 (Markstein's division with a fused multiply-add): the remainder of the first
// quotient is exact, so a quotient that fp32 can hold comes out exact, and any other rounded to nearest but for a
// hair's breadth around the middle of two numbers.
__device__ __forceinline__ float kv4_quotient(float a, float b, float y) {
    const float q = a * y;
    return fmaf(fmaf(-q, b, a), y, q);
}

// two fp32 numbers in a register pair, each operation one instruction for both
struct Kv4Two {
    unsigned long long v;
    __device__ Kv4Two(unsigned long long v) : v(v) {}
    __device__ Kv4Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ explicit Kv4Two(float2 a) : Kv4Two(a.x, a.y) {}
    __device__ friend Kv4Two operator+(Kv4Two a, Kv4Two b) { asm("add.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v)); return a; }
    __device__ friend Kv4Two operator*(Kv4Two a, Kv4Two b) { asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v)); return a; }
    __device__ uint32_t low() const { return (uint32_t)v; }
    __device__ uint32_t high() const { return (uint32_t)(v >> 32); }
};
__device__ __forceinline__ Kv4Two kv4_fma(Kv4Two a, Kv4Two b, Kv4Two c) {
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(a.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return a;
}
// the same quotients of two numbers: `minus_b` holds -b
__device__ __forceinline__ Kv4Two kv4_quotient(Kv4Two a, Kv4Two minus_b, Kv4Two y) {
    const Kv4Two q = a * y;
    return kv4_fma(kv4_fma(q, minus_b, a), y, q);
}

// ---- one row by eight neighbouring threads ----------------------------------------------------------------------------
// Thread r has the units (j, r) of all NB 32-dim blocks j: dims 32 j + 4 r .. + 3, x[2 j] and x[2 j + 1] in pairs.  Its codes
// are 2 NB neighbouring bytes of the stored row.  The range of a group is the minimum of (x, -x) over its blocks and, by
// three shuffles, over the eight threads, all of which call this; `row` < 0 stores nothing.
// A quotient on the border of two codes is common in 16-bit data and has to go to the even code, which a product with the
// reciprocal can miss; see kv4_quotient.  A sum with 1.5 * 2^23 then rounds it.  5 instructions for two elements where the
// compiler's division, good for all operands, takes some 20 for each.  Groups that need a clamp somewhere take the division.
template <typename T>
__device__ __noinline__ uint32_t kv4_codes_clamped(uint32_t x0, uint32_t x1, float base, float scale) {
    const float2 a = Kv4Pair<T>::wide(x0), c = Kv4Pair<T>::wide(x1);
    const float f[4] = {a.x, a.y, c.x, c.y};
    uint32_t code = 0;
    if (scale > 0.f)                         // false for a NaN too: its codes are 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = fminf(fmaxf(f[i], -KV4_LIMIT), KV4_LIMIT);
            code |= (uint32_t)min(max(__float2int_rn((v - base) / scale), 0), 15) << (4 * i);
        }
    return code;
}

template <typename T, int NB, int BPG>
__device__ __forceinline__ void kv4_store_row(const uint32_t (&x)[2 * NB], long row, int r, int32_t *codes, __half *params) {
    constexpr float MAGIC = 12582912.f;      // 1.5 * 2^23: a sum with it is rounded to a whole number, which its low bits hold
    uint32_t range[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) range[j] = pair_min<T>(x[2 * j], x[2 * j + 1]);      // for now both halves: minimum
    uint32_t upper[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) upper[j] = pair_max<T>(x[2 * j], x[2 * j + 1]);
    // blocks of a group
#pragma unroll
    for (int step = 1; step < 4; step <<= 1)
        if (BPG > step)
#pragma unroll
            for (int j = 0; j + step < NB; j += 2 * step) {
                range[j] = pair_min<T>(range[j], range[j + step]);
                upper[j] = pair_max<T>(upper[j], upper[j + step]);
            }
    uint32_t bits[NB];
    float bases[NB / BPG], scales[NB / BPG], inv = 0.f;      // BPG blocks are a group
    unsigned clamped = 0;                    // groups
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        float &base = bases[j / BPG], &scale = scales[j / BPG];
        if (j % BPG == 0) {                  // a new group
            // (minimum, -maximum) in one register
            uint32_t lo = pair_min<T>(range[j], range[j] >> 16 | range[j] << 16);
            uint32_t hi = pair_max<T>(upper[j], upper[j] >> 16 | upper[j] << 16) ^ 0x80008000u;
            uint32_t both = __byte_perm(lo, hi, 0x5410);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) both = pair_min<T>(both, __shfl_xor_sync(0xffffffffu, both, o));
            const float2 f = Kv4Pair<T>::wide(both);
            // min.NaN / max.NaN: a NaN passes the clamp
            float least, most;
            asm("{ .reg .f32 a; max.NaN.f32 a, %1, %2; min.NaN.f32 %0, a, %3; }" : "=f"(least) : "f"(f.x), "f"(-KV4_LIMIT), "f"(KV4_LIMIT));
            asm("{ .reg .f32 a; max.NaN.f32 a, %1, %2; min.NaN.f32 %0, a, %3; }" : "=f"(most) : "f"(-f.y), "f"(-KV4_LIMIT), "f"(KV4_LIMIT));
            const __half base_h = __float2half_rn(least);
            base = __half2float(base_h);
            const __half scale_h = __float2half_rn(kv4_quotient(most - base, 15.f, 1.f / 15.f));
            scale = __half2float(scale_h);
            // nothing to clamp: values inside the limits, and a scale that is rounded by 2^-11 at most
            clamped |= least == f.x && most == -f.y && scale >= 1.f / 8192.f ? 0u : 1u << (j / BPG);
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
            if (row >= 0 && r == j / BPG) reinterpret_cast<__half2 *>(params)[row * (NB / BPG) + j / BPG] = __halves2half2(scale_h, base_h);
        }
        uint32_t code = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Kv4Two a = Kv4Two(Kv4Pair<T>::wide(x[2 * j + i])) + Kv4Two(-base, -base);
            const Kv4Two c = kv4_quotient(a, Kv4Two(-scale, -scale), Kv4Two(inv, inv)) + Kv4Two(MAGIC, MAGIC);
            // the low bits of MAGIC are 0: only the nibble reaches the low 16 bits
            code += c.low() * (1u << (8 * i)) + c.high() * (16u << (8 * i));
        }
        bits[j] = code;
    }
    if (clamped)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (clamped >> (j / BPG) & 1) bits[j] = kv4_codes_clamped<T>(x[2 * j], x[2 * j + 1], bases[j / BPG], scales[j / BPG]);
    if (row < 0) return;
    unsigned char *to = reinterpret_cast<unsigned char *>(codes) + row * (16 * NB) + r * (2 * NB);
    if constexpr (NB % 2) {
#pragma unroll
        for (int j = 0; j < NB; ++j) reinterpret_cast<uint16_t *>(to)[j] = (uint16_t)bits[j];
    } else {
        uint32_t w[NB / 2];
#pragma unroll
        for (int j = 0; j < NB / 2; ++j) w[j] = __byte_perm(bits[2 * j], bits[2 * j + 1], 0x5410);
        if constexpr (NB == 8) *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (NB == 4) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
        else
#pragma unroll
            for (int j = 0; j < NB / 2; ++j) reinterpret_cast<uint32_t *>(to)[j] = w[j];
    }
}

template <typename T, int NB>
__device__ __forceinline__ void kv4_load_row(uint32_t (&x)[2 * NB], const T *row, int r) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const uint2 u = *reinterpret_cast<const uint2 *>(row + 32 * j + 4 * r);
        x[2 * j] = u.x;
        x[2 * j + 1] = u.y;
    }
}

// New rows [batch, tokens, heads, D] (token pitch stride_t elements) -> cache rows first[b] + t.  Eight threads a row of K and the
// same row of V, rows of a sequence (blockIdx.y) numbered (t, h).
// One sequence, 8192 tokens of 8 heads, D 128, bf16, groups of 128: 10.8 us, 6.5 us being the bytes at copy bandwidth; the issue of
// instructions bounds it (each element's quantisation, and a third of them for places and ranges).  With K and V in threads of
// their own, which search for their place twice, 16.4 us; with every operation of the quantisation on one number 11.9.  One token
// each of 64 sequences: 2.1 us, the time of a launch.
template <typename T, int NB, int BPG>
__global__ void __launch_bounds__(128)
kv4_append_kernel(const T *__restrict__ nk, const T *__restrict__ nv, Kv4Cache C, const int32_t *__restrict__ first,
                  const int32_t *__restrict__ new_lens, int tokens, long stride_kt, long stride_vt, int *status) {
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, r = threadIdx.x & 7;
    const long start = first[b];
    int n = tokens;
    if (new_lens) {
        n = new_lens[b];
        if (n > tokens) {
            n = tokens;
            if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(status, KV4_BAD_POSITION);
        }
    }
    const unsigned rows = C.heads * (unsigned)max(n, 0);
    for (unsigned i0 = (blockIdx.x * blockDim.x + threadIdx.x & ~31u) >> 3; i0 < rows; i0 += gridDim.x * blockDim.x >> 3) {
        const unsigned i = i0 + ((threadIdx.x & 31) >> 3);
        const bool live = i < rows;
        const unsigned th = live ? i : 0u, t = th / (unsigned)C.heads, h = th - t * C.heads;
        uint32_t x[2 * NB], y[2 * NB];
        const long at = (long)b * tokens + t, in_row = (long)h * (32 * NB);
        kv4_load_row<T, NB>(x, nk + at * stride_kt + in_row, r);
        kv4_load_row<T, NB>(y, nv + at * stride_vt + in_row, r);
        long row = -1;
        if (live) {
            const long pos = start + t;
            if ((unsigned long)pos < (unsigned long)C.capacity) {
                row = kv4_row(C, b, h, (int)pos);
                if (row < 0 && r == 0) atomicOr(status, KV4_BAD_BLOCK);
            } else if (r == 0) {
                atomicOr(status, KV4_BAD_POSITION);
            }
        }
        kv4_store_row<T, NB, BPG>(x, row, r, C.k_codes, C.k_params);
        kv4_store_row<T, NB, BPG>(y, row, r, C.v_codes, C.v_params);
    }
}

// A fused QKV row a sequence [q heads | k heads | v heads] -> q_out rotated, k rotated and quantised, v quantised.
// Rotation of the pairs (i, i + D/2) as in rope_full; the products and their sum are each rounded on their own, so that
// the key that is quantised does not depend on which of them a compiler contracts, and the key is rounded to its type
// first, as in the unfused sequence.  Eight threads a head; the other half of a pair is the same thread's where the
// number of blocks is even, and loaded again (from L1) where it is odd.
// 64 sequences of 32 + 2 x 8 heads: 2.0 us, 512 sequences 4.4 us: launch and three dependent loads (position, table row, qkv) bound it.
template <typename T, int NB, int BPG>
__global__ void __launch_bounds__(128)
kv4_rope_append_kernel(const T *__restrict__ qkv, const float *__restrict__ cos_t, const float *__restrict__ sin_t,
                       const int32_t *__restrict__ positions, T *__restrict__ q_out, Kv4Cache C, int32_t *__restrict__ lens_out, int hq,
                       int vec, int *status) {
    constexpr int D = 32 * NB, HALF = D / 2;
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, heads = hq + 2 * C.heads, r = threadIdx.x & 7;
    int pos = positions[b];
    // A position outside the cache: as in rope_kv_append_hm, nothing is stored, q is rotated with the nearest valid table
    // row, the length handed on stays within the cache and the status word says so.
    const bool in_range = (unsigned)pos < (unsigned)C.capacity;
    if (!in_range) {
        pos = pos < 0 ? 0 : C.capacity - 1;
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(status, KV4_BAD_POSITION);
    }
    if (lens_out && threadIdx.x == 0 && blockIdx.x == 0) lens_out[b] = pos + 1;
    const int h0 = (blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const bool live = h0 < heads;
    const int h = live ? h0 : 0;
    const T *row = qkv + ((size_t)b * heads + h) * D;
    uint32_t x[2 * NB];
    kv4_load_row<T, NB>(x, row, r);
    if (h < hq + C.heads) {
        const float *cr = cos_t + (size_t)pos * HALF, *sr = sin_t + (size_t)pos * HALF;
        uint32_t other[2 * NB];
        if constexpr (NB % 2) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int d = 32 * j + 4 * r;
                const uint2 u = *reinterpret_cast<const uint2 *>(row + (d < HALF ? d + HALF : d - HALF));
                other[2 * j] = u.x;
                other[2 * j + 1] = u.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) other[j] = x[(j + NB) % (2 * NB)];
        }
        uint32_t out[2 * NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int d = 32 * j + 4 * r;
            const bool upper = d >= HALF;
            const int p = d - (upper ? HALF : 0);
            float c[4], s[4];
            if (vec) {
                const float4 c4 = *reinterpret_cast<const float4 *>(cr + p), s4 = *reinterpret_cast<const float4 *>(sr + p);
                c[0] = c4.x; c[1] = c4.y; c[2] = c4.z; c[3] = c4.w;
                s[0] = s4.x; s[1] = s4.y; s[2] = s4.z; s[3] = s4.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) { c[e] = cr[p + e]; s[e] = sr[p + e]; }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 f = Kv4Pair<T>::wide(x[2 * j + e]), o = Kv4Pair<T>::wide(other[2 * j + e]);
                const float a0 = __fmul_rn(f.x, c[2 * e]), z0 = __fmul_rn(o.x, s[2 * e]);
                const float a1 = __fmul_rn(f.y, c[2 * e + 1]), z1 = __fmul_rn(o.y, s[2 * e + 1]);
                out[2 * j + e] = Kv4Pair<T>::pack(upper ? __fadd_rn(a0, z0) : __fsub_rn(a0, z0), upper ? __fadd_rn(a1, z1) : __fsub_rn(a1, z1));
            }
        }
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) x[j] = out[j];
        if (h < hq && live)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                *reinterpret_cast<uint2 *>(q_out + ((size_t)b * hq + h) * D + 32 * j + 4 * r) = make_uint2(x[2 * j], x[2 * j + 1]);
    }
    if (__all_sync(0xffffffffu, h < hq)) return;
    const bool is_v = h >= hq + C.heads;
    const long to = live && in_range && h >= hq ? kv4_row(C, b, is_v ? h - hq - C.heads : h - hq, pos) : -1;
    kv4_store_row<T, NB, BPG>(x, to, r, is_v ? C.v_codes : C.k_codes, is_v ? C.v_params : C.k_params);
}

// Rows first[b] + i of the cache, i < out_len and below context_lens[b] -> out [batch, heads, out_len, D]; rows behind
// them are left as they were.  Four threads a row: a thread's quarter of the codes (NB words) holds eight neighbouring dims of
// every block, 16 bytes of the output.  BOTH: of K and of V in turn, so that a place is looked up once and twice the bytes are under
// way; in a small launch K and V have threads of their own (kv4_read_launch).
// 4 sequences of 8192 positions, 8 heads, D 128, fp16: 29 us, 0.9 of the copy bandwidth, which bounds it; one of them 8.2 us (9.2
// not BOTH), 6.5 us being the bytes; a few hundred rows a sequence (paged, 16 sequences) 7.5 us (8.1) against 4 us of bytes, the
// start of the launch and the way through table, codes and parameters.
template <typename T, int NB, int BPG, bool BOTH>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Cache C, const int32_t *__restrict__ first, const int32_t *__restrict__ lens, T *__restrict__ k_out, T *__restrict__ v_out,
                int out_len, int *status) {
    constexpr int D = 32 * NB, TENSORS = BOTH ? 2 : 1;
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, t = threadIdx.x & 3;
    int len = lens[b];
    if (len > C.capacity) {
        len = C.capacity;
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(status, KV4_BAD_POSITION);
    }
    const long start = first ? (long)first[b] : 0l;
    const unsigned rows = (unsigned)max(min((long)out_len, len - start), 0l);     // of a head
    const long total = (long)rows * C.heads * (2 / TENSORS);
    for (long n = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 2; n < total; n += gridDim.x * blockDim.x >> 2) {
        const bool is_v = !BOTH && n & 1;
        const long hi = BOTH ? n : n >> 1;
        // (head, row) of a number below 2^32 by a 32-bit division, beyond that by a 64-bit one
        const int h = total >> 32 ? (int)(hi / rows) : (int)((unsigned)hi / rows);
        const unsigned i = (unsigned)(hi - (long)h * rows);
        const long pos = start + i;
        if (pos < 0) {
            if (t == 0) atomicOr(status, KV4_BAD_POSITION);
            continue;
        }
        const long row = kv4_row(C, b, h, (int)pos);
        if (row < 0) {
            if (t == 0) atomicOr(status, KV4_BAD_BLOCK);
            continue;
        }
        uint32_t w[TENSORS][NB];
        __half2 params[TENSORS][NB / BPG];
#pragma unroll
        for (int v = 0; v < TENSORS; ++v) {
            const uint32_t *from = reinterpret_cast<const uint32_t *>(v || is_v ? C.v_codes : C.k_codes) + row * (4 * NB) + t * NB;
            if constexpr (NB % 4 == 0) {
#pragma unroll
                for (int j = 0; j < NB; j += 4) {
                    const uint4 u = ldg_nc_v4(from + j);
                    w[v][j] = u.x; w[v][j + 1] = u.y; w[v][j + 2] = u.z; w[v][j + 3] = u.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < NB; ++j) w[v][j] = from[j];
            }
            const __half2 *at = reinterpret_cast<const __half2 *>(v || is_v ? C.v_params : C.k_params) + row * (NB / BPG);
#pragma unroll
            for (int g = 0; g < NB / BPG; ++g) params[v][g] = at[g];
        }
        const long to_row = (((long)b * C.heads + h) * out_len + i) * D + 8 * t;
#pragma unroll
        for (int v = 0; v < TENSORS; ++v) {
            T *to = (v || is_v ? v_out : k_out) + to_row;
            float2 p = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if (j % BPG == 0) {
                    p = __half22float2(params[v][j / BPG]);
                    p.x *= 16777216.f;       // the codes come as fp16 subnormals, c 2^-24: exact either way
                }
                // units (2 t, j) and (2 t + 1, j): dims 8 t .. + 3 in the low half, + 4 .. + 7 in the high one
                const uint32_t u = __byte_perm(w[v][j >> 1], w[v][(NB + j) >> 1], (j & 1 ? 0x32 : 0x10) | ((NB + j & 1 ? 0x76 : 0x54) << 8));
                float f[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 c = h2_to_f2((u >> (4 * e)) & 0x000f000fu);
                    f[e] = fmaf(c.x, p.x, p.y);
                    f[e + 4] = fmaf(c.y, p.x, p.y);
                }
                *reinterpret_cast<uint4 *>(to + 32 * j) = make_uint4(Kv4Pair<T>::pack(f[0], f[1]), Kv4Pair<T>::pack(f[2], f[3]),
                                                                     Kv4Pair<T>::pack(f[4], f[5]), Kv4Pair<T>::pack(f[6], f[7]));
            }
        }
    }
}

// calls f with the number of 32-dim blocks of a row and of a group as constants
template <typename F>
static void kv4_by_shape(int d, int g, F f) {
    using std::integral_constant;
    switch (d / 32 * 10 + g / 32) {
#define KV4_SHAPE(NB, BPG) \
    case NB * 10 + BPG: return f(integral_constant<int, NB>(), integral_constant<int, BPG>());
        KV4_SHAPE(1, 1) KV4_SHAPE(2, 1) KV4_SHAPE(2, 2) KV4_SHAPE(3, 1) KV4_SHAPE(4, 1) KV4_SHAPE(4, 2) KV4_SHAPE(4, 4) KV4_SHAPE(5, 1)
        KV4_SHAPE(6, 1) KV4_SHAPE(6, 2) KV4_SHAPE(7, 1) KV4_SHAPE(8, 1) KV4_SHAPE(8, 2) KV4_SHAPE(8, 4)
#undef KV4_SHAPE
    }
}

// blocks along x for `rows` rows a sequence: one pass over them while the grid fits the machine a few times over
static unsigned kv4_grid(long rows, int rows_per_block, long others) {
    const long blocks = (rows + rows_per_block - 1) / rows_per_block, cap = ((long)sm_count() * 64 + others - 1) / others;
    return (unsigned)(blocks < cap ? blocks : cap);
}

template <typename T>
static int kv4_append_launch(const char *name, const T *nk, const T *nv, const Kv4Cache &C, bool paged, const int32_t *first, const int32_t *new_lens,
                             int batch, int tokens, int stride_kt, int stride_vt, b200k_stream stream) {
    B200K_REQUIRE(nk && nv && first, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, paged);
    if (rc) return rc;
    B200K_REQUIRE(tokens >= 0 && (long)tokens * C.heads < (1l << 30) && stride_kt >= (long)C.heads * C.d && stride_vt >= (long)C.heads * C.d,
                  B200K_E_SHAPE,
                  "%s: tokens %d (tokens * heads below 2^30), strides %d and %d (at least heads * head_dim = %ld)", name, tokens, stride_kt, stride_vt,
                  (long)C.heads * C.d);
    B200K_REQUIRE(aligned16(nk) && aligned16(nv) && stride_kt % 8 == 0 && stride_vt % 8 == 0, B200K_E_ALIGN,
                  "%s: new_keys and new_values must be 16-byte aligned, their token strides multiples of 8", name);
    if (batch == 0 || tokens == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    const dim3 grid(kv4_grid((long)tokens * C.heads, 16, batch), batch);
    kv4_by_shape(C.d, C.g, [&](auto nb, auto bpg) {
        launch_kernel(kv4_append_kernel<T, nb(), bpg()>, grid, dim3(128), 0, to_stream(stream), nk, nv, C, first, new_lens, tokens, (long)stride_kt,
                      (long)stride_vt, status);
    });
    return launch_status(name);
}

template <typename T>
static int kv4_rope_append_launch(const char *name, const T *qkv, const float *cos_t, const float *sin_t, const int32_t *positions, T *q_out,
                                  const Kv4Cache &C, int32_t *lens_out, int hq, int batch, b200k_stream stream) {
    B200K_REQUIRE(qkv && cos_t && sin_t && positions && q_out, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, false);
    if (rc) return rc;
    B200K_REQUIRE(hq > 0 && hq + 2l * C.heads < (1l << 30), B200K_E_SHAPE, "%s: num_q_heads %d, num_kv_heads %d", name, hq, C.heads);
    B200K_REQUIRE(aligned16(qkv) && aligned16(q_out), B200K_E_ALIGN, "%s: qkv and q_out must be 16-byte aligned", name);
    if (batch == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    const int vec = aligned16(cos_t) && aligned16(sin_t);
    const dim3 grid(ceil_div(hq + 2 * C.heads, 16), batch);
    kv4_by_shape(C.d, C.g, [&](auto nb, auto bpg) {
        launch_kernel(kv4_rope_append_kernel<T, nb(), bpg()>, grid, dim3(128), 0, to_stream(stream), qkv, cos_t, sin_t, positions, q_out, C, lens_out, hq, vec,
                      status);
    });
    return launch_status(name);
}

template <typename T>
static int kv4_read_launch(const char *name, const Kv4Cache &C, bool paged, const int32_t *first, const int32_t *lens, T *k_out, T *v_out, int batch,
                           int out_len, b200k_stream stream) {
    B200K_REQUIRE(lens && k_out && v_out, B200K_E_NULL, "%s: NULL pointer", name);
    int rc = kv4_check(name, C, batch, paged);
    if (rc) return rc;
    B200K_REQUIRE(out_len >= 0 && out_len <= KV4_MAX_LEN, B200K_E_SHAPE, "%s: out_len %d", name, out_len);
    B200K_REQUIRE(aligned16(k_out) && aligned16(v_out), B200K_E_ALIGN, "%s: k_out and v_out must be 16-byte aligned", name);
    if (batch == 0 || out_len == 0) return 0;
    int *status = status_word();
    if (!status) return B200K_E_WORKSPACE;
    // K and V in threads of their own while these fit the machine at once (2048 an SM): latency counts then.  64 sequences of one
    // position of 8 heads 2.3 us (2.9 with both in a thread), 512 of four 3.4 (3.8); beyond that 8 of 1000 positions 6.7 us (6.0).
    const bool apart = 8.0 * batch * out_len * C.heads <= 2048.0 * sm_count();
    const long rows = (apart ? 2l : 1l) * out_len * C.heads;
    const int threads = 4 * rows <= 128 ? 64 : 256;             // a few rows a sequence: small blocks
    const dim3 grid(kv4_grid(rows, threads / 4, batch), batch);
    kv4_by_shape(C.d, C.g, [&](auto nb, auto bpg) {
        launch_kernel(apart ? kv4_read_kernel<T, nb(), bpg(), false> : kv4_read_kernel<T, nb(), bpg(), true>, grid, dim3(threads), 0, to_stream(stream),
                      C, first, lens, k_out, v_out, out_len, status);
    });
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
