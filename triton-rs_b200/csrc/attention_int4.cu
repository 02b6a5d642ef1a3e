// GQA decode attention over the 4-bit KV cache (format: kv_int4.cuh).
//
// The codes never become values.  With a row's scale s and base z per group,
//   q . K[p]        = sum_g s_pg (sum_{d in g} q_d c_pd) + z_pg (sum_{d in g} q_d)
//   sum_p w_p V[p]  = sum_p (w_p s_pg) c_pd + sum_p w_p z_pg
// so the matrix instructions multiply by the codes themselves and the scales go to the sums (K) and the probabilities (V).
// A masked nibble is already an fp16 number: bits 0-3 of a half are the subnormal c 2^-24, bits 4-7 are c 2^-20, both exact,
// so eight codes cost five instructions (and a byte permute where two positions have to share a register).  The factors of
// two go to q (K side) and to the output (V side).  Dequantising to fp16 first would take two more instructions for
// every pair of codes and round every value.
//
// mma.sync m16n8k16 in transposed form, as in the 16-bit kernel: positions (K) or dims (V) fill the 16 rows, up to 8 q heads
// of a GQA group the 8 columns; one query token a sequence cannot fill a 128-row tcgen05 tile.
//
// What bounds it: the bytes of the cache where contexts are long (74 x 8 contexts of 16384 positions, D 128, groups of 64:
// 246 us, 0.87 of the copy bandwidth), and just below that the issue of instructions: about 265 a warp for 16 positions of K
// and V, half of them on the integer pipe, at 0.6 a cycle and scheduler; HBM delivers 16 positions to an SM every 96 cycles.
// At 64 x 4096 positions (46 us of bytes) 69 us: starting takes 4 us, the joins of the CTAs 4, and the rest is the issue
// rate.  Groups of 32 take a fifth more instructions (86 us), groups of 128 a tenth fewer (59 us).
//
// Work is dealt out on the device, from the lengths, so a captured graph follows them; see the kernel's first part.  Each warp
// streams two 16-position tiles a stage through a ring of cp.async stages of its own, without a barrier between warps: four
// warps a CTA, four CTAs an SM at head_dim 128 keep 74 KB under way.  (Where two stages of two tiles took 64 us, before the sums
// were centred, three stages took 92: the shared memory then leaves no room for the fourth CTA; one tile a stage 68.)  Rows
// behind the context are not read.
#include "kv_int4.cuh"
#include "tma.cuh"

namespace b200k {

constexpr int A4_WARPS = 4, A4_THREADS = 32 * A4_WARPS, A4_STAGES = 2;
constexpr int A4_TILE = 16, A4_SUBS = 2;                // positions of a tile (the rows of an MMA), tiles of a stage
constexpr int A4_STEP = A4_SUBS * A4_TILE, A4_UNIT = A4_WARPS * A4_STEP;       // positions of a warp's stage, of a unit of work
constexpr int A4_MAX_CTAS = 640;                               // CTAs of a launch: one wave
constexpr int A4_FAN = 16;                                     // partial results that are joined at a time
constexpr unsigned A4_WHOLE = 2;                               // units of contexts that are never cut
constexpr int A4_HEADS = 8;                                    // columns of one MMA
constexpr float A4_MIDDLE = 7.5f;     // of the codes
constexpr float A4_LAZY = 6.f;        // the running maximum moves when a score passes it by 2^6: probabilities stay below 2^6
constexpr float A4_TOP = 512.f;       // 2^e times the largest value scale is set to [2^2, 2^3) and set again when it passes 2^9

struct Attn4Args {
    const void *q;                // [B, Hq, D]
    void *out;                    // [B, Hq, D]
    const int32_t *lens;
    Kv4Cache C;
    unsigned long long block_magic;   // floor(2^64 / block_size) + 1: pos / block_size = umul64hi(pos, magic) for pos < 2^32
    int batch, hq, head_blocks;   // head_blocks: blocks of 8 q heads a kv head has
    int bf16, out_kperm;
    float scale_log2e;
    int *status;
    int *counters;                // [level of the join][CTA][2], zero between launches
    float *parts;                 // [CTA][2][D * 8 + 16]
};

// ---- what a (head_dim, group) pair fixes -------------------------------------------------------------------------------
template <int NB_, int NG_>
struct A4 {
    static constexpr int NB = NB_, NG = NG_;                  // blocks of 32 dims, groups
    static constexpr int D = 32 * NB, G = D / NG;
    static constexpr int ROW = 16 * NB, PROW = 4 * NG;        // bytes of a row's codes, of its params
    static constexpr int PCOPY = NG % 4 == 0 ? 16 : NG % 2 == 0 ? 8 : 4;      // as wide as a row of params is aligned
    static constexpr int SUB = 2 * A4_TILE * (ROW + PROW) + 32;                // bytes of a tile in a stage; a multiple of 32: see at_k
    static constexpr int STAGE = A4_SUBS * SUB;
    static constexpr int MTILES = 2 * NB;
    static constexpr bool PURE = G == 32;                     // a group is one block: see kword()
    // With four groups the bases go through matrix instructions as well (a row's params are the 16 bytes that these want): two of
    // them, and 14 others, for 48 on scalars.  D 128, groups of 32, 64 x 4096: 78 us, 84 without (neither with SPLIT); with two
    // groups, where 16 instructions replace 24, 65.9 and 66.6, which is not worth rounding the probabilities that meet the bases to fp16.
    static constexpr bool BASES = NG == 4;
    static constexpr int PART = D * A4_HEADS + 16;            // floats of a partial result
    static constexpr int CTAS = NB <= 4 ? 4 : NB <= 5 ? 3 : 2;
    static constexpr int RING = A4_WARPS * A4_STAGES * STAGE;
    static constexpr int JOIN = A4_WARPS * D * A4_HEADS * 4;  // the warps' results
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;    // in turn
    // 16-byte chunk of a row in shared memory is chunk ^ swizzle(position): the K loads of a quarter warp (two rows of
    // opposite parity) and the V loads of a half warp (positions 0-3 or 4-7) then meet no bank twice
    __device__ static int swizzle(int pos) { return NB == 4 ? pos & 2 : NB == 8 ? ((pos & 3) << 1) | (pos & 1) : 0; }
};

__device__ __forceinline__ int a4_pos(int k) { return (k & 8) + ((k & 1) ? 4 + (((k & 7) >> 1) ^ 1) : (k & 7) >> 1); }   // position of MMA index k

__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void a4_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // sum from 0
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t a4_transpose(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float a4_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float a4_max_nan(float a, float b) {      // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <int BYTES>
__device__ __forceinline__ void a4_copy(uint32_t dst, const void *src, int bytes) {   // bytes = BYTES, or 0: zeros
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void a4_lds(uint32_t *w, uint32_t at) {    // N words of shared memory, as aligned as their number allows
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(at + 4 * i) : "memory");
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(at + 4 * i) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(at + 4 * i) : "memory");
    }
}
__device__ __forceinline__ void a4_ldm_trans(uint32_t &a, uint32_t &b, uint32_t at) {     // two 8 x 8 matrices of halves, transposed
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t a4_lds16(uint32_t at) {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
    return h;
}
template <int NG>
__device__ __forceinline__ void a4_params(float (&s)[NG], float (&z)[NG], const uint32_t *w) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float2 f = h2_to_f2(w[g]);
        s[g] = f.x; z[g] = f.y;
    }
}
// a value that is to be kept in its register: not to be worked out again wherever it is used
__device__ __forceinline__ uint32_t a4_keep(uint32_t x) {
    asm volatile("" : "+r"(x));
    return x;
}

// The eight codes of a word as four operand registers: nibbles 0 and 2 of both halves as c 2^-24, 1 and 3 as c 2^-20.  Four
// integer instructions and a subtraction (exact) on the other pipe: the integer one runs at half rate and is the busiest here.
__device__ __forceinline__ void a4_codes(uint32_t x, uint32_t &n0, uint32_t &n1, uint32_t &n2, uint32_t &n3, bool fifteen_minus = false) {
    const uint32_t y = __byte_perm(x, 0, 0x4341);
    if (fifteen_minus) {
        n0 = ~x & 0x000f000fu;
        n1 = ~x & 0x00f000f0u;
        n2 = ~y & 0x000f000fu;
        n3 = ~y & 0x00f000f0u;
        return;
    }
    n0 = x & 0x000f000fu;
    n1 = x & 0x00f000f0u;
    n3 = y & 0x00f000f0u;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(n2) : "r"(y), "r"(n3));
}

// Lane t of a K row holds units (2t, j) and (2t + 1, j), j = 0 .. NB-1, in this order, in NB words.  Word i of its operand: where
// a group spans several blocks, the two blocks of a word share a register (word i as loaded); where a group is one block,
// the two units of block i do.  Either way all products of one MMA belong to one group.
template <int NB, bool PURE>
__device__ __forceinline__ uint32_t a4_kword(const uint32_t (&w)[NB], int i) {
    if constexpr (!PURE) return w[i];
    const int a = i, b = NB + i;
    return __byte_perm(w[a >> 1], w[b >> 1], (a & 1 ? 0x32 : 0x10) | ((b & 1 ? 0x76 : 0x54) << 8));
}
// dims of the low and high half of nibble n of operand word i, for lane t
template <int NB, bool PURE>
__device__ __forceinline__ void a4_kdims(int i, int n, int t, int &lo, int &hi) {
    if constexpr (PURE) {
        lo = 32 * i + 8 * t + n;
        hi = lo + 4;
    } else {
        const int rho = 2 * t + (i >= NB / 2), jp = i % (NB / 2);
        lo = 64 * jp + 4 * rho + n;
        hi = lo + 32;
    }
}
template <int NB, int NG, bool PURE>
__device__ __forceinline__ constexpr int a4_kgroup(int i) { return PURE ? i : (i % (NB / 2)) * 2 * NG / NB; }

// The copies of a tile of which not all rows are there, or that spans blocks, or one of whose blocks the pool does not have: row
// by row, zeros for what is not there; a mask of the rows that are there goes to the tile's last words.
template <int NB, int NG>
__device__ __forceinline__ void a4_copy_edge(const Attn4Args &A, int b, int kvh, int p0, int len, uint32_t dst_codes, uint32_t dst_params,
                                             uint32_t mask) {
    using X = A4<NB, NG>;
    const Kv4Cache &C = A.C;
    const int lane = threadIdx.x & 31;
    auto row_of = [&](int row) { return p0 + row < len ? kv4_row(C, b, kvh, p0 + row) : -1l; };
#pragma unroll 1
    for (int c = lane; c < A4_TILE * NB; c += 32) {
        const long row = row_of(c / NB);
        const long off = max(row, 0l) * X::ROW + (c % NB) * 16;
        const uint32_t dst = dst_codes + (c - lane) * 16;
        a4_copy<16>(dst, (const unsigned char *)C.k_codes + off, row < 0 ? 0 : 16);
        a4_copy<16>(dst + A4_TILE * X::ROW, (const unsigned char *)C.v_codes + off, row < 0 ? 0 : 16);
    }
    const long row = row_of(lane & 15);
    const unsigned char *params = (const unsigned char *)(lane < 16 ? C.k_params : C.v_params) + max(row, 0l) * X::PROW;
#pragma unroll
    for (int c = 0; c < X::PROW; c += X::PCOPY) a4_copy<X::PCOPY>(dst_params + c, params + c, row < 0 ? 0 : X::PCOPY);
    const unsigned valid = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
    if (lane == 0) {
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(mask), "r"(valid) : "memory");
        const int rows = min(A4_TILE, len - p0);
        if (rows > 0 && __popc(valid) != rows) atomicOr(A.status, KV4_BAD_BLOCK);
    }
}

// A segment: units [u0, u1) of the n that a context (sequence b, kv head, q heads [h0, h0 + heads)) has.  The context is spread
// over `members` CTAs from c0 on.  `more`: another segment follows for this CTA.
struct Attn4Segment {
    int b, kvh, h0, heads, len, u0, u1, n, c0, members, more;
    unsigned seq_start;             // units before this sequence
    unsigned share, at, end;        // units of a CTA; those that follow this segment in this CTA: [at, end)
};

// SPLIT: the q heads of a kv head, 4 or fewer, stand in both halves of the columns.  The second half takes what the first half's
// probabilities times scales lose when they are rounded to fp16: nothing is lost then, and no instruction but those that
// part them is added.  For fp16 outputs; a bf16 output's own rounding is eight times larger.  With more heads an fp16 output is
// 3.0e-4 off (2.1e-4 from its own rounding), 3.1e-4 if the bases met rounded probabilities too.
enum { A4_PLAIN, A4_SPLIT, A4_EXACT_BASES };      // A4_EXACT_BASES: fp16 outputs of more than 4 heads do without BASES
template <int NB, int NG, int MODE>
__global__ void __launch_bounds__(A4_THREADS, A4<NB, NG>::CTAS)
attn4_kernel(const __grid_constant__ Attn4Args A) {
    using X = A4<NB, NG>;
    constexpr bool SPLIT = MODE == A4_SPLIT, BASES = X::BASES && MODE != A4_EXACT_BASES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(16) float sm_ref[A4_WARPS][A4_HEADS], sm_l[A4_WARPS][A4_HEADS], sm_top[A4_HEADS], sm_sum[A4_HEADS];
    __shared__ __align__(16) uint4 sm_q[NB][32];       // q as the B operand: word i of all lanes
    __shared__ float sm_qsum[NB][A4_HEADS], sm_fac[A4_HEADS], sm_wt[A4_FAN][A4_HEADS];
    __shared__ Attn4Segment sm_seg;
    __shared__ int sm_last;
    const Kv4Cache &C = A.C;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();

    // ---- the share of this CTA, by warp 0 (the host made sure that 32 bits hold all units) ----------------------------------------
    // Either one piece of one context, all contexts being cut into pieces of at most `share` units, no more pieces than CTAs; or
    // units [at, end) of all, which may begin and end within contexts: a CTA then joins and starts anew wherever it passes from
    // one to the next.  Pieces are taken where the largest is a sixth (and two units) over an equal share at most: one context of
    // 131071 positions 38.7 us in pieces, 43 cut evenly; 32 of 512 to 8192 positions, the pieces a third larger, groups of 32: 56 and
    // 54.7.  Twelve units over it are still better where more than every other CTA would start anew and four of five have a
    // piece: 40 sequences of 100 to 4000 positions 38.7 and 42.2 us, 100 of 4 kv heads up to 5000 44.6 and 50; but 50 of 1000 to
    // 3000, whole contexts for two of three CTAs, 46.4 and 38.9.
    const unsigned per_seq = C.heads * A.head_blocks;      // contexts of a sequence
    auto units_of = [&](int b) { return (unsigned)(max(min(A.lens[b], C.capacity), 0) + A4_UNIT - 1) / A4_UNIT; };
    auto place_heads = [&](Attn4Segment &d, unsigned ctx) {
        const unsigned hb = ctx % A.head_blocks, gqa = A.hq / C.heads;
        d.kvh = ctx / A.head_blocks;
        d.h0 = d.kvh * gqa + hb * A4_HEADS;
        d.heads = min((unsigned)A4_HEADS, gqa - hb * A4_HEADS);
        d.len = min(A.lens[d.b], C.capacity);
    };
    auto segment = [&](Attn4Segment d) {                   // the one that begins with unit d.at, of sequence d.b or a later one
        unsigned n = units_of(d.b);
#pragma unroll 1
        while (d.at >= d.seq_start + n * per_seq) {
            d.seq_start += n * per_seq;
            n = units_of(++d.b);
        }
        const unsigned ctx = (d.at - d.seq_start) / n, first = d.seq_start + ctx * n;       // units before this context
        place_heads(d, ctx);
        d.n = n;
        d.u0 = d.at - first;
        d.u1 = min(n, d.end - first);
        d.c0 = first / d.share;
        d.members = (first + n - 1) / d.share - d.c0 + 1;
        d.at = first + d.u1;
        d.more = d.at < d.end;
        sm_seg = d;
    };
    if (warp == 0) {
        unsigned total = 0, contexts = 0, longest = 0, share, at = 0, end = 0;
#pragma unroll 4
        for (int b = lane; b < A.batch; b += 32) {
            const unsigned n = units_of(b);
            total += n;
            contexts += n > 0;
            longest = max(longest, n);
        }
        total = __reduce_add_sync(0xffffffffu, total) * per_seq;
        contexts = __reduce_add_sync(0xffffffffu, contexts) * per_seq;
        longest = __reduce_max_sync(0xffffffffu, longest);
        share = max((total + gridDim.x - 1) / gridDim.x, 1u);
        // contexts of one or two units stay whole: nothing to join.  236 positions, 1 / 8 / 32 sequences: 6.9 / 9.6 / 10.7 us, cut
        // 8.1 / 10.1 / 11.6; three units 7.9 / 11.4 / 12.7 against 8.2 / 10.2 / 13.6, four 8.7 / 13.1 / 14.5 against 8.1 / 10.4 / 14.3
        if (longest <= A4_WHOLE && contexts <= gridDim.x) share = A4_WHOLE;
        bool cut = contexts > gridDim.x;                   // pieces will not do
        for (unsigned s = share; !cut && share > 1;) {     // with a unit for every CTA, units are the pieces
            unsigned pieces = 0;
#pragma unroll 4
            for (int b = lane; b < A.batch; b += 32) pieces += (units_of(b) + s - 1) / s;
            pieces = __reduce_add_sync(0xffffffffu, pieces) * per_seq;
            if (pieces <= gridDim.x) {
                cut = s > share + share / 6 + 2 && 5 * pieces < 4 * gridDim.x;
                if (!cut) share = s;
                break;
            }
            // a piece fewer for the longest context
            const unsigned parts = (longest + s - 1) / s;
            cut = parts < 2;
            if (!cut) s = (longest + parts - 2) / (parts - 1);
            cut = cut || s > share + share / 6 + (2 * contexts > gridDim.x ? 12 : 2);
        }
        // the sequence that this CTA's first unit, or its piece, belongs to
        if (cut) {
            at = share * blockIdx.x;
            end = min(at + share, total);
        }
        const unsigned mark = cut ? at : blockIdx.x;
        unsigned before = 0;
        if (lane == 0) sm_seg.n = 0;                       // nothing to do
        __syncwarp();
#pragma unroll 1
        for (int b0 = 0; b0 < A.batch && (!cut || at < end); b0 += 32) {
            const unsigned n = b0 + lane < A.batch ? units_of(b0 + lane) : 0u, parts = cut ? n : (n + share - 1) / share;
            const unsigned mine = parts * per_seq;
            unsigned upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > mark);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    Attn4Segment d = {};
                    d.b = b0 + lane;
                    d.seq_start = before + upto - mine;
                    if (cut) {
                        d.share = share;
                        d.at = at;
                        d.end = end;
                        segment(d);
                    } else {
                        const unsigned piece = mark - d.seq_start, ctx = piece / parts, part = piece % parts, size = (n + parts - 1) / parts;
                        place_heads(d, ctx);
                        d.n = n;
                        d.u0 = part * size;
                        d.u1 = min(n, (part + 1) * size);
                        d.c0 = blockIdx.x - part;
                        d.members = parts;
                        sm_seg = d;
                    }
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    } else {
#pragma unroll 1
        for (int b = blockIdx.x; b < A.batch; b += gridDim.x) {
            const int len = A.lens[b];
            if (len > C.capacity && tid == 32) atomicOr(A.status, KV4_BAD_POSITION);
            if (len <= 0)       // no keys: a zero output row
#pragma unroll 1
                for (int i = tid - 32; i < A.hq * X::D / 2; i += A4_THREADS - 32) reinterpret_cast<uint32_t *>(A.out)[(long)b * A.hq * X::D / 2 + i] = 0u;
        }
    }
    __syncthreads();
    if (sm_seg.n == 0) return;

    const uint32_t ring = smem_u32(smem) + warp * A4_STAGES * X::STAGE;
    // where this lane's first 16-byte piece goes in a tile of a stage, and its row of params: lanes 0-15 copy those of K, 16-31 those
    // of V, which stand beside them
    const uint32_t dst_codes = a4_keep(ring + (lane / NB) * X::ROW + ((lane % NB) ^ X::swizzle(lane / NB)) * 16);
    const uint32_t dst_params = a4_keep(ring + 2 * A4_TILE * X::ROW + ((lane & 15) * 2 + (lane >> 4)) * X::PROW);
    // where it reads: K rows kpos and kpos + 8 (chunk t of a row; two chunks at head_dim 256), their params, and its eighth of V
    // rows t, 4 + (t ^ 1) and these + 8
    const int kpos = a4_pos(r);
    const uint32_t at_k = a4_keep(ring + kpos * X::ROW + (NB == 4 ? (t ^ X::swizzle(kpos)) * 16 : NB == 8 ? ((2 * t) ^ X::swizzle(kpos)) * 16 : t * 4 * NB));
    const uint32_t at_p = a4_keep(ring + 2 * A4_TILE * X::ROW + kpos * 2 * X::PROW);
    auto piece_at = [&](int pos) { return ring + (A4_TILE + pos) * X::ROW + (((2 * NB * r >> 4) ^ X::swizzle(pos)) << 4) + (2 * NB * r & 15); };
    const uint32_t at_v0 = a4_keep(piece_at(t)), at_v1 = a4_keep(piece_at(4 + (t ^ 1)));
    // BASES: the params of V as a matrix [MMA index][scale, base of each group], and K's word of group t
    const uint32_t at_b = BASES ? a4_keep(ring + 2 * A4_TILE * X::ROW + (2 * a4_pos(lane & 15) + 1) * X::PROW) : 0;
    const uint32_t at_kz = BASES ? a4_keep(at_p + 4 * t) : 0;

    // ---- streaming a piece: tile i of this warp goes to stage i % STAGES ------------------------------------------------------------
    // 16 neighbouring rows are one linear part of the cache, so a tile that is whole and lies in one block takes nothing but
    // copies at fixed distances
    int tiles, whole;                      // stages of a segment; so many from the first on are whole (where blocks hold whole tiles)
    const unsigned char *src_k = nullptr, *src_v = nullptr, *src_p = nullptr;
    const bool paged = C.block_table != nullptr;
    auto copy_whole = [&](uint32_t stage, const unsigned char *k, const unsigned char *v, const unsigned char *p) {
#pragma unroll
        for (int c = 0; c < NB; c += 2)
            if (c + 1 < NB || lane < 16) {
                a4_copy<16>(dst_codes + stage + c * 256, k + c * 256, 16);
                a4_copy<16>(dst_codes + stage + A4_TILE * X::ROW + c * 256, v + c * 256, 16);
            }
#pragma unroll
        for (int c = 0; c < X::PROW; c += X::PCOPY) a4_copy<X::PCOPY>(dst_params + stage + c, p + c, X::PCOPY);
    };
    // returns whether the tiles need a look at their masks
    auto issue = [&](const Attn4Segment &d, int i, uint32_t stage) {
        bool fine = i < whole;
        if (fine) {
            if (paged) {
                // blocks of whole tiles: a tile lies in one block
                const int p0 = (d.u0 + i) * A4_UNIT + warp * A4_STEP;
                int lb = (int)__umul64hi((unsigned long long)p0, A.block_magic), slot = p0 - lb * C.block_size;
                const int32_t *table = C.block_table + (long)d.b * C.max_blocks;
                auto look_up = [&] {
                    const int blk = table[lb];
                    fine = fine && (unsigned)blk < (unsigned)C.num_blocks;
                    return ((long)blk * C.heads + d.kvh) * C.block_size + slot;
                };
                long row[A4_SUBS];
                row[0] = look_up();
#pragma unroll
                for (int s = 1; s < A4_SUBS; ++s) {
                    slot += A4_TILE;
                    if (slot == C.block_size) {
                        slot = 0;
                        ++lb;
                        row[s] = look_up();
                    } else {
                        row[s] = row[s - 1] + A4_TILE;
                    }
                }
                if (fine) {
#pragma unroll
                    for (int s = 0; s < A4_SUBS; ++s)
                        copy_whole(stage + s * X::SUB, src_k + row[s] * X::ROW, src_v + row[s] * X::ROW, src_p + row[s] * X::PROW);
                }
            } else {
#pragma unroll
                for (int s = 0; s < A4_SUBS; ++s)
                    copy_whole(stage + s * X::SUB, src_k + s * A4_TILE * X::ROW, src_v + s * A4_TILE * X::ROW, src_p + s * A4_TILE * X::PROW);
                src_k += A4_UNIT * X::ROW;
                src_v += A4_UNIT * X::ROW;
                src_p += A4_UNIT * X::PROW;
            }
        }
        const bool edge = !fine && i < tiles;
        if (edge)
#pragma unroll 1
            for (int s = 0; s < A4_SUBS; ++s)
                a4_copy_edge<NB, NG>(A, d.b, d.kvh, (d.u0 + i) * A4_UNIT + warp * A4_STEP + s * A4_TILE, d.len, dst_codes + stage + s * X::SUB,
                                     dst_params + stage + s * X::SUB, ring + stage + (s + 1) * X::SUB - 32);
        asm volatile("cp.async.commit_group;" ::: "memory");
        return edge;
    };
#pragma unroll 1
    for (;;) {
        const Attn4Segment &d = sm_seg;
        tiles = d.u1 - d.u0;
        whole = paged && C.block_size % A4_TILE ? 0 : min(max((d.len - (warp + 1) * A4_STEP + A4_UNIT) / A4_UNIT - d.u0, 0), tiles);
        const long row0 = paged ? 0l : ((long)d.b * C.heads + d.kvh) * C.capacity + d.u0 * A4_UNIT + warp * A4_STEP;
        src_k = (const unsigned char *)C.k_codes + row0 * X::ROW + lane * 16;
        src_v = (const unsigned char *)C.v_codes + row0 * X::ROW + lane * 16;
        src_p = (const unsigned char *)(lane < 16 ? C.k_params : C.v_params) + (row0 + (lane & 15)) * X::PROW;
        bool edge = issue(d, 0, 0);
        const uint32_t w_flip = t >= 2 ? 0x80000000u : 0u;
        const float w_all = t >= 2 ? 1.f : 0.f;

        // ---- q as the B operand, a word by each warp; scaled by a power of two to [2^14, 2^15) -------------------------------------------
        // (any 16-bit type then fits fp16 with all its bits, down to 2^-25 of the head's largest element; nibbles 1 and 3 carry
        // 2^4 more than 0 and 2, so their q is divided by 16)
        {
            // head r, lane t's dims: of operand word i 4 + 4 (two blocks), or 8 in a row (one block)
            const int hr = SPLIT ? r & 3 : r;
            const uint16_t *qrow = (const uint16_t *)A.q + ((long)d.b * A.hq + d.h0 + (hr < d.heads ? hr : 0)) * X::D;
            auto word = [&](int i) {
                int lo, hi;
                a4_kdims<NB, X::PURE>(i, 0, t, lo, hi);
                if constexpr (X::PURE) return *reinterpret_cast<const uint4 *>(qrow + lo);
                const uint2 u = *reinterpret_cast<const uint2 *>(qrow + lo), w = *reinterpret_cast<const uint2 *>(qrow + hi);
                return make_uint4(u.x, u.y, w.x, w.y);
            };
            uint32_t top2 = 0;                 // the largest magnitude: its bits order like the value, in either type
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint4 u = word(i);
                top2 = __vmaxu2(__vmaxu2(top2, u.x & 0x7fff7fffu), __vmaxu2(u.y & 0x7fff7fffu, __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu)));
            }
            top2 = max(top2 & 0xffffu, top2 >> 16);
            top2 = max(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
            top2 = max(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
            const float big = A.bf16 ? __uint_as_float(top2 << 16) : __half2float(__ushort_as_half((unsigned short)top2));
            const int k = min(14 - ((int)(__float_as_uint(big) >> 23) - 127), 126);
            const float up = hr < d.heads ? copysignf(__uint_as_float((uint32_t)(k + 127) << 23), A.scale_log2e) : 0.f, up16 = up * 0.0625f;
#pragma unroll 1
            for (int i = warp; i < NB; i += A4_WARPS) {
                const uint4 u = word(i);       // u.x, u.y: dims 0-3 of the low half, u.z, u.w of the high one
                float f[8];
                if (A.bf16) {
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e2 = 0; e2 < 4; ++e2) { f[2 * e2] = __uint_as_float(w[e2] << 16); f[2 * e2 + 1] = __uint_as_float(w[e2] & 0xffff0000u); }
                } else {
                    const float2 w[4] = {h2_to_f2(u.x), h2_to_f2(u.y), h2_to_f2(u.z), h2_to_f2(u.w)};
#pragma unroll
                    for (int e2 = 0; e2 < 4; ++e2) { f[2 * e2] = w[e2].x; f[2 * e2 + 1] = w[e2].y; }
                }
#pragma unroll
                for (int e2 = 0; e2 < 8; ++e2) f[e2] *= e2 & 1 ? up16 : up;
                if (hr >= d.heads) f[0] = f[1] = f[2] = f[3] = f[4] = f[5] = f[6] = f[7] = 0.f;     // another head's row stood in
                sm_q[i][lane] = make_uint4(f2_to_h2(f[0], f[4]), f2_to_h2(f[1], f[5]), f2_to_h2(f[2], f[6]), f2_to_h2(f[3], f[7]));
                float sum = fmaf((f[1] + f[5]) + (f[3] + f[7]), 16.f, (f[0] + f[4]) + (f[2] + f[6]));
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t == 0) sm_qsum[i][r] = sum * (1.f / 16777216.f);
            }
            // what a score is multiplied by; a q with an infinity or a NaN has no finite score: NaN
            if (warp == 0 && t == 0) sm_fac[r] = hr >= d.heads ? 0.f : big < INFINITY ? fabsf(A.scale_log2e) / fabsf(up) * 16777216.f : NAN;
        }
        __syncthreads();
        float qsum[NG][2];                     // of heads 2t and 2t + 1
        const float fac[2] = {sm_fac[2 * t], sm_fac[2 * t + 1]};
        uint32_t qz0 = 0, qz1 = 0;
        if constexpr (BASES) {
            // sum_g z_g (sum q) in one instruction: its k indices 2 t and 2 t + 1 meet (scale, base) of group t, so the operand has 0 and
            // the sum of q there, as two fp16 numbers (22 bits; 2^10 larger, so that the second is no subnormal) one after the other
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (a4_kgroup<NB, NG, X::PURE>(i) == t) sum += sm_qsum[i][r];
            sum *= 1024.f;
            const __half hi = __float2half_rn(sum), lo = __float2half_rn(sum - __half2float(hi));
            qz0 = (uint32_t)__half_as_ushort(hi) << 16;
            qz1 = (uint32_t)__half_as_ushort(lo) << 16;
        } else {
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
#pragma unroll
                for (int g = 0; g < NG; ++g) qsum[g][e2] = 0.f;
#pragma unroll
                for (int i = 0; i < NB; ++i) qsum[a4_kgroup<NB, NG, X::PURE>(i)][e2] += sm_qsum[i][2 * t + e2];
            }
        }

        // sacc: the sum of w (below), group 2 i in the first two registers, 2 i + 1 in the others
        // zacc: the sum of p (z + 7.5 s); BASES: in bacc that of lift p times scale (even r) or base (odd r) of group r / 2
        float oacc[X::MTILES][4], sacc[(NG + 1) / 2][4], zacc[NG][2], bacc[2] = {0.f, 0.f}, lift = 0.f, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < X::MTILES; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) oacc[i][j] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) zacc[g][0] = zacc[g][1] = sacc[g / 2][2 * (g & 1)] = sacc[g / 2][2 * (g & 1) + 1] = 0.f;
        if (NG & 1) sacc[NG / 2][2] = sacc[NG / 2][3] = 0.f;
        // top: the running maximum of the raw scores; a probability is 2^(score fac - ref), ref = top fac - e: the factor 2^e,
        // the same for all heads, keeps probability times value scale inside fp16 and cancels in the end
        float top[2] = {-1e30f, -1e30f}, ref[2] = {0.f, 0.f}, bar[2] = {-1e30f, -1e30f}, e = 0.f, most = -1.f;
        if (!(fac[0] > 0.f)) { top[0] = 0.f; bar[0] = INFINITY; }
        if (!(fac[1] > 0.f)) { top[1] = 0.f; bar[1] = INFINITY; }

        uint32_t stage = 0;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            const bool look = edge;               // some rows may have to be left out
            edge = issue(d, i + 1, stage ^ X::STAGE);
#pragma unroll
            for (int sub = 0; sub < A4_SUBS; ++sub) {
            const uint32_t st = stage + sub * X::SUB;
            bool ok0 = true, ok1 = true;
            if (look) {
                uint32_t valid;
                a4_lds<1>(&valid, ring + st + X::SUB - 32);
                ok0 = (valid >> kpos) & 1;
                ok1 = (valid >> (kpos + 8)) & 1;
            }

            // scores: rows r and r + 8 are positions kpos0 and kpos0 + 8, columns heads 2t and 2t + 1
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t pw0[2 * NG], pw1[2 * NG];     // params of these rows: K's, V's
            // with many groups V's words wait until they are needed: registers are short
            constexpr bool LATE = NG >= 4 && NB == 4;
            a4_lds<LATE ? NG : 2 * NG>(pw0, at_p + st);
            a4_lds<LATE ? NG : 2 * NG>(pw1, at_p + st + 16 * X::PROW);
            {
                uint32_t w0[NB], w1[NB];
                if constexpr (NB == 8) {
                    a4_lds<4>(w0, at_k + st);
                    a4_lds<4>(w0 + 4, (at_k ^ 16) + st);
                    a4_lds<4>(w1, at_k + st + 8 * X::ROW);
                    a4_lds<4>(w1 + 4, (at_k ^ 16) + st + 8 * X::ROW);
                } else {
                    a4_lds<NB>(w0, at_k + st);
                    a4_lds<NB>(w1, at_k + st + 8 * X::ROW);
                }
                if constexpr (BASES) {
                    uint32_t z0, z1;
                    float zq[4];
                    a4_lds<1>(&z0, at_kz + st);
                    a4_lds<1>(&z1, at_kz + st + 16 * X::PROW);
                    a4_mma0(zq, z0, z1, z0, z1, qz0, qz1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = zq[i] * (1.f / 1024.f);
                }
                float s0[NG], z0[NG], s1[NG], z1[NG];
                a4_params<NG>(s0, z0, pw0);
                a4_params<NG>(s1, z1, pw1);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float acc[4];
                    bool begun = false;
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        if (a4_kgroup<NB, NG, X::PURE>(j) != g) continue;
                        const uint32_t x = a4_kword<NB, X::PURE>(w0, j), y = a4_kword<NB, X::PURE>(w1, j);
                        uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
                        a4_codes(x, x0, x1, x2, x3);
                        a4_codes(y, y0, y1, y2, y3);
                        const uint4 q4 = sm_q[j][lane];
                        if (begun) a4_mma(acc, x0, y0, x1, y1, q4.x, q4.y);
                        else a4_mma0(acc, x0, y0, x1, y1, q4.x, q4.y);
                        begun = true;
                        a4_mma(acc, x2, y2, x3, y3, q4.z, q4.w);
                    }
                    if constexpr (!BASES) {
                        s[0] = fmaf(z0[g], qsum[g][0], s[0]);
                        s[1] = fmaf(z0[g], qsum[g][1], s[1]);
                        s[2] = fmaf(z1[g], qsum[g][0], s[2]);
                        s[3] = fmaf(z1[g], qsum[g][1], s[3]);
                    }
                    s[0] = fmaf(s0[g], acc[0], s[0]);
                    s[1] = fmaf(s0[g], acc[1], s[1]);
                    s[2] = fmaf(s1[g], acc[2], s[2]);
                    s[3] = fmaf(s1[g], acc[3], s[3]);
                }
            }
            constexpr int VW = NB % 2 == 0 ? NB / 2 : 1;
            uint32_t va[VW], vb[VW], vc[VW], vd[VW];
            auto load_v = [&] {
                a4_lds<VW>(va, at_v0 + st);
                a4_lds<VW>(vb, at_v1 + st);
                a4_lds<VW>(vc, at_v0 + st + 8 * X::ROW);
                a4_lds<VW>(vd, at_v1 + st + 8 * X::ROW);
            };
            if constexpr (LATE) {
                a4_lds<NG>(pw0 + NG, at_p + st + X::PROW);
                a4_lds<NG>(pw1 + NG, at_p + st + 17 * X::PROW);
            } else if constexpr (NB % 2 == 0) {
                load_v();
            }
            float vs0[NG], vz0[NG], vs1[NG], vz1[NG];
            a4_params<NG>(vs0, vz0, pw0 + NG);
            a4_params<NG>(vs1, vz1, pw1 + NG);
            if (look) {
                if (!ok0) s[0] = s[1] = -1e30f;
                if (!ok1) s[2] = s[3] = -1e30f;
            }
            float vmax = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) vmax = a4_max_nan(vmax, a4_max_nan(vs0[g], vs1[g]));
            if (__any_sync(0xffffffffu, fmaxf(s[0], s[2]) > bar[0] || fmaxf(s[1], s[3]) > bar[1] || !(vmax <= most))) {
                // a score or a value scale has outgrown what the probabilities are held against, or a value is NaN.  That must reach
                // its own group alone, but two groups share sacc and 0 NaN is NaN: through the bases, which are apart.
                if (vmax != vmax) {
                    vmax = 0.f;
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        if (vs0[g] != vs0[g]) { vz0[g] = vs0[g]; vs0[g] = 0.f; }
                        if (vs1[g] != vs1[g]) { vz1[g] = vs1[g]; vs1[g] = 0.f; }
                        vmax = fmaxf(vmax, fmaxf(vs0[g], vs1[g]));
                    }
                }
                float n0 = fmaxf(top[0], fmaxf(s[0], s[2])), n1 = fmaxf(top[1], fmaxf(s[1], s[3]));
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1) {
                    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
                    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
                    vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
                }
                const float e_was = e;
                if (vmax > most) {
                    // 2^e vmax in [2^2, 2^3): vmax is a positive fp16 number, so its exponent lies in -24 .. 15
                    const int ex = (int)(__float_as_uint(vmax) >> 23) - 127;
                    e = vmax > 0.f ? 2.f - (float)ex : 0.f;
                    most = vmax > 0.f ? A4_TOP * a4_exp2(-e) : 0.f;
                }
                const float f0 = fac[0], f1 = fac[1];
                const float r0 = f0 > 0.f ? n0 * f0 - e : -e, r1 = f1 > 0.f ? n1 * f1 - e : -e;
                const float a0 = top[0] <= -1e30f ? 0.f : a4_exp2(ref[0] - r0), a1 = top[1] <= -1e30f ? 0.f : a4_exp2(ref[1] - r1);
                if (f0 > 0.f) { top[0] = n0; bar[0] = n0 + A4_LAZY / f0; }
                if (f1 > 0.f) { top[1] = n1; bar[1] = n1 + A4_LAZY / f1; }
                ref[0] = r0;
                ref[1] = r1;
                l[0] *= a0;
                l[1] *= a1;
                if constexpr (BASES) {
                    const float back = a4_exp2(e_was - e);
                    bacc[0] *= a0 * back;
                    bacc[1] *= a1 * back;
                    lift = a4_exp2(9.f - e);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    zacc[g][0] *= a0;
                    zacc[g][1] *= a1;
                    sacc[g / 2][2 * (g & 1)] *= a0;
                    sacc[g / 2][2 * (g & 1) + 1] *= a1;
                }
#pragma unroll
                for (int m = 0; m < X::MTILES; ++m) { oacc[m][0] *= a0; oacc[m][1] *= a1; oacc[m][2] *= a0; oacc[m][3] *= a1; }
            }
            float p[4];
            p[0] = a4_exp2(fmaf(s[0], fac[0], -ref[0]));
            p[1] = a4_exp2(fmaf(s[1], fac[1], -ref[1]));
            p[2] = a4_exp2(fmaf(s[2], fac[0], -ref[0]));
            p[3] = a4_exp2(fmaf(s[3], fac[1], -ref[1]));
            if (look) {
                if (!ok0) p[0] = p[1] = 0.f;
                if (!ok1) p[2] = p[3] = 0.f;
            }
            l[0] += p[0] + p[2];
            l[1] += p[1] + p[3];
            // w = probability x value scale, rounded to fp16, is the B operand (SPLIT: its upper 11 bits in one column, the rest in
            // another).  With it
            //   sum p v = sum w (c - 7.5) + sum p (z + 7.5 s) = sum w c - 7.5 sum w + sum p (z + 7.5 s)
            // so that its rounding meets a code's distance from the middle, not the code; a product with ones gives sum w.  Every
            // other tile adds -w (15 - c) in place of w c: the codes are not centred, their sum would grow with the context, and
            // the tensor cores truncate.  Output error relative to 64 bits, fp16: 64 contexts of 4096 positions 6.3e-4 without
            // either, 3.1e-4 with the first or both, 2.1e-4 with SPLIT too, which is what rounding the output alone leaves; one of
            // 131071 positions 9.4e-4, 4.4e-4 with the first, 3.1e-4 with both, 2.1e-4 with SPLIT too.  SPLIT costs 4.5 % (64 x 4096: 67 ->
            // 70 us; as a branch in one kernel 72 and slower for every other call).  BASES: for the bases p is rounded to fp16 too, as
            // 2^9 of the largest (2^15 at most) whatever e is; the sums over a tile go to fp32, so that they do not grow in the
            // tensor cores either.
            constexpr uint32_t ONES = 0x3c003c00u;
            const float sign = sub & 1 ? -1.f : 1.f;
            uint32_t pb[NG][2];
            if constexpr (BASES) {
                uint32_t b0, b1;
                float x[4];
                a4_ldm_trans(b0, b1, at_b + st);
                a4_mma0(x, b0, 0u, b1, 0u, a4_transpose(f2_to_h2(p[0] * lift, p[1] * lift)), a4_transpose(f2_to_h2(p[2] * lift, p[3] * lift)));
                bacc[0] += x[0];
                bacc[1] += x[1];
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float y0 = fmaf(vs0[g], A4_MIDDLE, vz0[g]), y1 = fmaf(vs1[g], A4_MIDDLE, vz1[g]);
                float w[4] = {p[0] * (sign * vs0[g]), p[1] * (sign * vs0[g]), p[2] * (sign * vs1[g]), p[3] * (sign * vs1[g])};
                if constexpr (SPLIT)           // upper 11 bits, or x minus these
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = fmaf(w[i], w_all, __uint_as_float((__float_as_uint(w[i]) & 0xffffe000u) ^ w_flip));
                pb[g][0] = a4_transpose(f2_to_h2(w[0], w[1]));
                pb[g][1] = a4_transpose(f2_to_h2(w[2], w[3]));
                if constexpr (!BASES) {
                    zacc[g][0] = fmaf(p[0], y0, fmaf(p[2], y1, zacc[g][0]));
                    zacc[g][1] = fmaf(p[1], y0, fmaf(p[3], y1, zacc[g][1]));
                }
                if (g & 1) a4_mma(sacc[g / 2], 0u, ONES, 0u, ONES, pb[g][0], pb[g][1]);
                else a4_mma(sacc[g / 2], ONES, 0u, ONES, 0u, pb[g][0], pb[g][1]);
            }
            // output: rows r and r + 8 of m-tile 2 j + h are dims 32 j + 4 r + 2 h and + 1
            auto out_tiles = [&](int j, uint32_t x, uint32_t y) {
                const int g = j * NG / NB;
                uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
                a4_codes(x, x0, x1, x2, x3, sub & 1);
                a4_codes(y, y0, y1, y2, y3, sub & 1);
                a4_mma(oacc[2 * j], x0, x1, y0, y1, pb[g][0], pb[g][1]);
                a4_mma(oacc[2 * j + 1], x2, x3, y2, y3, pb[g][0], pb[g][1]);
            };
            if constexpr (NB % 2 == 0) {
                if constexpr (LATE) load_v();
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int sel = j & 1 ? 0x7632 : 0x5410;
                    out_tiles(j, __byte_perm(va[j >> 1], vb[j >> 1], sel), __byte_perm(vc[j >> 1], vd[j >> 1], sel));
                }
            } else {
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    out_tiles(j, a4_lds16(at_v0 + st + 2 * j) | a4_lds16(at_v1 + st + 2 * j) << 16,
                              a4_lds16(at_v0 + st + 8 * X::ROW + 2 * j) | a4_lds16(at_v1 + st + 8 * X::ROW + 2 * j) << 16);
            }
            }
            stage ^= X::STAGE;
        }

        // ---- join the warps ------------------------------------------------------------------------------------------------------
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
            l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
            if constexpr (!BASES)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    zacc[g][0] += __shfl_xor_sync(0xffffffffu, zacc[g][0], o);
                    zacc[g][1] += __shfl_xor_sync(0xffffffffu, zacc[g][1], o);
                }
        }
        if constexpr (BASES) {
            const float back = a4_exp2(e - 9.f);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    const int from = 8 * g + t;            // the lane that has the scale's sum; the base's is 4 on
                    zacc[g][e2] = fmaf(__shfl_sync(0xffffffffu, bacc[e2], from), A4_MIDDLE, __shfl_sync(0xffffffffu, bacc[e2], from + 4)) * back;
                }
        }
        if (lane < 4) {
            // a warp without positions has no say in the maximum
            *reinterpret_cast<float2 *>(&sm_ref[warp][2 * t]) = make_float2(l[0] != 0.f ? ref[0] : -INFINITY, l[1] != 0.f ? ref[1] : -INFINITY);
            *reinterpret_cast<float2 *>(&sm_l[warp][2 * t]) = make_float2(l[0], l[1]);
        }
        __syncthreads();                   // and every warp is done with its ring
        float *so = reinterpret_cast<float *>(smem);       // [warp][m-tile row][head], over the rings
        {
            float wgt[2], M[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < A4_WARPS; ++w) {
                M[0] = fmaxf(M[0], sm_ref[w][2 * t]);
                M[1] = fmaxf(M[1], sm_ref[w][2 * t + 1]);
            }
#pragma unroll
            for (int w = 0; w < A4_WARPS; ++w)
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    const float lw = sm_l[w][2 * t + e2], x = lw == 0.f ? 0.f : a4_exp2(sm_ref[w][2 * t + e2] - M[e2]);
                    L[e2] += lw * x;
                    if (w == warp) wgt[e2] = x;
                }
            if (tid < 4) {
                *reinterpret_cast<float2 *>(&sm_top[2 * t]) = make_float2(M[0], M[1]);
                *reinterpret_cast<float2 *>(&sm_sum[2 * t]) = make_float2(L[0], L[1]);
            }
            float *o0 = so + (warp * X::D + r) * A4_HEADS + 2 * t;
            const float own = SPLIT && t >= 2 ? 0.f : 1.f;         // the bases count once
#pragma unroll
            for (int m = 0; m < X::MTILES; ++m) {
                const int g = (m / 2) * NG / NB;
                const float za = fmaf(sacc[g / 2][2 * (g & 1)], -A4_MIDDLE, zacc[g][0] * own) * wgt[0];
                const float zb = fmaf(sacc[g / 2][2 * (g & 1) + 1], -A4_MIDDLE, zacc[g][1] * own) * wgt[1];
                float2 lo = make_float2(fmaf(oacc[m][0], 16777216.f * wgt[0], za), fmaf(oacc[m][1], 16777216.f * wgt[1], zb));
                float2 hi = make_float2(fmaf(oacc[m][2], 1048576.f * wgt[0], za), fmaf(oacc[m][3], 1048576.f * wgt[1], zb));
                if constexpr (SPLIT) {
                    lo.x += __shfl_xor_sync(0xffffffffu, lo.x, 2); lo.y += __shfl_xor_sync(0xffffffffu, lo.y, 2);
                    hi.x += __shfl_xor_sync(0xffffffffu, hi.x, 2); hi.y += __shfl_xor_sync(0xffffffffu, hi.y, 2);
                }
                *reinterpret_cast<float2 *>(o0 + m * 16 * A4_HEADS) = lo;
                *reinterpret_cast<float2 *>(o0 + (m * 16 + 8) * A4_HEADS) = hi;
            }
        }
        __syncthreads();
        const int two = d.heads > 4, quads = 1 + two;      // groups of four heads that exist
        // the sum over the warps of float4 i & two of m-tile row i >> two
        auto sum4 = [&](int i) {
            const float4 *s4 = reinterpret_cast<const float4 *>(so) + (i >> two) * 2 + (i & two);
            float4 o = s4[0];
#pragma unroll
            for (int w = 1; w < A4_WARPS; ++w) {
                const float4 x = s4[w * X::D * A4_HEADS / 4];
                o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
            }
            return o;
        };
        // ---- join the CTAs: partial results through the workspace, A4_FAN neighbours by the last of them to arrive, and so on with
        // these sums, always in CTA order -------------------------------------------------------------------------------------------
        bool last = true;
        if (d.u1 - d.u0 < d.n) {           // not the whole context was here
            const int c0 = d.c0;
            int members = d.members, me = blockIdx.x - c0, step = 1;
            // a CTA has two places: for a context that it continues, and for one that it begins
            auto place = [&](int c) { return (int)(c0 + c) * 2 + (c == 0); };
            int *counters = A.counters;
#pragma unroll 1
            while (members > 1) {
                const int lead = me / A4_FAN * A4_FAN, count = min(A4_FAN, members - lead);
                float *part = A.parts + (long)place(me * step) * X::PART;
#pragma unroll 1
                for (int i = tid; i < X::D * quads; i += A4_THREADS) reinterpret_cast<float4 *>(part)[(i >> two) * 2 + (i & two)] = sum4(i);
                if (tid < A4_HEADS) reinterpret_cast<float2 *>(part + X::D * A4_HEADS)[tid] = make_float2(sm_top[tid], sm_sum[tid]);
                __syncthreads();
                if (tid == 0) {
                    __threadfence();       // orders the whole block's stores: the barrier came before it
                    sm_last = atomicAdd(&counters[place(lead * step)], 1) == count - 1;
                    if (sm_last) counters[place(lead * step)] = 0;      // ready for the next launch
                    __threadfence();
                }
                __syncthreads();
                last = sm_last;
                if (!last) break;
                // every thread one (part, head): the weights 2^(m - M); every warp a quarter of the parts, all loads under way at once
                static_assert(A4_FAN * A4_HEADS == A4_THREADS && A4_FAN == 4 * A4_WARPS, "a thread for every part and head");
                auto part_at = [&](int c) { return A.parts + (long)place((lead + c) * step) * X::PART; };
                const int c = tid >> 3, h = tid & 7;
                float2 ml = make_float2(0.f, 0.f);
                if (c < count) ml = __ldcg(reinterpret_cast<const float2 *>(part_at(c) + X::D * A4_HEADS) + h);
                constexpr int DEEP = X::D / 32 < 4 ? X::D / 32 : 4;
#pragma unroll 1
                for (int i0 = lane; i0 < X::D * quads; i0 += 32 * DEEP) {
                    float4 x[DEEP][4];
#pragma unroll
                    for (int j = 0; j < DEEP; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int i = i0 + 32 * j;
                            x[j][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (warp * 4 + k < count && i < X::D * quads)
                                x[j][k] = __ldcg(reinterpret_cast<const float4 *>(part_at(warp * 4 + k)) + (i >> two) * 2 + (i & two));
                        }
                    if (i0 == lane) {
                        float M = ml.y == 0.f ? -INFINITY : ml.x;
                        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
                        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
                        if (lane < 8) sm_ref[warp][lane] = M;
                        __syncthreads();
#pragma unroll
                        for (int w = 0; w < A4_WARPS; ++w) M = fmaxf(M, sm_ref[w][h]);
                        const float wt = ml.y == 0.f ? 0.f : a4_exp2(ml.x - M);
                        float L = ml.y * wt;
                        sm_wt[c][h] = wt;
                        L += __shfl_xor_sync(0xffffffffu, L, 8);
                        L += __shfl_xor_sync(0xffffffffu, L, 16);
                        if (lane < 8) sm_l[warp][lane] = L;
                        __syncthreads();
                        if (tid < A4_HEADS) {
                            sm_top[tid] = M;
                            sm_sum[tid] = sm_l[0][tid] + sm_l[1][tid] + sm_l[2][tid] + sm_l[3][tid];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < DEEP; ++j) {
                        const int i = i0 + 32 * j, at4 = (i >> two) * 2 + (i & two);
                        if (i >= X::D * quads) break;
                        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float4 w = *reinterpret_cast<const float4 *>(&sm_wt[warp * 4 + k][4 * (at4 & 1)]);
                            o.x = fmaf(w.x, x[j][k].x, o.x); o.y = fmaf(w.y, x[j][k].y, o.y); o.z = fmaf(w.z, x[j][k].z, o.z); o.w = fmaf(w.w, x[j][k].w, o.w);
                        }
                        reinterpret_cast<float4 *>(so + warp * X::D * A4_HEADS)[at4] = o;
                    }
                }
                __syncthreads();
                me /= A4_FAN;
                members = (members + A4_FAN - 1) / A4_FAN;
                step *= A4_FAN;
                counters += 2 * A4_MAX_CTAS;       // a level's own counters
            }
        }
        if (last) {                        // the output rows of these heads
#pragma unroll 1
            for (int i = tid; i < X::D * quads; i += A4_THREADS) {
                const float4 o4 = sum4(i);
                const float o[4] = {o4.x, o4.y, o4.z, o4.w};
                const int idx = i >> two, m = idx >> 4, row = idx & 15, dim = 32 * (m >> 1) + 4 * (row & 7) + 2 * (m & 1) + (row >> 3);
                const int e7 = dim & 7, dd = A.out_kperm ? (dim & ~7) | (e7 < 4 ? 2 * e7 : 2 * e7 - 7) : dim;
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int h = 4 * (i & two) + e4;
                    if (h >= d.heads) break;
                    const float v = sm_sum[h] == 0.f ? 0.f : __fdividef(o[e4], sm_sum[h]);   // nothing but blocks outside the pool: 0
                    const long at_out = ((long)d.b * A.hq + d.h0 + h) * X::D + dd;
                    if (A.bf16) reinterpret_cast<__nv_bfloat16 *>(A.out)[at_out] = __float2bfloat16_rn(v);
                    else reinterpret_cast<__half *>(A.out)[at_out] = __float2half_rn(v);
                }
            }
        }
        if (!d.more) break;
        __syncthreads();                   // everybody has done with this segment
        if (tid == 0) segment(sm_seg);
        __syncthreads();
    }
}

// Workspace: the status word, the arrival counters from byte 256, and from 128 KiB the partial results.
constexpr size_t A4_COUNTERS_OFF = 256, A4_PARTS_OFF = 128 * 1024;
static size_t attn4_ws_bytes(int d) { return A4_PARTS_OFF + (size_t)A4_MAX_CTAS * 2 * (d * A4_HEADS + 16) * sizeof(float); }

template <int NB, int NG, int MODE>
static int attn4_launch_as(const char *name, const Attn4Args &A, long max_units, cudaStream_t st) {
    using X = A4<NB, NG>;
    static OncePerDevice once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(attn4_kernel<NB, NG, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, X::SMEM); });
    if (e != cudaSuccess) return fail((int)e, "%s: shared memory %d: %s", name, X::SMEM, cudaGetErrorString(e));
    const int wave = min(sm_count() * X::CTAS, A4_MAX_CTAS);
    launch_kernel(attn4_kernel<NB, NG, MODE>, dim3((unsigned)min(max_units, (long)wave)), dim3(A4_THREADS), X::SMEM, st, A);
    return launch_status(name);
}

template <int NB, int NG>
static int attn4_launch_shape(const char *name, const Attn4Args &A, long max_units, cudaStream_t st) {
    if (!A.bf16 && A.hq / A.C.heads <= 4) return attn4_launch_as<NB, NG, A4_SPLIT>(name, A, max_units, st);
    if constexpr (A4<NB, NG>::BASES)
        if (!A.bf16) return attn4_launch_as<NB, NG, A4_EXACT_BASES>(name, A, max_units, st);
    return attn4_launch_as<NB, NG, A4_PLAIN>(name, A, max_units, st);
}

static int attn4_launch(const char *name, const void *q, const Kv4Cache &C, bool paged, const int32_t *lens, void *out, int batch, int hq,
                        float scale, bool bf16, bool out_kperm, void *ws, size_t ws_bytes, bool own_ws, b200k_stream stream) {
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
    B200K_REQUIRE(ws && aligned16(ws) && ws_bytes >= attn4_ws_bytes(C.d), B200K_E_WORKSPACE, "%s: workspace %zu bytes, need %zu (16-byte aligned)", name,
                  ws_bytes, attn4_ws_bytes(C.d));
    Attn4Args A = {};
    A.q = q; A.out = out; A.lens = lens; A.C = C;
    A.block_magic = ~0ull / (unsigned)C.block_size + 1;      // used for multiples of 16 only
    A.batch = batch; A.hq = hq; A.head_blocks = ceil_div(hq / C.heads, A4_HEADS);
    A.bf16 = bf16; A.out_kperm = out_kperm;
    A.scale_log2e = scale * 1.4426950408889634f;
    A.status = (int *)ws;
    A.counters = (int *)((unsigned char *)ws + A4_COUNTERS_OFF);
    A.parts = (float *)((unsigned char *)ws + A4_PARTS_OFF);
    const long max_units = (long)batch * C.heads * A.head_blocks * (((long)C.capacity + A4_UNIT - 1) / A4_UNIT);
    B200K_REQUIRE(max_units < (1l << 31), B200K_E_SHAPE, "%s: batch * num_kv_heads * ceil(gqa / 8) * ceil(positions / 128) = %ld exceeds 31 bits", name, max_units);
    cudaStream_t st = to_stream(stream);
    switch (C.d / 32 * 1000 + C.d / C.g) {
        case 1001: return attn4_launch_shape<1, 1>(name, A, max_units, st);
        case 2001: return attn4_launch_shape<2, 1>(name, A, max_units, st);
        case 2002: return attn4_launch_shape<2, 2>(name, A, max_units, st);
        case 3003: return attn4_launch_shape<3, 3>(name, A, max_units, st);
        case 4001: return attn4_launch_shape<4, 1>(name, A, max_units, st);
        case 4002: return attn4_launch_shape<4, 2>(name, A, max_units, st);
        case 4004: return attn4_launch_shape<4, 4>(name, A, max_units, st);
        case 5005: return attn4_launch_shape<5, 5>(name, A, max_units, st);
        case 6003: return attn4_launch_shape<6, 3>(name, A, max_units, st);
        case 6006: return attn4_launch_shape<6, 6>(name, A, max_units, st);
        case 7007: return attn4_launch_shape<7, 7>(name, A, max_units, st);
        case 8002: return attn4_launch_shape<8, 2>(name, A, max_units, st);
        case 8004: return attn4_launch_shape<8, 4>(name, A, max_units, st);
        case 8008: return attn4_launch_shape<8, 8>(name, A, max_units, st);
    }
    return fail(B200K_E_SHAPE, "%s: head_dim %d, group_size %d", name, C.d, C.g);
}

// The head-major call with the output in the pre-permuted order the int4 GEMM wants, where asked for (used by the decode layer)
int batched_decode_attention_hm_int4_f16_layer(const __half *q, const int32_t *kc, const __half *kp, const int32_t *vc, const __half *vp,
                                               const int32_t *context_lens, __half *output, int batch, int hq, int hkv, int d, int g, int max_len,
                                               float scale, bool kperm, cudaStream_t st) {
    return attn4_launch("batched_decode_attention_hm_int4_f16", q, kv4_cache(kc, (const b200k_half *)kp, vc, (const b200k_half *)vp, hkv, d, g, max_len),
                        false, context_lens, output, batch, hq, scale, false, kperm, nullptr, 0, true, (b200k_stream)st);
}

}  // namespace b200k

using namespace b200k;

extern "C" size_t b200k_attention_int4_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int head_dim) {
    if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0) return 0;
    return attn4_ws_bytes(head_dim);
}

#define ATTN4_ENTRIES(SUF, ABI, IS_BF16)                                                                                                         \
    extern "C" int batched_decode_attention_hm_int4_##SUF##_ws(const ABI *q, const int32_t *k_codes, const b200k_half *k_params,             \
                                                               const int32_t *v_codes, const b200k_half *v_params,                          \
                                                               const int32_t *context_lens, ABI *output, int batch_size, int num_q_heads,   \
                                                               int num_kv_heads, int head_dim, int group_size, int max_len, float scale,    \
                                                               void *workspace, size_t workspace_bytes, b200k_stream stream) {              \
        return attn4_launch("batched_decode_attention_hm_int4_" #SUF, q,                                                                 \
                               kv4_cache(k_codes, k_params, v_codes, v_params, num_kv_heads, head_dim, group_size, max_len), false,         \
                               context_lens, output, batch_size, num_q_heads, scale, IS_BF16, false, workspace, workspace_bytes, workspace == nullptr, stream); \
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
        return attn4_launch("batched_decode_attention_paged_int4_" #SUF, q,                                                              \
                               kv4_pool(k_codes, k_params, v_codes, v_params, block_table, num_kv_heads, head_dim, group_size, block_size,  \
                                        num_blocks, max_blocks_per_seq), true, context_lens, output, batch_size, num_q_heads, scale,        \
                               IS_BF16, false, workspace, workspace_bytes, workspace == nullptr, stream);                                                   \
    }                                                                                                                                       \
    extern "C" int batched_decode_attention_paged_int4_##SUF(                                                                               \
        const ABI *q, const int32_t *k_codes, const b200k_half *k_params, const int32_t *v_codes, const b200k_half *v_params,               \
        const int32_t *block_table, const int32_t *context_lens, ABI *output, int batch_size, int num_q_heads, int num_kv_heads,            \
        int head_dim, int group_size, int block_size, int num_blocks, int max_blocks_per_seq, float scale, b200k_stream stream) {           \
        return batched_decode_attention_paged_int4_##SUF##_ws(q, k_codes, k_params, v_codes, v_params, block_table, context_lens, output,   \
                                                              batch_size, num_q_heads, num_kv_heads, head_dim, group_size, block_size,      \
                                                              num_blocks, max_blocks_per_seq, scale, nullptr, 0, stream);                   \
    }

ATTN4_ENTRIES(f16, b200k_half, false)
ATTN4_ENTRIES(bf16, b200k_bf16, true)
