// The 4-bit KV cache: its format, where a row stands, and the checks that every entry point makes.
//
// A row is one (position, kv head): D codes of 4 bits, D a multiple of 32 up to 256, and for every group of G
// consecutive dims (G = 32, 64 or 128, D % G == 0) a pair (scale, base) of fp16.  With x' = clamp(x, -LIMIT, LIMIT):
//   base  = fp16(min x')      scale = fp16((max x' - base) / 15)
//   code  = clamp(round_half_even((x' - base) / scale), 0, 15), 0 where scale = 0
//   value = code * scale + base
// Two fp16 a group cost 4 bytes (a quarter to a sixteenth of the codes); fp32 ones would double that for nothing, because
// the codes are chosen for the scale and base as stored.  LIMIT leaves room for the rounding of the scale, so that
// 15 * scale + base is finite in fp16.  A NaN makes scale and base NaN: its whole group reads back as NaN.
//
// Order of the codes: the row's D/4 units of four codes (16 bits; unit u = 8 j + r holds dims 4u .. 4u+3, the lowest in
// the lowest bits) stand at place r * (D/32) + j.  A contiguous eighth or quarter of a row then holds the same number of
// codes of every 32-dim block, hence of every group: a lane that loads such a piece in one access can feed the matrix
// instruction one group at a time, and the group's scale can be applied to the products instead of to every code.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace b200k {

constexpr float KV4_LIMIT = 65440.f;
constexpr long KV4_MAX_LEN = 1l << 30;      // positions of a sequence: sums of two of them stay in 32 bits
constexpr int KV4_BAD_POSITION = 4, KV4_BAD_BLOCK = 8;   // bits of the status word

struct Kv4Cache {
    int32_t *k_codes, *v_codes;      // [rows, D/8]
    __half *k_params, *v_params;     // [rows, D/G, 2]
    const int32_t *block_table;      // [batch, max_blocks], or nullptr: head-major [batch, heads, capacity]
    int heads, d, g;
    int block_size;                  // positions a block; head-major: the capacity, one block per sequence
    int num_blocks, max_blocks;
    int capacity;                    // positions a sequence can hold
};

// Row index of (b, h, pos), 0 <= pos < capacity; -1 when the block table names a block that the pool does not have.
__host__ __device__ __forceinline__ long kv4_row(const Kv4Cache &C, int b, int h, int pos) {
    if (!C.block_table) return ((long)b * C.heads + h) * C.capacity + pos;
    const int lb = pos / C.block_size;
    const int blk = C.block_table[(long)b * C.max_blocks + lb];
    if ((unsigned)blk >= (unsigned)C.num_blocks) return -1;
    return ((long)blk * C.heads + h) * C.block_size + (pos - lb * C.block_size);
}

static inline int kv4_check(const char *name, const Kv4Cache &C, int batch, bool paged) {
    B200K_REQUIRE(C.k_codes && C.k_params && C.v_codes && C.v_params && (!paged || C.block_table), B200K_E_NULL, "%s: NULL pointer", name);
    B200K_REQUIRE(C.heads > 0 && batch >= 0 && batch <= 65535, B200K_E_SHAPE, "%s: heads %d, batch %d", name, C.heads, batch);
    B200K_REQUIRE(C.d > 0 && C.d <= 256 && C.d % 32 == 0, B200K_E_SHAPE, "%s: head_dim %d (a multiple of 32 up to 256)", name, C.d);
    B200K_REQUIRE((C.g == 32 || C.g == 64 || C.g == 128) && C.d % C.g == 0, B200K_E_SHAPE,
                  "%s: group_size %d (32, 64 or 128, dividing head_dim %d)", name, C.g, C.d);
    if (paged)
        B200K_REQUIRE(C.block_size > 0 && C.num_blocks > 0 && C.max_blocks > 0 && (long)C.block_size * C.max_blocks <= KV4_MAX_LEN, B200K_E_SHAPE,
                      "%s: block_size %d, num_blocks %d, max_blocks_per_seq %d", name, C.block_size, C.num_blocks, C.max_blocks);
    else
        B200K_REQUIRE(C.capacity > 0 && C.capacity <= KV4_MAX_LEN, B200K_E_SHAPE, "%s: max_len %d", name, C.capacity);
    B200K_REQUIRE(aligned16(C.k_codes) && aligned16(C.v_codes) && aligned16(C.k_params) && aligned16(C.v_params), B200K_E_ALIGN,
                  "%s: codes and params must be 16-byte aligned", name);
    return 0;
}

static inline Kv4Cache kv4_cache(const int32_t *kc, const b200k_half *kp, const int32_t *vc, const b200k_half *vp, int heads, int d, int g, int max_len) {
    Kv4Cache C = {};
    C.k_codes = const_cast<int32_t *>(kc); C.v_codes = const_cast<int32_t *>(vc);
    C.k_params = (__half *)const_cast<b200k_half *>(kp); C.v_params = (__half *)const_cast<b200k_half *>(vp);
    C.heads = heads; C.d = d; C.g = g; C.block_size = C.capacity = max_len; C.max_blocks = 1;
    return C;
}
static inline Kv4Cache kv4_pool(const int32_t *kc, const b200k_half *kp, const int32_t *vc, const b200k_half *vp, const int32_t *table, int heads, int d,
                                int g, int block_size, int num_blocks, int max_blocks) {
    Kv4Cache C = kv4_cache(kc, kp, vc, vp, heads, d, g, 0);
    C.block_table = table; C.block_size = block_size; C.num_blocks = num_blocks; C.max_blocks = max_blocks;
    C.capacity = (int)min((long)block_size * max_blocks, KV4_MAX_LEN);
    return C;
}

}  // namespace b200k
