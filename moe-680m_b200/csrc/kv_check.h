// Argument checks of the cache and attention entry points, in plain C++ over plain values: every
// refusal happens here, before any CUDA call.
#pragma once
#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/moe_b200.h"

namespace moe {

// Sequences of one batch: the kernels keep their running counts in shared memory.
constexpr uint32_t kMaxBatchSeqs = 4096;

struct KvSpec {
    uint32_t type = 0, n_layers = 0, n_kv_heads = 0, head_dim = 0, page_size = 0, n_pages = 0;
    uint64_t k_off = 0, v_off = 0;
    uint64_t page_bytes() const { return 2ull * n_kv_heads * page_size * head_dim; }
    uint64_t layer_bytes() const { return page_bytes() * n_pages; }
    uint64_t pool_bytes() const { return layer_bytes() * n_layers; }
};

// One call on a batch: rows are q and out (attention) or k and v (append).
struct KvCall {
    uint32_t layer = 0, type = 0, n_seqs = 0, tokens = 0, max_pages = 0;
    uint64_t cu_off = 0, table_off = 0, lens_off = 0;
    uint64_t a_off = 0, a_stride = 0, a_width = 0;  // q, or k; width and stride in values
    uint64_t b_off = 0, b_stride = 0, b_width = 0;  // out, or v
};

inline int kv_refuse(std::string* err, int code, const std::string& what) {
    *err = what;
    return code;
}

inline bool kv_in_arena(uint64_t arena, uint64_t off, uint64_t bytes, uint64_t align) {
    return off != 0 && off % align == 0 && off <= arena && bytes <= arena - off;
}

inline bool kv_overlap(uint64_t a, uint64_t na, uint64_t b, uint64_t nb) { return a < b + nb && b < a + na; }

inline uint64_t kv_type_bytes(uint32_t type) { return type == MOE_T_F32 ? 4 : 2; }

inline int kv_check_spec(const KvSpec& s, uint64_t arena, std::string* err) {
    if (s.type != MOE_T_F16 && s.type != MOE_T_BF16)
        return kv_refuse(err, MOE_E_UNSUPPORTED, "cache type " + std::to_string(s.type) + ": MOE_T_F16 or MOE_T_BF16");
    if (s.head_dim != 64 && s.head_dim != 128)
        return kv_refuse(err, MOE_E_UNSUPPORTED, "head_dim " + std::to_string(s.head_dim) + ": 64 or 128");
    if (s.page_size != 16 && s.page_size != 32 && s.page_size != 64 && s.page_size != 128)
        return kv_refuse(err, MOE_E_UNSUPPORTED, "page_size " + std::to_string(s.page_size) + ": 16, 32, 64 or 128");
    if (s.n_layers == 0 || s.n_kv_heads == 0 || s.n_pages == 0 || s.n_layers > 65536 || s.n_kv_heads > 256)
        return kv_refuse(err, MOE_E_INVALID, "n_layers (1..65536), n_kv_heads (1..256) or n_pages (1..) invalid");
    // rows of a pool are addressed with 31 bits (rows, not bytes: up to 512 GB)
    const uint64_t page_rows = static_cast<uint64_t>(s.n_kv_heads) * s.page_size;
    if (s.n_pages > 0x7FFFFFFFull / page_rows || s.n_layers > 0x7FFFFFFFull / (page_rows * s.n_pages))
        return kv_refuse(err, MOE_E_UNSUPPORTED, "pool of 2^31 rows or more");
    if (!kv_in_arena(arena, s.k_off, s.pool_bytes(), 256) || !kv_in_arena(arena, s.v_off, s.pool_bytes(), 256))
        return kv_refuse(err, MOE_E_INVALID, "pool offset missing, not 256-byte aligned or outside the arena");
    if (kv_overlap(s.k_off, s.pool_bytes(), s.v_off, s.pool_bytes()))
        return kv_refuse(err, MOE_E_INVALID, "the key and value pools overlap");
    return MOE_OK;
}

// Bytes of `rows` rows of `width` values, `stride` values apart; 0 when a number is out of range.
inline uint64_t kv_rows_bytes(uint64_t rows, uint64_t stride, uint64_t width, uint64_t size) {
    if (stride < width || stride > (1ull << 40) || rows == 0) return 0;
    if (stride && rows - 1 > (~0ull / size - width) / stride) return 0;  // past 64 bits
    return ((rows - 1) * stride + width) * size;
}

// write_b: b is written (out); otherwise both are read.
inline int kv_check_call(const KvSpec& s, const KvCall& c, uint64_t arena, bool write_b, std::string* err) {
    if (c.layer >= s.n_layers) return kv_refuse(err, MOE_E_INVALID, "layer " + std::to_string(c.layer) + " of a cache with " + std::to_string(s.n_layers));
    if (c.type > MOE_T_BF16) return kv_refuse(err, MOE_E_INVALID, "unknown type " + std::to_string(c.type));
    if (c.type != MOE_T_F32 && c.type != s.type)
        return kv_refuse(err, MOE_E_UNSUPPORTED, "16-bit activations of another type than the cache's");
    if (c.n_seqs > kMaxBatchSeqs) return kv_refuse(err, MOE_E_UNSUPPORTED, "n_seqs " + std::to_string(c.n_seqs) + ": at most 4096");
    if (c.tokens > 0x7FFFFFFFu) return kv_refuse(err, MOE_E_UNSUPPORTED, "2^31 tokens or more");  // offsets have 31 bits
    if (c.cu_off == 0 && c.tokens != c.n_seqs)
        return kv_refuse(err, MOE_E_INVALID, "without offsets there is one token for each sequence");
    if (c.max_pages == 0 || static_cast<uint64_t>(c.max_pages) * s.page_size > 2147483392ull)
        return kv_refuse(err, MOE_E_INVALID, "max_pages invalid");
    if (!kv_in_arena(arena, c.table_off, 4ull * c.n_seqs * c.max_pages, 4) || !kv_in_arena(arena, c.lens_off, 4ull * c.n_seqs, 4) ||
        (c.cu_off && !kv_in_arena(arena, c.cu_off, 4ull * (c.n_seqs + 1), 4)))
        return kv_refuse(err, MOE_E_INVALID, "table, lens or offsets outside the arena or misaligned");
    const uint64_t size = kv_type_bytes(c.type), per16 = 16 / size;
    const uint64_t na = kv_rows_bytes(c.tokens, c.a_stride, c.a_width, size), nb = kv_rows_bytes(c.tokens, c.b_stride, c.b_width, size);
    if (na == 0 || nb == 0 || c.a_stride % per16 || c.b_stride % per16)
        return kv_refuse(err, MOE_E_INVALID, "row stride below the row's width or too large, or not a multiple of 16 bytes");
    if (!kv_in_arena(arena, c.a_off, na, 16) || !kv_in_arena(arena, c.b_off, nb, 16))
        return kv_refuse(err, MOE_E_INVALID, "rows outside the arena or not 16-byte aligned");
    const uint64_t pool = s.pool_bytes();
    if (write_b && (kv_overlap(c.b_off, nb, c.a_off, na) || kv_overlap(c.b_off, nb, s.k_off, pool) || kv_overlap(c.b_off, nb, s.v_off, pool)))
        return kv_refuse(err, MOE_E_INVALID, "the output overlaps the queries or the cache");
    if (!write_b && (kv_overlap(c.a_off, na, s.k_off, pool) || kv_overlap(c.a_off, na, s.v_off, pool) ||
                     kv_overlap(c.b_off, nb, s.k_off, pool) || kv_overlap(c.b_off, nb, s.v_off, pool)))
        return kv_refuse(err, MOE_E_INVALID, "the new rows overlap the cache");
    auto on_lists = [&](uint64_t off, uint64_t n) {
        return kv_overlap(off, n, c.table_off, 4ull * c.n_seqs * c.max_pages) || kv_overlap(off, n, c.lens_off, 4ull * c.n_seqs) ||
               (c.cu_off && kv_overlap(off, n, c.cu_off, 4ull * (c.n_seqs + 1)));
    };
    if (write_b ? on_lists(c.b_off, nb) : on_lists(s.k_off, pool) || on_lists(s.v_off, pool))
        return kv_refuse(err, MOE_E_INVALID, "what is written overlaps the page table, lengths or offsets");
    return MOE_OK;
}

inline int kv_check_tables(const KvSpec& s, uint64_t arena, uint32_t n, uint32_t max_pages, uint64_t table_off, uint64_t lens_off,
                           std::string* err) {
    if (n > kMaxBatchSeqs) return kv_refuse(err, MOE_E_UNSUPPORTED, "n_seqs " + std::to_string(n) + ": at most 4096");
    const uint64_t table = 4ull * max_pages * n, lens = 4ull * n, pool = s.pool_bytes();
    if (max_pages == 0 || !kv_in_arena(arena, table_off, table, 4) || !kv_in_arena(arena, lens_off, lens, 4) ||
        kv_overlap(table_off, table, lens_off, lens))
        return kv_refuse(err, MOE_E_INVALID, "table or lens offset invalid");
    for (uint64_t off : {s.k_off, s.v_off})
        if (kv_overlap(table_off, table, off, pool) || kv_overlap(lens_off, lens, off, pool))
            return kv_refuse(err, MOE_E_INVALID, "the table or the lengths overlap the cache");
    return MOE_OK;
}

inline int kv_check_heads(const KvSpec& s, const KvCall& c, uint32_t n_heads, float scale, std::string* err) {
    if (n_heads == 0 || n_heads > 4096 || n_heads % s.n_kv_heads != 0)
        return kv_refuse(err, MOE_E_INVALID, "n_heads " + std::to_string(n_heads) + ": a multiple of the cache's " +
                                                 std::to_string(s.n_kv_heads) + ", at most 4096");
    if (static_cast<uint64_t>(c.tokens) * n_heads > 0x7FFFFFFFull / 2) return kv_refuse(err, MOE_E_UNSUPPORTED, "2^30 query rows or more");
    if (!(scale > 0.f) || !std::isfinite(scale)) return kv_refuse(err, MOE_E_INVALID, "scale must be positive and finite");
    return MOE_OK;
}

// The decode kernel counts tiles of 32 tokens over all sequences and head blocks with 31 bits.
inline int kv_check_decode(const KvSpec& s, const KvCall& c, uint32_t n_heads, std::string* err) {
    const uint64_t group = n_heads / s.n_kv_heads, blocks = group > 8 ? (group + 15) / 16 : 1;
    const uint64_t tiles = (static_cast<uint64_t>(c.max_pages) * s.page_size + 31) / 32 * blocks * s.n_kv_heads;
    if (tiles > 0x7FFFFFFFull / c.n_seqs) return kv_refuse(err, MOE_E_UNSUPPORTED, "page tables of 2^36 tokens (times kv heads) or more");
    return MOE_OK;
}

}  // namespace moe
