// CPU checks of the cache and attention entry points at the ends of their ranges: sizes whose byte counts pass 64
// bits.  Prints "kv limits ok" and exits 0 on success.
//
// Build: c++ -std=c++17 -Wall -Wextra -Werror -I include tests/kv_limits_host.cpp -o kv_limits_host
#include <cstdio>
#include <cstdlib>

#include "../moe-680m_b200/csrc/kv_check.h"
#include "../moe-680m_b200/csrc/kv_pages.h"

#define EXPECT(cond)                                                          \
    do {                                                                      \
        if (!(cond)) {                                                        \
            std::fprintf(stderr, "line %d: %s (%s)\n", __LINE__, #cond, err.c_str()); \
            std::exit(1);                                                     \
        }                                                                     \
    } while (0)

static std::string err;

// Rows that a wrapped product of tokens, stride and size would place inside a small arena.
static void rows_past_64_bits() {
    const uint64_t arena = 1 << 20;
    moe::KvSpec s;
    s.type = MOE_T_F16; s.n_layers = 1; s.n_kv_heads = 1; s.head_dim = 64; s.page_size = 16; s.n_pages = 8;
    s.k_off = 256; s.v_off = 256 + s.pool_bytes();
    moe::KvCall c;
    const uint64_t top = s.v_off + s.pool_bytes();
    c.type = MOE_T_F32; c.n_seqs = 1; c.max_pages = 4; c.cu_off = top; c.table_off = top + 256; c.lens_off = top + 512;
    c.a_off = top + 1024; c.b_off = top + 65536; c.a_width = c.b_width = 64; c.a_stride = c.b_stride = 64; c.tokens = 2;
    EXPECT(moe::kv_check_call(s, c, arena, true, &err) == MOE_OK && moe::kv_check_call(s, c, arena, false, &err) == MOE_OK);
    // (tokens - 1) * stride * 4 = 2^64 in each, and 2^65, and just below 2^64
    const struct { uint32_t tokens; uint64_t stride; } wraps[] = {{(1u << 28) + 1, 1ull << 34}, {(1u << 22) + 1, 1ull << 40}, {(1u << 30) + 1, 1ull << 32},
                                                                  {(1u << 25) + 1, 1ull << 38}, {(1u << 29) + 1, 1ull << 34}, {1u << 28, 1ull << 34}};
    for (const auto& w : wraps) {
        for (const bool a : {true, false}) {
            moe::KvCall x = c;
            x.tokens = w.tokens;
            (a ? x.a_stride : x.b_stride) = w.stride;
            for (const bool write : {true, false}) EXPECT(moe::kv_check_call(s, x, arena, write, &err) == MOE_E_INVALID);
            x.a_stride = x.b_stride = w.stride;
            for (const bool write : {true, false}) EXPECT(moe::kv_check_call(s, x, arena, write, &err) == MOE_E_INVALID);
        }
    }
    // the same in 16-bit rows: the product passes 2^64 one power of two later
    moe::KvCall h = c;
    h.type = MOE_T_F16; h.tokens = (1u << 29) + 1; h.a_stride = h.b_stride = 1ull << 34;
    for (const bool write : {true, false}) EXPECT(moe::kv_check_call(s, h, arena, write, &err) == MOE_E_INVALID);
    // one row reaches its width however far the next would be
    c.tokens = 1; c.a_stride = c.b_stride = 1ull << 40;
    EXPECT(moe::kv_check_call(s, c, arena, true, &err) == MOE_OK);
}

// Offsets of packed tokens have 31 bits.
static void token_numbers() {
    const uint64_t arena = 1ull << 50;
    moe::KvSpec s;
    s.type = MOE_T_F16; s.n_layers = 1; s.n_kv_heads = 1; s.head_dim = 64; s.page_size = 16; s.n_pages = 8;
    s.k_off = 256; s.v_off = 256 + s.pool_bytes();
    moe::KvCall c;
    const uint64_t top = s.v_off + s.pool_bytes();
    c.type = MOE_T_F16; c.n_seqs = 1; c.max_pages = 4; c.cu_off = top; c.table_off = top + 256; c.lens_off = top + 512;
    c.a_off = top + 1024; c.b_off = 1ull << 45; c.a_width = c.b_width = 64; c.a_stride = c.b_stride = 64;
    for (const uint32_t n : {1u, 0x7FFFFFFFu, 0x80000000u, 0xFFFFFFFFu}) {
        c.tokens = n;
        for (const bool write : {true, false}) EXPECT(moe::kv_check_call(s, c, arena, write, &err) == (n >> 31 ? MOE_E_UNSUPPORTED : MOE_OK));
    }
}

int main() {
    rows_past_64_bits();
    token_numbers();
    std::puts("kv limits ok");
    return 0;
}
