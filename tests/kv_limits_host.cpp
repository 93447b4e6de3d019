// CPU checks of the cache and attention entry points at the ends of their ranges: sizes whose byte counts pass 64
// bits, and host memory or device copies that fail in the middle of a call.  Prints "kv limits ok" and exits 0 on success.
//
// Build: c++ -std=c++17 -Wall -Wextra -Werror -I include tests/kv_limits_host.cpp -o kv_limits_host
#include <cstdio>
#include <cstdlib>
#include <new>

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

// The allocation after `left` more fails (never, below zero).
static long left = -1;
__attribute__((noinline)) void* operator new(std::size_t n) {
    if (left == 0) throw std::bad_alloc();
    if (left > 0) --left;
    if (void* p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
__attribute__((noinline)) void operator delete(void* p) noexcept { std::free(p); }
__attribute__((noinline)) void operator delete(void* p, std::size_t) noexcept { std::free(p); }

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

// A cache of 12 pages of 16 with holes: living sequences a (2 pages, 20 tokens), c (3, 48), d (1, 5) around freed ones.
struct Holes {
    moe::KvPages kv{12, 16};
    uint64_t a, c, d;
    Holes() {
        uint64_t h[5];
        const uint64_t add[5] = {20, 40, 48, 16, 5};
        EXPECT(kv.create(5, h, &err) == MOE_OK && kv.extend(h, 5, add, &err) == MOE_OK);
        const uint64_t gone[2] = {h[1], h[3]};
        EXPECT(kv.free(gone, 2, &err) == MOE_OK);
        a = h[0]; c = h[2]; d = h[4];
    }
    std::vector<int32_t> state() {
        const uint64_t h[3] = {a, c, d};
        std::vector<int32_t> t;
        EXPECT(kv.tables(h, 3, 12, &t, &err) == MOE_OK);
        t.push_back(static_cast<int32_t>(kv.n_free()));
        return t;
    }
    // New pages are none that a living sequence has, and all free ones can be had.
    void still_sound() {
        const std::vector<int32_t> before = state();
        std::vector<int> users(12, 0);
        const uint32_t pages[3] = {2, 3, 1};
        for (int i = 0; i < 3; ++i)
            for (uint32_t j = 0; j < pages[i]; ++j) ++users[before[12 * i + j]];
        uint64_t x, all = 16ull * kv.n_free();
        std::vector<int32_t> t;
        EXPECT(kv.create(1, &x, &err) == MOE_OK && kv.extend(&x, 1, &all, &err) == MOE_OK && kv.n_free() == 0 && kv.tables(&x, 1, 12, &t, &err) == MOE_OK);
        for (uint64_t j = 0; j < all / 16; ++j) ++users[t[j]];
        for (int u : users) EXPECT(u == 1);
    }
};

// Every call does all of its work or, with an error, none: for each allocation that it makes, that one failing.
template <typename F>
static void failing_memory(F&& call) {
    for (long k = 0;; ++k) {
        EXPECT(k < 1000);
        Holes h;
        const std::vector<int32_t> before = h.state();
        bool threw = false;
        left = k;
        try {
            call(h);
        } catch (const std::bad_alloc&) {
            threw = true;
        }
        left = -1;
        if (!threw) return;  // it makes no more than k
        EXPECT(h.state() == before);
        h.still_sound();
    }
}

static void failures_leave_no_trace() {
    failing_memory([](Holes& h) { moe::KvPages::Moves m; h.kv.compact(&m); });
    failing_memory([](Holes& h) { const uint64_t add[2] = {30, 40}, s[2] = {h.a, h.d}; h.kv.extend(s, 2, add, &err); });
    failing_memory([](Holes& h) { const uint64_t p[3] = {h.a, h.c, h.a}; uint64_t kids[3]; moe::KvPages::Moves m; h.kv.fork(p, 3, kids, &m, &err); });
    failing_memory([](Holes& h) { uint64_t s[40]; h.kv.create(40, s, &err); });
    failing_memory([](Holes& h) { std::vector<int32_t> t; h.kv.tables(&h.a, 1, 12, &t, &err); });
    // a device copy that fails, or host memory that ends in it
    for (const bool throws : {false, true}) {
        Holes h;
        const std::vector<int32_t> before = h.state();
        const uint64_t p[3] = {h.a, h.c, h.a};
        uint64_t kids[3] = {7, 7, 7};
        auto copy = [&](const moe::KvPages::Moves& m) -> int {
            EXPECT(!m.empty());
            if (throws) throw std::bad_alloc();
            return MOE_E_CUDA;
        };
        for (const bool fork : {true, false}) {
            moe::KvPages::Moves m;
            int rc = MOE_E_CUDA;
            try {
                rc = fork ? h.kv.fork(p, 3, kids, &m, &err, copy) : h.kv.compact(&m, copy);
            } catch (const std::bad_alloc&) {
                EXPECT(throws);
            }
            EXPECT(rc == MOE_E_CUDA && kids[0] == 7 && kids[2] == 7 && h.state() == before);
        }
        h.still_sound();
    }
}

int main() {
    failures_leave_no_trace();
    rows_past_64_bits();
    token_numbers();
    std::puts("kv limits ok");
    return 0;
}
