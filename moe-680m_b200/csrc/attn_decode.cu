// Attention of one new token per sequence over its cached tokens (moe_attn_decode; moe-680m:
// shaders/attention.comp at M = 1, src/inference.rs:484-555).
//
// Each cached key and value is read once and takes part in 4 flops per query head of its group, so
// the pass is bound by HBM: sum(len) * Hkv * D * 4 bytes.  The layout of the work follows from that:
//   * the unit is a tile of 32 tokens of one (sequence, kv head); all units of the batch form one
//     flat list that is cut into equal parts, one per SM, however ragged the lengths are;
//   * a part's units go round its 4 warps; each warp feeds itself: its lane 0 copies the keys and
//     values of its next units into a 3-deep ring (TMA, a box of 16 rows per copy, 128-byte
//     swizzle: pages of 16 rows and more are whole boxes) while the warp works on the oldest, so
//     up to 192 KB per SM are in flight and no warp waits for another inside a sequence;
//   * the query heads of a group are the 16 rows of mma.sync.m16n8k16 tiles; a group of up to 8
//     heads leaves 8 rows, which carry the second 16-bit piece of f32 queries and of the
//     softmax weights, so both enter the products with twice a 16-bit type's precision at no cost
//     (groups above 8 take a second product): 22 bits (f16; weights times 2^15, so down to weights of 2^-18 of the
//     largest, and below that to 2^-40 of it) or 16 (bf16).  tcgen05 tiles have 128 rows: 120 of them would be empty;
//   * running maximum and sum per warp (f32, base 2); at the end of a sequence's part the warps hand
//     theirs over through shared memory to 4 more warps and go on with their next units, while those join
//     and store them (the copies never pause for it: 64 ragged sequences 181 -> 173 us);
//   * a sequence cut over several SMs leaves partial results (unnormalised sums, maximum, total) in a
//     workspace; the last part to arrive (a counter that it sets back to zero) joins them in order of
//     the parts, so the result does not depend on the order of arrival.
// Rows behind a sequence's end may hold anything: their scores are replaced, their values zeroed.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_cache.cuh"
#include "tc_ptx.cuh"

namespace moe {

namespace {

constexpr int kDWarps = 4;
constexpr int kDThreads = 64 * kDWarps;  // as many again that join
constexpr int kTile = 32;    // tokens per unit
constexpr int kBoxRows = 16; // rows per TMA box
// Fewest units a part is cut down to, 4 for each warp (one request of 500 tokens, 16 units of each of 2 kv
// heads: 10.2 us with 16, 8 or 4, 16.4 us with 32).
constexpr int kMinUnits = 16;

struct DecodeArgs {
    KvBatch b;
    AttnArgs a;
    float* part_o;       // [2 * grid][16][D]
    float2* part_ml;     // [2 * grid][16]
    // arrivals [3][grid] (an item's first 16 parts, later 16s, its 16s), zero between launches
    unsigned int* count;
    int group, head_blocks;  // query heads per kv head; blocks of 8 or 16 of them
    int layer_row;           // first pool row of the layer
};

template <typename C> struct Mma;
template <> struct Mma<__half> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Mma<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Walks the flat unit list: unit -> (sequence, head block, tile).
struct UnitIter {
    int s, hk, tile, nt;
    __device__ __forceinline__ void seek(const int* first, int n_seqs, int hh, int unit) {
        int lo = 0, hi = n_seqs;  // first[lo] * hh <= unit < first[hi] * hh
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] * hh <= unit) lo = mid; else hi = mid;
        }
        s = lo;
        nt = first[s + 1] - first[s];
        const int rem = unit - first[s] * hh;
        hk = rem / nt;
        tile = rem % nt;
    }
    // The caller keeps within the list, so a next non-empty sequence exists when it is needed.
    __device__ __forceinline__ void advance(const int* first, int hh, int by) {
        tile += by;
        while (tile >= nt) {
            tile -= nt;
            if (++hk == hh) {
                hk = 0;
                do { ++s; nt = first[s + 1] - first[s]; } while (nt == 0);
            }
        }
    }
};

template <typename A, typename C, int D, bool WIDE>
__global__ void __launch_bounds__(kDThreads, 1)
attn_decode_kernel(const DecodeArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr bool kSplitQ = sizeof(A) == 4;        // f32 queries: two 16-bit pieces
    constexpr int kTileBytes = kTile * D * 2;
    constexpr int kStages = D == 128 ? 3 : 6;
    constexpr int kBoxBytes = kBoxRows * D * 2;
    constexpr int kKS = D / 16;                     // products per score tile
    constexpr int kNT = D / 8;                      // output tiles
    constexpr int kRows = WIDE ? 16 : 8;
    // Weights e^(s - m) <= 1 enter the products times this.  An f16 piece below 2^-14 has the fewer bits the smaller it is
    // (the last is 2^-24), and beside one key far above the rest all other weights are that small, while the
    // total counts them in full: 8192 keys 18 below one whose value is zero, f32 result off by 9e-3 with weights times 1
    // and by 4e-6 so; 24 below, 1.5e-2 and 1.5e-5 (times unchanged).  O and the totals carry the factor alike and it
    // cancels.  bf16 has f32's range.
    constexpr float kLift = std::is_same<C, __half>::value ? 32768.f : 1.f;

    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* ring = sm;                                                   // [warp][stage]{K tile, V tile}
    float* mo = reinterpret_cast<float*>(ring + kDWarps * kStages * 2 * kTileBytes);  // [warp][8][D]
    float2* mml = reinterpret_cast<float2*>(mo + kDWarps * 8 * D);        // [warp][8] (maximum, total)
    uint64_t* full = reinterpret_cast<uint64_t*>(mml + kDWarps * 8);     // [warp][stage]
    uint64_t* join_full = full + kDWarps * kStages;                       // the warps' results are there / read
    uint64_t* join_free = join_full + 1;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(join_free + 1);
    int* last_flag = const_cast<int*>(abort_flag) + 1;
    int* wsum = last_flag + 1;                                            // [8] scan
    int* first = wsum + 10;                                                // [n_seqs + 1] tiles in front of each sequence

    const KvBatch& b = p.b;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int hh = b.n_kv_heads * p.head_blocks;

    if (tid < kDWarps * kStages) tc::mbar_init(&full[tid], 1);
    if (tid == 0) {
        tc::mbar_init(join_full, kDWarps);
        tc::mbar_init(join_free, kDWarps);
        *abort_flag = 0;
        first[0] = 0;
        tc::tma_prefetch_desc(&kmap);
        tc::tma_prefetch_desc(&vmap);
    }
    tc::fence_mbar_init();
    int carry = 0;
    for (int s0 = 0; s0 < b.n_seqs; s0 += kDThreads) {
        const int s = s0 + tid;
        const int len = s < b.n_seqs ? checked_len(b.lens[s], b, b.status) : 0;
        int x = (len + kTile - 1) / kTile;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        int before = carry;
        for (int i = 0; i < warp; ++i) before += wsum[i];
        if (s < b.n_seqs) first[s + 1] = before + x;
        for (int i = 0; i < kDThreads / 32; ++i) carry += wsum[i];
        __syncthreads();
    }

    // empty sequences: zeros
    A* out = static_cast<A*>(p.a.out);
    const int width = p.a.n_heads * D;
    for (int s = blockIdx.x; s < b.n_seqs; s += gridDim.x)
        if (first[s + 1] == first[s])
            for (int i = tid; i < width; i += kDThreads) out[static_cast<size_t>(s) * p.a.out_stride + i] = from_f32<A>(0.f);

    const long long units = static_cast<long long>(carry) * hh;
    const int parts = static_cast<int>(min(static_cast<long long>(gridDim.x), (units + kMinUnits - 1) / kMinUnits));
    if (static_cast<int>(blockIdx.x) >= parts) return;
    const int u0 = static_cast<int>(units * blockIdx.x / parts), u1 = static_cast<int>(units * (blockIdx.x + 1) / parts);

    // the items (sequence, head block) that the part touches, in order: fn(item, first unit, end unit)
    auto for_items = [&](auto&& fn) {
        UnitIter cur;
        cur.seek(first, b.n_seqs, hh, u0);
        int item_u = first[cur.s] * hh + cur.hk * cur.nt;
        while (item_u < u1) {
            const int end_u = item_u + cur.nt;
            fn(cur, item_u, end_u);
            item_u = end_u;
            if (item_u < u1) {
                cur.tile = cur.nt - 1;
                cur.advance(first, hh, 1);
            }
        }
    };
    auto head_of = [&](const UnitIter& it) { return it.hk / p.head_blocks * p.group + it.hk % p.head_blocks * kRows; };
    auto rows_of = [&](const UnitIter& it) { return min(kRows, p.group - it.hk % p.head_blocks * kRows); };
    constexpr int kR = WIDE ? 2 : 1;  // rows per lane: lane / 4 (and + 8)

    if (warp >= kDWarps) {
        // ---- join: 16 threads per row -------------------------------------------------------------
        const int jt = tid - 32 * kDWarps, k = jt & 15;
        auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kDWarps) : "memory"); };
        int round = 0;
        // arrival at a counter; true in every thread for the last of `of`
        auto last_of = [&](unsigned int* count, int of) {
            meet();
            if (jt == 0) {
                __threadfence();
                *last_flag = atomicAdd(count, 1u) == static_cast<unsigned>(of - 1);
                if (*last_flag) {
                    *count = 0;
                    __threadfence();
                }
            }
            meet();
            return *last_flag != 0;
        };
        for_items([&](const UnitIter& cur, int item_u, int end_u) {
            const int head0 = head_of(cur), n_rows = rows_of(cur);
            const bool whole = item_u >= u0 && end_u <= u1;
            const int slot = 2 * blockIdx.x + (item_u < u0 ? 0 : 1);
            A* to = out + static_cast<size_t>(cur.s) * p.a.out_stride + static_cast<size_t>(head0) * D + k * 4;
            for (int r = 0; r < kR; ++r, ++round) {  // rows 0-7, then 8-15
                const int jr = jt >> 4, row = 8 * r + jr;
                if (tc::mbar_wait_warp(join_full, round & 1, abort_flag) && row < n_rows) {
                    float2 ml[kDWarps];
                    float mx = -INFINITY, tot = 0.f, f[kDWarps];
#pragma unroll
                    for (int w = 0; w < kDWarps; ++w) {
                        ml[w] = mml[w * 8 + jr];
                        mx = fmaxf(mx, ml[w].x);
                    }
                    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
                    for (int w = 0; w < kDWarps; ++w) {
                        f[w] = ex2(ml[w].x - base);
                        tot = fmaf(ml[w].y, f[w], tot);
                    }
#pragma unroll
                    for (int d = 0; d < D; d += 64) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < kDWarps; ++w) {
                            const float4 x = *reinterpret_cast<const float4*>(mo + (w * 8 + jr) * D + k * 4 + d);
                            v.x = fmaf(x.x, f[w], v.x); v.y = fmaf(x.y, f[w], v.y);
                            v.z = fmaf(x.z, f[w], v.z); v.w = fmaf(x.w, f[w], v.w);
                        }
                        if (whole) store4(to + row * D + d, v, 1.f / tot);
                        else *reinterpret_cast<float4*>(p.part_o + (static_cast<size_t>(slot) * 16 + row) * D + k * 4 + d) = v;
                    }
                    if (!whole && k == 0) p.part_ml[slot * 16 + row] = make_float2(mx, tot);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(join_free);
            }
            if (whole) return;
            // The item's parts c0 .. c1 are joined 16 at a time, and then the 16s: one block would read all
            // of a long sequence's parts in 7 us.  What the parts c, c + step, ... (n of them) left goes to
            // `out` or, unnormalised, to the slot of part c.
            const int c0 = static_cast<int>(((item_u + 1ll) * parts - 1) / units), c1 = static_cast<int>((static_cast<long long>(end_u) * parts - 1) / units);
            auto slot_of = [&](int c, int row) { return static_cast<size_t>(2 * c + (c == c0 ? 1 : 0)) * 16 + row; };
            auto join = [&](int c, int step, int n, bool final) {
                for (int row = jt >> 4; row < kRows; row += 8) {
                    float m_all = -INFINITY, tot = 0.f;
                    float4 v[D / 64];
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    const bool there = row < n_rows;
                    for (int i0 = 0; i0 < n; i0 += 16) {
                        // thread k has the weight of the k-th part, and all their sums are loaded at once
                        const float2 ml = there && i0 + k < n ? __ldcg(&p.part_ml[slot_of(c + (i0 + k) * step, row)]) : make_float2(-INFINITY, 0.f);
                        float4 x[16][D / 64];
#pragma unroll
                        for (int i = 0; i < 16; ++i)
#pragma unroll
                            for (int d = 0; d < D / 64; ++d)
                                x[i][d] = there && i0 + i < n
                                              ? __ldcg(reinterpret_cast<const float4*>(p.part_o + slot_of(c + (i0 + i) * step, row) * D + k * 4 + 64 * d))
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
                        float mx = fmaxf(m_all, ml.x);
#pragma unroll
                        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const float base = mx == -INFINITY ? 0.f : mx, before = ex2(m_all - base), f = ex2(ml.x - base);
                        m_all = mx;
                        float sum = ml.y * f;
#pragma unroll
                        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        tot = fmaf(tot, before, sum);
#pragma unroll
                        for (int d = 0; d < D / 64; ++d) { v[d].x *= before; v[d].y *= before; v[d].z *= before; v[d].w *= before; }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float fi = __shfl_sync(0xffffffffu, f, (lane & 16) | i);
#pragma unroll
                            for (int d = 0; d < D / 64; ++d) {
                                v[d].x = fmaf(x[i][d].x, fi, v[d].x); v[d].y = fmaf(x[i][d].y, fi, v[d].y);
                                v[d].z = fmaf(x[i][d].z, fi, v[d].z); v[d].w = fmaf(x[i][d].w, fi, v[d].w);
                            }
                        }
                    }
                    if (!there) continue;
#pragma unroll
                    for (int d = 0; d < D / 64; ++d) {
                        if (final) store4(to + row * D + 64 * d, v[d], 1.f / tot);
                        else *reinterpret_cast<float4*>(p.part_o + slot_of(c, row) * D + k * 4 + 64 * d) = v[d];
                    }
                    if (!final) {
                        __syncwarp(0xffffu << (lane & 16));
                        if (k == 0) p.part_ml[slot_of(c, row)] = make_float2(m_all, tot);
                    }
                }
            };
            const int n = c1 - c0 + 1, mine = (static_cast<int>(blockIdx.x) - c0) / 16, c = c0 + 16 * mine, groups = (n + 15) / 16;
            if (!last_of(&p.count[mine == 0 ? c0 : gridDim.x + c], min(16, n - 16 * mine))) return;
            join(c, 1, min(16, n - 16 * mine), groups == 1);
            if (groups > 1 && last_of(&p.count[2 * gridDim.x + c0], groups)) join(c0, 16, groups, true);
            meet();
        });
        return;
    }

    uint8_t* my_ring = ring + warp * kStages * 2 * kTileBytes;
    uint64_t* my_full = full + warp * kStages;
    const int my_units = u1 - u0 > warp ? (u1 - u0 - warp + kDWarps - 1) / kDWarps : 0;

    // Copies of one unit's tile: box i (16 tokens) by lane i, keys and values.
    auto copy_box = [&](int slot, int box, int tile, int hk, int page) {
        uint8_t* dst = my_ring + slot * 2 * kTileBytes + box * kBoxBytes;
        const int row = p.layer_row + (static_cast<int>(checked_page(page, b.n_pages, b.status)) * b.n_kv_heads + hk / p.head_blocks) * b.page_size +
                        (tile * kTile + box * kBoxRows) % b.page_size;
        tc::tma_load_3d(dst, &kmap, 0, row, 0, &my_full[slot]);
        tc::tma_load_3d(dst + kTileBytes, &vmap, 0, row, 0, &my_full[slot]);
    };
    auto boxes_of = [&](int len, int tile) { return (min(kTile, len - tile * kTile) + kBoxRows - 1) / kBoxRows; };
    auto len_of = [&](int s) { return min(b.lens[s], b.max_pages * b.page_size); };  // a wrong one was reported above
    auto page_of = [&](int s, int tile, int box) {
        const int pg = (tile * kTile + box * kBoxRows) / b.page_size;
        return pg < b.max_pages ? b.table[static_cast<size_t>(s) * b.max_pages + pg] : 0;
    };
    UnitIter ahead;
    int issued = 0, ahead_len = 0, ahead_page = 0;
    if (my_units > 0) {
        // the ring's first units together: lane 2 i + box looks up and copies a box of unit i
        ahead.seek(first, b.n_seqs, hh, u0 + warp);
        UnitIter mine = ahead;
        for (issued = 0; issued < min(my_units, kStages);) {
            if (lane >> 1 == issued) mine = ahead;
            if (++issued < my_units) ahead.advance(first, hh, kDWarps);
        }
        const int n = issued, slot = lane >> 1, box = lane & 1;
        const int len = slot < n ? len_of(mine.s) : 0, page = slot < n ? page_of(mine.s, mine.tile, box) : 0;
        const int boxes = boxes_of(len, mine.tile);
        if (slot < n && box == 0) tc::mbar_arrive_expect_tx(&my_full[slot], static_cast<uint32_t>(2 * boxes * kBoxBytes));
        __syncwarp();
        if (slot < n && box < boxes) copy_box(slot, box, mine.tile, mine.hk, page);
        if (issued < my_units) {
            ahead_len = len_of(ahead.s);
            ahead_page = page_of(ahead.s, ahead.tile, lane & 1);
        }
    }
    auto issue = [&]() {  // the next unit into the slot just read; its page numbers are here already
        const int slot = issued % kStages, boxes = boxes_of(ahead_len, ahead.tile);
        if (lane == 0) tc::mbar_arrive_expect_tx(&my_full[slot], static_cast<uint32_t>(2 * boxes * kBoxBytes));
        __syncwarp();
        if (lane < boxes) copy_box(slot, lane, ahead.tile, ahead.hk, ahead_page);
        if (++issued < my_units) {
            const int s = ahead.s;
            ahead.advance(first, hh, kDWarps);
            if (ahead.s != s) ahead_len = len_of(ahead.s);
            ahead_page = page_of(ahead.s, ahead.tile, lane & 1);
        }
    };

    // byte offset of (row r of the lane's 8-row group, 16-byte chunk) inside a box: the swizzle
    // exchanges chunks by the row's low 3 bits
    const int lr = lane & 7;
    auto chunk_off = [&](int c) { return static_cast<uint32_t>((c >> 3) * (kBoxRows * 128) + lr * 128 + (((c & 7) ^ lr) << 4)); };

    int done = 0, round = 0;  // units this warp has finished; results handed over
    for_items([&](const UnitIter& cur, int item_u, int end_u) {
        const int ja = max(item_u, u0) - u0, jb = min(end_u, u1) - u0;
        const int len = len_of(cur.s), head0 = head_of(cur), n_rows = rows_of(cur);

        float o[kNT / 2][2][4];
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n / 2][n % 2][i] = 0.f;
        float m[kR], l[kR], sl[kR];
#pragma unroll
        for (int r = 0; r < kR; ++r) { m[r] = -INFINITY; l[r] = 0.f; sl[r] = p.a.scale * 1.4426950408889634f; }

        int j = ja + ((warp - ja) & (kDWarps - 1));
        if (j < jb) {
            // query fragments (rows behind the group are zero)
            uint32_t qa[kKS][4], qb[WIDE && kSplitQ ? kKS : 1][4];
            float qf[kR][kKS][4];
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                const int row = (lane >> 2) + 8 * r;
                const A* q = static_cast<const A*>(p.a.q) + static_cast<size_t>(cur.s) * p.a.q_stride +
                             static_cast<size_t>(head0 + row) * D + (lane & 3) * 2;
#pragma unroll
                for (int k = 0; k < kKS; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[r][k][i] = row < n_rows ? to_f32(q[16 * k + 8 * (i >> 1) + (i & 1)]) : 0.f;
                if constexpr (kSplitQ) {
                    if constexpr (std::is_same<C, __half>::value) {
                        // f16 pieces: the row's largest magnitude goes to [2^14, 2^15), undone in its score scale
                        float mx = 0.f;
#pragma unroll
                        for (int k = 0; k < kKS; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(qf[r][k][i]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const int e = row_exponent(mx);
                        sl[r] *= pow2(-e);
                        const float up = pow2(e);
#pragma unroll
                        for (int k = 0; k < kKS; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) qf[r][k][i] *= up;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kKS; ++k) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    qa[k][2 * h] = pack2<C>(qf[0][k][2 * h], qf[0][k][2 * h + 1]);
                    if constexpr (!WIDE) {
                        qa[k][2 * h + 1] = kSplitQ ? pack_rest<C>(qa[k][2 * h], qf[0][k][2 * h], qf[0][k][2 * h + 1]) : 0u;
                    } else {
                        qa[k][2 * h + 1] = pack2<C>(qf[kR - 1][k][2 * h], qf[kR - 1][k][2 * h + 1]);
                        if constexpr (kSplitQ) {
                            qb[k][2 * h] = pack_rest<C>(qa[k][2 * h], qf[0][k][2 * h], qf[0][k][2 * h + 1]);
                            qb[k][2 * h + 1] = pack_rest<C>(qa[k][2 * h + 1], qf[kR - 1][k][2 * h], qf[kR - 1][k][2 * h + 1]);
                        }
                    }
                }
            }
            for (; j < jb; j += kDWarps) {
                const int slot = done % kStages;
                if (!tc::mbar_wait_warp(&my_full[slot], (done / kStages) & 1, abort_flag)) break;
                const uint32_t kt = tc::smem_u32(my_ring + slot * 2 * kTileBytes), vt = kt + kTileBytes;
                const int t0 = (u0 + j - item_u) * kTile;  // the tile's first token
                const bool tail = t0 + kTile > len;
                if (tail) {
                    // values behind the end: zero (a weight of 0 times what lies there could be NaN)
                    uint8_t* v = my_ring + slot * 2 * kTileBytes + kTileBytes;
                    for (int i = lane; i < kTile * (D / 8); i += 32) {
                        const int row = i / (D / 8), c = i % (D / 8);
                        if (t0 + row >= len)
                            *reinterpret_cast<uint4*>(v + (row / kBoxRows) * kBoxBytes + (c >> 3) * (kBoxRows * 128) +
                                                      (row % kBoxRows) * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();  // ordered before the copy that reuses the slot
                    __syncwarp();
                }
                float s[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
#pragma unroll
                for (int c = 0; c < kKS / 2; ++c) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        uint32_t kb[4];
                        ldsm4(kb, kt + (t >> 1) * kBoxBytes + (t & 1) * 1024 + chunk_off(4 * c + (lane >> 3)));
                        Mma<C>::run(s[t], qa[2 * c], kb[0], kb[1]);
                        Mma<C>::run(s[t], qa[2 * c + 1], kb[2], kb[3]);
                        if constexpr (WIDE && kSplitQ) {
                            Mma<C>::run(s[t], qb[2 * c], kb[0], kb[1]);
                            Mma<C>::run(s[t], qb[2 * c + 1], kb[2], kb[3]);
                        }
                    }
                }
                // scores of row lane / 4 (+ 8 r), tokens t0 + 8 t + 2 (lane % 4) + {0, 1}
                float z[kR][8];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const bool seen = !tail || t0 + 8 * t + 2 * (lane & 3) + i < len;
                        if constexpr (WIDE) {
                            z[0][2 * t + i] = seen ? s[t][i] : -INFINITY;
                            z[kR - 1][2 * t + i] = seen ? s[t][2 + i] : -INFINITY;
                        } else {
                            z[0][2 * t + i] = seen ? (kSplitQ ? s[t][i] + s[t][2 + i] : s[t][i]) : -INFINITY;
                        }
                    }
                float alpha[kR];
#pragma unroll
                for (int r = 0; r < kR; ++r) {
                    float mx = z[r][0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, z[r][i]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[r], __fmul_rn(mx, sl[r]));
                    const float base = mn == -INFINITY ? 0.f : mn;
                    alpha[r] = ex2(m[r] - base);
                    m[r] = mn;
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // the product rounded as the maximum's was: what is left of the largest is 0 at any size
                        z[r][i] = ex2(__fsub_rn(__fmul_rn(z[r][i], sl[r]), base)) * kLift;
                        sum += z[r][i];
                    }
                    l[r] = fmaf(l[r], alpha[r], sum);
                }
                if (!kSplitQ && __any_sync(0xffffffffu, alpha[0] != 1.f || alpha[kR - 1] != 1.f)) {
#pragma unroll
                    for (int n = 0; n < kNT; ++n) {
                        float (&x)[4] = o[n / 2][n % 2];
                        x[0] *= alpha[0]; x[1] *= alpha[0];
                        x[2] *= alpha[kR - 1]; x[3] *= alpha[kR - 1];
                    }
                }
                // weights as two 16-bit pieces
                uint32_t pa[2][4], pb[WIDE ? 2 : 1][4];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int i = 4 * k + 2 * h;
                        pa[k][2 * h] = pack2<C>(z[0][i], z[0][i + 1]);
                        const uint32_t rest = pack_rest<C>(pa[k][2 * h], z[0][i], z[0][i + 1]);
                        if constexpr (WIDE) {
                            pa[k][2 * h + 1] = pack2<C>(z[kR - 1][i], z[kR - 1][i + 1]);
                            pb[k][2 * h] = rest;
                            pb[k][2 * h + 1] = pack_rest<C>(pa[k][2 * h + 1], z[kR - 1][i], z[kR - 1][i + 1]);
                        } else {
                            pa[k][2 * h + 1] = rest;
                        }
                    }
                // For f32 results a tile's products are summed apart and added to the rest by rounded additions: the
                // tensor core cuts off its sums, and over many tiles that shows (262144 tokens: error 1.4e-6 with
                // one sum, 5.9e-7 so; the time is the same).
                auto product = [&](float (&to)[2][4], int k, int n) {
                    uint32_t vb[4];
                    ldsm4t(vb, vt + k * kBoxBytes + ((lane >> 3) & 1) * 1024 + chunk_off(n + (lane >> 4)));
                    Mma<C>::run(to[0], pa[k], vb[0], vb[1]);
                    Mma<C>::run(to[1], pa[k], vb[2], vb[3]);
                    if constexpr (WIDE) {
                        Mma<C>::run(to[0], pb[k], vb[0], vb[1]);
                        Mma<C>::run(to[1], pb[k], vb[2], vb[3]);
                    }
                };
                if constexpr (kSplitQ) {
#pragma unroll
                    for (int n = 0; n < kNT; n += 2) {
                        float sum[2][4] = {};
                        product(sum, 0, n);
                        product(sum, 1, n);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[n / 2][h][i] = fmaf(o[n / 2][h][i], alpha[i < 2 ? 0 : kR - 1], sum[h][i]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int n = 0; n < kNT; n += 2) product(o[n / 2], k, n);
                }
                ++done;
                __syncwarp();  // every lane has read the slot
                if (issued < my_units) issue();
            }
        }

        // hand over: rows 0-7, then 8-15
#pragma unroll
        for (int r = 0; r < kR; ++r, ++round) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            tc::mbar_wait_warp(join_free, (round & 1) ^ 1, abort_flag);
            const int g = lane >> 2;
            if ((lane & 3) == 0) mml[warp * 8 + g] = make_float2(m[r], l[r]);
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
                const float (&x)[4] = o[n / 2][n % 2];
                const float2 v = WIDE ? make_float2(x[2 * r], x[2 * r + 1]) : make_float2(x[0] + x[2], x[1] + x[3]);
                *reinterpret_cast<float2*>(mo + (warp * 8 + g) * D + 8 * n + 2 * (lane & 3)) = v;
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(join_full);
        }
    });
    if (*abort_flag) {
        if (lane == 0) set_dev_error(b.status, kDevTimeout);
        // copies still in flight land before the block's shared memory goes away
        int alone = 0;
        for (int i = done; i < issued; ++i) tc::mbar_wait(&my_full[i % kStages], (i / kStages) & 1, &alone, 100000000ull);
    }
}

template <typename A, typename C, int D, bool WIDE>
void launch_t(const DecodeArgs& p, const CUtensorMap& k, const CUtensorMap& v, int grid, cudaStream_t s) {
    constexpr int kStages = D == 128 ? 3 : 6;
    const size_t smem = kDWarps * kStages * 2 * kTile * D * 2 + kDWarps * 8 * D * 4 + kDWarps * 8 * 8 + (kDWarps * kStages + 2) * 8 + 48 +
                        (static_cast<size_t>(p.b.n_seqs) + 1) * 4;
    static std::atomic<uint64_t> set{0};  // devices whose limit is raised
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(set.load() >> dev & 1)) {
        cudaFuncSetAttribute(attn_decode_kernel<A, C, D, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (dev < 64) set.fetch_or(1ull << dev);
    }
    attn_decode_kernel<A, C, D, WIDE><<<grid, kDThreads, smem, s>>>(p, k, v);
}

template <typename A, typename C>
void launch_d(const DecodeArgs& p, const CUtensorMap& k, const CUtensorMap& v, int grid, cudaStream_t s) {
    const bool wide = p.group > 8;
    if (p.b.head_dim == 64) {
        if (wide) launch_t<A, C, 64, true>(p, k, v, grid, s); else launch_t<A, C, 64, false>(p, k, v, grid, s);
    } else {
        if (wide) launch_t<A, C, 128, true>(p, k, v, grid, s); else launch_t<A, C, 128, false>(p, k, v, grid, s);
    }
}

}  // namespace

// part_o [2 * sm_count][16][128] f32, part_ml [2 * sm_count][16] float2, counters [3 * sm_count]
size_t attn_decode_ws_bytes(int sm_count) { return static_cast<size_t>(sm_count) * (2 * 16 * (128 * 4 + 8) + 12); }

void launch_attn_decode(const KvBatch& b, int act, const KvCache& kv, uint32_t layer, const AttnArgs& a, uint8_t* ws, int sm_count,
                        cudaStream_t s) {
    DecodeArgs p{};
    p.b = b;
    p.a = a;
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + static_cast<size_t>(sm_count) * 2 * 16 * 128 * 4);
    p.count = reinterpret_cast<unsigned int*>(ws + static_cast<size_t>(sm_count) * 2 * 16 * (128 * 4 + 8));
    p.group = a.n_heads / b.n_kv_heads;
    p.head_blocks = p.group > 8 ? (p.group + 15) / 16 : 1;
    p.layer_row = static_cast<int>(static_cast<uint64_t>(layer) * kv.spec.n_pages * kv.spec.n_kv_heads * kv.spec.page_size);
    // at most as many parts as the longest possible batch can be cut into
    const long long most = (static_cast<long long>(b.max_pages) * b.page_size + kTile - 1) / kTile * b.n_seqs * b.n_kv_heads * p.head_blocks;
    const int grid = static_cast<int>(std::max(1ll, std::min<long long>(sm_count, (most + kMinUnits - 1) / kMinUnits)));
    const CUtensorMap &k = kv.maps[0], &v = kv.maps[1];
    if (act == MOE_T_F32) {
        if (kv.spec.type == MOE_T_F16) launch_d<float, __half>(p, k, v, grid, s);
        else launch_d<float, __nv_bfloat16>(p, k, v, grid, s);
    } else if (act == MOE_T_F16) {
        launch_d<__half, __half>(p, k, v, grid, s);
    } else {
        launch_d<__nv_bfloat16, __nv_bfloat16>(p, k, v, grid, s);
    }
}

}  // namespace moe
