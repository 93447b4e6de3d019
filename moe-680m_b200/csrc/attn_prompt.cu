// Causal attention of packed prompt tokens over the paged cache (moe_attn_prompt; moe-680m:
// shaders/attention.comp, src/inference.rs:484-555, one sequence).
//
// 4 * D flops per (query row, visible key) against K and V tiles that many rows share: the work is
// matrix products, S = Q K^T and O += P V, with a softmax between them, on the tensor cores
// (tcgen05).  Layout of the work:
//   * a query row is one (token, head); the rows of a sequence's tokens and of the group's heads are
//     numbered together, so any group size fills the 128 rows of a tile and all of a group's heads
//     share the K and V tiles.  A CTA takes two such row tiles (256 rows; one with f32 queries of 128
//     columns) of one (sequence, kv head) and goes over the key tiles of 128 tokens that its last row sees, units with the most keys first;
//   * warp roles: 8 warps for the softmax (each thread a row, or two threads a row of a single tile), 2 that
//     issue products, one that loads K and V tiles by TMA, page by page, into a ring; the others look
//     over the V tiles at the causal edge;
//   * TMEM (512 columns): S of four steps of 64 keys (two for each of two tiles; one with 16-bit queries of 64
//     columns, whose CTAs have half the columns), O, and with f32 queries a
//     second O that takes O's sum every 8 steps.  The weights P go back over S as 16-bit values and are the
//     A operand of O += P V straight from TMEM; V is read as it lies in the page (MN-major), so nothing
//     is transposed.  While one step's softmax runs, the tensor core works on another's products;
//   * f32 queries enter as two 16-bit pieces (row scaled by a power of two for f16), and so do their
//     weights: twice the products, 22-bit (bf16: 16-bit) precision, for weights below 2^-16 of a row's largest
//     (f16) to 2^-38 of that; 16-bit queries' weights are one piece of their type;
//   * O is rescaled only when a row's maximum has grown by more than 2^8 (bf16) or 2^2 to 2^4 (f16, whose weights
//     are lifted towards the type's largest value) since the last time: until then its weights are that much above
//     1, which the 16-bit types and the f32 sums hold as exactly.
// A key that a row does not see must not touch it whatever it holds.  Scores are replaced, but a weight of 0 times
// an infinite or NaN value would be NaN; so in the tiles at the causal edge two warps put 0 in the place
// of such values (and of all rows behind the sequence's end) before the product, keep for each
// column the first key that had one, and the rows that do see it get NaN at the end.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_cache.cuh"
#include "tc_ptx.cuh"

namespace moe {

namespace {

constexpr int kRowTile = 128;
constexpr int kKeyTile = 128;  // keys of a K or V tile in shared memory
constexpr int kStep = 64;      // keys of a softmax step: two steps' S per row tile lie in TMEM
// Warps of a CTA with kTiles row tiles: 8 for the softmax (4 per tile, or two threads to each row of a single
// tile), 2 that issue products (one per tile; of a single tile one for S, one for O), a loading warp,
// 2 edge warps per tile (and one that fills the last warpgroup of two tiles).
template <int kTiles, bool kSlim> struct Roles {
    static constexpr int kMma = 8, kLoad = 10, kEdge = 11, kEdges = kSlim ? 1 : 2 * kTiles;
    static constexpr int kThreads = kSlim ? 384 : kTiles == 2 ? 512 : 416;
};
// Registers with two tiles: 512 threads * 128 at launch = 256 * 184 + 256 * 72.
constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;
// With f32 queries, steps that O is summed over by the tensor core before it is added to a second O: its
// sums are cut off, not rounded, at each of the products' additions (8192 keys, error of the output
// against 64 bits: 6.2e-6 in one O, 1.9e-6 in parts of 16 steps, 1.2e-6 of 8; the time is the same).
constexpr int kPart = 8;
// Log2 of how far a row's maximum may grow before O is rescaled, and of a factor that the weights have on their way into
// the products (O and the row's total carry it alike: it cancels).  An f16 piece below 2^-14 has the fewer bits the
// smaller it is (the last is 2^-24), and beside one key far above the rest all other weights are that small.
// Both together keep below f16's largest value, 2^15 in all.  8192 keys below one whose value is zero, error of an f32 result
// and time of 8192 tokens:   factor 2^0    2^7     2^11    2^13    2^14
//   18 below                  2.5e-1   5.2e-5  4.4e-6  3.8e-6  3.7e-6
//   20 below                  8.7e-1   5.8e-4  2.2e-5  6.5e-6  5.0e-6
//   f32 queries, D = 128      528 us   532     545     578     603
//   f16 queries, D = 64       133 us   134     135     139     143     (packed ragged prompts)
// (An operation more for each weight, where they are computed, has since made them 583 and 139.)  f16 results have 11
// bits and gain nothing from more than 2^11 (20 below: 4.7e-4 with 2^11 and 2^14).  bf16 has f32's range.
template <typename A, typename C> constexpr float kLift = std::is_same<C, __half>::value ? sizeof(A) == 4 ? 13.f : 11.f : 0.f;
template <typename A, typename C> constexpr float kRescaleAt = std::is_same<C, __half>::value ? 15.f - kLift<A, C> : 8.f;
struct PromptArgs {
    KvBatch b;
    AttnArgs a;
    int group;
    uint64_t group_inv;  // ceil(2^64 / group): row / group is the high half of row * group_inv (0: group 1)
    int unit_rows;       // rows of a CTA: two tiles, or one where that leaves at least half of the SMs idle
    int layer_row;
    int box_rows;  // rows per TMA box: page_size
    float zero;    // 0
};

struct Shared {  // behind Q and the ring
    uint64_t kv_full[8], kv_empty[8];
    // V tiles at the causal edge (256 rows see at most 3 in part): loaded, looked over.  Single use: the
    // edge warps join in the middle of the ring's phases, which a parity wait on kv_full could not tell apart
    uint64_t edge_full[4], edge_done[4];
    uint64_t q_full, s_full[4], p_full[4], o_full[2], drained[2];  // [row tile * kSBufs + step % kSBufs]
    uint64_t o_step[4];                                            // one row tile: O is up to this step
    uint32_t tmem;
    int abort_flag;
    int seq, unit, first_token, n_new;  // the unit found for this block; seq -1: none
    int bad;                            // some V value at the edge was replaced
    int wsum[16];
    float row[2][2][128];               // two threads to a row: what each tells the other,
    uint64_t meet[4];                   // and where they meet
    int bad_key[128];                   // per column: first key whose value was
};

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 2^x for x <= 16 on the FMA pipes: x = n + f, |f| <= 1/2 (rounding by adding 1.5 * 2^23, whose low bits then
// hold n), 2^f = 1 + f p(f) with p the degree-4 interpolation of (2^f - 1) / f at the Chebyshev
// points of [-1/2, 1/2] (relative error 2.6e-7), times 2^n as a float of its own bits, so that a NaN stays one.
// x <= -127 gives exactly 0 (2^n is 0 there).  One weight of 16
// goes this way with 16-bit queries, whose products take no longer than the special-function unit takes
// for all weights (8192 tokens, bf16: none 259 us, 1 of 16 242 us, 2 of 16 257 us); with f32 queries the
// products take twice as long and none does.
__device__ __forceinline__ float ex2_poly(float x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x));  // -127
    const float r = __fadd_rn(x, 12582912.f);
    const float f = __fsub_rn(x, __fadd_rn(r, -12582912.f));
    float p = fmaf(f, 0.0013381302f, 0.0096663684f);
    p = fmaf(p, f, 0.055503812f);
    p = fmaf(p, f, 0.2402235f);
    p = fmaf(p, f, 0.69314718f);
    p = fmaf(p, f, 1.f);
    return p * __int_as_float((__float_as_int(r) << 23) + 0x3F800000);
}

template <typename C> __host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
    return tc::idesc_f16(128, n) | (std::is_same<C, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u);
}

// kv_full waits etc. of whole warps
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Shared* sh) {
    return tc::mbar_wait_warp(bar, parity, &sh->abort_flag);
}

// f32 queries of 128 columns take one row tile per CTA: with two, TMEM has no room for a second O (8192
// tokens, weights not lifted: 455 us so, with an error of 6.2e-6; 521 us and 1.2e-6 with one).
template <typename A, int D> constexpr int kTilesOf = sizeof(A) == 4 && D == 128 ? 1 : 2;
// 16-bit queries of 64 columns: their CTAs take half of an SM's TMEM, registers and shared memory, so two run at
// once, with one place for S to each tile (9 ragged prompts up to 2500 tokens, 7 heads to a kv head, weights not
// lifted: 147 us as one CTA with two places, 132 so).
template <typename A, int D> constexpr bool kSlimOf = sizeof(A) == 2 && D == 64;
template <typename A, int D> constexpr int kBufsOf = kSlimOf<A, D> ? 4 : D == 64 ? 8 : 5;

template <typename A, typename C, int D>
__global__ void __launch_bounds__(Roles<kTilesOf<A, D>, kSlimOf<A, D>>::kThreads, kSlimOf<A, D> ? 2 : 1)
attn_prompt_kernel(const PromptArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr bool kSplit = sizeof(A) == 4;
    constexpr int kPieces = kSplit ? 2 : 1;
    constexpr int kHalves = D / 64;
    constexpr uint32_t kHalfBytes = 128 * 128;              // 128 rows x 64 values
    constexpr uint32_t kTileBytes = kHalves * kHalfBytes;   // a Q piece, K or V tile
    constexpr int kTiles = kTilesOf<A, D>, kBufs = kBufsOf<A, D>;
    constexpr bool kSlim = kSlimOf<A, D>;
    using R = Roles<kTiles, kSlim>;
    constexpr int kMmaWarp = R::kMma, kLoadWarp = R::kLoad, kEdgeWarp = R::kEdge, kThreads = R::kThreads;
    constexpr int kPer = 2 / kTiles;  // threads of a row
    // TMEM: S of the tiles' steps (256 columns), then each tile's O (and second O)
    constexpr int kSBufs = kSlim ? 1 : 4 / kTiles;  // S of this many steps per tile
    // Keys of an S product.  64 hold the tensor core for longer than they compute (they read 6 KB of shared memory,
    // 48 clocks, for 32 of arithmetic; 8192 tokens, bf16: 80 % busy, 66 % computing), but 128 need both steps' places at
    // once, and with two tiles nothing is then ahead of the softmax (250 us with 64, 282 with 128).  A single tile has
    // four places, so S of two steps goes at once, and two threads take a row, one for each step (8192
    // tokens, f32, weights not lifted: 527 us with a step at a time and a thread a row, 521 so; 37 tokens: 13.8 and 12.3).
    constexpr int kSKeys = kTiles == 2 ? kStep : 2 * kStep;
    constexpr uint32_t kOCol = kTiles * kSBufs * kStep, kOCols = kSplit ? 2 * D : kSlim ? D : 128, kTmemCols = kSlim ? 256 : 512;
    constexpr uint32_t kPCol = kSlim ? kStep / 2 : 0;  // P lies this far into S
    constexpr bool kHalfType = std::is_same<C, __half>::value;

    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* qs = sm;                                        // [tile][piece]
    uint8_t* ring = sm + kTiles * kPieces * kTileBytes;      // K0 V0 K1 V1 ... round kBufs buffers
    Shared* sh = reinterpret_cast<Shared*>(ring + kBufs * kTileBytes);
    const KvBatch& b = p.b;
    // the warp number from lane 0: the compiler then takes the roles' branches as warp-uniform
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int kvh = blockIdx.x % b.n_kv_heads, target = blockIdx.x / b.n_kv_heads;

    // ---- setup, and the block's unit ----------------------------------------------------------------
    if (warp == kLoadWarp && lane == 0) {
        for (int i = 0; i < kBufs; ++i) {
            tc::mbar_init(&sh->kv_full[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            tc::mbar_init(&sh->edge_full[i], 1);
            tc::mbar_init(&sh->edge_done[i], R::kEdges);
        }
        tc::mbar_init(&sh->q_full, 8);
        for (int i = 0; i < 4; ++i) {
            tc::mbar_init(&sh->s_full[i], 1);
            tc::mbar_init(&sh->p_full[i], 4);
            tc::mbar_init(&sh->meet[i], 2);
            tc::mbar_init(&sh->o_step[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            tc::mbar_init(&sh->o_full[t], 1);
            tc::mbar_init(&sh->drained[t], 1);
        }
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&kmap);
        tc::tma_prefetch_desc(&vmap);
    }
    if (tid == 0) {
        sh->seq = -1;
        sh->abort_flag = 0;
        sh->bad = 0;
    }
    if (tid < 128) sh->bad_key[tid] = 0x7FFFFFFF;
    // from lane 0, so that the compiler takes what follows (descriptors, trip counts) as warp-uniform
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    // a sequence's packed tokens; wrong offsets are reported and count as none
    auto tokens_of = [&](int s, int* t0) {
        *t0 = b.cu ? b.cu[s] : s;
        const int end = b.cu ? b.cu[s + 1] : s + 1;
        if (right_offsets(*t0, end, p.a.T)) return end - *t0;
        set_dev_error(b.status, kDevBadToken);
        return 0;
    };
    auto scan = [&](int x) {  // inclusive, over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += z;
        }
        return x;
    };
    const int unit_shift = p.unit_rows == 2 * kRowTile ? 8 : 7;
    auto count_units = [&](int n) { return static_cast<int>((static_cast<long long>(n) * p.group + p.unit_rows - 1) >> unit_shift); };
    int seq, unit, n_new, first_token, len;
    if (b.n_seqs <= 32) {
        // A sequence per lane, every warp for itself: the target-th unit in order of key tiles, most first, so that
        // the last CTAs are the shortest of the whole batch (f16, 64 columns, 7 heads to a kv head: 9 prompts up to 2500
        // tokens 129 us, in batch order 137; 32 up to 1000 111 and 119; f32, 128 columns, 8 heads to each of 2 kv
        // heads: 32 up to 1000 211 both ways, 32 up to 300 78 and 72).  Larger batches are taken in their own
        // order: CTAs are many enough (64 up to 1000 tokens: 213 us and 420, twice the 32's).
        int t0 = 0, n = 0, l = 0;
        if (lane < b.n_seqs) {
            l = checked_len(b.lens[lane], b, b.status);
            n = tokens_of(lane, &t0);
        }
        const int x = count_units(n);
        auto at_least = [&](int tiles) {  // the lane's units with that many key tiles: its last ones
            const long long hidden = 128ll * (tiles - 1) - (l - n);  // token positions that see less
            if (tiles == 0 || hidden <= 0) return x;
            const long long r = hidden * p.group;
            return r < static_cast<long long>(n) * p.group ? x - static_cast<int>(r >> unit_shift) : 0;
        };
        if (target >= __reduce_add_sync(0xffffffffu, x)) return;
        int lo = 0, hi = __reduce_max_sync(0xffffffffu, (l + kKeyTile - 1) / kKeyTile) + 1;
        while (hi - lo > 1) {  // more than target units have lo tiles, no more than target have hi
            const int mid = (lo + hi) >> 1;
            if (__reduce_add_sync(0xffffffffu, at_least(mid)) > target) lo = mid; else hi = mid;
        }
        const int more = at_least(hi), same = at_least(lo) - more, left = target - __reduce_add_sync(0xffffffffu, more), y = scan(same);
        const int from = __ffs(__ballot_sync(0xffffffffu, left < y)) - 1;
        auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
        seq = from;
        unit = of(x - more - 1 - (left - (y - same)));
        n_new = of(n);
        first_token = of(t0);
        len = of(l);
    } else {
        int carry = 0;
        for (int s0 = 0; s0 < b.n_seqs; s0 += kThreads) {
            const int s = s0 + tid;
            int t0 = 0;
            const int n = s < b.n_seqs ? tokens_of(s, &t0) : 0, x = count_units(n), y = scan(x);
            if (lane == 31) sh->wsum[warp] = y;
            __syncthreads();
            int before = carry + y - x;
            for (int i = 0; i < warp; ++i) before += sh->wsum[i];
            for (int i = 0; i < kThreads / 32; ++i) carry += sh->wsum[i];
            if (target >= before && target < before + x) {  // a sequence's units from its end
                sh->seq = s;
                sh->unit = x - 1 - (target - before);
                sh->first_token = t0;
                sh->n_new = n;
            }
            __syncthreads();
            if (target < carry && target > 0) break;  // the first unit's blocks look over all offsets
        }
        if (sh->seq < 0) return;
        seq = uniform(sh->seq);
        unit = uniform(sh->unit);
        n_new = uniform(sh->n_new);
        first_token = uniform(sh->first_token);
        len = uniform(checked_len(b.lens[seq], b, b.status));
    }
    if (warp == kMmaWarp) tc::tmem_alloc(&sh->tmem, kTmemCols);
    const int row0 = unit * p.unit_rows;                   // of the sequence's n_new * group rows
    const int rows = static_cast<int>(min(static_cast<long long>(n_new) * p.group - row0, static_cast<long long>(p.unit_rows)));
    auto token_of = [&](int row) { return p.group_inv ? static_cast<int>(__umul64hi(row0 + row, p.group_inv)) : row0 + row; };
    // keys that a row sees: its token's position + 1 (could be <= 0)
    auto visible = [&](int row) { return len - n_new + token_of(row) + 1; };
    const int n_keys = uniform(visible(rows - 1));                    // of the last row
    const int n_tiles = n_keys > 0 ? (n_keys + kKeyTile - 1) / kKeyTile : 0;
    const int n_keys0 = uniform(rows > kRowTile ? visible(kRowTile - 1) : n_keys);  // of the first tile's last row
    // key tiles and steps of each row tile
    const int keys_of[2] = {max(n_keys0, 0), rows > kRowTile ? max(n_keys, 0) : 0};
    const int tiles_of[2] = {(keys_of[0] + kKeyTile - 1) / kKeyTile, (keys_of[1] + kKeyTile - 1) / kKeyTile};
    const int edge = uniform(max(0, visible(0)) / kKeyTile);          // first tile that some row sees only in part
    if (warp == kLoadWarp && lane == 0) {
        // both row tiles' product warps give a buffer back
        for (int i = 0; i < kBufs; ++i) tc::mbar_init(&sh->kv_empty[i], max(1, (tiles_of[0] > 0) + (tiles_of[1] > 0)));
        tc::fence_mbar_init();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = kSlim ? uniform(static_cast<int>(sh->tmem)) : 0;  // all 512 columns start at 0

    if (warp >= kMmaWarp) {
        if constexpr (kTiles == 2 && !kSlim) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ---- loads: buffer i holds K of tile i / 2 (i even) or V (i odd) ----------------------
            int i = 0;
            for (; i < 2 * n_tiles; ++i) {
                const int buf = i % kBufs;
                if (i >= kBufs && !wait(&sh->kv_empty[buf], (i / kBufs - 1) & 1, sh)) break;
                const int j = i >> 1;
                const int need = min(kKeyTile, n_keys - j * kKeyTile);
                const int boxes = (need + p.box_rows - 1) / p.box_rows;
                const bool at_edge = (i & 1) && j >= edge;
                uint64_t* bar = at_edge ? &sh->edge_full[j - edge] : &sh->kv_full[buf];
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(bar, static_cast<uint32_t>(boxes * p.box_rows * 128 * kHalves));
                    if (at_edge) tc::mbar_arrive(&sh->kv_full[buf]);  // the ring's phase goes on; nobody waits for it
                }
                __syncwarp();
                if (lane < boxes * kHalves) {  // at most 8 * 2
                    const int box = lane / kHalves, half = lane % kHalves;
                    const int t = j * kKeyTile + box * p.box_rows;
                    const uint32_t page = checked_page(b.table[static_cast<size_t>(seq) * b.max_pages + t / b.page_size], b.n_pages, b.status);
                    const int row = p.layer_row + (static_cast<int>(page) * b.n_kv_heads + kvh) * b.page_size + t % b.page_size;
                    tc::tma_load_3d(ring + buf * kTileBytes + half * kHalfBytes + box * p.box_rows * 128, (i & 1) ? &vmap : &kmap, 0, row, half, bar);
                }
                __syncwarp();
            }
            if (sh->abort_flag) {  // copies still in flight land before the block ends
                volatile int alone = 0;
                for (int k = max(0, i - kBufs); k < i; ++k) {
                    const bool at_edge = (k & 1) && (k >> 1) >= edge;
                    tc::mbar_wait(at_edge ? &sh->edge_full[(k >> 1) - edge] : &sh->kv_full[k % kBufs], at_edge ? 0 : (k / kBufs) & 1, &alone, 100000000ull);
                }
            }
        } else if (warp < kLoadWarp) {
            // ---- products ------------------------------------------------------------------------------
            const int mma = warp - kMmaWarp, t = kTiles == 2 ? mma : 0, n = (keys_of[t] + kStep - 1) / kStep;
            const uint32_t idesc_s = idesc<C>(kSKeys, false), idesc_o = idesc<C>(D, true);
            const uint64_t qd = tc::sw128_desc(tc::smem_u32(qs) + t * kPieces * kTileBytes);
            const uint64_t kd = tc::sw128_desc(tc::smem_u32(ring)), vd = tc::sw128_desc_mn(tc::smem_u32(ring), kHalfBytes);
            const uint32_t s_at = tmem + t * kSBufs * kStep, o_at = tmem + kOCol + t * kOCols;
            uint64_t *s_full = sh->s_full + t * kSBufs, *p_full = sh->p_full + t * kSBufs;
            auto scores = [&](int i) {  // S(i) = Q K^T, then its tile's buffer back after the tile's last
                const int buf = 2 * (i >> 1) % kBufs;
                const uint64_t k_at = kd + (buf * kTileBytes + (i & 1) * (kStep * 128) >> 4);
#pragma unroll
                for (int h = 0; h < kPieces; ++h)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t o = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
                        // the second piece first: fewer of the additions, each cut off at the sum's size, are at full size
                        tc::mma_ss(s_at + (i % kSBufs) * kStep, qd + (kPieces - 1 - h) * (kTileBytes >> 4) + o, k_at + o, idesc_s, (h | k) != 0);
                    }
                tc::mma_commit(&s_full[i % kSBufs]);
                if (kTiles == 1 || (i & 1) || i + 1 == n) tc::mma_commit(&sh->kv_empty[buf]);
            };
            auto product = [&](int i) {  // O += P(i) V, then its tile's buffer back after the tile's last
                const int vbuf = (2 * (i >> 1) + 1) % kBufs, ksteps = min(kStep, n_keys - i * kStep + 15) / 16;
                const uint64_t v_at = vd + (vbuf * kTileBytes + (i & 1) * (kStep * 128) >> 4);
#pragma unroll
                for (int h = 0; h < kPieces; ++h)
#pragma unroll
                    for (int k = 0; k < kStep / 16; ++k)
                        if (k < ksteps)
                            tc::mma_ts(o_at, s_at + (i % kSBufs) * kStep + kPCol + h * 32 + k * 8, v_at + k * (2048 >> 4), idesc_o,
                                       ((kSplit ? i % kPart : i) | h | k) != 0);
                if ((i & 1) || i + 1 == n) tc::mma_commit(&sh->kv_empty[vbuf]);
            };
            auto wait_k = [&](int j) { return wait(&sh->kv_full[2 * j % kBufs], (2 * j / kBufs) & 1, sh); };
            auto wait_v = [&](int j) {
                return j < edge ? wait(&sh->kv_full[(2 * j + 1) % kBufs], ((2 * j + 1) / kBufs) & 1, sh) : wait(&sh->edge_done[j - edge], 0, sh);
            };
            auto wait_p = [&](int i) { return wait(&p_full[i % kSBufs], (i / kSBufs) & 1, sh); };
            bool ok = true;
            if constexpr (kTiles == 2) {
                // S(0), S(1), then O += P(i) V, S(i + 2) into the place of P(i); with one place S(0), O += P(i) V, S(i + 1)
                if (n > 0 && (ok = wait(&sh->q_full, 0, sh) && wait_k(0))) {
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        scores(0);
                        if (!kSlim && n > 1) scores(1);
                    }
                    __syncwarp();
                }
                for (int i = 0; ok && i < n; ++i) {
                    const int j = i >> 1;
                    if (!(i & 1)) ok = wait_v(j) && (kSlim || i + 2 >= n || wait_k(j + 1));
                    if (kSlim && ok && (i & 1) && i + 1 < n) ok = wait_k(j + 1);
                    if (!ok || !(ok = wait_p(i))) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        product(i);
                        if (i + kSBufs < n) scores(i + kSBufs);
                        else if (i + 1 < n) tc::mma_commit(&s_full[i % kSBufs]);  // no step i + 2: O is up to step i
                        else tc::mma_commit(&sh->o_full[t]);
                    }
                    __syncwarp();
                }
            } else if (mma == 0) {
                // S(i) and S(i + 1) into the places of P(i - 4) and P(i - 3), whose products are then done; so V of all
                // tiles but the last two in front has come, and a wait for K's phase cannot be taken for the one before
                ok = n == 0 || wait(&sh->q_full, 0, sh);
                for (int i = 0; ok && i < n; i += 2) {
                    if (i >= kSBufs)
                        ok = wait(&sh->o_step[i % kSBufs], (i / kSBufs - 1) & 1, sh) && wait(&sh->o_step[i % kSBufs + 1], (i / kSBufs - 1) & 1, sh);
                    if (!ok || !(ok = wait_k(i >> 1))) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) scores(i);
                    __syncwarp();
                }
            } else {
                // P(i) first: then K of its tile has come, and V's phase is the one waited for
                for (int i = 0; ok && i < n; ++i) {
                    ok = wait_p(i) && ((i & 1) || wait_v(i >> 1));
                    if (!ok) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        product(i);
                        tc::mma_commit(i + 1 < n ? &sh->o_step[i % kSBufs] : &sh->o_full[t]);
                    }
                    __syncwarp();
                }
            }
            // buffers that only the other row tile reads
            for (int i = 2 * tiles_of[t]; ok && n > 0 && i < 2 * n_tiles; ++i) {
                ok = wait(&sh->kv_full[i % kBufs], (i / kBufs) & 1, sh);
                if (ok && lane == 0) tc::mbar_arrive(&sh->kv_empty[i % kBufs]);
            }
            if (!ok) {  // given up: products in flight end before their memory goes away
                volatile int alone = 0;
                if (tc::elect_one()) tc::mma_commit(&sh->drained[mma]);
                tc::mbar_wait(&sh->drained[mma], 0, &alone, 100000000ull);
            }
        } else if (warp < kEdgeWarp + R::kEdges) {
            // ---- V at the causal edge ------------------------------------------------------------
            for (int j = edge; j < n_tiles; ++j) {
                const int buf = (2 * j + 1) % kBufs;
                if (!wait(&sh->edge_full[j - edge], 0, sh)) break;
                uint8_t* v = ring + buf * kTileBytes;
                const int used = (min(kKeyTile, n_keys - j * kKeyTile) + 15) / 16 * 16;  // rows of the product
                const int held = len - j * kKeyTile;                                        // rows of the sequence
                constexpr uint32_t kExp = kHalfType ? 0x7C00u : 0x7F80u;
                // 16 bytes per lane, a group of 4 rows x 128 bytes per step; 4 steps' loads ahead of their checks
#pragma unroll 1
                for (int half = 0; half < kHalves; ++half) {
                    uint8_t* at = v + half * kHalfBytes + lane * 16;
#pragma unroll 1
                    for (int r0 = (warp - kEdgeWarp) * 16; r0 < used; r0 += 16 * R::kEdges) {
                        uint4 x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint4*>(at + (r0 + 4 * k) * 128);
                        uint32_t flags = 0;  // chunks with an exponent of ones
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
                            bool any = false;
#pragma unroll
                            for (int i = 0; i < 4; ++i) any |= (w[i] & kExp) == kExp || (w[i] & (kExp << 16)) == (kExp << 16);
                            if (r0 + 4 * k + (lane >> 3) >= held) *reinterpret_cast<uint4*>(at + (r0 + 4 * k) * 128) = make_uint4(0, 0, 0, 0);
                            else flags |= any << k;
                        }
                        while (flags) {
                            const int k = __ffs(flags) - 1, r = r0 + 4 * k + (lane >> 3);
                            flags &= flags - 1;
                            uint16_t* e = reinterpret_cast<uint16_t*>(at + (r0 + 4 * k) * 128);
#pragma unroll 1
                            for (int i = 0; i < 8; ++i) {
                                if ((e[i] & kExp) != kExp) continue;
                                sh->bad = 1;
                                atomicMin(&sh->bad_key[half * 64 + ((lane & 7) ^ (r & 7)) * 8 + i], j * kKeyTile + r);
                                e[i] = 0;
                            }
                        }
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh->edge_done[j - edge]);
            }
        }
    } else {
        // ---- softmax: one row per thread, or two threads a row, of which one takes the even steps -----------
        if constexpr (kTiles == 2 && !kSlim) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = kTiles == 2 ? warp >> 2 : 0, g = kTiles == 2 ? 0 : warp >> 2, r = tid & 127;
        const int row = t * kRowTile + r;
        int met = 0;
        auto meet = [&]() {  // the rows' other warp: what either did before is done
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh->meet[warp & 3]);
            return wait(&sh->meet[warp & 3], met++ & 1, sh);
        };
        auto other = [&](float mine, float* theirs) {
            float* at = sh->row[met & 1][0] + r;
            at[g * 128] = mine;
            const bool there = meet();
            *theirs = at[(g ^ 1) * 128];
            return there;
        };
        bool ok = true;
        const bool live = row < rows;
        const int local = token_of(row), token = first_token + local, head = kvh * p.group + row0 + row - local * p.group;
        const int vis = live ? visible(row) : 0;
        float sl = p.a.scale * 1.4426950408889634f;
        // The warp's 32 query rows to shared memory as 16-bit pieces, kRowsPer whole rows per load (a
        // thread reading its own row would touch 32 lines per load);
        // rows behind the last are zero.
        constexpr int kLanesPer = D * sizeof(A) / 16, kRowsPer = 32 / kLanesPer, kVals = 16 / sizeof(A);
        const size_t q_off = static_cast<size_t>(token) * p.a.q_stride + static_cast<size_t>(head) * D;
        {
            const int part = lane % kLanesPer;  // the lane's 16 bytes of a row
            if constexpr (!kSplit) {
                // asynchronous copies: all rows in flight
#pragma unroll 4
                for (int i = 0; i < 32; i += kRowsPer) {
                    const int src = i + lane / kLanesPer, rr = (warp & 3) * 32 + src, c = part * kVals / 8;
                    const size_t off = __shfl_sync(0xffffffffu, q_off, src);
                    const int there = __shfl_sync(0xffffffffu, live, src);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 ::"r"(tc::smem_u32(qs + t * kPieces * kTileBytes + (c >> 3) * kHalfBytes + rr * 128 + (((c & 7) ^ (rr & 7)) << 4))),
                                   "l"(static_cast<const A*>(p.a.q) + (there ? off + part * kVals : 0)), "r"(there * 16) : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
                constexpr int kSteps = 32 / kRowsPer / kPer, kBatch = kSteps < 8 ? kSteps : 8;  // a group's share of the rows
                uint4 in[kBatch], ahead[kBatch];  // a batch of rows is loaded while the one before is worked on
                auto load = [&](int i0, uint4 (&to)[kBatch]) {
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int src = (g * kSteps + i0 + k) * kRowsPer + lane / kLanesPer;  // row of the warp
                        const size_t off = __shfl_sync(0xffffffffu, q_off, src);
                        const bool there = __shfl_sync(0xffffffffu, live, src);
                        to[k] = there ? __ldg(reinterpret_cast<const uint4*>(static_cast<const A*>(p.a.q) + off) + part) : make_uint4(0, 0, 0, 0);
                    }
                };
                load(0, ahead);
#pragma unroll 1
                for (int i0 = 0; i0 < kSteps; i0 += kBatch) {
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) in[k] = ahead[k];
                    if (i0 + kBatch < kSteps) load(i0 + kBatch, ahead);
#pragma unroll
                    for (int k0 = 0; k0 < kBatch; ++k0) {
                        const int i = (g * kSteps + i0 + k0) * kRowsPer, src = i + lane / kLanesPer;
                        alignas(16) A x[kVals];
                        *reinterpret_cast<uint4*>(x) = in[k0];
                        const int rr = (warp & 3) * 32 + src;
                        const int c = part * kVals / 8;  // 16-byte chunk of 16-bit values
                        uint8_t* at = qs + t * kPieces * kTileBytes + (c >> 3) * kHalfBytes + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
                        float f[4] = {to_f32(x[0]), to_f32(x[1]), to_f32(x[2]), to_f32(x[3])};
                        if constexpr (kHalfType) {
                            // the row's largest magnitude goes to [2^14, 2^15), undone in its score scale
                            float mx = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
                            if constexpr (kLanesPer == 32) {  // magnitudes order as their bits do
                                mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
                            } else {
#pragma unroll
                                for (int o = 1; o < kLanesPer; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                            }
                            const int e = row_exponent(mx);
#pragma unroll
                            for (int k = 0; k < 4; ++k) f[k] *= pow2(e);
#pragma unroll
                            for (int k = 0; k < kRowsPer; ++k) {
                                const int ek = __shfl_sync(0xffffffffu, e, k * kLanesPer);
                                if (lane == i + k) sl *= pow2(-ek);
                            }
                        }
                        uint2 hi, lo;
                        hi.x = pack2<C>(f[0], f[1]); hi.y = pack2<C>(f[2], f[3]);
                        lo.x = pack_rest<C>(hi.x, f[0], f[1]); lo.y = pack_rest<C>(hi.y, f[2], f[3]);
                        *reinterpret_cast<uint2*>(at + (part & 1) * 8) = hi;
                        *reinterpret_cast<uint2*>(at + kTileBytes + (part & 1) * 8) = lo;
                    }
                }
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh->q_full);
            if constexpr (kPer == 2 && kHalfType) {  // the scale of a row that the other group has loaded
                float theirs;
                ok = other(sl, &theirs);
                if (lane / (32 / kPer) != g) sl = theirs;
            }
        }
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // the warp's 32 TMEM lanes
        const uint32_t s_at = tmem + t * kSBufs * kStep + lanes, o_at = tmem + kOCol + t * kOCols + lanes;
        const int n = (keys_of[t] + kStep - 1) / kStep;
        const int part = max(0, visible(t * kRowTile)) / kStep;  // first step that a row of this tile sees in part
        float m = -INFINITY, l = 0.f;
        for (int i0 = 0; ok && i0 < n; i0 += kPer) {
            const int i = i0 + g;  // this thread's step
            ok = wait(&sh->s_full[t * kSBufs + i0 % kSBufs], (i0 / kSBufs) & 1, sh);
            if (!ok) break;
            tc::tc_fence_after();
            const uint32_t at = s_at + (i % kSBufs) * kStep;
            // kHeld of the step's scores at a time: those of the rows' last keys, with one place for S, are held from the
            // maximum to the weights, the others read twice, and weights go where scores are held or spent
            constexpr int kHeld = kSlim ? kStep / 2 : kStep;
            uint32_t raw[kHeld];
            float* z = reinterpret_cast<float*>(raw);
            auto take = [&](int c0) {
#pragma unroll
                for (int c = 0; c < kHeld; c += 32) tc::tmem_ld32(at + c0 + c, raw + c);
                tc::tmem_wait_ld();
                if (i >= part) {
                    const int seen = vis - i * kStep - c0;
#pragma unroll
                    for (int c = 0; c < kHeld; ++c)
                        if (c >= seen) z[c] = -INFINITY;
                }
            };
            float mz = -INFINITY;
#pragma unroll
            for (int c0 = 0; c0 < kStep; c0 += kHeld) {
                take(c0);
                float mx[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
                for (int c = 4; c < kHeld - 4; c += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], z[c + k]), z[c + 4 + k]);
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], z[kHeld - 4 + k]);
                const float mc = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                mz = c0 == 0 ? mc : fmaxf(mz, mc);
            }
            if constexpr (kPer == 2) {
                float theirs;
                if (!(ok = other(mz, &theirs))) break;
                mz = fmaxf(mz, theirs);
            }
            const float m_new = fmaxf(m, __fmul_rn(mz, sl));
            const bool grown = __any_sync(0xffffffffu, m_new - m > kRescaleAt<A, C>), part_end = kSplit && i0 > 0 && i0 % kPart == 0;
            if (grown || part_end) {
                float f = 1.f;
                if (grown) {
                    f = ex2(m - (m_new == -INFINITY ? 0.f : m_new));
                    m = m_new;
                    l *= f;
                }
                if (i0 > 0) {
                    // O holds the steps in front: with two tiles once S(i + 1), issued behind their last product, is there
                    if constexpr (kSlim) ok = true;  // S(i) was issued behind their last product
                    else if constexpr (kTiles == 2) ok = wait(&sh->s_full[t * kSBufs + ((i + 1) & 1)], ((i + 1) >> 1) & 1, sh);
                    else ok = wait(&sh->o_step[(i0 - 1) % kSBufs], ((i0 - 1) / kSBufs) & 1, sh);
                    if (!ok) break;
                    tc::tc_fence_after();
#pragma unroll 1
                    for (int c = g * (D / kPer); c < (g + 1) * (D / kPer); c += 16) {
                        uint32_t o[16], o2[16];
                        tc::tmem_ld16(o_at + c, o);
                        if (kSplit && i0 > kPart) tc::tmem_ld16(o_at + D + c, o2);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float x = __uint_as_float(o[k]), y = kSplit && i0 > kPart ? __uint_as_float(o2[k]) : 0.f;
                            o[k] = __float_as_uint(x * f);
                            o2[k] = __float_as_uint((part_end ? x + y : y) * f);
                        }
                        if (!part_end) tc::tmem_st16(o_at + c, o);  // else the next product writes it anew
                        if (kSplit && i0 >= kPart) tc::tmem_st16(o_at + D + c, o2);
                    }
                    if constexpr (kPer == 2) {  // both halves of O, before either's weights are taken
                        tc::tmem_wait_st();
                        tc::tc_fence_before();
                        if (!(ok = meet())) break;
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m;
            float2 sum[2] = {both(0.f), both(0.f)};
            // An f16 weight keeps within the type however large the scores: their products with the scale are rounded as the
            // maximum's was (from 2^24 on the exact product is units away from it), and a factor that next to the maximum
            // rounds up is left out.  Product and sum are two operations (f16, 64 columns: 139 us, 136 as one; f32, 128
            // columns: 583, 578); the product as one with a 0 that the compiler does not know, or it would join them.
            float nb = kLift<A, C> - base;
            if (kHalfType && nb + base > kLift<A, C>) nb = -base;
            const float2 sl2 = both(sl), nb2 = both(nb), zero2 = both(p.zero);
#pragma unroll
            for (int c0 = kStep - kHeld; c0 >= 0; c0 -= kHeld) {
                if (c0 + kHeld < kStep) take(c0);
#pragma unroll
                for (int c = 0; c < kHeld; c += 32) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 x = make_float2(z[c + 2 * k], z[c + 2 * k + 1]);
                        x = kHalfType ? add2(fma2(x, sl2, zero2), nb2) : fma2(x, sl2, nb2);
                        x = make_float2(ex2(x.x), !kSplit && k % 8 == 0 ? ex2_poly(x.y) : ex2(x.y));
                        sum[k & 1] = add2(sum[k & 1], x);
                        hi[k] = pack2<C>(x.x, x.y);
                        if constexpr (kSplit) lo[k] = pack_rest<C>(hi[k], x.x, x.y);
                    }
                    tc::tmem_st16(at + kPCol + (c0 + c) / 2, hi);
                    if constexpr (kSplit) tc::tmem_st16(at + 32 + (c0 + c) / 2, lo);
                }
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tc::tmem_wait_st();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh->p_full[t * kSBufs + i % kSBufs]);
        }
        // ---- output ------------------------------------------------------------------------------
        if (n > 0 && ok) ok = wait(&sh->o_full[t], 0, sh);
        if constexpr (kPer == 2) {
            float theirs = 0.f;
            ok = ok && other(l, &theirs);
            l += theirs;
        }
        if (ok) {
            tc::tc_fence_after();
            // each thread's row goes through shared memory (Q of this tile is done with), 16-byte chunks
            // exchanged by the row's number, and leaves as whole rows
            constexpr int kChunks = kLanesPer;
            uint8_t* stage = qs + t * kPieces * kTileBytes + (warp & 3) * 32 * kChunks * 16;
            const bool bad = sh->bad != 0;
            const float inv = vis > 0 ? 1.f / l : 1.f;
#pragma unroll 1
            for (int c = g * (D / kPer); c < (g + 1) * (D / kPer); c += 16) {
                uint32_t o[16], o2[16];
                if (n > 0) {
                    tc::tmem_ld16(o_at + c, o);
                    if (kSplit && n > kPart) tc::tmem_ld16(o_at + D + c, o2);
                    tc::tmem_wait_ld();
                }
                float* f = reinterpret_cast<float*>(o);
                if (kSplit && n > kPart) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) f[i] += __uint_as_float(o2[i]);
                }
                if (vis <= 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) f[i] = 0.f;
                } else if (bad) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (vis > sh->bad_key[c + i]) f[i] = NAN;
                }
#pragma unroll
                for (int i = 0; i < 16; i += kVals) {
                    alignas(16) A x[kVals];
#pragma unroll
                    for (int k = 0; k < kVals; k += 4) store4(x + k, make_float4(f[i + k], f[i + k + 1], f[i + k + 2], f[i + k + 3]), inv);
                    *reinterpret_cast<uint4*>(stage + (lane * kChunks + (((c + i) / kVals) ^ (lane & (kChunks - 1)))) * 16) = *reinterpret_cast<uint4*>(x);
                }
            }
            if constexpr (kPer == 2) meet(); else __syncwarp();  // a meeting missed: reported
            const size_t out_off = static_cast<size_t>(token) * p.a.out_stride + static_cast<size_t>(head) * D;
            const int part = lane % kLanesPer;
#pragma unroll 4
            for (int i = g * (32 / kPer); i < (g + 1) * (32 / kPer); i += kRowsPer) {
                const int src = i + lane / kLanesPer;
                const size_t off = __shfl_sync(0xffffffffu, out_off, src);
                const bool there = __shfl_sync(0xffffffffu, live, src);
                const uint4 x = *reinterpret_cast<const uint4*>(stage + (src * kChunks + (part ^ (src & (kChunks - 1)))) * 16);
                if (there) *(reinterpret_cast<uint4*>(static_cast<A*>(p.a.out) + off) + part) = x;
            }
        }
        tc::tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::tc_fence_after();
        tc::tmem_dealloc(sh->tmem, kTmemCols);
    }
    if (tid == 0 && sh->abort_flag) set_dev_error(b.status, kDevTimeout);
}

// No batch of T tokens in n_seqs sequences has more units.
long long units_of(const KvBatch& b, const AttnArgs& a, int group, int unit_rows) {
    const long long rows = static_cast<long long>(a.T) * group;
    return (b.n_seqs == 1 ? (rows + unit_rows - 1) / unit_rows : rows / unit_rows + std::min(b.n_seqs, a.T)) * b.n_kv_heads;
}

template <typename A, typename C, int D>
void launch_t(const PromptArgs& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
    constexpr size_t kTile = static_cast<size_t>(D / 64) * 128 * 128;
    constexpr int kTiles = kTilesOf<A, D>;
    constexpr size_t kSmem = (kTiles * (sizeof(A) == 4 ? 2 : 1) + kBufsOf<A, D>) * kTile + sizeof(Shared);
    static_assert(kSmem <= 232448, "shared memory");
    static std::atomic<uint64_t> set{0};  // devices whose limit is raised
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(set.load() >> dev & 1)) {
        cudaFuncSetAttribute(attn_prompt_kernel<A, C, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
        if (dev < 64) set.fetch_or(1ull << dev);
    }
    const unsigned grid = static_cast<unsigned>(units_of(p.b, p.a, p.group, p.unit_rows));
    attn_prompt_kernel<A, C, D><<<grid, Roles<kTiles, kSlimOf<A, D>>::kThreads, kSmem, s>>>(p, k, v);
}

template <typename A, typename C>
void launch_d(const PromptArgs& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
    if (p.b.head_dim == 64) launch_t<A, C, 64>(p, k, v, s); else launch_t<A, C, 128>(p, k, v, s);
}

}  // namespace

void launch_attn_prompt(const KvBatch& b, int act, const KvCache& kv, uint32_t layer, const AttnArgs& a, int sm_count, cudaStream_t s) {
    PromptArgs p{};
    p.b = b;
    p.a = a;
    p.group = a.n_heads / b.n_kv_heads;
    p.group_inv = p.group == 1 ? 0 : ~0ull / p.group + 1;
    // one row tile per CTA while twice the CTAs still run at once: a key step of one tile takes less time than
    // one of two (512 tokens, 8 query heads to each of 2 kv heads, f16: 21.5 us as 32 CTAs, 19.5 us as 64)
    p.unit_rows = (act == MOE_T_F32 && b.head_dim == 128) || 2 * units_of(b, a, p.group, 2 * kRowTile) <= sm_count ? kRowTile : 2 * kRowTile;
    p.layer_row = static_cast<int>(static_cast<uint64_t>(layer) * kv.spec.n_pages * kv.spec.n_kv_heads * kv.spec.page_size);
    p.box_rows = static_cast<int>(kv.spec.page_size);
    p.zero = 0.f;
    const CUtensorMap &k = kv.maps[2], &v = kv.maps[3];
    if (act == MOE_T_F32) {
        if (kv.spec.type == MOE_T_F16) launch_d<float, __half>(p, k, v, s);
        else launch_d<float, __nv_bfloat16>(p, k, v, s);
    } else if (act == MOE_T_F16) {
        launch_d<__half, __half>(p, k, v, s);
    } else {
        launch_d<__nv_bfloat16, __nv_bfloat16>(p, k, v, s);
    }
}

}  // namespace moe
