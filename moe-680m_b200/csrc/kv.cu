// Paged key-value cache kernels: append of new rows, whole-page copies (fork, compaction), table
// upload.  moe-680m writes its cache with shaders/kv_write.comp (one sequence, quantised rows); the
// pages and their sharing have no counterpart there.
#include <cuda_runtime.h>

#include <algorithm>

#include "kv_cache.cuh"

namespace moe {

namespace {

// ---- append -------------------------------------------------------------------------------
// Pure movement: T * Hkv * D values of K and of V read once and stored as 16 bits.  A warp per token: it
// finds the token's sequence, position and page once (a thread per 16 bytes, each finding them for itself,
// took 9.7 us for 8192 tokens of 8 heads in 11 sequences, against 8.4), and its lanes then take 16 bytes of
// K and of V at a time, four of each in flight.
template <typename A, typename C>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvBatch b, const A* __restrict__ k, const A* __restrict__ v,
                                                        uint64_t stride, int T, C* __restrict__ kp, C* __restrict__ vp) {
    if (blockIdx.x == gridDim.x - 1 && b.cu) {
        // A block more than the tokens take, off their path: offsets that do not ascend or that leave the rows.  (A
        // token's own search meets only some of them.)
        for (int i = threadIdx.x; i < b.n_seqs; i += 256)
            if (!right_offsets(b.cu[i], b.cu[i + 1], T)) set_dev_error(b.status, kDevBadToken);
        return;
    }
    // a batch has up to 2^31 - 1 tokens: the token's number, not its thread's, fits 32 bits
    const unsigned token = blockIdx.x * 8u + threadIdx.x / 32u;
    if (token >= static_cast<unsigned>(T)) return;
    const int t = static_cast<int>(token), lane = threadIdx.x & 31;
    const int s = warp_seq_of_token(b, t, lane);
    if (s < 0) return;
    const int from = b.cu ? b.cu[s] : t, to = b.cu ? b.cu[s + 1] : t + 1;
    if (!right_offsets(from, to, T) || t < from || t >= to) {
        set_dev_error(b.status, kDevBadToken);
        return;
    }
    const int n_after = to - t;  // tokens from this one to its sequence's end
    const long long pos = static_cast<long long>(b.lens[s]) - n_after;
    if (pos < 0 || pos >= static_cast<long long>(b.max_pages) * b.page_size) {
        set_dev_error(b.status, kDevBadToken);
        return;
    }
    const int p = b.table[static_cast<size_t>(s) * b.max_pages + pos / b.page_size];
    if (static_cast<uint32_t>(p) >= b.n_pages) {
        set_dev_error(b.status, kDevBadPage);
        return;
    }
    const int per_row = b.head_dim / 8, per_tok = per_row * b.n_kv_heads;
    const size_t src = static_cast<size_t>(t) * stride;
    const size_t row0 = static_cast<size_t>(p) * b.n_kv_heads * b.page_size + pos % b.page_size;  // of head 0
#pragma unroll 4
    for (int e = lane; e < per_tok; e += 32) {
        const int h = e / per_row, d = (e % per_row) * 8;
        const size_t from = src + static_cast<size_t>(h) * b.head_dim + d;
        const size_t to = (row0 + static_cast<size_t>(h) * b.page_size) * b.head_dim + d;
        alignas(16) A in[2][8];
        alignas(16) C out[2][8];
#pragma unroll
        for (int j = 0; j < static_cast<int>(8 * sizeof(A) / 16); ++j) {
            reinterpret_cast<uint4*>(in[0])[j] = __ldg(reinterpret_cast<const uint4*>(k + from) + j);
            reinterpret_cast<uint4*>(in[1])[j] = __ldg(reinterpret_cast<const uint4*>(v + from) + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            out[0][j] = from_f32<C>(to_f32(in[0][j]));
            out[1][j] = from_f32<C>(to_f32(in[1][j]));
        }
        *reinterpret_cast<uint4*>(kp + to) = *reinterpret_cast<uint4*>(out[0]);
        *reinterpret_cast<uint4*>(vp + to) = *reinterpret_cast<uint4*>(out[1]);
    }
}

template <typename A, typename C>
void append_t(const KvBatch& b, const void* k, const void* v, uint64_t stride, int T, void* kp, void* vp, cudaStream_t s) {
    kv_append_kernel<A, C><<<(static_cast<unsigned>(T) + 7) / 8 + (b.cu ? 1 : 0), 256, 0, s>>>(
        b, static_cast<const A*>(k), static_cast<const A*>(v), stride, T, static_cast<C*>(kp), static_cast<C*>(vp));
}

// ---- page copies --------------------------------------------------------------------------
// The page list travels in the kernel parameters: no staging copy, no wait.
constexpr int kCopyList = 448;
struct CopyList {
    uint2 move[kCopyList];  // (from, to)
};

// blockIdx.y: move; blockIdx.z: layer and pool (K, V); the x blocks share a page's bytes.
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ CopyList list, uint4* __restrict__ k,
                                                      uint4* __restrict__ v, uint64_t layer_vecs, uint32_t page_vecs) {
    const uint2 m = list.move[blockIdx.y];
    uint4* pool = ((blockIdx.z & 1) ? v : k) + (blockIdx.z >> 1) * layer_vecs;
    const uint4* src = pool + static_cast<uint64_t>(m.x) * page_vecs;
    uint4* dst = pool + static_cast<uint64_t>(m.y) * page_vecs;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < page_vecs; i += gridDim.x * blockDim.x) dst[i] = __ldg(src + i);
}

// ---- table upload -------------------------------------------------------------------------
constexpr int kTableList = 960;
struct TableList {
    int32_t v[kTableList];
};
__global__ void kv_table_kernel(const __grid_constant__ TableList list, int n, int at, int n_table, int32_t* __restrict__ table,
                                int32_t* __restrict__ lens) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int j = at + i;
    if (j < n_table) table[j] = list.v[i]; else lens[j - n_table] = list.v[i];
}

}  // namespace

void launch_kv_append(const KvBatch& b, int act, int cache, const void* k, const void* v, uint64_t stride, int T, void* kp,
                      void* vp, cudaStream_t s) {
    if (act == MOE_T_F32) {
        if (cache == MOE_T_F16) append_t<float, __half>(b, k, v, stride, T, kp, vp, s);
        else append_t<float, __nv_bfloat16>(b, k, v, stride, T, kp, vp, s);
    } else if (act == MOE_T_F16) {
        append_t<__half, __half>(b, k, v, stride, T, kp, vp, s);
    } else {
        append_t<__nv_bfloat16, __nv_bfloat16>(b, k, v, stride, T, kp, vp, s);
    }
}

int launch_kv_copy(const std::pair<uint32_t, uint32_t>* moves, size_t n, void* k, void* v, int n_layers, uint64_t layer_bytes,
                   uint64_t page_bytes, cudaStream_t s) {
    const uint32_t vecs = static_cast<uint32_t>(page_bytes / 16);
    int launches = 0;
    for (size_t at = 0; at < n; at += kCopyList, ++launches) {
        CopyList list;
        const unsigned m = static_cast<unsigned>(std::min<size_t>(kCopyList, n - at));
        for (unsigned i = 0; i < m; ++i) list.move[i] = make_uint2(moves[at + i].first, moves[at + i].second);
        for (int l = 0; l < n_layers; l += 16384) {  // the grid's z extent is limited
            const unsigned z = static_cast<unsigned>(std::min(16384, n_layers - l));
            kv_copy_kernel<<<dim3((vecs + 1023) / 1024, m, 2 * z), 256, 0, s>>>(
                list, reinterpret_cast<uint4*>(static_cast<uint8_t*>(k) + l * layer_bytes),
                reinterpret_cast<uint4*>(static_cast<uint8_t*>(v) + l * layer_bytes), layer_bytes / 16, vecs);
        }
    }
    return launches;
}

cudaError_t launch_kv_tables(const std::vector<int32_t>& rows, uint32_t n_seqs, int32_t* table, int32_t* lens, cudaStream_t s,
                             int* launches) {
    const size_t n = rows.size(), n_table = n - n_seqs;
    *launches = 0;
    if (n > 8 * static_cast<size_t>(kTableList)) {
        // pageable source: the copies have left `rows` when cudaMemcpyAsync returns
        cudaError_t e = cudaMemcpyAsync(table, rows.data(), n_table * 4, cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaMemcpyAsync(lens, rows.data() + n_table, n_seqs * 4ull, cudaMemcpyHostToDevice, s);
        return e;
    }
    for (size_t at = 0; at < n; at += kTableList, ++*launches) {
        TableList list;
        const int m = static_cast<int>(std::min<size_t>(kTableList, n - at));
        std::copy(rows.begin() + static_cast<long>(at), rows.begin() + static_cast<long>(at) + m, list.v);
        kv_table_kernel<<<(m + 255) / 256, 256, 0, s>>>(list, m, static_cast<int>(at), static_cast<int>(n_table), table, lens);
    }
    return cudaSuccess;
}

}  // namespace moe
