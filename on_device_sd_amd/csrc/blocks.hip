// Copies of whole cache blocks, in all layers and all tensors of a cache by one launch: what a fork (the last, part-filled block of a
// sequence gets a copy) and compaction (blocks move to free places, block tables follow) need.  A byte mover: 2 bytes of traffic for
// every byte of a block, which is the bound: 1.57 GB in and out in 320 us, 4.9 TB/s.  A fork is one launch, 6 us for 12 MB.
//
// The lists of block numbers come from the host and travel as kernel arguments, so there is no copy to wait for and nothing to
// allocate; they are frozen where the call is captured into a graph.  No block is both read and written, so the order does not matter.
#include "common.h"

#define BLK_TENSORS ODSD_COPY_TENSORS
#define BLK_PAIRS 384        // pairs of a launch
#define BLK_CHUNK 16384      // bytes of a workgroup

struct BlkTensor {
    char *base;
    int64_t layer_bytes;     // from one layer's blocks to the next's
    uint32_t block_bytes, layers;
    uint32_t first_wg;       // its first workgroup
    uint32_t unit;           // bytes of an access: 16, 4, 2 or 1
    uint32_t per_inverse;    // small blocks: ceil(2^32 / units of one), 0 for 1
};
struct BlkParams {
    BlkTensor t[BLK_TENSORS];
    int n_tensors, n_pairs;
    uint32_t pairs_inverse;  // ceil(2^32 / n_pairs), 0 for 1
    uint32_t copy_wgs;       // workgroups that copy; those behind them rename table entries
    int32_t *tables;
    int64_t n_entries;
    int32_t src[BLK_PAIRS], dst[BLK_PAIRS];
};

// n / d with d's inverse, for n d < 2^32
__device__ __forceinline__ uint32_t blk_divide(const uint32_t n, const uint32_t inverse) { return inverse ? __umulhi(n, inverse) : n; }
template <typename V>
__device__ __forceinline__ void blk_copy(const BlkTensor &t, const BlkParams &p, const uint32_t wg) {
    constexpr uint32_t SZ = (uint32_t)sizeof(V);
    if (t.block_bytes >= BLK_CHUNK / 2) {
        // a piece of one block
        const uint32_t pieces = (t.block_bytes + BLK_CHUNK - 1) / BLK_CHUNK;
        const uint32_t which = wg / pieces, piece = wg - which * pieces, layer = which / (uint32_t)p.n_pairs, pair = which - layer * (uint32_t)p.n_pairs;
        const char *from = t.base + layer * t.layer_bytes + (uint64_t)(uint32_t)p.src[pair] * t.block_bytes;
        char *to = t.base + layer * t.layer_bytes + (uint64_t)(uint32_t)p.dst[pair] * t.block_bytes;
        const uint32_t end = min(t.block_bytes, (piece + 1) * BLK_CHUNK);
        for (uint32_t b = piece * BLK_CHUNK + threadIdx.x * SZ; b < end; b += 256 * SZ) *(V *)(to + b) = *(const V *)(from + b);
    } else {
        // Blocks are small: units of all of them one after the other.  The workgroup's first unit is divided out once; from there on the
        // numbers are small enough for a multiplication.  (Four units of a thread on their way together, which the compiler would not do by itself:
        // 1900 blocks of 2 KB of 24 layers 113 / 109 us; for blocks of several KB it changes nothing.)
        const uint32_t per = t.block_bytes / SZ;
        const uint64_t all = (uint64_t)per * p.n_pairs * t.layers, first = (uint64_t)wg * (BLK_CHUNK / SZ);
        const uint32_t here = (uint32_t)min((uint64_t)(BLK_CHUNK / SZ), all - first);
        const uint32_t which0 = (uint32_t)(first / per), at0 = (uint32_t)(first - (uint64_t)which0 * per);
        const uint32_t layer0 = which0 / (uint32_t)p.n_pairs, pair0 = which0 - layer0 * (uint32_t)p.n_pairs;
        for (uint32_t i = threadIdx.x; i < here; i += 4 * 256) {
            V v[4];
            char *to[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint32_t at = at0 + min(i + 256 * u, here - 1), block = blk_divide(at, t.per_inverse);
                const uint32_t pairs = pair0 + block, layer = blk_divide(pairs, p.pairs_inverse), pair = pairs - layer * (uint32_t)p.n_pairs;
                char *b = t.base + (layer0 + layer) * t.layer_bytes + (uint64_t)(at - block * per) * SZ;
                v[u] = *(const V *)(b + (uint64_t)(uint32_t)p.src[pair] * t.block_bytes);
                to[u] = b + (uint64_t)(uint32_t)p.dst[pair] * t.block_bytes;
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u)
                if (i + 256 * u < here) *(V *)to[u] = v[u];
        }
    }
}

__global__ __launch_bounds__(256) void copy_blocks_kernel(const BlkParams p) {
    if (blockIdx.x >= p.copy_wgs) {             // block tables: an entry that names a moved block names its new place
        const int64_t i = (int64_t)(blockIdx.x - p.copy_wgs) * 256 + threadIdx.x;
        if (i >= p.n_entries) return;
        const int32_t was = p.tables[i];
        int32_t now = was;
        for (int k = 0; k < p.n_pairs; ++k) now = was == p.src[k] ? p.dst[k] : now;
        if (now != was) p.tables[i] = now;
        return;
    }
    int k = 0;
    while (k + 1 < p.n_tensors && blockIdx.x >= p.t[k + 1].first_wg) ++k;
    const BlkTensor t = p.t[k];
    const uint32_t wg = blockIdx.x - t.first_wg;
    if (t.unit == 16) blk_copy<uint4_t>(t, p, wg);
    else if (t.unit == 4) blk_copy<uint32_t>(t, p, wg);
    else if (t.unit == 2) blk_copy<uint16_t>(t, p, wg);
    else blk_copy<uint8_t>(t, p, wg);
}

extern "C" int odsd_copy_blocks(void *const *tensors, const int64_t *block_bytes, const int64_t *layer_bytes,
                                const int32_t *layers, int32_t n_tensors, const int32_t *src, const int32_t *dst,
                                int32_t n_pairs, int32_t n_blocks, int32_t *block_tables, int64_t n_entries, void *stream) {
    if (n_tensors < 0 || n_pairs < 0 || n_blocks < 0 || n_entries < 0) return ODSD_ERR_SHAPE;
    if (n_tensors > BLK_TENSORS || n_entries > (1LL << 31)) return ODSD_ERR_UNSUPPORTED;
    if (n_pairs == 0 || (n_tensors == 0 && !block_tables)) return ODSD_OK;
    if (!src || !dst || (n_tensors && (!tensors || !block_bytes || !layer_bytes || !layers))) return ODSD_ERR_NULL;
    for (int i = 0; i < n_pairs; ++i)
        if (src[i] < 0 || src[i] >= n_blocks || dst[i] < 0 || dst[i] >= n_blocks) return ODSD_ERR_SHAPE;
    BlkParams p{};
    auto inverse = [](const uint32_t d) { return d > 1 ? (uint32_t)(((1ULL << 32) + d - 1) / d) : 0u; };
    p.n_tensors = n_tensors;
    const int most = min(n_pairs, BLK_PAIRS);
    for (int k = 0; k < n_tensors; ++k) {
        if (!tensors[k]) return ODSD_ERR_NULL;
        if (block_bytes[k] <= 0 || layers[k] < 0 || (layers[k] > 1 && layer_bytes[k] < block_bytes[k] * n_blocks)) return ODSD_ERR_SHAPE;
        // (32 bits for the bytes of a block and for the blocks that a launch copies)
        if (block_bytes[k] > 0x40000000LL || (int64_t)layers[k] * most > 0x7fffffffLL) return ODSD_ERR_UNSUPPORTED;
        const uint64_t all = (uint64_t)(uintptr_t)tensors[k] | (uint64_t)block_bytes[k] | (layers[k] > 1 ? (uint64_t)layer_bytes[k] : 0u);
        p.t[k] = BlkTensor{(char *)tensors[k], layer_bytes[k], (uint32_t)block_bytes[k], (uint32_t)layers[k], 0,
                           (uint32_t)(all & 15u ? all & 3u ? all & 1u ? 1 : 2 : 4 : 16), 0};
        p.t[k].per_inverse = inverse(p.t[k].block_bytes / p.t[k].unit);
    }
    p.tables = block_tables;
    p.n_entries = block_tables ? n_entries : 0;
    const int64_t table_wgs = (p.n_entries + 255) / 256;
    auto workgroups = [&](const int pairs) {    // of a launch; every tensor's first on the way
        int64_t wgs = 0;
        for (int k = 0; k < n_tensors; ++k) {
            const int64_t blocks = (int64_t)p.t[k].layers * pairs, bytes = p.t[k].block_bytes;
            p.t[k].first_wg = (uint32_t)wgs;
            wgs += bytes >= BLK_CHUNK / 2 ? blocks * ((bytes + BLK_CHUNK - 1) / BLK_CHUNK) : (blocks * bytes + BLK_CHUNK - 1) / BLK_CHUNK;
        }
        return wgs;
    };
    if ((workgroups(most) + table_wgs) >= (1LL << 24)) return ODSD_ERR_UNSUPPORTED;
    for (int at = 0; at < n_pairs; at += BLK_PAIRS) {
        p.n_pairs = min(n_pairs - at, BLK_PAIRS);
        p.pairs_inverse = inverse((uint32_t)p.n_pairs);
        for (int i = 0; i < p.n_pairs; ++i) {
            p.src[i] = src[at + i];
            p.dst[i] = dst[at + i];
        }
        p.copy_wgs = (uint32_t)workgroups(p.n_pairs);
        if (p.copy_wgs + table_wgs == 0) continue;
        copy_blocks_kernel<<<(unsigned)(p.copy_wgs + table_wgs), 256, 0, (hipStream_t)stream>>>(p);
        ODSD_CHECK_LAUNCH();
    }
    return ODSD_OK;
}
