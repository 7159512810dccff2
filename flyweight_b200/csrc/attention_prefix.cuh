// What the kernels of attention over a shared prefix have in common: the batch as they see it.
//
// The tokens [group_start[g], group_start[g + 1]) belong to requests whose first group_pages[g] pages are the same ones;
// the block-table row of the group's first token that belongs to a request names them.  A token sees the keys up to its own
// position: those of the shared pages, then its request's own from position 64 * group_pages[g] on.
#pragma once

#include "common.cuh"

namespace fwb {
namespace prefix {

constexpr int PAGE = 64;
constexpr int MAX_SPLITS = 64;           // slices of a group's shared pages

struct Batch {
    const int* positions;        // [T]
    const int* tok_seg;          // [T]
    const int* block_table;      // [n_segments][max_pages]
    const int* group_start;      // [n_groups + 1], rising
    const int* group_pages;      // [n_groups]
    int T, n_segments, n_groups, max_pages, num_pages;

    __device__ __forceinline__ int start_of(int g) const {
        const int t = group_start[g];
        return t < 0 ? 0 : t > T ? T : t;
    }
    __device__ __forceinline__ int pages_of(int g) const {
        const int n = group_pages[g];
        return n < 0 ? 0 : n > max_pages ? max_pages : n;
    }
    // the block-table row of a token, null for a token of no request
    __device__ __forceinline__ const int* row_of(int token) const {
        const int seg = tok_seg[token];
        return seg < 0 || seg >= n_segments ? nullptr : block_table + (size_t)seg * max_pages;
    }
    // the last key that a token at this position sees: -1 (none) in front of the first one, wherever
    __device__ __forceinline__ int last_key(int position) const {
        return position < 0 ? -1 : position < max_pages * PAGE ? position : max_pages * PAGE - 1;
    }
    __device__ __forceinline__ bool is_page(int page) const { return page >= 0 && page < num_pages; }
};

// The token tile `index` when every group's tokens are cut into tiles of `per_tile`: its group's tokens and pages, its own
// first token and tokens (0: no such tile).  Asked by whole warps; everything it reads is asked for at once.
struct TokenTile {
    int group_first, group_end, pages, first, count;
};
__device__ __forceinline__ TokenTile token_tile(const Batch& b, int index, int per_tile) {
    const int lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < b.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int first = g < b.n_groups ? b.start_of(g) : 0, pages = g < b.n_groups ? b.pages_of(g) : 0;
        int n = g < b.n_groups ? b.start_of(g + 1) - first : 0;
        n = n < 0 ? 0 : n;
        const int tiles = (n + per_tile - 1) / per_tile;
        int upto = tiles;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, offset);
            if (lane >= offset) upto += other;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, index < upto);
        if (behind) {
            const int owner = __ffs(behind) - 1;
            const int inside = index - (__shfl_sync(0xffffffffu, upto, owner) - __shfl_sync(0xffffffffu, tiles, owner));
            TokenTile t;
            t.group_first = __shfl_sync(0xffffffffu, first, owner);
            t.pages = __shfl_sync(0xffffffffu, pages, owner);
            t.group_end = t.group_first + __shfl_sync(0xffffffffu, n, owner);
            t.first = t.group_first + inside * per_tile;
            const int left = t.group_end - t.first;
            t.count = left < per_tile ? left : per_tile;
            return t;
        }
        index -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return TokenTile{0, 0, 0, 0, 0};
}
// The block-table row that names the shared pages of a tile's group (null: none of its tokens belongs to a request).  Asked by whole warps.
__device__ __forceinline__ const int* shared_row(const Batch& b, const TokenTile& tile) {
    const int lane = threadIdx.x & 31;
    for (int t0 = tile.group_first; t0 < tile.group_end; t0 += 32) {
        const int seg = t0 + lane < tile.group_end ? b.tok_seg[t0 + lane] : -1;
        const unsigned there = __ballot_sync(0xffffffffu, seg >= 0 && seg < b.n_segments);
        if (there) return b.block_table + (size_t)__shfl_sync(0xffffffffu, seg, __ffs(there) - 1) * b.max_pages;
    }
    return nullptr;
}
// The most such tiles a batch can have, from what the host knows.
inline long most_token_tiles(int T, int n_groups, int per_tile) {
    const long most = ((long)T + (long)n_groups * (per_tile - 1)) / per_tile;
    return most < T ? most : T;
}

// A token as the own kernels see it: its group's shared pages (-1: it is in no group), its block-table row and the last key it
// sees.  Asked by whole warps; the group's arrays and the token's are asked for at once.
struct Token {
    int pages, last;
    int first, end;              // its group's tokens
    const int* table;
};
__device__ __forceinline__ Token token_of(const Batch& b, int token) {
    const int lane = threadIdx.x & 31;
    const int seg = b.tok_seg[token], position = b.positions[token];
    Token t{-1, -1, 0, 0, nullptr};
    for (int g0 = 0; g0 <= b.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int start = g <= b.n_groups ? b.start_of(g) : b.T;
        const bool begun = g <= b.n_groups && start <= token;
        const int pages = g < b.n_groups ? b.pages_of(g) : -1;       // (behind the last group: in none)
        const int n = __popc(__ballot_sync(0xffffffffu, begun));
        if (n > 0) t.pages = __shfl_sync(0xffffffffu, pages, n - 1), t.first = __shfl_sync(0xffffffffu, start, n - 1);
        if (n < 32) {
            t.end = __shfl_sync(0xffffffffu, start, n);
            break;
        }
    }
    if (seg >= 0 && seg < b.n_segments) {
        t.table = b.block_table + (size_t)seg * b.max_pages;
        t.last = b.last_key(position);
    }
    return t;
}

// How a group's shared pages are cut into at most `splits` slices: pages a slice.
__host__ __device__ __forceinline__ int pages_per_slice(int pages, int splits) { return (pages + splits - 1) / splits; }

// The bfloat16 form on tensor cores (host functions, attention_prefix_tcgen05.cu): whether it takes the shape, and its launch.
bool tensor_cores_take(const void* q, const void* k_pool, const void* v_pool, const void* out, const void* part_o, const Batch& b, int nkv, int hd);
int launch_tensor_cores(const Batch& b, const void* q, const void* k_pool, const void* v_pool, void* out, float* part_o, float* part_ml,
                        const float* sink, int nh, int nkv, int hd, int splits, int own_slices, bool neighbours, float scale, float softcap,
                        cudaStream_t stream);

}  // namespace prefix
}  // namespace fwb
