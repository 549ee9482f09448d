// Attention of new tokens over a key/value cache: what its kernels share.
//
// Query token i of a sequence with n new tokens and `len` keys (the new ones
// included) sits at position p = len - n + i and sees key j when
//     j < min(e, len)  and  (j >= e - window  or  j < sinks),   e = (p / block + 1) * block
// (block 1: causal; a larger block sees to its own end). Query heads share key
// heads in groups of G, and the (token, head) pairs of a group are the rows of
// one problem: row r is token r / G, head kvh * G + r % G. The keys a tile of
// rows needs are walked in tiles; a tile that no row sees is not read.
//
// The keys lie in pages ([pages, kv_heads, page_size, 128] with a page table)
// or, without a table, in one "page" a sequence ([B, kv_heads, keys, 128]).
#pragma once

#include <cuda.h>

#include <type_traits>

#include "common.cuh"

namespace abx {

struct ChunkArgs {
    const void* q;
    void* o;
    float* lse;            // nullptr: not written
    int64_t q_seq, q_head, q_token;  // strides in elements; q_seq is 0 when tokens are packed
    int64_t o_seq, o_head, o_token;
    int64_t l_seq, l_head, l_token;
    float* part_o;         // [splits, rows_total, 128] f32, normalised by the split's own sum
    float* part_lse;       // [splits, rows_total] base 2; -inf: the split saw nothing, +inf: see chunk_part
    const int32_t* starts;   // [seqs + 1] or nullptr (every sequence has `tokens` tokens)
    const int32_t* lengths;  // [seqs] or nullptr (every sequence has `keys` keys)
    const int32_t* table;    // [seqs, table_width] or nullptr (sequence s is page s)
    int32_t seqs, heads, kv_heads, group;
    int32_t tokens;        // per sequence, or, packed, of all sequences
    int32_t longest;       // tokens of the longest sequence
    int32_t keys;          // per sequence, or, paged, at most (table_width * page_size)
    int32_t table_width, page_size, pages;
    int32_t page_shift;    // log2 of page_size, -1: not a power of two
    int32_t window, sinks, block;  // window: kNoWindow without one
    int32_t tile_rows;     // rows of a tile: 16 or 32 (chunk_token.cu), 256 (chunk_tile.cu)
    int32_t splits;        // CTAs that share the keys of one row tile
    int32_t cluster;       // 1: the splits of a row tile form a cluster and join their rows themselves
    int32_t span;          // key tiles of one split, or 0: the row tile's keys in equal parts
    int32_t units;         // > 0: a grid of one dimension, `units` row tiles a key head, and from the
    int32_t whole_jobs;    // whole_jobs-th on each row tile as two of half its rows (the tile kernel)
    int32_t sorted;        // 1: ragged sequences, the longest first; a grid of one dimension of splits, key heads and row
                           // tiles, the first fastest (the tile kernel)
    int32_t q_map;         // 1: maps.q describes the queries (the tile kernel, group divides 128)
    int64_t rows_total;    // tokens of all sequences * heads
    float kappa;           // 128^-0.5 * log2(e)
    int* error;
};

constexpr int32_t kNoWindow = 0x7fffffff;  // above every block's end
constexpr int32_t kMaxCacheKeys = 0x3fffffff;
constexpr int kMaxCluster = 8;
constexpr int kChunkTokenKeys = 64;  // keys of a tile of each kernel
constexpr int kChunkTileKeys = 128;
constexpr int kChunkBoxKeys = 64;    // keys of a TMA box at most: a tile of the one kernel, half a tile of the other

// One tile of rows of one sequence.
struct ChunkUnit {
    int32_t seq;    // -1: none (past the last tile)
    int32_t row0;   // first row
    int32_t n;      // the sequence's new tokens
    int32_t len;    // its keys
    int32_t first;  // its first token in the packed arrays (0 when not packed)
};

// Tokens [a, b) and key count of packed sequence s, clipped to what the buffers hold.
__device__ __forceinline__ void chunk_sequence(const ChunkArgs& a, int s, int32_t& first, int32_t& n, int32_t& len,
                                               bool& bad) {
    const int32_t s0 = __ldg(a.starts + s), s1 = __ldg(a.starts + s + 1), l = __ldg(a.lengths + s);
    first = min(max(s0, 0), a.tokens);
    const int32_t last = min(max(s1, first), a.tokens);
    n = last - first;
    len = min(max(l, 0), a.keys);
    bad = s0 != first || s1 != last || l != len || n > a.longest;
    if (n > a.longest) n = 0;  // more tokens than the launch covers: reported and not computed
}

// The row tile that unit u of the grid works on; called by whole warps. Tiles of
// a sequence come last first: under a causal mask the longest rows start first. sorted: of every 32 sequences
// those with the most keys come first.
__device__ __forceinline__ ChunkUnit chunk_unit(const ChunkArgs& a, int u, int tile_rows, bool sorted) {
    ChunkUnit r{-1, 0, 0, 0, 0};
    if (a.starts == nullptr) {
        const int tiles = (a.tokens * a.group + tile_rows - 1) / tile_rows;
        r.seq = u / tiles;
        r.row0 = (tiles - 1 - (u - r.seq * tiles)) * tile_rows;
        r.n = a.tokens;
        r.len = a.keys;
        return r;
    }
    const int lane = threadIdx.x & 31;
    int before = 0;
#pragma unroll 1
    for (int base = 0; base < a.seqs; base += 32) {
        const int s = base + lane;
        int32_t first = 0, n = 0, len = 0, tiles = 0;
        if (s < a.seqs) {
            bool bad;
            chunk_sequence(a, s, first, n, len, bad);
            if (bad) raise_device_error(a.error, ABX_ERR_INVALID_ARGUMENT);
            tiles = static_cast<int32_t>((static_cast<int64_t>(n) * a.group + tile_rows - 1) / tile_rows);
        }
        const int all = __reduce_add_sync(0xffffffffu, tiles);
        if (before + all > u) {
            int ahead = before;  // tiles of the sequences before this lane's
            if (sorted) {
#pragma unroll 1
                for (int o = 0; o < 32; ++o) {
                    const int other = __shfl_sync(0xffffffffu, len, o), its = __shfl_sync(0xffffffffu, tiles, o);
                    if (other > len || (other == len && o < lane)) ahead += its;
                }
            } else {
                int sum = tiles;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int other = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += other;
                }
                ahead += sum - tiles;
            }
            const int at = __ffs(__ballot_sync(0xffffffffu, u >= ahead && u - ahead < tiles)) - 1;
            const int tiles_before = __shfl_sync(0xffffffffu, ahead, at);
            tiles = __shfl_sync(0xffffffffu, tiles, at);
            r.seq = base + at;
            r.row0 = (tiles - 1 - (u - tiles_before)) * tile_rows;
            r.n = __shfl_sync(0xffffffffu, n, at);
            r.len = __shfl_sync(0xffffffffu, len, at);
            r.first = __shfl_sync(0xffffffffu, first, at);
            return r;
        }
        before += all;
    }
    return r;
}

// Token and head of row `row`, then of every `step`-th row after it.
struct RowWalk {
    int32_t token, head, group, last, token_step, head_step;
    __device__ __forceinline__ RowWalk(const ChunkArgs& a, int kvh, int row, int step)
        : token(row / a.group), head(kvh * a.group + row - token * a.group), group(a.group), last((kvh + 1) * a.group),
          token_step(step / a.group), head_step(step - token_step * a.group) {}
    __device__ __forceinline__ void next() {
        token += token_step;
        head += head_step;
        if (head >= last) {
            head -= group;
            ++token;
        }
    }
};

// Keys [0, sink) and [low, end) are what a query sees.
struct Seen {
    int32_t sink, low, end;
};

__device__ __forceinline__ Seen chunk_seen(const ChunkArgs& a, const ChunkUnit& u, int row) {
    const int32_t p = u.len - u.n + row / a.group;
    const int32_t e = p < 0 ? 0 : (a.block == 1 ? p + 1 : (p / a.block + 1) * a.block);
    Seen s;
    s.end = min(e, u.len);
    s.low = min(max(e - a.window, 0), s.end);
    s.sink = min(a.sinks, s.low);
    return s;
}

// The key tiles of a tile of rows: `head` of them from key 0 on (sinks), the others from key `base` on.
struct KeyTiles {
    int32_t head, base, count;
    Seen first, last;  // of the first and the last row: every bound grows with the row
    template <int kKeys>
    __device__ __forceinline__ int32_t key(int i) const {
        return i < head ? i * kKeys : base + (i - head) * kKeys;
    }
    // Whether any row of the tile sees key j.
    __device__ __forceinline__ bool any(int32_t j) const {
        return j < last.end && (j >= first.low || j < last.sink);
    }
};

// Contiguous keys are walked from the first that is seen (a window's tiles are then one fewer on average); in
// pages, tiles start where pages do.
template <int kKeys>
__device__ __forceinline__ KeyTiles chunk_tiles(const ChunkArgs& a, const Seen& first, const Seen& last) {
    KeyTiles t;
    t.first = first;
    t.last = last;
    const int32_t low = min(first.low, last.end);
    t.base = a.table == nullptr ? low : low / kKeys * kKeys;
    t.head = (last.sink + kKeys - 1) / kKeys;
    if (t.head * kKeys > t.base) t.head = t.base = 0;  // the sinks' tiles reach the window's: all from key 0
    t.count = t.head + (last.end - t.base + kKeys - 1) / kKeys;
    return t;
}

// The part [begin, end) of `count` key tiles that split `s` takes. Returns whether the first split
// has them all: it then writes the result itself and kWhole as its partial lse, and the others write nothing.
constexpr float kWhole = INFINITY;
__device__ __forceinline__ bool chunk_part(const ChunkArgs& a, int count, int s, int& begin, int& end) {
    if (a.span > 0) {
        begin = min(s * a.span, count);
        end = min(begin + a.span, count);
        return count <= a.span;
    } else {
        const int each = count / a.splits, more = count - each * a.splits;  // the first `more` parts take one more
        begin = each * s + min(s, more);
        end = begin + each + (s < more);
        return a.splits == 1;
    }
}

// Page of the `box` keys from j on for the K/V tensor maps: `pages` (which reads
// zeros) where no row sees any of them (their page may be long gone) or the table names no page.
__device__ __forceinline__ int32_t chunk_page(const ChunkArgs& a, const ChunkUnit& u, const KeyTiles& t, int32_t j,
                                              int32_t box) {
    if (a.table == nullptr) return u.seq;
    if (j >= t.last.end || (j + box <= t.first.low && j >= t.last.sink)) return a.pages;
    const int32_t at = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
    const int32_t page = __ldg(a.table + static_cast<int64_t>(u.seq) * a.table_width + at);
    if (page < 0 || page >= a.pages) {
        raise_device_error(a.error, ABX_ERR_INVALID_ARGUMENT);
        return a.pages;
    }
    return page;
}

// The row of key j in its page.
__device__ __forceinline__ int32_t chunk_page_row(const ChunkArgs& a, int32_t j) {
    return a.table == nullptr ? j : a.page_shift >= 0 ? j & (a.page_size - 1) : j % a.page_size;
}

// Of K and V: [128, tokens of a page, kv_heads, pages], 64 columns x `rows` tokens a box, 128-byte swizzle.
struct ChunkMaps {
    CUtensorMap k, v;
    CUtensorMap q;  // [128, heads, tokens, sequences], 64 columns x group heads x 128 / group tokens (with q_map)
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z, int32_t w,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// The same by one lane of a converged warp, all operands alike in the warp: the lanes' own coordinates would be
// taken one lane after the other (95 cycles a box against 40).
__device__ __forceinline__ void tma_load_4d_elect(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z, int32_t w,
                                                  uint32_t bar) {
    asm volatile(
        "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
        "@e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];\n}\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// All threads of all CTAs of the cluster; what they wrote before is seen after.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// This CTA's shared address `at`, read in CTA `rank` of the cluster.
__device__ __forceinline__ float cluster_load(uint32_t at, int rank) {
    float x;
    asm volatile("{\n.reg .u32 p;\nmapa.shared::cluster.u32 p, %1, %2;\nld.shared::cluster.f32 %0, [p];\n}\n"
                 : "=f"(x) : "r"(at), "r"(rank) : "memory");
    return x;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t at, int rank) {
    float4 x;
    asm volatile("{\n.reg .u32 p;\nmapa.shared::cluster.u32 p, %4, %5;\nld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n}\n"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at), "r"(rank) : "memory");
    return x;
}

// Weights are held 2^kLift above the row's reference: fp16 ends at 2^-24, which many small weights of a long row
// would reach together (the reference is within 2^8 of the largest, so 2^15 stays below fp16's 2^16).
template <class T>
constexpr float kLift = std::is_same<T, half>::value ? 7.f : 0.f;

// 16-bit pairs of the two element types.
template <class T>
struct Pair;
template <>
struct Pair<bf16> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&p);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
};
template <>
struct Pair<half> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __half2 p = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&p);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
};

// Chooses the kernel (tile_rows) and the splits of a call.
void chunk_layout(ChunkArgs& args);
int64_t chunk_units(const ChunkArgs& args);  // row tiles of a key head, at most
int chunk_tile_keys(const ChunkArgs& args);

// The launchers. Arguments are validated by the C ABI layer.
cudaError_t launch_chunk(const ChunkArgs& args, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream);
cudaError_t launch_chunk_token(const ChunkArgs& args, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream);
cudaError_t launch_chunk_tile(const ChunkArgs& args, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream);
cudaError_t launch_chunk_join(const ChunkArgs& args, bool fp16, cudaStream_t stream);

}  // namespace abx
