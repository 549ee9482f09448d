// Which kernel takes a chunk call, how its keys are shared out to CTAs, and how the shares are joined.
#include <algorithm>

#include "chunk.cuh"

namespace abx {
namespace {

constexpr int kSms = 148;
// Below this many parts of one length, at most eight of them form a cluster (no workspace, one launch);
// from it on, leaving SMs idle would cost more. Four streams of one token over 4,100 keys (9 parts, or 8 in
// a cluster): 22.5 us joined by a second kernel, 20.6 us in the cluster.
constexpr int kClusterUpTo = 16;
// Waves of CTAs for ragged sequences: 48 of up to 16,000 keys take 277 / 266 / 265 / 268 / 282 us with
// 4 / 6 / 8 / 12 / 20, and 292 us with clusters of 7 equal parts (a cluster waits for its slowest CTA).
constexpr int kRaggedWaves = 8;
// ... unless no part of the longest has more tiles than this without them: a part of 16 tiles takes 12 us, a join
// with its launch 8 us more.
constexpr int kRaggedTiles = 16;
// Waves of row tiles up to which a last wave that leaves half the SMs idle may be taken in halves: half a row tile
// takes 0.77 of a whole one's time, so that saves a quarter of a wave at most. 12 heads, 3,600 tokens on themselves (1.2
// waves): 115 us whole, 102.5 us; 24 heads, 1,700 causal (1.1): 48.4 / 41; 16 heads on 4, 8,191 in a window of 1,024
// (3.5): 87.6 / 84.1.
constexpr int kHalvesUpTo = 5;

// Whether the call's row tiles, each taken by the SM that is free first, end sooner when those from job `whole` on
// are taken as two halves. Not always: short row tiles (the first tokens under a causal mask) may fill the last wave
// already, and halves cost half as much again (4 heads, 20,000 tokens in a window of 2,000: 97.7 us whole, 105 us).
bool halves_end_sooner(const ChunkArgs& a, int jobs, int whole) {
    constexpr int kLongest = 64, kRing = 128;  // ticks of the longest row tile
    const int units = jobs / a.kv_heads, half = a.tile_rows / 2, rows = std::min(a.longest * a.group, units * a.tile_rows);
    const int per = (rows + a.tile_rows - 1) / a.tile_rows;  // row tiles of a sequence, the last first
    // In 1/13 of a whole tile's step on 128 keys: about three steps to start and end, and ten for half the rows.
    auto cost = [&](int row0, int count) -> int {
        const int past = std::min(row0 + count, rows);
        if (past <= row0) return 0;
        auto end = [&](int row) {
            const int p = a.keys - a.longest + row / a.group;
            return p < 0 ? 0 : std::min(a.block == 1 ? p + 1 : (p / a.block + 1) * a.block, a.keys);
        };
        const int low = std::max(end(row0) - a.window, 0), keys = end(past - 1) - low + std::min(a.sinks, low);
        return 39 + (keys + kChunkTileKeys - 1) / kChunkTileKeys * (past - row0 <= half ? 10 : 13);
    };
    int of[kHalvesUpTo * kSms], longest = 1;
    for (int x = 0; x < per; ++x) longest = std::max(longest, of[x] = cost((per - 1 - x) * a.tile_rows, a.tile_rows));
    const float scale = static_cast<float>(kLongest - 1) / longest;
    auto ticks = [&](int c) { return c == 0 ? 0 : static_cast<int>(c * scale) + 1; };
    for (int x = 0; x < per; ++x) of[x] = ticks(of[x]);
    struct Sms {
        int16_t free[kRing] = {kSms};  // that become free at a tick
        int now = 0, end = 0;
        void run(int t) {
            if (t == 0) return;
            while (free[now % kRing] == 0) ++now;
            --free[now % kRing];
            ++free[(now + t) % kRing];
            end = std::max(end, now + t);
        }
    } with, without;
    int x = 0;  // the row tile of its sequence
    for (int j = 0; j < whole; ++j, x = x + 1 == per ? 0 : x + 1) without.run(of[x]);
    with = without;
    for (int j = whole; j < jobs; ++j, x = x + 1 == per ? 0 : x + 1) {
        const int row0 = (per - 1 - x) * a.tile_rows;
        without.run(of[x]);
        with.run(ticks(cost(row0, half)));
        with.run(ticks(cost(row0 + half, half)));
    }
    return with.end < without.end;
}

// Whether a call over ragged sequences computes packed token `token`: it lies in a sequence, and that has no more
// tokens than the launch covers. The splits wrote nothing for any other row, so a join leaves it alone.
__device__ __forceinline__ bool chunk_covers(const ChunkArgs& a, int64_t token) {
    int lo = 0, hi = a.seqs;
    if (token < __ldg(a.starts) || token >= __ldg(a.starts + hi)) return false;
    while (hi - lo > 1) {  // starts[lo] <= token < starts[hi]
        const int mid = (lo + hi) >> 1;
        if (__ldg(a.starts + mid) <= token)
            lo = mid;
        else
            hi = mid;
    }
    int32_t first, n, len;
    bool bad;
    chunk_sequence(a, lo, first, n, len, bad);
    return token < first + n;
}

// Joins the splits of each row: o = sum_s 2^(lse_s - lse) o_s. A block a row, four dims a lane, each warp an
// eighth of the splits; reads splits * 516 bytes a row.
template <class T>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChunkArgs a) {
    constexpr int kWarps = 8;
    __shared__ float4 part[kWarps][32];
    __shared__ float2 stat[kWarps];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x;
    const int64_t token = row / a.heads;
    const int head = static_cast<int>(row - token * a.heads);
    int64_t seq = 0, at = token;
    bool mine = true;
    if (a.starts == nullptr) {
        seq = token / a.tokens;
        at = token - seq * a.tokens;
    } else {
        mine = chunk_covers(a, token);  // else left as it was; read while the last splits still run
    }
    cudaGridDependencySynchronize();
    if (!mine) return;
    if (a.span > 0 && a.part_lse[row] == kWhole) return;  // written by its only split
    // This warp's splits w, w + 8, ..: 32 at a time, their sums' weights against a running maximum.
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = w; base < a.splits; base += 32 * kWarps) {
        const int s = base + lane * kWarps;
        const float x = s < a.splits ? a.part_lse[s * a.rows_total + row] : -INFINITY;
        float next = x;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, d));
        next = fmaxf(next, top);
        if (next == -INFINITY && !__any_sync(0xffffffffu, isnan(x))) continue;
        const float scale = next == top ? 1.f : exp2f(top - next), f = exp2f(x - next);  // a NaN stays one
        top = next;
        sum = sum * scale + f;
        acc.x *= scale, acc.y *= scale, acc.z *= scale, acc.w *= scale;
        const int count = min(32, (a.splits - base + kWarps - 1) / kWarps);
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(
                a.part_o + (static_cast<int64_t>(base + i * kWarps) * a.rows_total + row) * 128 + 4 * lane);
            const float fi = __shfl_sync(0xffffffffu, f, i);
            acc.x += fi * v.x;
            acc.y += fi * v.y;
            acc.z += fi * v.z;
            acc.w += fi * v.w;
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    part[w][lane] = acc;
    if (lane == 0) stat[w] = make_float2(top, sum);
    __syncthreads();
    if (w != 0) return;
    top = -INFINITY;
    bool reached = false;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        top = fmaxf(top, stat[i].x);
        reached |= stat[i].y != 0.f;
    }
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (reached) {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float f = exp2f(stat[i].x - top);
            const float4 v = part[i][lane];
            sum += f * stat[i].y;
            acc.x += f * v.x;
            acc.y += f * v.y;
            acc.z += f * v.z;
            acc.w += f * v.w;
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const uint2 pair = make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + seq * a.o_seq + head * a.o_head + at * a.o_token + 4 * lane) = pair;
    if (a.lse != nullptr && lane == 0)
        a.lse[seq * a.l_seq + head * a.l_head + at * a.l_token] = sum == 0.f ? -INFINITY : top + log2f(sum);
}

// The same for many rows: eight lanes a row, 16 dims a lane, so that a warp has four rows in flight and all loads of
// a row's splits (eight at a time) go out together.
template <class T>
__global__ void __launch_bounds__(256) chunk_join_rows_kernel(const ChunkArgs a) {
    const int lane = threadIdx.x & 7;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 3);
    const int64_t token = row / a.heads;
    const int head = static_cast<int>(row - token * a.heads);
    int64_t seq = 0, at = token;
    bool mine = row < a.rows_total;
    if (a.starts == nullptr) {
        seq = token / a.tokens;
        at = token - seq * a.tokens;
    } else {
        mine = mine && chunk_covers(a, token);  // else left as it was; read while the last splits still run
    }
    cudaGridDependencySynchronize();
    if (mine && a.span > 0) mine = a.part_lse[row] != kWhole;  // written by its only split
    const unsigned lanes = 0xffu << (threadIdx.x & 24);
    if (!mine) return;  // whole groups of eight lanes
    float top = -INFINITY, sum = 0.f;
    float4 acc[4] = {};
    for (int base = 0; base < a.splits; base += 8) {
        const float x = base + lane < a.splits ? a.part_lse[static_cast<int64_t>(base + lane) * a.rows_total + row] : -INFINITY;
        float next = x;
#pragma unroll
        for (int d = 4; d > 0; d /= 2) next = fmaxf(next, __shfl_xor_sync(lanes, next, d));
        next = fmaxf(next, top);
        if (next == -INFINITY && !__any_sync(lanes, isnan(x))) continue;
        const float scale = next == top ? 1.f : exp2f(top - next), f = exp2f(x - next);  // a NaN stays one
        top = next;
        sum = sum * scale + f;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k].x *= scale, acc[k].y *= scale, acc[k].z *= scale, acc[k].w *= scale;
        const int count = min(8, a.splits - base);
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
            const float4* from =
                reinterpret_cast<const float4*>(a.part_o + (static_cast<int64_t>(base + i) * a.rows_total + row) * 128) + lane;
            const float fi = __shfl_sync(lanes, f, i, 8);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 v = from[8 * k];
                acc[k].x += fi * v.x;
                acc[k].y += fi * v.y;
                acc[k].z += fi * v.z;
                acc[k].w += fi * v.w;
            }
        }
    }
#pragma unroll
    for (int d = 4; d > 0; d /= 2) sum += __shfl_xor_sync(lanes, sum, d);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.o) + seq * a.o_seq + head * a.o_head + at * a.o_token + 4 * lane;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint2*>(out + 32 * k) =
            make_uint2(Pair<T>::pack(acc[k].x * inv, acc[k].y * inv), Pair<T>::pack(acc[k].z * inv, acc[k].w * inv));
    if (a.lse != nullptr && lane == 0)
        a.lse[seq * a.l_seq + head * a.l_head + at * a.l_token] = sum == 0.f ? -INFINITY : top + log2f(sum);
}

// The join starts while the last CTAs of the splits still run, and waits for them itself.
template <class Kernel>
cudaError_t launch_join(Kernel kernel, int rows, const ChunkArgs& a, cudaStream_t stream) {
    const int64_t blocks = ceil_div(a.rows_total, rows);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.blockDim = dim3(256);
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, a);
}

}  // namespace

int64_t chunk_units(const ChunkArgs& a) {
    const int64_t units = a.seqs * ceil_div(static_cast<int64_t>(a.longest) * a.group, a.tile_rows);
    if (a.starts == nullptr) return units;
    const int64_t ragged = static_cast<int64_t>(a.tokens) * a.group / a.tile_rows + a.seqs;
    return ragged < units ? ragged : units;
}

void chunk_layout(ChunkArgs& a) {
    const int64_t rows = static_cast<int64_t>(a.longest) * a.group;
    a.tile_rows = rows <= 16 ? 16 : 32;
    if (rows > 32) {
        // More rows than one tile of the few-row kernel: it still is the faster one while all its CTAs run at once
        // and have little to do (it starts in 6 us where the tile kernel takes 10). us of the few-row / the tile kernel,
        // by 64-key steps: 8 heads on 2, 100 tokens on 100 keys 9.9 / 13.2 (52 steps), 200 on 200 12.0 / 14.8
        // (200), 100 on 2,000 16.7 / 20.5 (832), 40 on 8,000 24.8 / 20.9 (1,250); 12 heads, 100 on 2,000 36 / 19 (1,536).
        const int64_t ctas = chunk_units(a) * a.kv_heads;
        const int64_t steps = ctas * ceil_div(a.keys, kChunkTokenKeys) / (a.starts != nullptr && a.seqs > 1 ? 2 : 1);
        if (ctas > kSms || steps > 5 * kSms) a.tile_rows = 256;
    }
    const int tile_keys = chunk_tile_keys(a);
    const int64_t ctas = chunk_units(a) * a.kv_heads;
    // Keys that one row tile can see, in tiles; the lengths themselves are known on the device only.
    int64_t keys = a.keys;
    if (a.window != kNoWindow) {
        const int64_t seen = static_cast<int64_t>(a.window) + a.sinks + a.block + a.tile_rows + 3 * tile_keys;
        if (seen < keys) keys = seen;
    }
    const int64_t tiles = ceil_div(keys, tile_keys);
    if (a.tile_rows < 256) {
        // CTAs that fit the GPU at a time, and the parts of a row tile's keys that one wave of them has room for; no
        // part under four tiles.
        const int64_t slots = kSms * (a.tile_rows == 16 ? 2 : 1);
        const bool ragged = a.starts != nullptr && a.seqs > 1;
        const int64_t most = ceil_div(tiles, 4), room = slots / ctas < most ? slots / ctas : most;
        const int64_t joined = room < kMaxCluster ? room : kMaxCluster;
        a.span = 0;
        if (room < kClusterUpTo && (!ragged || ceil_div(tiles, joined < 1 ? 1 : joined) <= kRaggedTiles)) {
            a.splits = static_cast<int32_t>(joined < 1 ? 1 : joined);  // equal parts, joined in a cluster
            a.cluster = a.splits > 1;
        } else if (!ragged) {
            a.splits = static_cast<int32_t>(room);  // few and long: equal parts, joined through the workspace
        } else {
            // Ragged and long: equal spans, joined through the workspace, that come to several waves if all sequences
            // were as long as the table allows (the lengths are on the device), so that they still balance.
            const int64_t want = ceil_div(slots * kRaggedWaves, ctas), parts = want > most ? most : want;
            a.span = static_cast<int32_t>(ceil_div(tiles, parts));
            a.splits = static_cast<int32_t>(ceil_div(tiles, a.span));
        }
        return;
    }
    // Equal parts, as many as make the waves of CTAs (one an SM) shortest: a part costs its tiles and
    // about three more to start and end, joining costs a write and a read of each part's rows. Ragged: equal spans. The
    // longest sequences come first, so the end is the longest job's, or the mean SM's and some of a job; the lengths,
    // known on the device only, are taken as half the table's on average. Nine of 30 to 701 tokens over up to 8,000
    // keys, 16 heads on 4: 159 us (one part) against 186 in the order of the sequences (two parts).
    const bool ragged = a.starts != nullptr && a.seqs > 1;
    a.sorted = ragged;
    a.span = 0;
    a.splits = 1;
    double best = 0;
    for (int s = 1; s <= (ragged ? 32 : 16) && s <= tiles && (s == 1 || !ragged || 8 * (s - 1) < tiles); ++s) {
        const double part = static_cast<double>(ceil_div(tiles, s)) + 3;
        const double join = s == 1 ? 0 : 2 + s * static_cast<double>(a.rows_total) * 1032 / 11e6;  // in tiles of 1.7 us
        const double cost = join + (ragged ? std::max(part, ctas * (0.5 * tiles + 3) / kSms + part / 3) : ceil_div(ctas * s, kSms) * part);
        if (s == 1 || cost < 0.97 * best) {
            best = cost;
            a.splits = s;
        }
    }
    if (ragged) {
        a.span = static_cast<int32_t>(ceil_div(tiles, a.splits));
        a.splits = static_cast<int32_t>(ceil_div(tiles, a.span));
    }
}

int chunk_tile_keys(const ChunkArgs& a) { return a.tile_rows < 256 ? kChunkTokenKeys : kChunkTileKeys; }

cudaError_t launch_chunk(const ChunkArgs& a, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream) {
    if (a.tile_rows < 256) return launch_chunk_token(a, maps, fp16, box_rows, stream);
    ChunkArgs b = a;
    const int64_t ctas = chunk_units(a) * a.kv_heads, over = ctas % kSms;
    if (a.splits == 1 && !a.sorted && over > 0 && 2 * over <= kSms && ctas <= kHalvesUpTo * kSms &&
        halves_end_sooner(a, static_cast<int>(ctas), static_cast<int>(ctas - over))) {
        b.units = static_cast<int32_t>(ctas / a.kv_heads);
        b.whole_jobs = static_cast<int32_t>(ctas - over);
    }
    return launch_chunk_tile(b, maps, fp16, box_rows, stream);
}

cudaError_t launch_chunk_join(const ChunkArgs& a, bool fp16, cudaStream_t stream) {
    // A block a row while there are few rows: the splits' loads are what a row waits for.
    if (a.rows_total <= 8 * kSms)
        return fp16 ? launch_join(chunk_join_kernel<half>, 1, a, stream) : launch_join(chunk_join_kernel<bf16>, 1, a, stream);
    return fp16 ? launch_join(chunk_join_rows_kernel<half>, 32, a, stream)
                : launch_join(chunk_join_rows_kernel<bf16>, 32, a, stream);
}

}  // namespace abx
