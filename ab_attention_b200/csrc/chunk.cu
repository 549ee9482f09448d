// Which kernel takes a chunk call, how its keys are shared out to CTAs, and how the shares are joined.
#include "chunk.cuh"

namespace abx {
namespace {

constexpr int kSms = 148;

// Joins the splits of each row: o = sum_s 2^(lse_s - lse) o_s. One warp a row, four dims a lane;
// reads splits * 516 bytes a row.
template <class T>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChunkArgs a) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= a.rows_total) return;
    const int64_t token = row / a.heads;
    const int head = static_cast<int>(row - token * a.heads);
    int64_t seq = 0, at = token;
    if (a.starts == nullptr) {
        seq = token / a.tokens;
        at = token - seq * a.tokens;
    } else if (token < __ldg(a.starts) || token >= __ldg(a.starts + a.seqs)) {
        return;  // in no sequence: left as it was
    }
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * a.rows_total + row]);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float x = a.part_lse[s * a.rows_total + row];
        if (x == -INFINITY) continue;
        const float f = exp2f(x - top);
        const float4 v = *reinterpret_cast<const float4*>(a.part_o + (s * a.rows_total + row) * 128 + 4 * lane);
        sum += f;
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 pair = make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + seq * a.o_seq + head * a.o_head + at * a.o_token + 4 * lane) = pair;
    if (a.lse != nullptr && lane == 0)
        a.lse[seq * a.l_seq + head * a.l_head + at * a.l_token] = sum == 0.f ? -INFINITY : top + log2f(sum);
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
    a.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 256;
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
        // Equal spans: about eight CTAs an SM if every sequence were as long as its table allows, so a
        // ragged batch still balances; no span under four tiles.
        const int64_t span = ceil_div(ctas * tiles, kSms * 8);
        a.span = static_cast<int32_t>(span < 4 ? 4 : span);
        a.splits = static_cast<int32_t>(ceil_div(tiles, a.span));
        return;
    }
    // Equal parts, as many as make the waves of CTAs (one an SM) shortest: a part costs its tiles and
    // about three more to start and end, joining costs a write and a read of each part's rows.
    a.span = 0;
    a.splits = 1;
    double best = 0;
    for (int s = 1; s <= 16 && s <= tiles; ++s) {
        const double waves = static_cast<double>(ceil_div(ctas * s, kSms));
        const double join = s == 1 ? 0 : 2 + s * static_cast<double>(a.rows_total) * 1032 / 11e6;  // in tiles of 1.7 us
        const double cost = waves * (static_cast<double>(ceil_div(tiles, s)) + 3) + join;
        if (s == 1 || cost < 0.97 * best) {
            best = cost;
            a.splits = s;
        }
    }
}

int chunk_tile_keys(const ChunkArgs& a) { return a.tile_rows < 256 ? kChunkTokenKeys : kChunkTileKeys; }

cudaError_t launch_chunk(const ChunkArgs& a, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream) {
    return a.tile_rows < 256 ? launch_chunk_token(a, maps, fp16, box_rows, stream)
                             : launch_chunk_tile(a, maps, fp16, box_rows, stream);
}

cudaError_t launch_chunk_join(const ChunkArgs& a, bool fp16, cudaStream_t stream) {
    const int64_t blocks = ceil_div(a.rows_total, 8);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    if (fp16)
        chunk_join_kernel<half><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    else
        chunk_join_kernel<bf16><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace abx
