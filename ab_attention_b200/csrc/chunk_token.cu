// Few rows against many keys: attention of single tokens (and of a few) over the cache.
//
// One CTA takes one tile of 16 or 32 rows ((token, head) pairs that share a key
// head) and a part of its keys, so each key is read once for all heads of its
// group. It is bound by reading K and V: a ring of three 64-key tiles (32 KB each)
// filled by TMA keeps up to 192 KB in flight an SM (two CTAs of 16 rows). The four
// consumer warps take 16 keys of every tile each, with a softmax of their own (running
// maximum and sum in 32 bits), so the loop has no barrier among them; they are joined
// once, at the end, through shared memory. mma.sync, not tcgen05: at most 32 rows would
// fill a quarter of a 128-row tile, and the products are 30% of the tensor pipe as it is.
// P goes into its product as two terms of the element type, rounded and rest: 3% of the
// time, and the rounding of the weights no longer shows in short outputs.
// With few sequences the keys are split over CTAs as well, joined in a cluster (up to
// eight) or by a second kernel. One token of 12 heads over 131,001 keys in pages
// of 16: 131 us (6.1 TB/s, 94% of the copy rate); 48 ragged sequences, 32 heads on 8:
// 268 us (5.9 TB/s).
#include <type_traits>

#include "chunk.cuh"
#include "tcgen05.cuh"

namespace abx {
namespace {

constexpr int kKeys = kChunkTokenKeys;          // keys of a tile
constexpr int kWarpKeys = 16;
constexpr int kWarps = kKeys / kWarpKeys;       // consumers
constexpr int kThreads = (kWarps + 1) * 32;     // and the loader
constexpr int kStages = 3;
constexpr uint32_t kSlab = kKeys * 128;         // 64 keys x 64 columns
constexpr uint32_t kOperand = 2 * kSlab;        // K or V of a tile
constexpr uint32_t kStage = 2 * kOperand;
constexpr uint64_t kWaitLimit = 400ull * 1000 * 1000;
constexpr float kGrow = 8.0f;  // log2: rows are rescaled only when their maximum grows by more

template <int MT>
struct Layout {
    static constexpr int rows = 16 * MT;
    static constexpr uint32_t q = kStages * kStage;
    static constexpr uint32_t stats = q + rows * 256;              // m, l of each warp and row
    static constexpr uint32_t bars = stats + kWarps * rows * 8;
    static constexpr uint32_t abort_flag = bars + 8 * (3 * kStages);
    static constexpr uint32_t bytes = abort_flag + 16 + 1024;
    static_assert((kWarps + 1) * rows * 128 * 4 + rows * 4 <= kStages * kStage, "the join reuses the ring");
};

template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, bf16>::value) {
        mma_bf16_16816(d, a, b0, b1);
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// Byte offset of 16-byte chunk c (0..15) of row r in a swizzled tile whose 64-column slabs are `slab` bytes.
__device__ __forceinline__ uint32_t chunk_at(int r, int c, uint32_t slab) {
    return (c >> 3) * slab + r * 128 + (((c ^ r) & 7) << 4);
}

template <class T, int MT>
__global__ void __launch_bounds__(kThreads) chunk_token_kernel(const ChunkArgs a, const __grid_constant__ ChunkMaps maps,
                                                              const int box_rows) {
    using L = Layout<MT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* mem = smem_raw + (base - raw);
    const uint32_t bars = base + L::bars;
    auto k_full = [&](int st) { return bars + 8u * st; };
    auto v_full = [&](int st) { return bars + 8u * (kStages + st); };
    auto empty = [&](int st) { return bars + 8u * (2 * kStages + st); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + L::abort_flag);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.z, kvh = blockIdx.y;
    const ChunkUnit u = chunk_unit(a, blockIdx.x, L::rows, false);
    if (u.seq < 0) return;  // past the last tile
    const int rows = min(L::rows, u.n * a.group - u.row0);
    const KeyTiles t = chunk_tiles<kKeys>(a, chunk_seen(a, u, u.row0), chunk_seen(a, u, u.row0 + rows - 1));
    int begin, end;
    const bool whole = chunk_part(a, t.count, split, begin, end);
    if (whole && split > 0) return;
    const int n = end - begin;

    cudaTriggerProgrammaticLaunchCompletion();  // the join may come onto the GPU; it waits for this grid's end
    if (tid == 0) {
        *abort_flag = 0;
        for (int st = 0; st < kStages; ++st) {
            tc::mbar_init(k_full(st), 1);
            tc::mbar_init(v_full(st), 1);
            tc::mbar_init(empty(st), kWarps);
        }
        tc::mbar_init_fence();
    }
    if (warp == kWarps && lane < 2) prefetch_map(lane ? &maps.v : &maps.k);
    __syncthreads();

    float* stat_m = reinterpret_cast<float*>(mem + L::stats);
    float* stat_l = stat_m + kWarps * L::rows;
    float o[MT][16][4];
    if (warp == kWarps) {
        // ---- loader: one box a lane ----
        const int boxes = kKeys / box_rows;  // of one slab
        const int op = lane / (2 * boxes), rest = lane % (2 * boxes), slab = rest & 1, box = rest >> 1;
        const uint32_t to = op * kOperand + slab * kSlab + box * box_rows * 128;
        auto key = [&](int i) { return t.key<kKeys>(begin + i) + box * box_rows; };
        int32_t page = lane < 4 * boxes && n > 0 ? chunk_page(a, u, t, key(0), box_rows) : 0;
        int issued = 0;
        for (int i = 0; i < n; ++i) {
            const int st = i % kStages, use = i / kStages;
            // the next tile's page is looked up while this one waits for its place
            const int32_t next = lane < 4 * boxes && i + 1 < n ? chunk_page(a, u, t, key(i + 1), box_rows) : 0;
            const bool free_ok =
                use == 0 || tc::mbar_wait_suspend(empty(st), (use - 1) & 1, abort_flag, kWaitLimit);
            if (!__all_sync(0xffffffffu, free_ok)) break;
            issued = i + 1;
            if (lane == 0) {
                tc::mbar_arrive_expect_tx(k_full(st), kOperand);
                tc::mbar_arrive_expect_tx(v_full(st), kOperand);
            }
            __syncwarp();
            if (lane < 4 * boxes)
                tma_load_4d(base + st * kStage + to, op ? &maps.v : &maps.k, 64 * slab, chunk_page_row(a, key(i)),
                            kvh, page, op ? v_full(st) : k_full(st));
            page = next;
            __syncwarp();
        }
        if (lane == 0) {  // every copy has landed before the ring is used for anything else
            for (int st = 0; st < kStages && st < issued; ++st) {
                const int last = (issued - 1 - st) / kStages;
                tc::mbar_wait_suspend(k_full(st), last & 1, abort_flag, kWaitLimit, /*honor_abort=*/false);
                tc::mbar_wait_suspend(v_full(st), last & 1, abort_flag, kWaitLimit, /*honor_abort=*/false);
            }
        }
        __syncwarp();
    } else {
        // ---- consumers: keys [16 * warp, 16 * warp + 16) of every tile ----
        float m[MT][2], l[MT][2];
        Seen seen[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                m[i][h] = -INFINITY;
                l[i][h] = 0.f;
                seen[i][h] = chunk_seen(a, u, u.row0 + min(16 * i + 8 * h + (lane >> 2), rows - 1));
            }
#pragma unroll
            for (int d = 0; d < 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][d][e] = 0.f;
        }
        // The rows' queries, zeros past the last row (the first tiles are on their way meanwhile).
        if (n > 0) {
            for (int i = tid; i < L::rows * 16; i += kWarps * 32) {
                const int r = i >> 4, c = i & 15;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (r < rows) {
                    const int token = (u.row0 + r) / a.group, head = kvh * a.group + (u.row0 + r) % a.group;
                    x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + u.seq * a.q_seq + head * a.q_head +
                                                        (u.first + token) * a.q_token + c * 8);
                }
                *reinterpret_cast<uint4*>(mem + L::q + chunk_at(r, c, L::rows * 128)) = x;
            }
        }
        asm volatile("bar.sync 1, %0;\n" ::"n"(kWarps * 32) : "memory");
        const int mat = lane >> 3, mr = lane & 7;
        auto load_q = [&](uint32_t (&qa)[4], int x, int step) {
            ldmatrix_x4(qa, base + L::q + chunk_at(16 * x + (mat & 1) * 8 + mr, 2 * step + (mat >> 1), L::rows * 128));
        };
        uint32_t q1[MT == 1 ? 8 : 1][4];  // 16 rows stay in registers; 32 are read again for each tile
        if constexpr (MT == 1) {
#pragma unroll
            for (int step = 0; step < 8; ++step) load_q(q1[step], 0, step);
        }
        for (int i = 0; i < n; ++i) {
            const int st = i % kStages;
            const uint32_t phase = (i / kStages) & 1;
            const uint32_t kbase = base + st * kStage, vbase = kbase + kOperand;
            const int32_t k0 = t.key<kKeys>(begin + i) + warp * kWarpKeys;
            if (!tc::mbar_wait_warp_suspend(k_full(st), phase, abort_flag, kWaitLimit)) break;
            // S = Q K^T for 16 keys (two 8-key column tiles), dims in eight steps of 16.
            float s[MT][2][4];
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[x][y][e] = 0.f;
#pragma unroll
            for (int step = 0; step < 8; ++step) {
                uint32_t kb[4];
                ldmatrix_x4(kb, kbase + chunk_at(warp * kWarpKeys + (mat >> 1) * 8 + mr, 2 * step + (mat & 1), kSlab));
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    uint32_t q2[4];
                    if constexpr (MT > 1) load_q(q2, x, step);
                    const uint32_t (&qa)[4] = MT == 1 ? q1[step] : q2;
                    mma_16816<T>(s[x][0], qa, kb[0], kb[1]);
                    mma_16816<T>(s[x][1], qa, kb[2], kb[3]);
                }
            }
            // Keys that a row does not see -> -inf (only where the tile is not seen whole by all rows).
            if (k0 + kWarpKeys > t.first.end || (k0 < t.last.low && k0 + kWarpKeys > t.first.sink)) {
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int32_t j = k0 + 8 * y + 2 * (lane & 3) + (e & 1);
                            const Seen& w = seen[x][e >> 1];
                            if (!(j < w.end && (j >= w.low || j < w.sink))) s[x][y][e] = -INFINITY;
                        }
            }
            uint32_t p[MT][4], rest[MT][4];
#pragma unroll
            for (int x = 0; x < MT; ++x) {
                // The maximum is kept as the bare score: s - m is exact where it matters, so the
                // largest weight of a row is 1 (or 2^8 at most) however large the scores are, times 2^kLift.
                float top[2];
                bool grow = false;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v = fmaxf(fmaxf(s[x][0][2 * h], s[x][0][2 * h + 1]), fmaxf(s[x][1][2 * h], s[x][1][2 * h + 1]));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                    top[h] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                    grow |= (top[h] - m[x][h]) * a.kappa > kGrow;
                }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float next = fmaxf(m[x][h], top[h]);
                        const float scale = next == -INFINITY ? 1.f : exp2f((m[x][h] - next) * a.kappa);
                        m[x][h] = next;
                        l[x][h] *= scale;
#pragma unroll
                        for (int d = 0; d < 16; ++d) {
                            o[x][d][2 * h] *= scale;
                            o[x][d][2 * h + 1] *= scale;
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float shift = m[x][h] == -INFINITY ? 0.f : m[x][h];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float p0 = exp2f(fmaf(s[x][y][2 * h] - shift, a.kappa, kLift<T>));
                        const float p1 = exp2f(fmaf(s[x][y][2 * h + 1] - shift, a.kappa, kLift<T>));
                        l[x][h] += p0 + p1;
                        p[x][2 * y + h] = Pair<T>::pack(p0, p1);
                        const float2 r = Pair<T>::unpack(p[x][2 * y + h]);
                        rest[x][2 * y + h] = Pair<T>::pack(p0 - r.x, p1 - r.y);
                    }
                }
            }
            if (!tc::mbar_wait_warp_suspend(v_full(st), phase, abort_flag, kWaitLimit)) break;
            // V rows that no row sees (a page's stale tail) must not meet P = 0 as NaN or infinity.
            if (!(t.any(k0) && t.any(k0 + kWarpKeys - 1)) ||
                (k0 < t.first.low && k0 + kWarpKeys > t.last.sink)) {
                for (int x = lane; x < kWarpKeys * 16; x += 32)
                    if (!t.any(k0 + (x >> 4)))
                        *reinterpret_cast<uint4*>(mem + st * kStage + kOperand +
                                                  chunk_at(warp * kWarpKeys + (x >> 4), x & 15, kSlab)) =
                            make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            // O += P V: V as [key][dim], transposed by the load; 16 dims a step.
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                uint32_t vb[4];
                ldmatrix_x4_trans(vb, vbase + chunk_at(warp * kWarpKeys + (mat & 1) * 8 + mr, 2 * d + (mat >> 1), kSlab));
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    mma_16816<T>(o[x][2 * d], p[x], vb[0], vb[1]);
                    mma_16816<T>(o[x][2 * d + 1], p[x], vb[2], vb[3]);
                    mma_16816<T>(o[x][2 * d], rest[x], vb[0], vb[1]);
                    mma_16816<T>(o[x][2 * d + 1], rest[x], vb[2], vb[3]);
                }
            }
            // The next copy into this stage is another proxy's write: an arrival alone does not keep it behind the
            // warp's reads (and clears). Without the fence, reads that waited behind other traffic of the SM, a storm
            // of atomics say, found the tile three on.
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(empty(st));
        }
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], 1);
                l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], 2);
                if ((lane & 3) == 0) {
                    const int r = 16 * x + 8 * h + (lane >> 2);
                    stat_m[warp * L::rows + r] = m[x][h] * a.kappa - kLift<T>;
                    stat_l[warp * L::rows + r] = l[x][h];
                }
            }
    }
    __syncthreads();  // the ring is free
    float* part = reinterpret_cast<float*>(mem);  // [warp][row][128]
    if (warp < kWarps && n > 0) {
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int d = 0; d < 16; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float2*>(part + (warp * L::rows + 16 * x + 8 * h + (lane >> 2)) * 128 + 8 * d +
                                               2 * (lane & 3)) = make_float2(o[x][d][2 * h], o[x][d][2 * h + 1]);
    }
    __syncthreads();
    // The CTA's own result, where the other CTAs of its cluster read it.
    float* share = part + kWarps * L::rows * 128;  // [row][128]
    float* share_lse = share + L::rows * 128;
    // Join the warps: weight 2^(m_w - m); a row that nothing reached gives zeros and -inf.
    for (int i = tid; i < rows * 32; i += kThreads) {
        const int r = i >> 5, c = (i & 31) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n > 0) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat_m[w * L::rows + r]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = stat_m[w * L::rows + r];
                const float f = mw == -INFINITY ? 0.f : exp2f(mw - top);
                const float4 x = *reinterpret_cast<const float4*>(part + (w * L::rows + r) * 128 + c);
                sum += f * stat_l[w * L::rows + r];
                acc.x += f * x.x;
                acc.y += f * x.y;
                acc.z += f * x.z;
                acc.w += f * x.w;
            }
        }
        // NaN (from a NaN among the row's own inputs) passes through.
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float lse = sum == 0.f ? -INFINITY : top + log2f(sum);
        const int token = (u.row0 + r) / a.group, head = kvh * a.group + (u.row0 + r) % a.group;
        if (a.cluster) {
            *reinterpret_cast<float4*>(share + r * 128 + c) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            if (c == 0) share_lse[r] = lse;
        } else if (!whole) {
            const int64_t tokens_before = a.starts ? u.first : static_cast<int64_t>(u.seq) * a.tokens;
            const int64_t at = split * a.rows_total + (tokens_before + token) * a.heads + head;
            *reinterpret_cast<float4*>(a.part_o + at * 128 + c) =
                make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            if (c == 0) a.part_lse[at] = lse;
        } else {
            uint2 pair = make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
            *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + u.seq * a.o_seq + head * a.o_head +
                                      (u.first + token) * a.o_token + c) = pair;
            if (a.lse != nullptr && c == 0) a.lse[u.seq * a.l_seq + head * a.l_head + (u.first + token) * a.l_token] = lse;
            if (a.splits > 1 && c == 0) a.part_lse[static_cast<int64_t>(u.first + token) * a.heads + head] = kWhole;
        }
    }
    if (a.cluster) {
        // Up to eight splits form a cluster: its CTAs join the rows over distributed shared memory, each
        // every splits-th row.
        cluster_sync();
        for (int r = split + a.splits * warp; r < rows; r += a.splits * (kWarps + 1)) {
            const uint32_t at = smem_addr(share + r * 128 + 4 * lane), at_lse = smem_addr(share_lse + r);
            float lse[kMaxCluster];
            float4 x[kMaxCluster];
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int s = 0; s < kMaxCluster; ++s)
                if (s < a.splits) {
                    lse[s] = cluster_load(at_lse, s);
                    x[s] = cluster_load4(at, s);
                }
            bool reached = false;
#pragma unroll
            for (int s = 0; s < kMaxCluster; ++s)
                if (s < a.splits) {
                    top = fmaxf(top, lse[s]);
                    reached |= lse[s] != -INFINITY;  // a NaN reaches too, and stays one
                }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            if (reached) {
#pragma unroll
                for (int s = 0; s < kMaxCluster; ++s)
                    if (s < a.splits) {
                        const float f = exp2f(lse[s] - top);
                        sum += f;
                        acc.x += f * x[s].x;
                        acc.y += f * x[s].y;
                        acc.z += f * x[s].z;
                        acc.w += f * x[s].w;
                    }
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int token = (u.row0 + r) / a.group, head = kvh * a.group + (u.row0 + r) % a.group;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + u.seq * a.o_seq + head * a.o_head +
                                      (u.first + token) * a.o_token + 4 * lane) =
                make_uint2(Pair<T>::pack(acc.x * inv, acc.y * inv), Pair<T>::pack(acc.z * inv, acc.w * inv));
            if (a.lse != nullptr && lane == 0)
                a.lse[u.seq * a.l_seq + head * a.l_head + (u.first + token) * a.l_token] =
                    sum == 0.f ? -INFINITY : top + log2f(sum);
        }
        cluster_sync();  // nobody leaves while its rows are read
    }
    if (tid == 0 && *abort_flag) raise_device_error(a.error, ABX_ERR_DEVICE_TIMEOUT);
}

template <class T, int MT>
cudaError_t launch(const ChunkArgs& a, const ChunkMaps& maps, int box_rows, cudaStream_t stream) {
    using L = Layout<MT>;
    auto kernel = chunk_token_kernel<T, MT>;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(L::bytes));
    if (err != cudaSuccess) return err;
    const int64_t units = chunk_units(a);
    if (units > 0x7fffffff || a.splits > 65535) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = cluster.val.clusterDim.y = 1;
    cluster.val.clusterDim.z = a.cluster ? a.splits : 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(units), a.kv_heads, a.splits);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = L::bytes;
    config.stream = stream;
    config.attrs = &cluster;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, a, maps, box_rows);
}

}  // namespace

cudaError_t launch_chunk_token(const ChunkArgs& a, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream) {
    const bool narrow = a.tile_rows == 16;
    if (fp16) return narrow ? launch<half, 1>(a, maps, box_rows, stream) : launch<half, 2>(a, maps, box_rows, stream);
    return narrow ? launch<bf16, 1>(a, maps, box_rows, stream) : launch<bf16, 2>(a, maps, box_rows, stream);
}

}  // namespace abx
