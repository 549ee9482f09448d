// Many rows against many keys: attention of chunks of tokens on the tensor cores (tcgen05).
//
// One CTA takes 256 rows (two groups of 128, one TMEM lane and one softmax thread a
// row) of one key head and walks the 128-key tiles that any of them sees; K and V
// tiles are read once for both groups. Per tile and group:
//     S = Q K^T (TMEM, f32)  ->  P = 2^((s - m) * kappa) (registers, then shared memory, 16 bits)  ->  O += P V (TMEM, f32)
// A softmax thread takes its whole S row into registers at once, which frees the S
// columns: the product for the next tile runs while this tile's exponentials do,
// because P goes to shared memory and not over S. A group's chain is then its
// softmax alone, and the two groups share the tensor pipe and the exponential unit.
// Bounds for a tile of both groups, in SM cycles: tensor pipe 2,048 (four products of
// 128^3), exponential unit 2,048 (32,768 at 16 a cycle), shared memory 3,072 (operands
// 2,048, P 512, incoming K and V 512).
//
// The maximum of a row is raised lazily (only when it grows by more than 2^8, so P stays
// in fp16's range and O is rarely rescaled); sums and O are f32. P is rounded to the
// element type for its product, as V is given in it; the row's sum takes P unrounded.
#include "chunk.cuh"
#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace abx {
namespace {

constexpr int kGroups = 2;
constexpr int kGroupRows = 128;
constexpr int kKeys = kChunkTileKeys;
constexpr int kMmaWarp = 8;   // one warp a group
constexpr int kLoadWarp = 10;
constexpr int kThreads = 12 * 32;
constexpr int kSoftmaxRegs = 208;
constexpr int kOtherRegs = 72;
constexpr int kStages = 3;    // 32 KB tiles, K and V in the order of use
constexpr uint32_t kSlab = 128 * 128;      // 128 rows x 64 columns
constexpr uint32_t kOperand = 2 * kSlab;
constexpr uint32_t kOffQ = 0;
constexpr uint32_t kOffP = kOffQ + kGroups * kOperand;
constexpr uint32_t kOffRing = kOffP + kGroups * kOperand;
constexpr uint32_t kOffBars = kOffRing + kStages * kOperand;
constexpr int kBarFull = 0;
constexpr int kBarEmpty = kBarFull + kStages;
constexpr int kBarQ = kBarEmpty + kStages;       // [group] the rows' queries are in shared memory
constexpr int kBarS = kBarQ + kGroups;           // [group] S(t) is in TMEM
constexpr int kBarSFree = kBarS + kGroups;       // [group] S(t) is in registers
constexpr int kBarP = kBarSFree + kGroups;       // [group] P(t) is in shared memory
constexpr int kBarO = kBarP + kGroups;           // [group] O holds tile t, P(t) is free
constexpr int kBarDrain = kBarO + kGroups;       // [group]
constexpr int kBarTurn = kBarDrain + kGroups;    // [group] the other group is past its exponentials
constexpr int kNumBars = kBarTurn + kGroups;
constexpr uint32_t kOffTmem = kOffBars + 8 * kNumBars;
constexpr uint32_t kOffAbort = kOffTmem + 4;
constexpr uint32_t kSmemBytes = kOffAbort + 4 + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory exceeds the per-block limit");
constexpr uint32_t kTmemColumns = 512;
__device__ __forceinline__ constexpr uint32_t col_o(int g) { return 128u * static_cast<uint32_t>(g); }
__device__ __forceinline__ constexpr uint32_t col_s(int g) { return 256u + 128u * static_cast<uint32_t>(g); }
constexpr uint64_t kWaitLimit = 400ull * 1000 * 1000;
constexpr float kGrow = 8.0f;               // log2
constexpr float kLargeScore = 1048576.0f;   // log2: above, s * kappa - m * kappa is off by more than a few units

// Instruction descriptor: f32 accumulators, A and B of type T (f16 is type 0, bf16 type 1), M = N = 128.
template <class T>
__host__ __device__ constexpr uint32_t idesc(int b_mn_major) {
    return std::is_same<T, bf16>::value ? tc::idesc_bf16_f32(128, 128, 0, b_mn_major)
                                        : tc::idesc_bf16_f32(128, 128, 0, b_mn_major) & ~((1u << 7) | (1u << 10));
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The place of K(t) and V(t) of `n` tiles in the order of use: K0 K1 V0 K2 V1 .. V(n-1).
__device__ __forceinline__ int item_k(int t) { return t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int item_v(int t, int n) { return t + 1 < n ? 2 * t + 2 : 2 * n - 1; }

// The lowest x of 32 bits.
__device__ __forceinline__ uint32_t low_bits(int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; }

template <class T>
__global__ void __launch_bounds__(kThreads, 1) chunk_tile_kernel(const ChunkArgs a, const __grid_constant__ ChunkMaps maps,
                                                                const int box_rows) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* mem = smem_raw + (base - raw);
    auto bar = [&](int i) { return base + kOffBars + 8u * i; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + kOffAbort);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mem + kOffTmem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // Tiles of rows fastest, then splits, then key heads: CTAs that run at the same time share K and V in L2.
    const int kvh = blockIdx.z, split = blockIdx.y;
    const ChunkUnit u = chunk_unit(a, blockIdx.x, kGroups * kGroupRows);
    if (u.seq < 0) return;
    const int rows = min(kGroups * kGroupRows, u.n * a.group - u.row0);
    const int groups = rows > kGroupRows ? 2 : 1;
    const KeyTiles t = chunk_tiles<kKeys>(a, u, u.row0, u.row0 + rows - 1);
    int begin, end;
    chunk_part(a, t.count, split, begin, end);
    const int n = end - begin;

    cudaTriggerProgrammaticLaunchCompletion();  // the join may come onto the GPU; it waits for this grid's end
    // The rows' queries, 16 threads a row, all loads in flight at once while the CTA sets up; zeros past
    // the last row.
    uint4 q_part[kGroupRows / 8];
    if (warp < kMmaWarp) {
        const int row0 = (tid >> 7) * kGroupRows + ((tid & 127) >> 4);
        RowWalk at(a, kvh, u.row0 + row0, 8);
        const T* q = static_cast<const T*>(a.q) + u.seq * a.q_seq + u.first * a.q_token + (tid & 15) * 8;
#pragma unroll
        for (int i = 0; i < kGroupRows / 8; ++i) {
            q_part[i] = make_uint4(0, 0, 0, 0);
            if (n > 0 && row0 + i * 8 < rows)
                q_part[i] = __ldg(reinterpret_cast<const uint4*>(q + at.head * a.q_head + at.token * a.q_token));
            at.next();
        }
    }
    if (tid == 0) {
        *abort_flag = 0;
        for (int st = 0; st < kStages; ++st) {
            tc::mbar_init(bar(kBarFull + st), 1);
            tc::mbar_init(bar(kBarEmpty + st), groups);
        }
        for (int g = 0; g < kGroups; ++g) {
            tc::mbar_init(bar(kBarQ + g), kGroupRows);
            tc::mbar_init(bar(kBarS + g), 1);
            tc::mbar_init(bar(kBarSFree + g), kGroupRows);
            tc::mbar_init(bar(kBarP + g), kGroupRows);
            tc::mbar_init(bar(kBarO + g), 1);
            tc::mbar_init(bar(kBarDrain + g), 1);
            tc::mbar_init(bar(kBarTurn + g), kGroupRows);
        }
        tc::mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        tc::tmem_alloc(smem_addr(tmem_slot), kTmemColumns);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ---- loader: K and V tiles in the order of use, one box a lane ----
            const int boxes = kKeys / box_rows;  // of a 64-column slab
            int issued = 0;
            for (int i = 0; i < 2 * n; ++i) {
                const int st = i % kStages, use = i / kStages;
                const bool is_v = i == 2 * n - 1 || (i > 0 && (i & 1) == 0);
                const int tile = i == 0 ? 0 : i == 2 * n - 1 ? n - 1 : is_v ? i / 2 - 1 : (i + 1) / 2;
                const int32_t j = t.tile(begin + tile) * kKeys + (lane >> 1) * box_rows;
                const int32_t page = lane < 2 * boxes ? chunk_page(a, u, t, j, box_rows) : 0;
                const bool free_ok =
                    use == 0 || tc::mbar_wait_suspend(bar(kBarEmpty + st), (use - 1) & 1, abort_flag, kWaitLimit);
                if (!__all_sync(0xffffffffu, free_ok)) break;
                issued = i + 1;
                if (lane == 0) tc::mbar_arrive_expect_tx(bar(kBarFull + st), kOperand);
                __syncwarp();
                if (lane < 2 * boxes)
                    tma_load_4d(base + kOffRing + st * kOperand + (lane & 1) * kSlab + (lane >> 1) * box_rows * 128,
                                is_v ? &maps.v : &maps.k, 64 * (lane & 1), a.table ? j % a.page_size : j, kvh, page,
                                bar(kBarFull + st));
                __syncwarp();
            }
            if (lane == 0)
                for (int st = 0; st < kStages && st < issued; ++st)
                    tc::mbar_wait_suspend(bar(kBarFull + st), ((issued - 1 - st) / kStages) & 1, abort_flag, kWaitLimit,
                                          /*honor_abort=*/false);
            __syncwarp();
        } else if (warp < kMmaWarp + groups && n > 0) {
            // ---- products of group g: S(t + 1) as soon as S(t) is in registers, then O += P(t) V(t) ----
            const int g = warp - kMmaWarp;
            const uint64_t qdesc = tc::smem_desc(base + kOffQ + g * kOperand, 16, 1024, tc::kSwizzle128B);
            const uint64_t pdesc = tc::smem_desc(base + kOffP + g * kOperand, 16, 1024, tc::kSwizzle128B);
            auto full = [&](int item) {
                return tc::mbar_wait_warp_suspend(bar(kBarFull + item % kStages), (item / kStages) & 1, abort_flag, kWaitLimit);
            };
            auto issue_s = [&](int item) {
                const uint64_t kdesc = tc::smem_desc(base + kOffRing + (item % kStages) * kOperand, 16, 1024, tc::kSwizzle128B);
#pragma unroll
                for (int s = 0; s < 8; ++s) {  // 16 dims a step: 32 bytes on inside a 64-column slab
                    const uint32_t off = ((s >> 2) * kSlab + (s & 3) * 32) >> 4;
                    tc::mma_ss_elect(tmem + col_s(g), qdesc + off, kdesc + off, idesc<T>(0), s > 0 ? 1u : 0u);
                }
                tc::mma_commit_elect(bar(kBarS + g));
                tc::mma_commit_elect(bar(kBarEmpty + item % kStages));
            };
            bool ok = tc::mbar_wait_warp_suspend(bar(kBarQ + g), 0, abort_flag, kWaitLimit) && full(0);
            if (ok) {
                tc::fence_after_sync();
                issue_s(0);
            }
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) {
                    if (!full(item_k(i + 1)) ||
                        !tc::mbar_wait_warp_suspend(bar(kBarSFree + g), i & 1, abort_flag, kWaitLimit)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    issue_s(item_k(i + 1));
                }
                const int item = item_v(i, n);
                if (!full(item) || !tc::mbar_wait_warp_suspend(bar(kBarP + g), i & 1, abort_flag, kWaitLimit)) {
                    ok = false;
                    break;
                }
                tc::fence_after_sync();
                const uint64_t vdesc =
                    tc::smem_desc(base + kOffRing + (item % kStages) * kOperand, kSlab, 1024, tc::kSwizzle128B);
#pragma unroll
                for (int s = 0; s < 8; ++s)  // 16 keys a step; V rows as they lie (MN-major)
                    tc::mma_ss_elect(tmem + col_o(g), pdesc + (((s >> 2) * kSlab + (s & 3) * 32) >> 4),
                                     vdesc + ((s * 16 * 128) >> 4), idesc<T>(1), (i > 0 || s > 0) ? 1u : 0u);
                tc::mma_commit_elect(bar(kBarO + g));
                tc::mma_commit_elect(bar(kBarEmpty + item % kStages));
            }
            tc::mma_commit_elect(bar(kBarDrain + g));
            if (lane == 0) tc::mbar_wait_suspend(bar(kBarDrain + g), 0, abort_flag, kWaitLimit, /*honor_abort=*/false);
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        const int g = warp >> 2, r = tid & 127;
        const int g_row0 = u.row0 + g * kGroupRows;
        const int g_rows = min(kGroupRows, rows - g * kGroupRows);  // at most 0: the group has no rows
        if (g_rows > 0) {
            if (n > 0) {
                uint8_t* to = mem + kOffQ + g * kOperand + ((r & 15) >> 3) * kSlab + (r >> 4) * 128 + (((r ^ (r >> 4)) & 7) << 4);
#pragma unroll
                for (int i = 0; i < kGroupRows / 8; ++i) *reinterpret_cast<uint4*>(to + i * 1024) = q_part[i];
                tc::fence_proxy_async_smem();
                tc::mbar_arrive(bar(kBarQ + g));
            }
            const Seen mine = chunk_seen(a, u, g_row0 + min(r, g_rows - 1));
            const Seen lo = chunk_seen(a, u, g_row0), hi = chunk_seen(a, u, g_row0 + g_rows - 1);
            const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t s_col = lane_base + col_s(g), o_col = lane_base + col_o(g);
            uint8_t* p_row = mem + kOffP + g * kOperand + r * 128;
            float m = -INFINITY;   // the row's reference, a bare score
            float mk = 0.f;        // m * kappa, 0 while m is -inf
            float l = 0.f;
            bool ok = true;
            for (int i = 0; i < n; ++i) {
                const int32_t k0 = t.tile(begin + i) * kKeys;
                if (!tc::mbar_wait_warp_suspend(bar(kBarS + g), i & 1, abort_flag, kWaitLimit)) {
                    ok = false;
                    break;
                }
                tc::fence_after_sync();
                uint32_t r0[32], r1[32], r2[32], r3[32];
                tc::tmem_ld32(s_col, r0);
                tc::tmem_ld32(s_col + 32, r1);
                tc::tmem_ld32(s_col + 64, r2);
                tc::tmem_ld32(s_col + 96, r3);
                tc::tmem_wait_ld();
                tc::tmem_reg_fence(r0);
                tc::tmem_reg_fence(r1);
                tc::tmem_reg_fence(r2);
                tc::tmem_reg_fence(r3);
                tc::fence_before_sync();
                tc::mbar_arrive(bar(kBarSFree + g));
                // Keys that the row does not see -> -inf (only in tiles that some row does not see whole).
                if (k0 + kKeys > lo.end || (k0 < hi.low && k0 + kKeys > lo.sink)) {
                    auto hide = [&](uint32_t (&x)[32], int first) {
                        const uint32_t see = low_bits(mine.end - first) & (~low_bits(mine.low - first) | low_bits(mine.sink - first));
                        if (__all_sync(0xffffffffu, see == 0xffffffffu)) return;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(see & (1u << e))) x[e] = 0xff800000u;
                    };
                    hide(r0, k0);
                    hide(r1, k0 + 32);
                    hide(r2, k0 + 64);
                    hide(r3, k0 + 96);
                }
                float top;
                {
                    float x0 = __uint_as_float(r0[0]), x1 = __uint_as_float(r1[0]), x2 = __uint_as_float(r2[0]),
                          x3 = __uint_as_float(r3[0]);
#pragma unroll
                    for (int e = 1; e < 31; e += 2) {
                        x0 = max3f(x0, __uint_as_float(r0[e]), __uint_as_float(r0[e + 1]));
                        x1 = max3f(x1, __uint_as_float(r1[e]), __uint_as_float(r1[e + 1]));
                        x2 = max3f(x2, __uint_as_float(r2[e]), __uint_as_float(r2[e + 1]));
                        x3 = max3f(x3, __uint_as_float(r3[e]), __uint_as_float(r3[e + 1]));
                    }
                    x0 = max3f(x0, x1, __uint_as_float(r0[31]));
                    x2 = max3f(x2, x3, __uint_as_float(r1[31]));
                    top = max3f(fmaxf(x0, x2), __uint_as_float(r2[31]), __uint_as_float(r3[31]));
                }
                const bool grow = (top - m) * a.kappa > kGrow;
                float shift = mk;
                if (__any_sync(0xffffffffu, grow || !(fabsf(mk) < kLargeScore))) {
                    const float next = grow ? top : m;
                    const float scale = grow ? exp2f((m - next) * a.kappa) : 1.0f;
                    m = next;
                    mk = m == -INFINITY ? 0.f : m * a.kappa;
                    l *= scale;
                    if (i > 0 && __any_sync(0xffffffffu, grow)) {
                        if (!tc::mbar_wait_warp_suspend(bar(kBarO + g), (i - 1) & 1, abort_flag, kWaitLimit)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {
                            uint32_t o[16];
                            tc::tmem_ld16(o_col + c, o);
                            tc::tmem_wait_ld();
                            tc::tmem_reg_fence(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale);
                            tc::tmem_st16(o_col + c, o);
                        }
                        tc::tmem_wait_st();
                    }
                    // x = s * kappa - m * kappa in one FMA. Its rounding is common to the row and falls out of
                    // o = O / l, unless the scores are so large that it reaches whole units.
                    shift = mk;
                    if (!(fabsf(mk) < kLargeScore)) {
                        shift = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            r0[e] = __float_as_uint(__uint_as_float(r0[e]) - m);
                            r1[e] = __float_as_uint(__uint_as_float(r1[e]) - m);
                            r2[e] = __float_as_uint(__uint_as_float(r2[e]) - m);
                            r3[e] = __float_as_uint(__uint_as_float(r3[e]) - m);
                        }
                    }
                }
                // P's place is free once the product of the tile before is done.
                if (i > 0 && !tc::mbar_wait_warp_suspend(bar(kBarO + g), (i - 1) & 1, abort_flag, kWaitLimit)) {
                    ok = false;
                    break;
                }
                // The groups take turns at the exponential unit: while one's exponentials run, the other
                // reads, finds maxima and hands over.
                if (groups == 2 && (g == 1 || i > 0) &&
                    !tc::mbar_wait_warp_suspend(bar(kBarTurn + g), (g == 1 ? i : i - 1) & 1, abort_flag, kWaitLimit)) {
                    ok = false;
                    break;
                }
                {
                    const uint64_t kappa2 = pack2(a.kappa, a.kappa), shift2 = pack2(-shift, -shift);
                    uint64_t sum0 = kZeros2, sum1 = kZeros2;
                    auto weights = [&](const uint32_t (&x)[32], uint32_t (&p)[16]) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint64_t s2 = (static_cast<uint64_t>(x[2 * e + 1]) << 32) | x[2 * e];
                            const float2 y = unpack2(fma2(s2, kappa2, shift2));
                            const float p0 = exp2f(y.x), p1 = exp2f(y.y);
                            if (e & 1)
                                sum1 = add2(sum1, pack2(p0, p1));
                            else
                                sum0 = add2(sum0, pack2(p0, p1));
                            p[e] = Pair<T>::pack(p0, p1);
                        }
                    };
                    auto store = [&](const uint32_t (&p)[16], int quarter) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4*>(p_row + (quarter >> 1) * kSlab + ((((4 * quarter + c) ^ r) & 7) << 4)) =
                                make_uint4(p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
                    };
                    uint32_t p0[16], p1[16];
                    weights(r0, p0);
                    store(p0, 0);
                    weights(r1, p1);
                    store(p1, 1);
                    weights(r2, p0);
                    store(p0, 2);
                    if (groups == 2) tc::mbar_arrive(bar(kBarTurn + 1 - g));
                    weights(r3, p1);
                    store(p1, 3);
                    const float2 y = unpack2(add2(sum0, sum1));
                    l += y.x + y.y;
                }
                // V rows that no row sees (a page's stale tail) must not meet P = 0 as NaN or infinity. Both
                // groups clear them, each before its own product.
                if (!t.any(k0) || !t.any(k0 + kKeys - 1) || (k0 < t.first.low && k0 + kKeys > t.last.sink)) {
                    const int item = item_v(i, n);
                    if (!tc::mbar_wait_warp_suspend(bar(kBarFull + item % kStages), (item / kStages) & 1, abort_flag, kWaitLimit)) {
                        ok = false;
                        break;
                    }
                    if (!t.any(k0 + r)) {
                        uint8_t* v_row = mem + kOffRing + (item % kStages) * kOperand + r * 128;
#pragma unroll
                        for (int c = 0; c < 16; ++c)  // in an order without bank conflicts
                            *reinterpret_cast<uint4*>(v_row + (c >> 3) * kSlab + (((c ^ r) & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                }
                tc::fence_proxy_async_smem();
                tc::fence_before_sync();
                tc::mbar_arrive(bar(kBarP + g));
            }
            // o = O / l, lse = m * kappa + log2(l); a row that nothing reached gives zeros and -inf.
            if (ok && n > 0) ok = tc::mbar_wait_warp_suspend(bar(kBarO + g), (n - 1) & 1, abort_flag, kWaitLimit);
            if (ok) {
                tc::fence_after_sync();
                const bool none = l == 0.f;
                const float inv = none ? 0.f : 1.f / l;
                const float lse = none ? -INFINITY : mk + log2f(l);
                const int64_t tokens_before = a.starts ? u.first : static_cast<int64_t>(u.seq) * a.tokens;
                const int64_t part = split * a.rows_total + tokens_before * a.heads;
                if (r < g_rows) {
                    const RowWalk at(a, kvh, g_row0 + r, 0);
                    if (a.splits > 1)
                        a.part_lse[part + static_cast<int64_t>(at.token) * a.heads + at.head] = lse;
                    else if (a.lse != nullptr)
                        a.lse[u.seq * a.l_seq + at.head * a.l_head + (u.first + at.token) * a.l_token] = lse;
                }
                // A row is a lane here; through shared memory (the group's Q and P are done with) its
                // columns go out 16 bytes a thread, whole rows at a time.
                const int shift_rows = a.splits > 1 ? 5 : 4;  // 32 or 16 threads a row
                const uint32_t q_row = kOffQ + g * kOperand, p_base = kOffP + g * kOperand;
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t o[32];
                    if (n > 0) {
                        tc::tmem_ld32(o_col + c, o);
                        tc::tmem_wait_ld();
                        tc::tmem_reg_fence(o);
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = none || n == 0 ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                    if (a.splits > 1) {  // f32: columns 0-63 in Q's place, 64-127 in P's, 256 bytes a row
                        uint8_t* to = mem + (c < 64 ? q_row : p_base) + r * 256;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4*>(to + (((((c & 32) + e) >> 2) ^ (r & 15)) << 4)) =
                                make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    } else {
                        uint8_t* to = mem + p_base + r * 256;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            auto two = [&](int i) { return Pair<T>::pack(__uint_as_float(o[e + i]), __uint_as_float(o[e + i + 1])); };
                            *reinterpret_cast<uint4*>(to + ((((c + e) >> 3) ^ (r & 15)) << 4)) = make_uint4(two(0), two(2), two(4), two(6));
                        }
                    }
                }
                asm volatile("bar.sync %0, %1;\n" ::"r"(1 + g), "n"(kGroupRows) : "memory");
                const int step = kGroupRows >> shift_rows, first = r >> shift_rows, c = r & ((1 << shift_rows) - 1);
                RowWalk at(a, kvh, g_row0 + first, step);
#pragma unroll 4
                for (int row = first; row < g_rows; row += step, at.next()) {
                    const uint32_t from = (a.splits > 1 && c < 16 ? q_row : p_base) + row * 256 + (((c & 15) ^ (row & 15)) << 4);
                    const uint4 x = *reinterpret_cast<const uint4*>(mem + from);
                    if (a.splits > 1)
                        *reinterpret_cast<uint4*>(a.part_o + (part + static_cast<int64_t>(at.token) * a.heads + at.head) * 128 + 4 * c) = x;
                    else
                        *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + u.seq * a.o_seq + at.head * a.o_head +
                                                  (u.first + at.token) * a.o_token + 8 * c) = x;
                }
            }
        }
    }

    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemColumns);
    }
    if (tid == 0 && *abort_flag) raise_device_error(a.error, ABX_ERR_DEVICE_TIMEOUT);
}

template <class T>
cudaError_t launch(const ChunkArgs& a, const ChunkMaps& maps, int box_rows, cudaStream_t stream) {
    auto kernel = chunk_tile_kernel<T>;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes));
    if (err != cudaSuccess) return err;
    cudaFuncAttributes attr{};
    if ((err = cudaFuncGetAttributes(&attr, kernel)) != cudaSuccess) return err;
    // setmaxnreg hands out what the launch allocated, never more.
    if (attr.numRegs * kThreads < 8 * 32 * kSoftmaxRegs + (kThreads - 8 * 32) * kOtherRegs) return cudaErrorInvalidConfiguration;
    const int64_t units = chunk_units(a);
    if (units > 0x7fffffff || a.splits > 65535) return cudaErrorInvalidConfiguration;
    kernel<<<dim3(static_cast<unsigned>(units), a.splits, a.kv_heads), kThreads, kSmemBytes, stream>>>(a, maps, box_rows);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_tile(const ChunkArgs& a, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream) {
    return fp16 ? launch<half>(a, maps, box_rows, stream) : launch<bf16>(a, maps, box_rows, stream);
}

}  // namespace abx
