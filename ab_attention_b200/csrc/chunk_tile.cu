// Many rows against many keys: attention of chunks of tokens on the tensor cores (tcgen05).
//
// A CTA takes 256 rows (two groups of 128, one TMEM lane and one softmax thread a
// row) of one key head and walks the 128-key tiles that any of them sees; K and V
// tiles are read once for both groups. Per tile and group:
//     S = Q K^T (TMEM, f32)  ->  P = 2^((s - m) * kappa) (registers, then shared memory, 16 bits)  ->  O += P V (TMEM, f32)
// A softmax thread takes its whole S row into registers at once, which frees the S
// columns: the product for the next tile runs while this tile's exponentials do,
// because P goes to shared memory and not over S. A group's chain is then its
// softmax alone, about 3,240 cycles a tile: S read 150, maximum 360, exponentials
// 1,550, stores and fence 120, and some 200 to 300 for each of three waits.
//
// The groups take turns at the exponentials. In phase, both groups' ran at half the
// rate and the unit idled through the rest of the tile (3,850 cycles); in turns one
// group's other steps fill the other's. Bounds for a tile of both groups, in SM
// cycles: tensor pipe 2,048 (four products of 128^3), exponential unit 2,048 (32,768 at
// 16 a cycle), shared memory half as much again (3,072: operands 2,048, P 512, incoming K and V
// 512), and that is what a step of 3,130 cycles is bound by.
// Measured for 3,600 rows x 12 heads over 75,600 keys (1,672 GFLOP): 1.41 to 1.45 ms alone
// (1,180 TFLOP/s, tensor pipe 61 and exponential unit 64% busy), 1.62 ms back to back, where the
// power cap (980 W) takes the clock to 1.58 GHz; cuDNN's attention on the same call: 1.78 and 1.81 ms.
// Cycles still count under the cap: over 75,520 rows cuDNN has 1,356 TFLOP/s at 1.43 GHz,
// this kernel 1,168 at 1.55.
//
// CTAs are persistent: near the end of its rows a CTA asks the grid's launch control for
// the place of a CTA that has not started and goes on with that. Set-up and hand-over
// between two tiles of rows otherwise cost 15,000 cycles (five tiles of keys): now the
// next queries (TMA), keys and first scores arrive during the last tile, and four
// warps of their own write finished rows during the next one. 8,191 tokens in a
// window of 1,024 (ten tiles of keys each): 140 us with one CTA a tile of rows, 104 us so.
// The code is kept small (90 KB; 159 KB cost 3 to 10%): a change of jobs runs code that
// is not in the instruction cache.
//
// Keys are walked in halves of a tile (a box of 64), whatever lies between two: a window's sinks share a
// tile with its last keys, which makes nine tiles of those ten (96 us).
//
// The maximum of a row is raised lazily (only when it grows by more than 2^8, so P stays
// in fp16's range and O is rarely rescaled); sums and O are f32. P is rounded to the
// element type for its product, as V is given in it: half a unit of each weight, which
// shows as an error of 1.4 times the result's own rounding. The row's sum takes P unrounded.
#include "chunk.cuh"
#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace abx {
namespace {

constexpr int kGroups = 2;
constexpr int kGroupRows = 128;
constexpr int kKeys = kChunkTileKeys;
constexpr int kHalf = kChunkBoxKeys;  // the keys of a tile's halves need not adjoin: a window's sinks and its last keys share one
constexpr int kMmaWarp = 8;    // one warp a group
constexpr int kLoadWarp = 10;  // one for K, one for V
constexpr int kOutWarp = 12;   // four warps: finished rows; the first also finds the next job and loads its queries
constexpr int kThreads = 16 * 32;
// 512 threads start with 128 registers each. The split with no spills anywhere; 168/88, 184/72 and 192/64 measured
// 1 to 2% slower.
constexpr int kSoftmaxRegs = 176;
constexpr int kOtherRegs = 80;
constexpr int kAskAhead = 4;  // tiles before a job's end at which the next is asked for
constexpr int kVStages = 2;    // K has one: both groups are soon done with it
constexpr uint32_t kSlab = 128 * 128;      // 128 rows x 64 columns
constexpr uint32_t kOperand = 2 * kSlab;
constexpr uint32_t kOffQ = 0;
constexpr uint32_t kOffP = kOffQ + kGroups * kOperand;
constexpr uint32_t kOffK = kOffP + kGroups * kOperand;
constexpr uint32_t kOffV = kOffK + kOperand;
constexpr uint32_t kOffBars = kOffV + kVStages * kOperand;
constexpr int kBarK = 0;                         // K(t) is in shared memory
constexpr int kBarKFree = 1;                     // ... and read by both groups
constexpr int kBarV = 2;                         // [stage] the same of V(t)
constexpr int kBarVFree = kBarV + kVStages;      // [stage]
constexpr int kBarQ = kBarVFree + kVStages;      // [group] the rows' queries are in shared memory
constexpr int kBarS = kBarQ + kGroups;           // [group] S(t) is in TMEM
constexpr int kBarSFree = kBarS + kGroups;       // [group] S(t) is in registers
constexpr int kBarP = kBarSFree + kGroups;       // [group] P(t) is in shared memory
constexpr int kBarO = kBarP + kGroups;           // [group] O holds tile t, P(t) is free
constexpr int kBarTurn = kBarO + kGroups;        // [group] the other group is past its exponentials
constexpr int kBarSum = kBarTurn + kGroups;      // [group] a job's sums are in shared memory
constexpr int kBarOFree = kBarSum + kGroups;     // [group] ... and its O has been read
constexpr int kBarQFree = kBarOFree + kGroups;   // [group] a job's last scores are done with the queries
constexpr int kBarAsk = kBarQFree + kGroups;     // a job is near its end
constexpr int kBarDrain = kBarAsk + 1;           // [group]
constexpr int kBarJob = kBarDrain + kGroups;     // [slot] a job is written
constexpr int kBarJobFree = kBarJob + 2;         // [slot] ... and done with by all 16 warps
constexpr int kBarNext = kBarJobFree + 2;        // the answer to the request for another CTA's place
constexpr int kNumBars = kBarNext + 1;
constexpr uint32_t kOffNext = kOffBars + (8 * kNumBars + 15) / 16 * 16;  // 16 bytes: the answer
constexpr uint32_t kOffJobs = kOffNext + 16;

// One row tile with its part of the keys, as the first output warp writes it for all.
struct Job {
    ChunkUnit u;
    KeyTiles t;
    Seen low[kGroups], high[kGroups];  // of the first and last row of each group
    int32_t kvh, split, rows, whole;
    int32_t begin, n;                  // key tiles of two halves each (t counts halves); n < 0: no more jobs
};
constexpr uint32_t kOffTmem = kOffJobs + 2 * sizeof(Job);
constexpr uint32_t kOffAbort = kOffTmem + 4;
constexpr uint32_t kOffSums = (kOffAbort + 4 + 15) / 16 * 16;  // [group][row]: m * kappa, l
constexpr uint32_t kSmemBytes = kOffSums + kGroups * kGroupRows * 8;
static_assert(kSmemBytes <= 227 * 1024, "shared memory exceeds the per-block limit");
constexpr uint32_t kTmemColumns = 512;
static_assert(kKeys == 2 * kHalf, "a tile is two boxes of keys");
__device__ __forceinline__ constexpr uint32_t col_o(int g) { return 128u * static_cast<uint32_t>(g); }
__device__ __forceinline__ constexpr uint32_t col_s(int g) { return 256u + 128u * static_cast<uint32_t>(g); }
constexpr uint64_t kWaitLimit = 400ull * 1000 * 1000;  // cycles, of the waits at a CTA's end
constexpr int kPolls = 1 << 22;
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

// One lane of a converged warp, always the same.
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e != 0;
}

// A value that is the same in all lanes, so that the compiler may keep it in a uniform register.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ void store_shared(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The lowest x of 32 bits.
__device__ __forceinline__ uint32_t low_bits(int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; }

// Asks for the place of a CTA of this grid that has not started; the 16-byte answer lands at `to`.
__device__ __forceinline__ void ask_next(uint32_t to, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(to), "r"(bar)
                 : "memory");
}
// The answer: whether there was one, and its block index.
__device__ __forceinline__ bool read_next(uint32_t from, int& x, int& y, int& z) {
    uint32_t got, bx, by, bz;
    asm volatile(
        "{\n"
        ".reg .b128 answer;\n"
        ".reg .pred p;\n"
        "ld.shared.b128 answer, [%4];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, answer;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "mov.u32 %1, 0;\n"
        "mov.u32 %2, 0;\n"
        "mov.u32 %3, 0;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, answer;\n"
        "}\n"
        : "=r"(got), "=r"(bx), "=r"(by), "=r"(bz)
        : "r"(from)
        : "memory");
    x = static_cast<int>(bx), y = static_cast<int>(by), z = static_cast<int>(bz);
    return got != 0;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) chunk_tile_kernel(const ChunkArgs a, const __grid_constant__ ChunkMaps maps,
                                                                const int box_rows) {
    extern __shared__ __align__(1024) uint8_t mem[];
    const uint32_t base = smem_addr(mem);
    if ((base & 1023u) != 0) {  // swizzled tiles start on 1,024 bytes; there is no room to round up
        if (threadIdx.x == 0) raise_device_error(a.error, ABX_ERR_CUDA);
        return;
    }
    auto bar = [&](int i) { return base + kOffBars + 8u * i; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + kOffAbort);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mem + kOffTmem);
    Job* jobs = reinterpret_cast<Job*>(mem + kOffJobs);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        *abort_flag = 0;
        tc::mbar_init(bar(kBarK), 1);
        tc::mbar_init(bar(kBarKFree), kGroups);
        for (int st = 0; st < kVStages; ++st) {
            tc::mbar_init(bar(kBarV + st), 1);
            tc::mbar_init(bar(kBarVFree + st), kGroups);
        }
        for (int g = 0; g < kGroups; ++g) {
            tc::mbar_init(bar(kBarQ + g), 1);
            tc::mbar_init(bar(kBarS + g), 1);
            tc::mbar_init(bar(kBarSFree + g), kGroupRows);
            tc::mbar_init(bar(kBarP + g), kGroupRows);
            tc::mbar_init(bar(kBarO + g), 1);
            tc::mbar_init(bar(kBarTurn + g), kGroupRows);
            tc::mbar_init(bar(kBarSum + g), kGroupRows);
            tc::mbar_init(bar(kBarOFree + g), kGroupRows);
            tc::mbar_init(bar(kBarQFree + g), 1);
            tc::mbar_init(bar(kBarDrain + g), 1);
            tc::mbar_init(bar(kBarJob + g), 1);
            tc::mbar_init(bar(kBarJobFree + g), 16);
        }
        tc::mbar_init(bar(kBarNext), 1);
        tc::mbar_init(bar(kBarAsk), 1);
        tc::mbar_init_fence();
    }
    if (warp == kOutWarp && lane < (a.q_map ? 3 : 2)) prefetch_map(lane == 0 ? &maps.k : lane == 1 ? &maps.v : &maps.q);
    if (warp == kMmaWarp) {
        tc::tmem_alloc(smem_addr(tmem_slot), kTmemColumns);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // Waits are bounded by their polls (each may suspend the warp for a while): the library's wait by the clock is
    // four times the code, and at some 40 places it alone would fill a third of the instruction cache.
    auto wait = [&](int b, int phase) {
        if (__all_sync(0xffffffffu, tc::mbar_try_wait_suspend(bar(b), phase & 1))) return true;
#pragma unroll 1
        for (int spin = 0; spin < kPolls; ++spin) {
            if (__all_sync(0xffffffffu, tc::mbar_try_wait_suspend(bar(b), phase & 1))) return true;
            if ((spin & 15) == 15 && *abort_flag) break;
        }
        *abort_flag = 1;
        return false;
    };
    auto there = [&](int b, int phase) { return __all_sync(0xffffffffu, tc::mbar_try_wait(bar(b), phase & 1)) != 0; };
    // For waits of a tile's length and more: the warp sleeps through them and leaves the issue slots alone.
    auto wait_long = [&](int b, int phase) {
#pragma unroll 1
        for (int spin = 0; spin < kPolls; ++spin) {
            if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar(b), phase & 1, tc::kLongWaitHintNs))) return true;
            if (*abort_flag) break;
        }
        *abort_flag = 1;
        return false;
    };
    // The j-th job's slot, once it is written; done_with() gives it back (once a warp).
    auto job_ready = [&](int j) { return wait_long(kBarJob + (j & 1), j >> 1); };
    auto done_with = [&](int j) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar(kBarJobFree + (j & 1)));
    };
    // All counters run on over the jobs of the CTA: `keys` key tiles, `tiles` those of a group, `rounds` its jobs.

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (warp >= kLoadWarp && warp < kOutWarp) {
            // ---- loaders of K and of V; lane b looks up the page of box b ----
            const bool is_v = warp > kLoadWarp;
            const CUtensorMap* const map = is_v ? &maps.v : &maps.k;
            const int boxes = kKeys / box_rows;  // of a 64-column slab
            int keys = 0;
            bool ok = true;
#pragma unroll 1
            for (int j = 0; ok; ++j) {
                if (!job_ready(j)) break;
                const Job& job = jobs[j & 1];
                const int n = job.n;
                if (n < 0) break;
                const ChunkUnit u = job.u;
                const KeyTiles t = job.t;
                const int begin = job.begin, kvh = job.kvh;
                done_with(j);
                int32_t page = 0, row = 0;
                const int half = lane * box_rows >= kHalf, in_half = lane * box_rows - half * kHalf;
                auto look_up = [&](int i) {
                    if (lane >= boxes) return;
                    const int32_t k = t.key<kHalf>(2 * (begin + i) + half) + in_half;
                    page = chunk_page(a, u, t, k, box_rows);
                    row = chunk_page_row(a, k);
                };
                if (n > 0) look_up(0);
#pragma unroll 1
                for (int i = 0; i < n; ++i, ++keys) {
                    const int st = is_v ? keys % kVStages : 0, use = is_v ? keys / kVStages : keys;
                    if (use > 0 && !wait((is_v ? kBarVFree : kBarKFree) + st, use - 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t to = base + (is_v ? kOffV : kOffK) + st * kOperand, full = bar((is_v ? kBarV : kBarK) + st);
                    if (lane == 0) tc::mbar_arrive_expect_tx(full, kOperand);
                    __syncwarp();
#pragma unroll 1
                    for (int b = 0; b < boxes; ++b) {
                        const int32_t p = __shfl_sync(0xffffffffu, page, b), y = __shfl_sync(0xffffffffu, row, b);
                        tma_load_4d_elect(to + b * box_rows * 128, map, 0, y, kvh, p, full);
                        tma_load_4d_elect(to + kSlab + b * box_rows * 128, map, 64, y, kvh, p, full);
                    }
                    if (i + 1 < n) look_up(i + 1);  // while that tile's place is still taken
                }
            }
            // Every copy has landed before the CTA ends.
            if (lane == 0) {
                if (!is_v && keys > 0)
                    tc::mbar_wait_suspend(bar(kBarK), (keys - 1) & 1, abort_flag, kWaitLimit, /*honor_abort=*/false);
                for (int x = max(keys - kVStages, 0); is_v && x < keys; ++x)
                    tc::mbar_wait_suspend(bar(kBarV + x % kVStages), (x / kVStages) & 1, abort_flag, kWaitLimit,
                                          /*honor_abort=*/false);
            }
            __syncwarp();
        } else if (warp >= kOutWarp) {
            // ---- the first of them: jobs. This CTA's own place in the grid, then the places of CTAs that have not
            // started. Tiles of rows fastest, then key heads, then splits: CTAs that run at the same time share K and V
            // in L2. Ragged sequences go by length instead, so that no long job starts among the last ----
            int x = blockIdx.x, y = blockIdx.y, z = blockIdx.z;
            int asked[kGroups] = {0, 0};  // rounds of queries
            int questions = 0;
            ChunkUnit u;                  // the latest job
            KeyTiles t;
            Seen bound{};                 // of the row that this lane stands for
            int rows = 0, begin = 0, n = 0;
            bool whole = false;
            auto work_out = [&]() {
                int most = kGroups * kGroupRows, second = 0;
                if (a.sorted) {
                    z = x % a.splits;
                    x /= a.splits;
                    y = x % a.kv_heads;
                    x /= a.kv_heads;
                } else if (a.units > 0) {
                    const int past = x - a.whole_jobs;
                    if (past >= 0) {
                        most = kGroupRows;
                        second = past & 1;
                        x = a.whole_jobs + (past >> 1);
                    }
                    y = x / a.units;
                    x -= y * a.units;
                }
                u = chunk_unit(a, x, kGroups * kGroupRows, a.sorted != 0);
                u.row0 += second * kGroupRows;
                rows = u.seq < 0 ? 0 : max(min(most, u.n * a.group - u.row0), 0);
                n = begin = 0;
                whole = false;
                if (rows == 0) return;
                // A lane for each row that matters: the tile's first and last, the groups' first and last.
                const int which = lane < 2 ? (lane == 0 ? 0 : rows - 1)
                                           : (lane & 2 ? (lane & 1) * kGroupRows : min(((lane & 1) + 1) * kGroupRows, rows) - 1);
                bound = chunk_seen(a, u, u.row0 + min(which, rows - 1));
                auto of = [&](int from) {
                    return Seen{__shfl_sync(0xffffffffu, bound.sink, from), __shfl_sync(0xffffffffu, bound.low, from),
                                __shfl_sync(0xffffffffu, bound.end, from)};
                };
                t = chunk_tiles<kHalf>(a, of(0), of(1));
                int end;
                whole = chunk_part(a, (t.count + 1) / 2, z, begin, end);
                n = end - begin;
                if (whole && z > 0) rows = n = 0;  // nothing to do
            };
            auto publish = [&](int j) {
                const int groups = rows > kGroupRows ? 2 : 1;
                if (j >= 2 && !wait_long(kBarJobFree + (j & 1), (j >> 1) - 1)) return false;
                Job& job = jobs[j & 1];
                if (lane == 0) {
                    job.u = u;
                    job.t = t;
                    job.kvh = y;
                    job.split = z;
                    job.rows = rows;
                    job.whole = whole;
                    job.begin = begin;
                    job.n = n;
                }
                if (lane >= 2 && lane < 4) job.low[lane & 1] = bound;
                if (lane >= 4 && lane < 6) job.high[lane & 1] = bound;
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(bar(kBarJob + (j & 1)));
                if (n == 0) return true;
                // The rows' queries, as soon as the last scores of the job before are done with theirs: by TMA, or
                // 16 lanes a row, zeros past the last row (rows past it are never stored).
#pragma unroll 1
                for (int g = 0; g < groups; ++g) {
                    if (asked[g] > 0 && !wait_long(kBarQFree + g, asked[g] - 1)) return false;
                    ++asked[g];
                    if (a.q_map) {  // two boxes: the heads of 128 / group tokens are the rows in order
                        if (lane == 0) tc::mbar_arrive_expect_tx(bar(kBarQ + g), kOperand);
                        __syncwarp();
                        const int32_t token = u.first + (u.row0 + g * kGroupRows) / a.group;
#pragma unroll 1
                        for (int slab = 0; slab < 2; ++slab)
                            tma_load_4d_elect(base + kOffQ + g * kOperand + slab * kSlab, &maps.q, 64 * slab, y * a.group, token,
                                              a.starts ? 0 : u.seq, bar(kBarQ + g));
                        continue;
                    }
                    const int c = lane & 15, row0 = g * kGroupRows + (lane >> 4);
                    RowWalk at(a, y, u.row0 + row0, 2);
                    const T* q = static_cast<const T*>(a.q) + u.seq * a.q_seq + u.first * a.q_token + c * 8;
                    const uint32_t to = base + kOffQ + g * kOperand + (c >> 3) * kSlab;
#pragma unroll 2
                    for (int i = 0; i < kGroupRows; i += 2, at.next()) {
                        const int row = i + (lane >> 4);
                        const bool valid = row0 + i < rows;
                        tc::cp_async_16_zfill(to + row * 128 + (((c ^ row) & 7) << 4),
                                              valid ? q + at.head * a.q_head + at.token * a.q_token : q, valid);
                    }
                    cp_async_commit();
                }
                if (!a.q_map) {
                    if (groups == 2) {
                        cp_async_wait<1>();
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(bar(kBarQ));
                    }
                    cp_async_wait<0>();
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar(kBarQ + groups - 1));
                }
                return true;
            };
            // Job j: the CTA's own place, then one asked for shortly before the end of the job before it, not sooner: a
            // place taken early would wait behind that job while other SMs run dry.
            auto find = [&](int j) {
                if (n > 0 && !wait_long(kBarAsk, asked[0] - 1)) return false;
                bool more = true, own = j == 0;
#pragma unroll 1
                for (rows = 0; more && rows == 0; own = false) {  // places with nothing to do are passed over
                    if (!own) {
                        if (lane == 0) {
                            tc::mbar_arrive_expect_tx(bar(kBarNext), 16);
                            ask_next(base + kOffNext, bar(kBarNext));
                        }
                        bool ok =
                            tc::mbar_wait_suspend(bar(kBarNext), questions & 1, abort_flag, kWaitLimit, /*honor_abort=*/false);
                        ok = __all_sync(0xffffffffu, ok);
                        ++questions;
                        more = read_next(base + kOffNext, x, y, z);
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (!ok) return false;
                    }
                    if (more) work_out();
                }
                if (more) return publish(j);
                if (j >= 2 && !wait_long(kBarJobFree + (j & 1), (j >> 1) - 1)) return false;
                if (lane == 0) {
                    jobs[j & 1].n = -1;
                    tc::mbar_arrive(bar(kBarJob + (j & 1)));
                }
                return true;
            };
            // ---- all four: finished rows: o = O / l, lse = m * kappa + log2(l); a row that nothing reached gives
            // zeros and -inf. A row is a lane; the softmax is at the next job meanwhile ----
            const int r = tid & 127;
            int tiles[kGroups] = {0, 0}, rounds[kGroups] = {0, 0};
            bool ok = true;
#pragma unroll 1
            for (int j = -1; ok; ++j) {
                int n = 0, rows = 0;
                bool whole = false;
                int32_t first = 0, kvh = 0, row0 = 0;
                int64_t seq = 0, part = 0;
                if (j >= 0) {
                    if (!job_ready(j)) break;
                    const Job& job = jobs[j & 1];
                    n = job.n, rows = job.rows, whole = job.whole != 0;
                    if (n < 0) break;
                    first = job.u.first, kvh = job.kvh, row0 = job.u.row0, seq = job.u.seq;
                    part = job.split * a.rows_total + (a.starts ? first : seq * a.tokens) * a.heads;
                    done_with(j);
                }
                if (warp == kOutWarp && !find(j + 1)) break;
#pragma unroll 1
                for (int g = 0; g * kGroupRows < rows; ++g) {
                    float mk = 0.f, l = 0.f;
                    if (n > 0) {
                        if (!wait_long(kBarSum + g, rounds[g]) || !wait_long(kBarO + g, tiles[g] + n - 1)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
                        const float2 sums = *reinterpret_cast<const float2*>(mem + kOffSums + (g * kGroupRows + r) * 8);
                        mk = sums.x, l = sums.y;
                    }
                    const bool none = l == 0.f, valid = g * kGroupRows + r < rows;
                    const float inv = none ? 0.f : 1.f / l;
                    const RowWalk at(a, kvh, row0 + g * kGroupRows + r, 0);
                    const int64_t part_row = part + static_cast<int64_t>(at.token) * a.heads + at.head;
                    T* out = static_cast<T*>(a.o) + seq * a.o_seq + at.head * a.o_head + (first + at.token) * a.o_token;
                    const uint32_t o_col = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + col_o(g);
#pragma unroll 1
                    for (int c = 0; c < 128; c += 16) {
                        uint32_t o[16];
                        if (n > 0) {
                            tc::tmem_ld16(o_col + c, o);
                            tc::tmem_wait_ld();
                            tc::tmem_reg_fence(o);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                        if (valid && !whole) {
#pragma unroll
                            for (int e = 0; e < 16; e += 4)
                                *reinterpret_cast<uint4*>(a.part_o + part_row * 128 + c + e) =
                                    make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        } else if (valid) {
                            auto two = [&](int e) { return Pair<T>::pack(__uint_as_float(o[e]), __uint_as_float(o[e + 1])); };
                            *reinterpret_cast<uint4*>(out + c) = make_uint4(two(0), two(2), two(4), two(6));
                            *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(two(8), two(10), two(12), two(14));
                        }
                        __syncwarp();  // TMEM is read by whole warps
                    }
                    if (n > 0) {
                        tc::fence_before_sync();
                        tc::mbar_arrive(bar(kBarOFree + g));
                        tiles[g] += n;
                        ++rounds[g];
                    }
                    if (valid) {
                        const float lse = none ? -INFINITY : mk + log2f(l);
                        if (a.splits > 1) a.part_lse[part_row] = whole ? kWhole : lse;
                        if (whole && a.lse != nullptr)
                            a.lse[seq * a.l_seq + at.head * a.l_head + (first + at.token) * a.l_token] = lse;
                    }
                }
            }
            // Queries that were asked for have landed before the CTA ends.
            for (int g = 0; g < kGroups; ++g)
                if (a.q_map && lane == 0 && asked[g] > 0)
                    tc::mbar_wait_suspend(bar(kBarQ + g), (asked[g] - 1) & 1, abort_flag, kWaitLimit, /*honor_abort=*/false);
            __syncwarp();
        } else {
            // ---- products of group g: S(t + 1) as soon as S(t) is in registers, then O += P(t) V(t) ----
            const int g = uniform(warp) - kMmaWarp;
            const uint32_t tm = uniform(tmem);
            const uint64_t qdesc = tc::smem_desc(base + kOffQ + g * kOperand, 16, 1024, tc::kSwizzle128B);
            const uint64_t pdesc = tc::smem_desc(base + kOffP + g * kOperand, 16, 1024, tc::kSwizzle128B);
            int keys = 0, tiles = 0, rounds = 0;
            const uint64_t kdesc = tc::smem_desc(base + kOffK, 16, 1024, tc::kSwizzle128B);
            auto issue_s = [&]() {
                if (elected()) {
#pragma unroll
                    for (int s = 0; s < 8; ++s) {  // 16 dims a step: 32 bytes on inside a 64-column slab
                        const uint32_t off = ((s >> 2) * kSlab + (s & 3) * 32) >> 4;
                        tc::mma_ss(tm + col_s(g), qdesc + off, kdesc + off, idesc<T>(0), s > 0 ? 1u : 0u);
                    }
                    tc::mma_commit(bar(kBarS + g));
                    tc::mma_commit(bar(kBarKFree));
                }
                __syncwarp();
            };
            bool ok = true, early = false;  // early: S(0) of the job is on its way
#pragma unroll 1
            for (int j = 0; ok; ++j) {
                if (!job_ready(j)) break;
                const int n = jobs[j & 1].n, groups = jobs[j & 1].rows > kGroupRows ? 2 : 1;
                if (n < 0) break;
                done_with(j);
                if (n == 0) continue;
                if (g >= groups) {  // the tiles of the other group alone
#pragma unroll 1
                    for (int i = 0; i < n && ok; ++i, ++keys) {
                        ok = wait(kBarK, keys);
                        if (ok && lane == 0) tc::mbar_arrive(bar(kBarKFree));
                        ok = ok && wait(kBarV + keys % kVStages, keys / kVStages);
                        if (ok && lane == 0) tc::mbar_arrive(bar(kBarVFree + keys % kVStages));
                    }
                    continue;
                }
#pragma unroll 1
                for (int i = early ? 0 : -1; i < n; ++i) {
                    if (g == 0 && lane == 0 && i == max(n - kAskAhead, 0)) tc::mbar_arrive(bar(kBarAsk));
                    __syncwarp();
                    if (i + 1 == n) {
                        // The first scores of the next job before this one's last product, which still waits for its P:
                        // if that job, its queries and its first keys are there.
                        early = false;
                        if (there(kBarJob + ((j + 1) & 1), (j + 1) >> 1)) {
                            const int n2 = jobs[(j + 1) & 1].n, groups2 = jobs[(j + 1) & 1].rows > kGroupRows ? 2 : 1;
                            if (n2 > 0 && g < groups2 && there(kBarQ + g, rounds + 1) && there(kBarK, keys + n)) {
                                if (!wait(kBarSFree + g, tiles + i)) {
                                    ok = false;
                                    break;
                                }
                                tc::fence_after_sync();
                                issue_s();
                                if (n2 == 1) tc::mma_commit_elect(bar(kBarQFree + g));
                                early = true;
                            }
                        }
                    } else {
                        if ((i < 0 && !wait(kBarQ + g, rounds)) || !wait(kBarK, keys + i + 1) ||
                            (tiles + i >= 0 && !wait(kBarSFree + g, tiles + i))) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
                        issue_s();
                        if (i + 2 == n) tc::mma_commit_elect(bar(kBarQFree + g));
                    }
                    if (i < 0) continue;
                    const int st = uniform((keys + i) % kVStages);
                    if (!wait(kBarV + st, (keys + i) / kVStages) || (i == 0 && rounds > 0 && !wait(kBarOFree + g, rounds - 1)) || !wait(kBarP + g, tiles + i)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    const uint64_t vdesc =
                        tc::smem_desc(base + kOffV + st * kOperand, kSlab, 1024, tc::kSwizzle128B);
                    if (elected()) {
#pragma unroll
                        for (int s = 0; s < 8; ++s)  // 16 keys a step; V rows as they lie (MN-major)
                            tc::mma_ss(tm + col_o(g), pdesc + (((s >> 2) * kSlab + (s & 3) * 32) >> 4), vdesc + ((s * 16 * 128) >> 4),
                                       idesc<T>(1), (i > 0 || s > 0) ? 1u : 0u);
                        tc::mma_commit(bar(kBarO + g));
                        tc::mma_commit(bar(kBarVFree + st));
                    }
                    __syncwarp();
                }
                keys += n;
                tiles += n;
                ++rounds;
            }
            tc::mma_commit_elect(bar(kBarDrain + g));
            if (lane == 0) tc::mbar_wait_suspend(bar(kBarDrain + g), 0, abort_flag, kWaitLimit, /*honor_abort=*/false);
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        const int g = warp >> 2, r = tid & 127;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_col = lane_base + col_s(g), o_col = lane_base + col_o(g);
        const uint32_t p_row = base + kOffP + g * kOperand + r * 128;
        int keys = 0, tiles = 0, turns = 0, rounds = 0;
        bool ok = true;
#pragma unroll 1
        for (int j = 0; ok; ++j) {
            if (!job_ready(j)) break;
            const Job& job = jobs[j & 1];
            const int n = job.n;
            if (n < 0) break;
            const int groups = job.rows > kGroupRows ? 2 : 1;
            const int g_row0 = job.u.row0 + g * kGroupRows;
            const int g_rows = min(kGroupRows, job.rows - g * kGroupRows);
            if (g_rows <= 0 || n == 0) {  // the group has no rows, or nothing to do for them
                keys += n;
                done_with(j);
                continue;
            }
            const Seen mine = chunk_seen(a, job.u, g_row0 + min(r, g_rows - 1));
            // Halves in [whole_low, whole_end) or below whole_sink are seen whole by all rows of the group.
            const int32_t whole_end = job.low[g].end, whole_low = job.high[g].low, whole_sink = job.low[g].sink;
            const int32_t head = job.t.head, after = job.t.base - head * kHalf, begin = job.begin;
            float m = -INFINITY;   // the row's reference, a bare score
            float mk = 0.f;        // m * kappa - kLift, 0 while m is -inf
            float l = 0.f;
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const int h = 2 * (begin + i);
                const int32_t k0 = h * kHalf + (h < head ? 0 : after), k1 = (h + 1) * kHalf + (h + 1 < head ? 0 : after);
                if (!wait(kBarS + g, tiles + i)) {
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
                const bool partly = max(k0, k1) + kHalf > whole_end || (k0 < whole_low && k0 + kHalf > whole_sink) ||
                                    (k1 < whole_low && k1 + kHalf > whole_sink);
                if (partly) {
                    auto hide = [&](uint32_t (&x)[32], int first) {
                        const uint32_t see = low_bits(mine.end - first) & (~low_bits(mine.low - first) | low_bits(mine.sink - first));
                        if (__all_sync(0xffffffffu, see == 0xffffffffu)) return;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(see & (1u << e))) x[e] = 0xff800000u;
                    };
                    hide(r0, k0);
                    hide(r1, k0 + 32);
                    hide(r2, k1);
                    hide(r3, k1 + 32);
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
                    mk = m == -INFINITY ? 0.f : m * a.kappa - kLift<T>;
                    l *= scale;
                    if (i > 0 && __any_sync(0xffffffffu, grow)) {
                        if (!wait(kBarO + g, tiles + i - 1)) {
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
                        shift = -kLift<T>;
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
                if (tiles + i > 0 && !wait(kBarO + g, tiles + i - 1)) {
                    ok = false;
                    break;
                }
                // The groups take turns at the exponential unit: while one's exponentials run, the other
                // reads, finds maxima and hands over.
                if (groups == 2 && turns + i + g > 0 && !wait(kBarTurn + g, turns + i + g - 1)) {
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
                            store_shared(p_row + (quarter >> 1) * kSlab + ((((4 * quarter + c) ^ r) & 7) << 4), p[4 * c], p[4 * c + 1],
                                         p[4 * c + 2], p[4 * c + 3]);
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
                const KeyTiles& t = job.t;
                auto gaps = [&](int32_t k) {  // of a half
                    return !t.any(k) || !t.any(k + kHalf - 1) || (k < t.first.low && k + kHalf > t.last.sink);
                };
                if (partly && (gaps(k0) || gaps(k1))) {
                    const int st = (keys + i) % kVStages;
                    if (!wait(kBarV + st, (keys + i) / kVStages)) {
                        ok = false;
                        break;
                    }
                    if (!t.any((r < kHalf ? k0 : k1 - kHalf) + r)) {
                        const uint32_t v_row = base + kOffV + st * kOperand + r * 128;
#pragma unroll
                        for (int c = 0; c < 16; ++c)  // in an order without bank conflicts
                            store_shared(v_row + (c >> 3) * kSlab + (((c ^ r) & 7) << 4), 0, 0, 0, 0);
                    }
                }
                tc::fence_proxy_async_smem();
                tc::fence_before_sync();
                tc::mbar_arrive(bar(kBarP + g));
            }
            // The job before has had its sums read.
            if (!ok || (rounds > 0 && !wait(kBarOFree + g, rounds - 1))) break;
            *reinterpret_cast<float2*>(mem + kOffSums + (g * kGroupRows + r) * 8) = make_float2(mk, l);
            tc::mbar_arrive(bar(kBarSum + g));
            keys += n;
            tiles += n;
            if (groups == 2) turns += n;
            ++rounds;
            done_with(j);
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
    if (a.sorted && units * a.kv_heads * a.splits > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const dim3 grid = a.sorted      ? dim3(static_cast<unsigned>(units * a.kv_heads * a.splits))
                      : a.units > 0 ? dim3(static_cast<unsigned>(2 * units * a.kv_heads - a.whole_jobs))
                                    : dim3(static_cast<unsigned>(units), a.kv_heads, a.splits);
    kernel<<<grid, kThreads, kSmemBytes, stream>>>(a, maps, box_rows);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_tile(const ChunkArgs& a, const ChunkMaps& maps, bool fp16, int box_rows, cudaStream_t stream) {
    return fp16 ? launch<half>(a, maps, box_rows, stream) : launch<bf16>(a, maps, box_rows, stream);
}

}  // namespace abx
