// Rotary positions over several axes (time, height, width), and the append to a paged cache.
//
// Each pair (a, b) of a row's dims turns by angle = position[axis] * frequency:
//     a' = a cos - b sin,   b' = a sin + b cos            (the turn back: -sin).
// Bound by HBM: a row is read once and written once. The angles are the same for
// every head of a token, so eight threads take one token, compute its 64 sines
// and cosines once (eight each) and walk the heads; the position times the
// frequency is taken in 64 bits in units of pi and reduced there (a position of 2^28
// is off by 2^-23 radians at most), and no table of angles is read from memory.
// A thread holds the 16-byte chunks l and l + 8 of a row: pairs of neighbours
// lie inside a chunk, pairs (i, i + 64) in its two chunks. With few tokens the heads are shared out to more thread
// groups instead, which then compute the same angles again.
#include "rotary.cuh"

namespace abx {
namespace {

constexpr int kThreads = 128;
constexpr int kLanes = 8;                       // threads of a token
constexpr int kGroups = kThreads / kLanes;
// Heads in flight, blocks an SM and thread groups an SM, without and with a cache. Measured (us, one
// B200): 75,600 tokens x 24 heads / 2 x 10,799 x 80 heads / 10,800 x 36 rows into pages: 150 / 142 / 45 for
// (4, 4, 160), 155 / 156 / 39 for (2, 6, 64), 43 for (2, 6, 128) into pages; blocks of 256 threads 152 / 146 / 39; a
// register limit that spills costs up to 2x.
constexpr int kUnroll[2] = {4, 2};
constexpr int kBlocks[2] = {4, 6};
constexpr int kWant[2] = {160, 64};

template <class T>
struct Vec {  // eight elements
    uint4 raw[sizeof(T) / 2];
};

template <class T>
__device__ __forceinline__ float to_f(T x) {
    return static_cast<float>(x);
}
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ half from_f<half>(float x) {
    return __float2half_rn(x);
}

template <class T>
__device__ __forceinline__ Vec<T> load8(const T* p) {
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) v.raw[i] = reinterpret_cast<const uint4*>(p)[i];
    return v;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const Vec<T>& v) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = v.raw[i];
}

template <class T>
__device__ __forceinline__ void turn(Vec<T>& lo, Vec<T>& hi, const float (&cs)[8], const float (&sn)[8], bool halves) {
    T* a = reinterpret_cast<T*>(&lo);
    T* b = reinterpret_cast<T*>(&hi);
    if (halves) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = to_f(a[i]), y = to_f(b[i]);
            a[i] = from_f<T>(x * cs[i] - y * sn[i]);
            b[i] = from_f<T>(x * sn[i] + y * cs[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = to_f(a[2 * i]), y0 = to_f(a[2 * i + 1]);
            a[2 * i] = from_f<T>(x0 * cs[i] - y0 * sn[i]);
            a[2 * i + 1] = from_f<T>(x0 * sn[i] + y0 * cs[i]);
            const float x1 = to_f(b[2 * i]), y1 = to_f(b[2 * i + 1]);
            b[2 * i] = from_f<T>(x1 * cs[4 + i] - y1 * sn[4 + i]);
            b[2 * i + 1] = from_f<T>(x1 * sn[4 + i] + y1 * cs[4 + i]);
        }
    }
}

template <class T, bool kPaged>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? kBlocks[kPaged] : 1) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    constexpr int kHeads = kUnroll[kPaged];
    __shared__ double freq[kPairs];
    __shared__ uint8_t axis[kPairs];
    if (threadIdx.x < kPairs) {
        freq[threadIdx.x] = a.freq[threadIdx.x];
        axis[threadIdx.x] = a.axis[threadIdx.x];
    }
    __syncthreads();
    const int lane = threadIdx.x % kLanes;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kLanes;
    // Slices of a token are far apart, so neighbouring groups take neighbouring tokens.
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
    const int slice = static_cast<int>(group / rows);
    if (slice >= a.slices) return;
    const int64_t row = group - slice * rows;
    const int batch = static_cast<int>(row / a.tokens), token = static_cast<int>(row - static_cast<int64_t>(batch) * a.tokens);
    const int h0 = static_cast<int>(static_cast<int64_t>(a.heads) * slice / a.slices);
    const int h1 = static_cast<int>(static_cast<int64_t>(a.heads) * (slice + 1) / a.slices);

    float cs[8], sn[8];
    if (a.positions != nullptr) {
        const int32_t* at = a.positions + batch * a.p_batch + static_cast<int64_t>(token) * a.axes;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pair = a.halves ? 8 * lane + i : (i < 4 ? 4 * lane + i : 32 + 4 * lane + i - 4);
            const double half_turns = static_cast<double>(__ldg(at + axis[pair])) * freq[pair];
            sincospif(static_cast<float>(half_turns - 2.0 * rint(0.5 * half_turns)), &sn[i], &cs[i]);
            sn[i] *= a.sign;
        }
    }
    // Where a paged row of this token goes: -1 when it has no place in the cache.
    int64_t page = -1, slot = 0;
    if constexpr (kPaged) {
        int lo = 0, hi = a.seqs;  // the last sequence that starts at or before the token
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(a.starts + mid + 1) > token)
                hi = mid;
            else
                lo = mid + 1;
        }
        if (lo < a.seqs && token >= __ldg(a.starts + lo)) {  // else in no sequence: not written
            const int64_t pos = static_cast<int64_t>(__ldg(a.lengths + lo)) - __ldg(a.starts + lo + 1) + token;
            if (pos >= 0 && pos < static_cast<int64_t>(a.table_width) * a.page_size) {
                page = __ldg(a.table + static_cast<int64_t>(lo) * a.table_width + pos / a.page_size);
                slot = pos % a.page_size;
            }
            if (page < 0 || page >= a.pages) {
                page = -1;
                raise_device_error(a.error, ABX_ERR_INVALID_ARGUMENT);
            }
        }
    }

    int first = 0;  // head of all jobs that the job starts with
    for (int j = 0; j < a.jobs; first += a.job[j++].heads) {
        const RotaryJob& job = a.job[j];
        const int begin = max(h0 - first, 0), end = min(h1 - first, job.heads);
        if (begin >= end) continue;
        const T* src = static_cast<const T*>(job.src) + batch * job.s_batch + begin * job.s_head + token * job.s_token + 8 * lane;
        T* dst;
        if (kPaged && job.paged) {
            if (page < 0) continue;
            dst = static_cast<T*>(job.dst) + page * job.d_batch + begin * job.d_head + slot * job.d_token + 8 * lane;
        } else {
            dst = static_cast<T*>(job.dst) + batch * job.d_batch + begin * job.d_head + token * job.d_token + 8 * lane;
        }
        for (int h = begin; h < end; h += kHeads) {
            Vec<T> lo[kHeads], hi[kHeads];
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
                if (h + i < end) {
                    lo[i] = load8(src + i * job.s_head);
                    hi[i] = load8(src + i * job.s_head + 64);
                }
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
                if (h + i < end) {
                    if (job.turn) turn(lo[i], hi[i], cs, sn, a.halves != 0);
                    store8(dst + i * job.d_head, lo[i]);
                    store8(dst + i * job.d_head + 64, hi[i]);
                }
            src += kHeads * job.s_head;
            dst += kHeads * job.d_head;
        }
    }
}

template <class T>
void launch(const RotaryArgs& a, unsigned blocks, cudaStream_t stream) {
    if (a.table != nullptr)
        rotary_kernel<T, true><<<blocks, kThreads, 0, stream>>>(a);
    else
        rotary_kernel<T, false><<<blocks, kThreads, 0, stream>>>(a);
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& args, int dtype, cudaStream_t stream) {
    RotaryArgs a = args;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
    // With few tokens the heads are shared out to more thread groups, at most one a head.
    const int64_t want = ceil_div(148 * kWant[a.table != nullptr], rows);
    a.slices = static_cast<int32_t>(want < 1 ? 1 : want > a.heads ? a.heads : want);
    const int64_t blocks = ceil_div(rows * a.slices, kGroups);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    if (dtype == 0)
        launch<bf16>(a, static_cast<unsigned>(blocks), stream);
    else if (dtype == 1)
        launch<half>(a, static_cast<unsigned>(blocks), stream);
    else
        launch<float>(a, static_cast<unsigned>(blocks), stream);
    return cudaGetLastError();
}

}  // namespace abx
