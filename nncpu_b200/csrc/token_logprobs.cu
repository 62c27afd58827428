// Log probabilities of given tokens, the distribution's entropy and its best alternatives, row by row of logits:
//   M = max x, S = sum e^(x - M):  log p(t) = x_t - M - ln S,  entropy = ln S - sum e^(x - M) (x - M) / S,
//   the k best by (x descending, index ascending).
// A NaN counts as -inf, as everywhere in the choice of a token (crates/nncpu/src/model/forward.rs:1003-1011); a lane of -inf has
// probability 0 and adds nothing to the entropy.
//
// One pass over the logits, which is what bounds it: a thread keeps (maximum, sum, weighted sum) of what it has seen and
// follows the maximum 16 logits (32 of bfloat16) at a time.  Alternatives ride along: a warp keeps its best 32 as sorted keys
// (the order of the logit's bits above the complement of the index), one a lane, and a bar that a logit must reach to be
// looked at: the k-th best of what any warp of the block has sorted, or the least of what the warps offer now and then, each the
// ceil(k / warps)-th largest of its lanes' maxima so far, whichever is higher.  At least k logits reach either, and few more.  Those
// that do gather in shared memory and are sorted into the list 32 at a time.
// (300 rows of 50 257, three sets of them in turn: without alternatives 16.7 us, one 23.5, 20 25.9; 14 instructions a logit and some ten
// more with alternatives fill half of the issue slots.  With offers at the first turn alone 25.7 and 29.8; one list a block 52.  64
// rows of 151 936: 12.1 and, with 20, 19.6.  1 001 rows of those: 100, bytes, 608 MB at 6 080 GB/s.)
// Where there are few rows several blocks, a cluster, share one, each a stretch of it, and meet in distributed shared memory.

#include <math.h>

#define NN_LIB token_logprobs
#include "common.cuh"

namespace {

struct Rows {
    const void* logits;      // [n, vocab]
    const int* targets;      // [n]
    float* logprobs;         // [n]
    float* entropy;          // [n]
    float* top;              // [n, k] or null
    int* ids;                // [n, k]
    int n, vocab, k;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 16;      // blocks of a cluster
constexpr int kVectors = 4;         // 16-byte vectors of a thread's turn
constexpr int kStages = 3;          // turns in flight
constexpr int kBelow = (int)0x80000000;      // a bar below everything
constexpr int kRing = kStages * kVectors * kThreads * 16;
typedef unsigned long long Key;

__device__ __forceinline__ Key key_of(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.0f);     // (zeros of both signs are equal)
    return (Key)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logit_of(Key key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// A logit's place in the order, as an integer.
__device__ __forceinline__ int ordered(float x) { return (int)((uint32_t)(key_of(x, 0) >> 32) ^ 0x80000000u); }

// A warp's keys, one a lane, into descending order.
__device__ __forceinline__ Key step(Key a, int stride, bool larger, int lane) {
    const Key b = __shfl_xor_sync(0xffffffffu, a, stride);
    return larger == (a > b) ? a : b;
}
__device__ __forceinline__ Key sort32(Key a, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1)
            a = step(a, stride, ((lane & stride) == 0) == ((lane & size) == 0 || size == 32), lane);
    return a;
}
// The best 32 of two descending lists, descending.
__device__ __forceinline__ Key merge32(Key a, Key b, int lane) {
    b = __shfl_xor_sync(0xffffffffu, b, 31);
    a = a > b ? a : b;
#pragma unroll
    for (int stride = 16; stride > 0; stride >>= 1) a = step(a, stride, (lane & stride) == 0, lane);
    return a;
}

struct Sums {
    float m, s, e;      // maximum, sum of w = e^(x - m), sum of w (x - m)
};
// Those of a warp's lanes, joined: every lane gets them.
__device__ __forceinline__ Sums join_lanes(Sums a) {
    const float m = warp_max(a.m), d = a.m - m;
    const float f = a.m == -INFINITY ? 0.0f : expf(d);
    a.e = warp_sum(f == 0.0f ? 0.0f : f * fmaf(a.s, d, a.e));
    a.s = warp_sum(f * a.s);
    a.m = m;
    return a;
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_of(const void* local, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return at;
}
__device__ __forceinline__ float ld_remote(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ Key ld_remote_key(uint32_t at) {
    Key v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}

template <bool BF16, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) rows_kernel(const Rows p, int splits) {
    constexpr int E = BF16 ? 8 : 4;              // logits of a vector
    __shared__ Key waiting[TOP ? kWarps : 1][64];
    __shared__ Key lists[TOP ? kWarps : 1][32];
    __shared__ Sums sums[kWarps];
    __shared__ Sums whole;
    __shared__ int bar_bits;                     // the bar, as an integer of the same order
    __shared__ int offers[kWarps];               // a logit that ceil(k / kWarps) lanes of a warp have reached, as such integers
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t row = blockIdx.x / splits;
    const int split = blockIdx.x % splits;
    const int size = BF16 ? 2 : 4;
    const char* base = reinterpret_cast<const char*>(p.logits) + row * p.vocab * size;
    // vectors lie on 16-byte boundaries; vector v holds logits E v - shift to E v - shift + E - 1 of the row
    const int shift = (int)((uintptr_t)base % 16) / size;
    const int n_vec = (p.vocab + shift + E - 1) / E;
    const int v0 = (int)((long)n_vec * split / splits), v1 = (int)((long)n_vec * (split + 1) / splits);
    if (TOP) {
        if (tid == 0) bar_bits = kBelow;
        if (lane == 0) offers[warp] = kBelow;
        __syncthreads();
    }
    Sums mine{-INFINITY, 0.0f, 0.0f};
    Key list = 0;                                // this lane's of the warp's best 32
    Key last = 0;                                // the k-th of them
    int n_waiting = 0;
    unsigned turn_number = 0;
    auto settle = [&]() {                        // sorts what waits into the list
        __syncwarp();
        Key got = lane < n_waiting ? waiting[warp][lane] : 0;
        list = merge32(list, sort32(got, lane), lane);
        if (n_waiting > 32) {
            got = 32 + lane < n_waiting ? waiting[warp][32 + lane] : 0;
            list = merge32(list, sort32(got, lane), lane);
        }
        n_waiting = 0;
        last = __shfl_sync(0xffffffffu, list, p.k - 1);
        if (last != 0 && lane == 0) atomicMax(&bar_bits, (int)((uint32_t)(last >> 32) ^ 0x80000000u));
        __syncwarp();
    };
    // Turns ahead lie in shared memory, every thread's own: [kStages][kVectors][kThreads] vectors.  (One that is not the row's alone
    // is not asked for; its logits are read one by one.)
    extern __shared__ uint4 ring[];
    auto ask = [&](int v, int stage) {
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            const int at = v + u * kThreads + tid, i = at * E - shift;
            if (at < v1 && i >= 0 && i + E <= p.vocab)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(ring + (stage * kVectors + u) * kThreads + tid)), "l"(base + (long)i * size) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int stage = 0;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) ask(v0 + s * kThreads * kVectors, s);
    for (int v = v0; v < v1; v += kThreads * kVectors) {
        float x[kVectors * E];
        ask(v + (kStages - 1) * kThreads * kVectors, stage == 0 ? kStages - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            const int at = v + u * kThreads + tid, i = at * E - shift;
            if (at < v1 && i >= 0 && i + E <= p.vocab) {
                const uint4 w = ring[(stage * kVectors + u) * kThreads + tid];
                if constexpr (BF16) {
                    const float2 a = two_bf16(w.x), b = two_bf16(w.y), c = two_bf16(w.z), d = two_bf16(w.w);
                    x[u * E] = a.x; x[u * E + 1] = a.y; x[u * E + 2] = b.x; x[u * E + 3] = b.y;
                    x[u * E + 4] = c.x; x[u * E + 5] = c.y; x[u * E + 6] = d.x; x[u * E + 7] = d.y;
                } else {
                    x[u * E] = __uint_as_float(w.x); x[u * E + 1] = __uint_as_float(w.y);
                    x[u * E + 2] = __uint_as_float(w.z); x[u * E + 3] = __uint_as_float(w.w);
                }
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    x[u * E + j] = at < v1 && i + j >= 0 && i + j < p.vocab ? ld_f(base, (size_t)(i + j), BF16 ? DT_BF16 : DT_F32) : -INFINITY;
            }
        }
        const uint4* turn = ring + stage * kVectors * kThreads + tid;
        stage = stage == kStages - 1 ? 0 : stage + 1;
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < kVectors * E; ++j) mx = fmaxf(mx, x[j]);      // (a NaN is dropped)
        const float m = fmaxf(mine.m, mx);
        if (m > -INFINITY) {
            const float d = mine.m - m;
            if (d < 0.0f) {
                const float f = mine.m == -INFINITY ? 0.0f : expf(d);
                mine.e = mine.m == -INFINITY ? 0.0f : f * fmaf(mine.s, d, mine.e);
                mine.s *= f;
                mine.m = m;
            }
            float s = 0.0f, e = 0.0f;
#pragma unroll
            for (int j = 0; j < kVectors * E; ++j) {
                // 2^-150 and less is 0, and 0 times its finite y adds nothing; -inf and NaN come to y = -1000 or so
                const float y = fmaxf(x[j] - m, -1000.0f), w = fast_exp2(y * 1.4426950408889634f);
                s += w;
                e = fmaf(w, y, e);
            }
            mine.s += s;
            mine.e += e;
        }
        if (TOP) {
            // At turns 0, 1, 2, 4, 8, ... : k logits or more reach what every warp offers, since each has that many lanes whose own maximum
            // does.  (What another warp has not written yet is less, and as good a bar.)
            if ((turn_number & (turn_number - 1)) == 0) {
                int reach = ordered(mine.m), offer = __reduce_max_sync(0xffffffffu, reach);
                for (int k = kWarps; k < p.k; k += kWarps) {
                    const unsigned has = __ballot_sync(0xffffffffu, reach == offer);
                    if (lane == __ffs(has) - 1) reach = kBelow;
                    offer = __reduce_max_sync(0xffffffffu, reach);
                }
                volatile int* o = offers;
                if (lane == 0) o[warp] = offer;
                if (turn_number == 0) __syncthreads();
                else __syncwarp();
                offer = __reduce_min_sync(0xffffffffu, o[lane % kWarps]);
                if (lane == 0) atomicMax(&bar_bits, offer);
                __syncwarp();
            }
            ++turn_number;
            const int bits = *reinterpret_cast<volatile int*>(&bar_bits);
            const float bar = bits == kBelow ? -INFINITY : logit_of((Key)((uint32_t)bits ^ 0x80000000u) << 32);
            unsigned pass = 0;
            if (__any_sync(0xffffffffu, mx >= bar))
#pragma unroll
                for (int j = 0; j < kVectors * E; ++j) pass |= (x[j] < bar ? 0u : 1u) << j;        // (a NaN passes, as -inf)
            while (__any_sync(0xffffffffu, pass != 0)) {
                const int j = __ffs(pass) - 1;           // one of each lane's at a time
                const int at = v + j / E * kThreads + tid, i = at * E - shift + j % E;
                bool looks = pass != 0 && at < v1 && i >= 0 && i < p.vocab;
                pass &= pass - 1;
                Key key = 0;
                if (looks) {
                    const int i0 = i - j % E;
                    float c = i0 >= 0 && i0 + E <= p.vocab ? ld_f(turn + j / E * kThreads, (size_t)(j % E), BF16 ? DT_BF16 : DT_F32)
                                                           : ld_f(base, (size_t)i, BF16 ? DT_BF16 : DT_F32);
                    if (c != c) c = -INFINITY;
                    key = key_of(c, i);
                    looks = key > last;
                }
                const unsigned got = __ballot_sync(0xffffffffu, looks);
                if (looks) waiting[warp][n_waiting + __popc(got & ((1u << lane) - 1))] = key;
                n_waiting += __popc(got);
                if (n_waiting >= 32) settle();
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // -- the warps of a block, then the blocks of a row
    mine = join_lanes(mine);
    if (lane == 0) sums[warp] = mine;
    if (TOP) {
        if (n_waiting > 0) settle();
        lists[warp][lane] = list;
    }
    __syncthreads();
    if (TOP)
        for (int half = kWarps / 2; half > 0; half >>= 1) {
            if (warp < half) lists[warp][lane] = merge32(lists[warp][lane], lists[warp + half][lane], lane);
            __syncthreads();
        }
    if (warp == 0) {
        Sums a = lane < kWarps ? sums[lane] : Sums{-INFINITY, 0.0f, 0.0f};
        a = join_lanes(a);
        if (lane == 0) whole = a;
    }
    if (splits > 1) {
        cluster_barrier();
        if (TOP && split == 0) {
            if (warp < splits) list = ld_remote_key(remote_of(&lists[0][lane], warp));
            if (warp + kWarps < splits) list = merge32(list, ld_remote_key(remote_of(&lists[0][lane], warp + kWarps)), lane);
        }
        if (split == 0 && warp == 0) {
            Sums a{-INFINITY, 0.0f, 0.0f};
            if (lane < splits) {
                const uint32_t at = remote_of(&whole, lane);
                a = Sums{ld_remote(at), ld_remote(at + 4), ld_remote(at + 8)};
            }
            a = join_lanes(a);
            if (lane == 0) sums[0] = a;
        }
        cluster_barrier();          // what other blocks left has been read
        if (split != 0) return;
        if (TOP && warp < splits) lists[warp][lane] = list;
        __syncthreads();
        if (TOP)
            for (int half = min(splits, kWarps) / 2; half > 0; half >>= 1) {
                if (warp < half) lists[warp][lane] = merge32(lists[warp][lane], lists[warp + half][lane], lane);
                __syncthreads();
            }
        if (tid == 0) whole = sums[0];
    }
    __syncthreads();
    if (warp != 0) return;
    const Sums a = whole;
    const float logs = a.m == -INFINITY ? 0.0f : (float)log((double)a.s);
    if (lane == 0) {
        const int t = p.targets[row];
        float x = t < 0 || t >= p.vocab ? __int_as_float(0x7FC00000) : ld_f(p.logits, row * p.vocab + t, BF16 ? DT_BF16 : DT_F32);
        if (t >= 0 && t < p.vocab && x != x) x = -INFINITY;
        p.logprobs[row] = x != x ? x : a.m == INFINITY ? a.m - a.m : x == -INFINITY ? x : (x - a.m) - logs;
        p.entropy[row] = a.m == -INFINITY ? 0.0f : a.m == INFINITY ? a.m - a.m : logs - a.e / a.s;
    }
    if (TOP && lane < p.k) {
        const Key key = lists[0][lane];
        const float x = logit_of(key);
        p.ids[row * p.k + lane] = (int)~(uint32_t)key;
        p.top[row * p.k + lane] = a.m == INFINITY ? a.m - a.m : x == -INFINITY ? x : (x - a.m) - logs;
    }
}

}  // namespace

// Blocks that share a row.  Few rows: as many as give the device's SMs two blocks each (8 rows of 151 936, best 5: 1 block 33 us, 4 16.5,
// 8 or 16 12.4).  A few hundred: one, because a cluster's own cost is that of some 10 000 logits (300 rows of 50 257, best 20: 1
// block 25.9 us, 2 28.6, 4 34.1).  Many long rows: two, which end together more nearly (1 001 rows of 151 936: 1 block 102 us, 2 98.8, 4 107).
static int splits_of(int n, int vocab) {
    if (n >= 5L * sm_count()) return vocab >= 1 << 16 ? 2 : 1;
    int s = 1;
    while (s < kMaxSplits && 2L * n * s <= 2L * sm_count() && vocab / (2 * s) >= 4 * kThreads) s *= 2;
    return s;
}

extern "C" int nncpu_token_logprobs(const void* logits, int dt, const int* targets, float* logprobs, float* entropy, float* top, int* ids,
                                    int n, int vocab, int k, cudaStream_t stream) {
    NN_CHECK(n >= 0 && vocab > 0 && vocab < (1 << 30), "token_logprobs: %d rows of %d logits", n, vocab);
    NN_CHECK(k >= 0 && k <= vocab && k <= kMaxTop, "token_logprobs: the best %d of %d (at most %d)", k, vocab, kMaxTop);
    NN_CHECK((uintptr_t)logits % (dt == DT_BF16 ? 2 : 4) == 0, "token_logprobs: logits do not start on a number's boundary");
    if (n == 0) return 0;
    const Rows p{logits, targets, logprobs, entropy, top, ids, n, vocab, k};
    const auto kernel = dt == DT_BF16 ? (k ? rows_kernel<true, true> : rows_kernel<true, false>) : (k ? rows_kernel<false, true> : rows_kernel<false, false>);
    static bool done[4][64];
    if (first_use_on_this_device(done[(dt == DT_BF16 ? 2 : 0) + (k ? 1 : 0)])) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        const cudaError_t e2 = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
        NN_CHECK(e2 == cudaSuccess, "token_logprobs: shared memory: %s", cudaGetErrorString(e2));
        NN_CHECK(e == cudaSuccess, "token_logprobs: clusters of %d: %s", kMaxSplits, cudaGetErrorString(e));
    }
    const int splits = splits_of(n, vocab);
    NN_CHECK((long)n * splits < (1L << 31), "token_logprobs: %d rows", n);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kRing;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, splits);
    NN_CHECK(e == cudaSuccess, "token_logprobs: launch failed: %s", cudaGetErrorString(e));
    return 0;
}
