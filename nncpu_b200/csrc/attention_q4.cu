// Causal attention over the 4-bit cache (cache_q4.cuh says how its pages lie), token by token: every token of the step attends to
// the pages of its sequence up to its own position (crates/nncpu/src/model/forward.rs:383-426).
//
//   any_kernel: any type of queries, any whole number of 32-lane groups; 32-bit arithmetic on numbers taken out of the pages.
//     A block takes one token, up to eight query heads of one key/value head and a split of their pages, turns a page of keys and
//     then one of values into 32-bit numbers in shared memory and works on those.
// Splits meet in merge_kernel, in the order of their keys.

#include <math.h>

#define NN_LIB attention_q4
#include "common.cuh"
#include "cache_q4.cuh"

namespace {

struct AttnQ4 {
    const void* q;             // [n, n_heads D]
    int dt;                    // type of q and out
    const uint8_t* k_pages;    // [n_pages, n_kv, 40 D]
    const uint8_t* v_pages;
    int n_pages;
    const int* block_table;
    int bt_stride;
    const int* tok_seq;
    const int* tok_pos;
    void* out;                 // [n, n_heads D]
    float* part;               // partial outputs [n, n_heads, n_splits, D], then (maximum, sum) pairs
    int n, n_heads, n_kv, D;
    float scale;
    int window, keep;
    float slope_base;
    const float* sinks;
    float cap;
    const float* head_gate;
    int gate_ld;
    int n_splits;
};

constexpr int kAnyHeads = 8;      // query heads of a block
constexpr int kAnyThreads = 128;

__device__ __forceinline__ float slope_of(const AttnQ4& p, int h) {
    return p.slope_base != 0.0f ? exp2f(-p.slope_base * (float)(h + 1) / (float)p.n_heads) : 0.0f;
}

// What an output row is multiplied by: one over the softmax's denominator, times the head's gate.
__device__ __forceinline__ float closing_factor(const AttnQ4& p, int t, int h, float m, float l) {
    if (p.sinks != nullptr) l += expf(p.sinks[h] - m);
    float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (p.head_gate != nullptr) inv *= 1.0f / (1.0f + expf(0.0f - p.head_gate[(size_t)t * p.gate_ld + h]));
    return inv;
}

// Pages of a token's walk that split s takes: [first, end).
__device__ __forceinline__ int2 split_pages(int n_walk, int n_splits, int s) {
    const int per = (n_walk + n_splits - 1) / n_splits;
    return make_int2(min(n_walk, s * per), min(n_walk, (s + 1) * per));
}

__global__ void __launch_bounds__(kAnyThreads) any_kernel(const AttnQ4 p) {
    extern __shared__ float any_smem[];
    const int D = p.D, NG = D / kGroup, ld = D + 1, tid = threadIdx.x;
    float* tile = any_smem;                    // [64][D + 1]
    float* qs = tile + kPage * ld;             // [kAnyHeads][D]
    float* ps = qs + kAnyHeads * D;            // [kAnyHeads][64] scores, then weights
    float* stat = ps + kAnyHeads * kPage;      // [kAnyHeads][3]: maximum, sum, correction
    const int t = blockIdx.x / p.n_splits, split = blockIdx.x % p.n_splits;
    const int group = p.n_heads / p.n_kv, chunks = (group + kAnyHeads - 1) / kAnyHeads;
    const int kvh = blockIdx.y / chunks, h0 = kvh * group + blockIdx.y % chunks * kAnyHeads;
    const int nh = min(kAnyHeads, (kvh + 1) * group - h0);
    const int seq = p.tok_seq[t], pos = p.tok_pos[t];
    const bool idle = seq < 0 || pos < 0;
    const int first = idle ? 0 : first_visible_key(pos, p.window);
    const PageWalk walk(first, idle ? 0 : pos, p.keep);
    const int2 mine = idle ? make_int2(0, 0) : split_pages(walk.n, p.n_splits, split);
    for (int i = tid; i < nh * D; i += kAnyThreads) qs[i] = idle ? 0.0f : ld_f(p.q, ((size_t)t * p.n_heads + h0) * D + i, p.dt) * p.scale;
    if (tid < kAnyHeads) {
        stat[tid * 3] = -INFINITY;
        stat[tid * 3 + 1] = 0.0f;
    }
    float acc[kAnyHeads][2];
#pragma unroll
    for (int h = 0; h < kAnyHeads; ++h) acc[h][0] = acc[h][1] = 0.0f;
    for (int i = mine.x; i < mine.y; ++i) {
        const int pi = walk.page(i), page = pi < p.bt_stride ? p.block_table[(size_t)seq * p.bt_stride + pi] : -1;
        if (page < 0 || page >= p.n_pages) continue;      // no such page: nothing is seen of it
        const int key0 = pi * kPage;
        const size_t at = ((size_t)page * p.n_kv + kvh) * q4_page_bytes(D);
        const uint8_t* kb = p.k_pages + at;
        const uint8_t* vb = p.v_pages + at;
        auto seen = [&](int key) { return key <= pos && (key >= first || key < p.keep); };
        __syncthreads();
        for (int w = tid; w < kPage * 4 * NG; w += kAnyThreads) {        // a word: eight lanes of one key
            const int row = w / (4 * NG), c = w % (4 * NG) / NG, g = w % NG;
            const uint32_t u = reinterpret_cast<const uint32_t*>(kb)[w];
            const float2 dm = __half22float2(reinterpret_cast<const __half2*>(kb + q4_scales_at(D))[row * NG + g]);
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[row * ld + 32 * g + 8 * c + j] = q4_number(u >> (4 * j) & 15, dm);
        }
        __syncthreads();
        for (int k = tid; k < nh * kPage; k += kAnyThreads) {
            const int h = k / kPage, row = k % kPage;
            float z = -INFINITY;
            if (seen(key0 + row)) {
                z = 0.0f;
                for (int d = 0; d < D; ++d) z = fmaf(qs[h * D + d], tile[row * ld + d], z);
                if (p.cap != 0.0f) z = p.cap * tanhf(z / p.cap);
                z -= slope_of(p, h0 + h) * (float)(pos - key0 - row);
            }
            ps[k] = z;
        }
        __syncthreads();
        // weights against the running maximum: a warp a head
        for (int h = tid >> 5; h < nh; h += kAnyThreads / 32) {
            const int lane = tid & 31;
            const float a = ps[h * kPage + lane], b = ps[h * kPage + 32 + lane];
            const float m0 = stat[h * 3], m1 = fmaxf(m0, warp_max(fmaxf(a, b)));
            const float ea = m1 == -INFINITY ? 0.0f : expf(a - m1), eb = m1 == -INFINITY ? 0.0f : expf(b - m1);
            const float sum = warp_sum(ea + eb);
            ps[h * kPage + lane] = ea;
            ps[h * kPage + 32 + lane] = eb;
            __syncwarp();
            if (lane == 0) {
                const float corr = m1 == -INFINITY ? 1.0f : expf(m0 - m1);
                stat[h * 3] = m1;
                stat[h * 3 + 1] = fmaf(stat[h * 3 + 1], corr, sum);
                stat[h * 3 + 2] = corr;
            }
        }
        // values: what no query may see counts as zero whatever lies there
        for (int w = tid; w < kPage * 4 * NG; w += kAnyThreads) {        // a word: four lanes of two positions
            const int g = w % NG, pr = w / NG % 4, r = w / (4 * NG) % 8, row = w / (32 * NG) * 8 + 2 * pr;
            const uint32_t u = reinterpret_cast<const uint32_t*>(vb)[w];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 dm = __half22float2(reinterpret_cast<const __half2*>(vb + q4_scales_at(D))[(row + k) * NG + g]);
                const bool use = seen(key0 + row + k);
#pragma unroll
                for (int j = 0; j < 4; ++j) tile[(row + k) * ld + 32 * g + 4 * r + j] = use ? q4_number(u >> (16 * k + 4 * j) & 15, dm) : 0.0f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = tid + e * kAnyThreads;
            if (d >= D) continue;
#pragma unroll
            for (int h = 0; h < kAnyHeads; ++h)
                if (h < nh) acc[h][e] *= stat[h * 3 + 2];
            for (int row = 0; row < kPage; ++row) {
                const float v = tile[row * ld + d];
#pragma unroll
                for (int h = 0; h < kAnyHeads; ++h)
                    if (h < nh) acc[h][e] = fmaf(ps[h * kPage + row], v, acc[h][e]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kAnyHeads; ++h) {
        if (h >= nh) break;
        const float m = stat[h * 3], l = stat[h * 3 + 1];
        const size_t row = (size_t)t * p.n_heads + h0 + h;
        if (p.n_splits == 1) {
            const float f = idle ? 0.0f : closing_factor(p, t, h0 + h, m, l);
            for (int e = 0; e < 2; ++e) {
                const int d = tid + e * kAnyThreads;
                if (d < D) st_f(p.out, row * D + d, p.dt, acc[h][e] * f);
            }
        } else {
            float* o = p.part + (row * p.n_splits + split) * D;
            for (int e = 0; e < 2; ++e) {
                const int d = tid + e * kAnyThreads;
                if (d < D) o[d] = acc[h][e];
            }
            if (tid == 0) {
                float* ml = p.part + (size_t)p.n * p.n_heads * p.n_splits * D + (row * p.n_splits + split) * 2;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// grid = (n_heads, n): a block a row of a head.
__global__ void __launch_bounds__(kAnyThreads) merge_any_kernel(const AttnQ4 p) {
    const int h = blockIdx.y, t = blockIdx.x;
    const size_t row = (size_t)t * p.n_heads + h;
    const float* ml = p.part + (size_t)p.n * p.n_heads * p.n_splits * p.D + row * p.n_splits * 2;
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < p.n_splits; ++s) m = fmaxf(m, ml[2 * s]);
    for (int s = 0; s < p.n_splits; ++s) l = fmaf(ml[2 * s + 1], ml[2 * s] == -INFINITY ? 0.0f : expf(ml[2 * s] - m), l);
    const bool idle = p.tok_seq[t] < 0 || p.tok_pos[t] < 0;
    const float f = idle ? 0.0f : closing_factor(p, t, h, m, l);
    for (int d = threadIdx.x; d < p.D; d += kAnyThreads) {
        float o = 0.0f;
        for (int s = 0; s < p.n_splits; ++s)
            o = fmaf(p.part[(row * p.n_splits + s) * p.D + d], ml[2 * s] == -INFINITY ? 0.0f : expf(ml[2 * s] - m), o);
        st_f(p.out, row * p.D + d, p.dt, o * f);
    }
}

}  // namespace

// Splits of a token's pages: enough blocks for the device, each with at least two pages of the longest token.
static int any_splits(int n, int n_heads, int n_kv, int longest) {
    const int group = n_heads / n_kv;
    const long blocks = (long)n * n_kv * ((group + kAnyHeads - 1) / kAnyHeads);
    const long want = (4L * sm_count() + blocks - 1) / blocks, room = (longest / kPage + 1 + 1) / 2;
    const long s = want < room ? want : room;
    return s < 1 ? 1 : (s > 64 ? 64 : (int)s);
}

static bool sizes_ok(int n, int n_heads, int n_kv, int D) {
    return n >= 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && D >= 32 && D <= 256 && D % 32 == 0;
}

// Floats of scratch for a call of these sizes, `longest` the most keys that a token may see.
extern "C" long nncpu_attention_q4_scratch(int n, int n_heads, int n_kv, int D, int dt, int longest) {
    if (n <= 0 || !sizes_ok(n, n_heads, n_kv, D)) return 0;
    const int s = any_splits(n, n_heads, n_kv, longest);
    return s > 1 ? (long)n * n_heads * s * (D + 2) : 0;
}

extern "C" int nncpu_attention_q4(const void* q, int dt, const uint8_t* k_pages, const uint8_t* v_pages, int n_pages,
                                  const int* block_table, int bt_stride, const int* tok_seq, const int* tok_pos, void* out, float* part,
                                  long part_floats, int n, int n_heads, int n_kv, int D, float scale, int window, int keep,
                                  float slope_base, const float* sinks, float cap, const float* head_gate, int gate_ld, int longest,
                                  cudaStream_t stream) {
    NN_CHECK(sizes_ok(n, n_heads, n_kv, D), "attention_q4: %d tokens, %d heads over %d of %d lanes (whole groups of 32, at most 256)", n, n_heads, n_kv, D);
    NN_CHECK(cap >= 0.0f && keep >= 0 && (keep == 0 || window > 0) && (head_gate == nullptr || gate_ld >= n_heads),
             "attention_q4: cap %f, %d kept keys, gate rows of %d", cap, keep, gate_ld);
    NN_CHECK(bt_stride > 0 && n_pages > 0 && longest > 0, "attention_q4: %d pages, tables of %d, at most %d keys", n_pages, bt_stride, longest);
    const long need = nncpu_attention_q4_scratch(n, n_heads, n_kv, D, dt, longest);
    NN_CHECK(need <= part_floats, "attention_q4: %ld floats of scratch, %ld are needed", part_floats, need);
    if (n == 0) return 0;
    AttnQ4 p{q, dt, k_pages, v_pages, n_pages, block_table, bt_stride, tok_seq, tok_pos, out, part, n, n_heads, n_kv, D, scale, window, keep,
             slope_base, sinks, cap, head_gate, gate_ld, any_splits(n, n_heads, n_kv, longest)};
    const int group = n_heads / n_kv, chunks = (group + kAnyHeads - 1) / kAnyHeads;
    const size_t smem = sizeof(float) * ((size_t)kPage * (D + 1) + (size_t)kAnyHeads * (D + kPage + 3));
    NN_CHECK((long)n * p.n_splits < (1L << 31) && n_kv * chunks <= 65535 && n_heads <= 65535, "attention_q4: %d tokens in %d splits", n, p.n_splits);
    static bool done[64];
    if (first_use_on_this_device(done)) {
        const cudaError_t e = cudaFuncSetAttribute(any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
        NN_CHECK(e == cudaSuccess, "attention_q4: shared memory: %s", cudaGetErrorString(e));
    }
    any_kernel<<<dim3((unsigned)(n * p.n_splits), (unsigned)(n_kv * chunks)), kAnyThreads, smem, stream>>>(p);
    NN_LAUNCH_OK("attention_q4");
    if (p.n_splits > 1) {
        merge_any_kernel<<<dim3((unsigned)n, (unsigned)n_heads), kAnyThreads, 0, stream>>>(p);
        NN_LAUNCH_OK("attention_q4 (merge)");
    }
    return 0;
}
