// Causal attention over the 4-bit cache (cache_q4.cuh says how its pages lie), token by token: every token of the step attends to
// the pages of its sequence up to its own position (crates/nncpu/src/model/forward.rs:383-426).
//
//   stream_kernel: bfloat16 queries, heads of up to 128 lanes, score caps of up to 4 096, on the tensor cores, straight from the codes
//     (see there).
//   any_kernel: any type of queries, any whole number of 32-lane groups, any cap; 32-bit arithmetic on numbers taken out of the pages.
//     A block takes one token, up to eight query heads of one key/value head and a split of their pages.
// Parts of a token's keys meet in a second kernel, in the order of the keys.

#include <math.h>

#define NN_LIB attention_q4
#define NN_LAUNCH_OVERLAP
#include "common.cuh"
#include "cache_q4.cuh"

namespace {

struct AttnQ4 {
    const void* q;             // [n, n_heads D]
    int dt;                    // type of q and out
    const uint8_t* k_pages;    // [n_pages, n_kv, 40 D]
    const uint8_t* v_pages;
    int n_pages;
    const int* block_table;    // [bt_rows, bt_stride]
    int bt_rows, bt_stride;
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

// ---------------------------------------------------------------------------
// stream_kernel.  With a key j's lanes k = d_g c + m_g (g the lane's group of 32) and likewise for values,
//   score_j = sum_g d_jg (sum_x q_x c_jx) + sum_g m_jg (sum_x q_x),    out_x = sum_j (p_j d_jg) (c_jx - 8) + sum_j p_j (m_jg + 8 d_jg),
// so the tensor cores multiply the codes themselves, whole numbers and exact in float16: 16 keys are the rows of
// m16n8k16 (a group of lanes is two of its steps), the query heads that share the key/value head its columns.
//   * A code becomes a float16 number without a conversion: 0x6400 | c is 1024 + c, and with the code four bits further up
//     0x5400 | 16 c is 64 + c; one AND-OR (and a shift every other time) makes two of them.
//   * A key group's sum, in 32 bits, is multiplied by d.  The rest, sum_g m_g (sum q) less what the 1024 and 64 added,
//     sum_g d_g off_g, is itself a product of a key's eight numbers (d_0, m_0, d_1, ...) with numbers of the query: one more
//     tensor-core step per 16 keys, the query's side in two float16 parts (22 bits).
//   * Of the values 1032 or 72 is subtracted at once, which is exact: a sum over thousands of keys of numbers around 1024
//     would lose what is left of c - 8.  sum_j p_j d_jg and sum_j p_j m_jg are a tensor-core step as well.
//   * Queries enter as float16 times a power of two per head that makes the greatest at most 1 (exact for all but what is
//     2^-14 below it).  Weights are float16 with 11 bits: p is taken against a reference below the maximum so that p and p d
//     lie in float16's middle, and the reference moves when a weight passes 2^15 or a step passes what it allows.  (What is less than
//     2^-36 of the greatest weight counts for nothing, 2^-22 where a step of the values is thousands.)
// Rounded below 32 bits are: a weight p, and p d, both to 11 bits.
//
// A block is two warps, each of which takes one half of every page: it brings its 32 keys' codes and scales (5 KB for D = 128) to its
// own ring in shared memory by 16-byte cp.async (with the copy engine's untiled copies, asked for by one lane, 64 sequences of up to
// 8 000 keys took 115 us instead of 98) and shares nothing with the other until a pair's pages are done, when the first adds
// what the second leaves in shared memory.
//
// The pages of all (token, key/value head) pairs lie in one row, of which every block takes an equal share, wherever that
// begins and ends: unequal sequences cost nothing, and there is one wave of blocks.  A pair that lies within one block is finished by it; of
// the others every block leaves its part (its first and its last pair at most) in scratch for stream_merge_kernel.  Where there are few
// pairs of not too many pages (CLUSTER), a cluster of blocks shares each of them instead, and its parts meet in distributed
// shared memory: one launch, and no way through global memory.
//
// Bound where there is much to read by the fixed latency between a warp's instructions, some 300 for 16 keys, at three warps a scheduler: 55 % of
// the issue slots, 27 % of the tensor pipe and 60 % of DRAM are used.  64 sequences of up to 8 000 keys, 32 heads over 8 of 128 lanes, 70 us
// for 328 MB (4 700 GB/s); 64 of 4 000 each 73 us where bfloat16 takes 154.  One sequence of 2 500 keys takes 9.7 us, launch and
// latency; 12.0 where the call is told of 32 768 keys (the row, see cluster_of).
// ---------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStreamWarps = 2;
constexpr int kStreamStages = 2;            // pages of a warp's ring (with 3, 16 unequal sequences took 26.0 us instead of 24.6, 64 long ones 72.2 instead of 70.7)
constexpr int kTiles = 2;                   // tensor-core tiles of 16 keys that a warp has of a page

struct Stream {
    int heads;              // query heads of a pair (a part of those that share a key/value head where these are many)
    int chunks;             // such parts of a key/value head
    int pairs;              // n_kv * chunks: pairs of a tile
    int tile;               // tokens of a tile: 1, or (cu not null) several neighbours of the step's one sequence
    int tiles;              // tiles of the step
    const int* cu;          // or null: the first token of the step's one sequence, and the first behind it
    int min_places;         // places of the row that a block takes at least
    int blocks;             // blocks of the launch
    float scale2;           // scale * log2(e)
    ScoreCap cap;
    int cluster;            // CLUSTER: blocks that share a pair
    int2* parts;            // [tiles, pairs]: the first block that has a part of a pair, and the last
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ldmatrix, two 8x8 tiles transposed: lane l of the first 16 gives the address of row l.
__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t& a, uint32_t& b, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t local, uint32_t rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float low_half(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFF))); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Codes I and I + 4 of a word as float16 numbers: 1024 + c for even I, 64 + c for odd I.
template <int I>
__device__ __forceinline__ uint32_t codes_at(uint32_t w) {
    uint32_t d;
    if (I >= 2) w >>= 8;
    if (I % 2 == 0) asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(d) : "r"(w));     // (a & b) | c
    else asm("lop3.b32 %0, %1, 0x00F000F0, 0x54005400, 0xEA;" : "=r"(d) : "r"(w));
    return d;
}
// The same as c - 8.
template <int I>
__device__ __forceinline__ uint32_t centred_at(uint32_t w) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(codes_at<I>(w)), "r"(I % 2 == 0 ? 0x64086408u : 0x54805480u));
    return d;
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// A tile: its first token, how many it has (0: it is of no sequence), the positions of the first and the last, the first key that one of
// them sees.
struct Tile {
    int t0, count, pos, last, first;
};
template <bool TILED>
__device__ __forceinline__ Tile tile_of(const AttnQ4& p, const Stream& st, int i) {
    Tile w{i, 1, 0, 0, 0};
    if (TILED && st.cu != nullptr) {
        w.t0 = max(0, st.cu[0]) + i * st.tile;
        w.count = max(0, min(st.tile, min(st.cu[1], p.n) - w.t0));
    }
    if (w.count > 0) {
        w.pos = p.tok_pos[w.t0];
        const int seq = p.tok_seq[w.t0];        // (both asked for at once)
        if (min(w.pos, seq) < 0 || seq >= p.bt_rows) w.count = 0;
    }
    w.last = w.pos + w.count - 1;
    w.first = first_visible_key(w.pos, p.window);
    return w;
}
// The pages that a tile sees.
template <bool TILED>
__device__ __forceinline__ int pages_of(const AttnQ4& p, const Stream& st, int i) {
    const Tile w = tile_of<TILED>(p, st, i);
    return w.count > 0 ? PageWalk(w.first, w.last, p.keep).n : 0;
}

// How the row of pairs is cut.  A pair is kPairCost places and then its pages, one place each: what a block does once for a pair (queries
// in, parts out) takes about as long as that many pages, so that blocks with several short pairs end with the others.
constexpr unsigned kPairCost = 3;
struct Row {
    unsigned places, blocks, each, more;         // a block has `each` places, the first `more` blocks one more
    __device__ __forceinline__ unsigned start(unsigned b) const { return each * b + min(b, more); }
    __device__ __forceinline__ int block_of(unsigned place) const {
        const unsigned at = more * (each + 1);
        return place < at ? place / (each + 1) : more + (place - at) / each;
    }
};
// (Every warp by itself, 32 tokens at a time; `mine`: the pages of tile `lane`, which are asked for once.)
template <bool TILED>
__device__ __forceinline__ Row row_of(const AttnQ4& p, const Stream& st, int lane, int mine) {
    unsigned sum = mine > 0 ? mine + kPairCost : 0;
    for (int t = lane + 32; t < st.tiles; t += 32) {
        const int n = pages_of<TILED>(p, st, t);
        sum += n > 0 ? n + kPairCost : 0;
    }
    Row row;
    row.places = __reduce_add_sync(0xffffffffu, sum) * st.pairs;
    row.blocks = min((row.places + st.min_places - 1) / st.min_places, (unsigned)st.blocks);
    row.each = row.blocks > 0 ? row.places / row.blocks : 0;
    row.more = row.places - row.each * row.blocks;
    return row;
}

// Where a block is: page i of the n that pair y of tile t walks through, and how many places are left to it.
struct Place {
    int t, y, i, n, left;
    // to the next pair with pages
    template <bool TILED>
    __device__ __forceinline__ void next_pair(const AttnQ4& p, const Stream& st) {
        i = 0;
        left -= kPairCost;
        if (++y == st.pairs) {
            y = 0;
            do { ++t; } while (t < st.tiles && (n = pages_of<TILED>(p, st, t)) == 0);
        }
    }
};
template <bool TILED>
__device__ __forceinline__ Place place_of(const AttnQ4& p, const Stream& st, unsigned place, int left, int lane, int mine) {
    unsigned before = 0;
    for (int t0 = 0;; t0 += 32) {
        const int n = t0 == 0 ? mine : t0 + lane < st.tiles ? pages_of<TILED>(p, st, t0 + lane) : 0;
        const unsigned places = n > 0 ? n + kPairCost : 0;
        unsigned upto = places;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, before + upto * st.pairs > place);
        if (beyond != 0 || t0 + 32 >= st.tiles) {
            const int l = beyond != 0 ? __ffs(beyond) - 1 : 31;
            const unsigned of_pair = __shfl_sync(0xffffffffu, places, l);
            const unsigned rest = place - before - (__shfl_sync(0xffffffffu, upto, l) - of_pair) * st.pairs;
            Place w;
            w.t = t0 + l;
            w.n = __shfl_sync(0xffffffffu, n, l);
            w.y = of_pair > 0 ? rest / of_pair : 0;
            w.i = (int)(rest - w.y * of_pair) - (int)kPairCost;
            w.left = left + min(w.i, 0);          // (the places before the pair's first page)
            w.i = max(w.i, 0);
            return w;
        }
        before += __shfl_sync(0xffffffffu, upto, 31) * st.pairs;
    }
}

// The reference lies `room` below the greatest score when it moves, so that weights start at 2^room; it moves when one passes
// 2^(room + kLag).  With steps of at most 1 room is 11: weights of 2^11 to 2^15 and what is 2^-25 of them are normal numbers of
// float16, and so is p d.  Greater steps (they are at most 8 736: numbers lie within +-65 504) leave less.
constexpr float kLag = 4.0f;
__device__ __forceinline__ float headroom(float d_max) { return d_max <= 1.0f ? 11.0f : 11.0f - ceilf(log2f(d_max)); }

// Tiles of no sequence are in one part, and (token by token) zeros.
template <int D, bool TILED>
__device__ __forceinline__ void zero_rows(const AttnQ4& p, const Stream& st) {
    for (int t = blockIdx.x; t < st.tiles; t += gridDim.x) {
        if (pages_of<TILED>(p, st, t) > 0) continue;
        for (int i = threadIdx.x; st.cu == nullptr && i < p.n_heads * D / 8; i += 32 * kStreamWarps)
            reinterpret_cast<uint4*>(p.out)[(size_t)t * p.n_heads * D / 8 + i] = make_uint4(0, 0, 0, 0);
        for (int i = threadIdx.x; i < st.pairs; i += 32 * kStreamWarps) st.parts[(size_t)t * st.pairs + i] = make_int2(0, 0);
    }
}

template <int NG, int NT, bool CLUSTER>
__global__ void __launch_bounds__(32 * kStreamWarps, NT == 1 ? 6 : 4) stream_kernel(const AttnQ4 p, const Stream st) {
    constexpr int D = 32 * NG, COLS = 8 * NT;
    constexpr bool TILED = NT == 2;       // a tile may have several tokens
    constexpr int kCodes = 256 * NG, kScales = 64 * NG;          // bytes of a tile's 16 keys
    constexpr int kVCodes = kTiles * kCodes, kKScales = 2 * kVCodes, kVScales = kKScales + kTiles * kScales, kStage = 2 * kTiles * (kCodes + kScales);
    constexpr unsigned kPageBytes = 40 * D;
    extern __shared__ __align__(128) uint8_t stream_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    uint8_t* ring = stream_smem + warp * kStreamStages * kStage;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    float* meet = reinterpret_cast<float*>(stream_smem + kStreamWarps * kStreamStages * kStage);   // [COLS][D + 4]: lanes, reference, sum
    wait_for_previous_kernels();
    let_next_kernel_start();
    const int my_pages = CLUSTER ? 0 : lane < st.tiles ? pages_of<TILED>(p, st, lane) : 0;
    Row row{};
    Place here;
    if (CLUSTER) {
        const int pair = blockIdx.x / st.cluster, rank = blockIdx.x - pair * st.cluster;
        here.t = pair / st.pairs;
        here.y = pair - here.t * st.pairs;
        here.n = pages_of<TILED>(p, st, here.t);
        here.i = here.n * rank / st.cluster;
        here.left = here.n * (rank + 1) / st.cluster - here.i;
    } else {
        row = row_of<TILED>(p, st, lane, my_pages);
        if ((int)blockIdx.x >= row.blocks) {
            zero_rows<D, TILED>(p, st);
            return;
        }
        const unsigned first_place = row.start(blockIdx.x);
        here = place_of<TILED>(p, st, first_place, (int)(row.start(blockIdx.x + 1) - first_place), lane, my_pages);
    }
    Place ahead = here;
    // The columns of a pair are its tile's tokens times its heads.  Their queries, as they lie: column r of each eight, lanes 32 g + 8 c to + 7.
    const int group = p.n_heads / p.n_kv;
    uint4 raw[NT][NG];
    auto ask_queries = [&]() {
        const int kvh = here.y / st.chunks, part = here.y - kvh * st.chunks, heads = min(st.heads, group - part * st.heads);
        const Tile w = here.left > 0 ? tile_of<TILED>(p, st, here.t) : Tile{0, 0, 0, 0, 0};
        const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + ((size_t)w.t0 * p.n_heads + kvh * group + part * st.heads) * D + 8 * c;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int at = !TILED || st.tile == 1 ? 0 : (8 * nt + r) / heads, h = 8 * nt + r - at * heads;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                raw[nt][g] = make_uint4(0, 0, 0, 0);
                if (at < w.count && h < heads) raw[nt][g] = *reinterpret_cast<const uint4*>(q + ((size_t)at * p.n_heads + h) * D + 32 * g);
            }
        }
    };
    ask_queries();
    unsigned there = 0;                     // bit s: stage s holds a page (and not one that is missing)
    int ids = -1, id_at = 0, id_end = 0;    // lane l holds the page l of the next 32 of the pair that is being fetched; the next one, and how many
    const uint8_t *kc = nullptr, *vc = nullptr, *ks = nullptr, *vs = nullptr;   // this lane's first 16 bytes of a page: codes and scales
    const unsigned stride = (unsigned)p.n_kv * kPageBytes;

    // asks for this warp's keys of the next page (nothing for a page that is not there)
    auto fetch = [&](int stage) {
        if (ahead.left > 0) {
            if (id_at == id_end) {
                const Tile w = tile_of<TILED>(p, st, ahead.t);
                const PageWalk walk(w.first, w.last, p.keep);
                id_at = 0;
                id_end = min(32, ahead.n - ahead.i);
                const int pi = walk.page(min(ahead.i + lane, ahead.n - 1));
                ids = pi < p.bt_stride ? p.block_table[(size_t)p.tok_seq[w.t0] * p.bt_stride + pi] : -1;
                if (ids >= p.n_pages) ids = -1;
                const size_t head = (size_t)(ahead.y / st.chunks) * kPageBytes + lane * 16;
                kc = p.k_pages + head + warp * kTiles * kCodes;
                vc = p.v_pages + head + warp * kTiles * kCodes;
                ks = p.k_pages + head + 32 * D + warp * kTiles * kScales;
                vs = p.v_pages + head + 32 * D + warp * kTiles * kScales;
            }
            const int id = __shfl_sync(0xffffffffu, ids, id_at++);
            if (id >= 0) {
                there |= 1u << stage;
                const size_t at = (size_t)(unsigned)id * stride;
                const uint32_t dst = ring_at + stage * kStage + lane * 16;
#pragma unroll
                for (int k = 0; k < kTiles * NG / 2; ++k) cp_async16(dst + k * 512, kc + at + k * 512);
#pragma unroll
                for (int k = 0; k < kTiles * NG / 2; ++k) cp_async16(dst + kVCodes + k * 512, vc + at + k * 512);
                if (NG == 4 || lane < 8 * NG) {
                    cp_async16(dst + kKScales, ks + at);
                    cp_async16(dst + kVScales, vs + at);
                }
            } else {
                there &= ~(1u << stage);
            }
            --ahead.left;
            if (++ahead.i == ahead.n && !CLUSTER) ahead.template next_pair<TILED>(p, st);
        }
        cp_async_commit();
    };
    static_assert(kTiles == 2, "a tile's copies are counted in whole rounds of a warp");
#pragma unroll
    for (int s = 0; s < kStreamStages - 1; ++s) fetch(s);

    int stage = 0;
    while (here.left > 0) {
        // -- a pair, or the part of it that lies here
        const int t = here.t, y = here.y, from = here.i, take = min(here.n - from, here.left);
        const int n_pages = here.n;
        const bool whole = !CLUSTER && take == n_pages;
        const int kvh = y / st.chunks, h0 = kvh * group + (y - kvh * st.chunks) * st.heads, heads = min(st.heads, (kvh + 1) * group - h0);
        const Tile tile = tile_of<TILED>(p, st, t);
        const int count = TILED ? tile.count : 1, t0 = TILED ? tile.t0 : t, nh = heads * count;      // tokens, and columns
        const int pos = tile.pos, last = TILED ? tile.last : pos, first = tile.first, first_last = TILED ? first_visible_key(last, p.window) : first;
        const PageWalk walk(first, last, p.keep);
        // this thread's columns 2 c and 2 c + 1 of each eight: which token of the tile
        int tok[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) tok[nt][e] = !TILED || st.tile == 1 ? 0 : min((8 * nt + 2 * c + e) / heads, count - 1);
        // Queries as the right-hand operand: head r of the column tile, the lanes of word (c, g), in the order of the codes' pairs.
        uint32_t qb[NT][NG][4];
        uint32_t qhi[NT], qlo[NT];     // the right-hand operand of (d_c, m_c): (-off, sum of q) of group c and head r, in two parts
        float col[NT][2];              // what scores of heads 2 c and 2 c + 1 are multiplied by
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint4 (&w)[NG] = raw[nt];
            float top = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float2 a = two_bf16(w[g].x), b = two_bf16(w[g].y), e = two_bf16(w[g].z), f = two_bf16(w[g].w);
                top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))),
                                       fmaxf(fmaxf(fabsf(e.x), fabsf(e.y)), fmaxf(fabsf(f.x), fabsf(f.y)))));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e with top < 2^e (from the exponent's bits; of zeros and the smallest numbers 2^-99)
            const int e = min(max((int)(__float_as_uint(top) >> 23), 27) - 126, 126);
            const float down = __int_as_float((127 - e) << 23), up = __int_as_float((127 + e) << 23);
            float qs = 0.0f, off = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float2 a = two_bf16(w[g].x), b = two_bf16(w[g].y), x = two_bf16(w[g].z), y = two_bf16(w[g].w);
                qb[nt][g][0] = pack_f16(a.x * down, x.x * down);
                qb[nt][g][1] = pack_f16(a.y * down, x.y * down);
                qb[nt][g][2] = pack_f16(b.x * down, y.x * down);
                qb[nt][g][3] = pack_f16(b.y * down, y.y * down);
                // the sums are those of the numbers as they are multiplied
                const float2 t0 = __half22float2(*reinterpret_cast<const __half2*>(&qb[nt][g][0])), t1 = __half22float2(*reinterpret_cast<const __half2*>(&qb[nt][g][1]));
                const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&qb[nt][g][2])), t3 = __half22float2(*reinterpret_cast<const __half2*>(&qb[nt][g][3]));
                float even = (t0.x + t0.y) + (t2.x + t2.y), odd = (t1.x + t1.y) + (t3.x + t3.y);
#pragma unroll
                for (int k = 1; k <= 2; k <<= 1) {
                    even += __shfl_xor_sync(0xffffffffu, even, k);
                    odd += __shfl_xor_sync(0xffffffffu, odd, k);
                }
                if (g == c) {
                    qs = even + odd;
                    off = 0.0f - (1024.0f * even + 64.0f * odd);
                }
            }
            qhi[nt] = pack_f16(off, qs);
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&qhi[nt]));
            qlo[nt] = pack_f16(off - hi.x, qs - hi.y);
            const float by = st.cap.out > 0.0f ? up : up * st.scale2;
            col[nt][0] = __shfl_sync(0xffffffffu, by, 8 * c);
            col[nt][1] = __shfl_sync(0xffffffffu, by, 8 * c + 4);
        }
        float o[NT][2 * NG][4];
        // row r: sum of p d (r even) or p m (r odd) of group r / 2; row 8: of p; heads 2 c and 2 c + 1
        float od[NT][4];
        float m[NT][2];                       // the weights' reference (0 until a key has been seen)
        float d_max = 1.0f, room = 11.0f;     // greatest step that the references leave room for, and how much that is
        unsigned seen = 0;                    // bit 2 nt + e: this thread's column e of the eight has seen a key
        bool all_seen = false;                // every column of the warp has
        const uint32_t ones = r == 0 ? 0x3C003C00u : 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k) o[nt][k][0] = o[nt][k][1] = o[nt][k][2] = o[nt][k][3] = 0.0f;
            od[nt][0] = od[nt][1] = od[nt][2] = od[nt][3] = 0.0f;
            m[nt][0] = m[nt][1] = 0.0f;
        }
        int pi = walk.page(from);
        for (int i = 0; i < take; ++i) {
            cp_async_wait<kStreamStages - 2>();
            __syncwarp();
            uint8_t* at = ring + stage * kStage;
            const bool missing = (there >> stage & 1) == 0;
            fetch(stage == 0 ? kStreamStages - 1 : stage - 1);
            stage = stage == kStreamStages - 1 ? 0 : stage + 1;
            const int key0 = pi * kPage + 16 * kTiles * warp;
            pi = from + i + 1 == walk.n_kept ? walk.lo : pi + 1;
            if (missing || key0 > last || (key0 + 16 * kTiles - 1 < first && key0 >= p.keep)) continue;      // none of these keys is seen
            const bool full = key0 >= first_last && key0 + 16 * kTiles - 1 <= pos;                          // all of them by all
            if (!full) {
                // what is not seen may hold anything, NaN too: its weight will be zero, and so must its numbers be
                const int key = key0 + lane;
                if (key > last || (key < first && key >= p.keep))
#pragma unroll
                    for (int g = 0; g < NG; ++g) *reinterpret_cast<uint32_t*>(at + kVScales + lane * 4 * NG + g * 4) = 0;
                __syncwarp();
            }
            // -- scores
            float z[kTiles][NT][4];
            uint32_t sd[kTiles][2];
            float step = 0.0f;
#pragma unroll
            for (int kt = 0; kt < kTiles; ++kt) {
                const uint8_t* kcode = at + kt * kCodes + r * 16 * NG + c * 4 * NG;
                const uint8_t* kscale = at + kKScales + kt * kScales + r * 4 * NG;
                uint32_t kw[2][NG], kd[2][NG], dm[2] = {0, 0};
                lds_words<NG>(kw[0], kcode);
                lds_words<NG>(kw[1], kcode + 128 * NG);
                lds_words<NG>(kd[0], kscale);
                lds_words<NG>(kd[1], kscale + 32 * NG);
                if (NG == 4 || c < NG) {
                    dm[0] = *reinterpret_cast<const uint32_t*>(kscale + c * 4);
                    dm[1] = *reinterpret_cast<const uint32_t*>(kscale + 32 * NG + c * 4);
                }
                // row r of the values' (d, m): those of keys 2 c, 2 c + 1 and of 2 c + 8, 2 c + 9
                if constexpr (NG == 4) {
                    ldmatrix_x2_trans(sd[kt][0], sd[kt][1], (uint32_t)__cvta_generic_to_shared(at) + kVScales + kt * kScales + (lane & 15) * 16);
                } else {
                    sd[kt][0] = sd[kt][1] = 0;
                    if (r < 2 * NG) {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(at + kVScales + kt * kScales) + 4 * c * NG + r;
                        sd[kt][0] = h[0] | (uint32_t)h[2 * NG] << 16;
                        sd[kt][1] = h[16 * NG] | (uint32_t)h[18 * NG] << 16;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    z[kt][nt][0] = z[kt][nt][1] = z[kt][nt][2] = z[kt][nt][3] = 0.0f;
                    mma_f16(z[kt][nt], dm[0], dm[1], dm[0], dm[1], qhi[nt], qlo[nt]);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t a[2][4] = {{codes_at<0>(kw[0][g]), codes_at<0>(kw[1][g]), codes_at<1>(kw[0][g]), codes_at<1>(kw[1][g])},
                                              {codes_at<2>(kw[0][g]), codes_at<2>(kw[1][g]), codes_at<3>(kw[0][g]), codes_at<3>(kw[1][g])}};
                    const float d0 = low_half(kd[0][g]), d1 = low_half(kd[1][g]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(acc, a[0][0], a[0][1], a[0][2], a[0][3], qb[nt][g][0], qb[nt][g][1]);
                        mma_f16(acc, a[1][0], a[1][1], a[1][2], a[1][3], qb[nt][g][2], qb[nt][g][3]);
                        z[kt][nt][0] = fmaf(acc[0], d0, z[kt][nt][0]);
                        z[kt][nt][1] = fmaf(acc[1], d0, z[kt][nt][1]);
                        z[kt][nt][2] = fmaf(acc[2], d1, z[kt][nt][2]);
                        z[kt][nt][3] = fmaf(acc[3], d1, z[kt][nt][3]);
                    }
                }
                const float2 f = __half22float2(__hmax2(*reinterpret_cast<const __half2*>(&sd[kt][0]), *reinterpret_cast<const __half2*>(&sd[kt][1])));
                step = fmaxf(step, fmaxf(f.x, f.y));
            }
            if (r & 1) step = 0.0f;
            // -- weights: first what 2 is raised to
            bool moves = step > d_max;
            if (full && p.slope_base == 0.0f && st.cap.out == 0.0f) {
#pragma unroll
                for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            z[kt][nt][e] = fmaf(z[kt][nt][e], col[nt][e & 1], 0.0f - m[nt][e & 1]);
                            moves |= z[kt][nt][e] > room + kLag;
                        }
            } else {
#pragma unroll
                for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + 16 * kt + r + 8 * (e >> 1), at_pos = TILED ? pos + tok[nt][e & 1] : pos;
                            float v = z[kt][nt][e] * col[nt][e & 1];
                            if (st.cap.out > 0.0f) v = capped_score(v, st.cap);
                            if (p.slope_base != 0.0f)
                                v -= slope_of(p, h0 + 8 * nt + 2 * c + (e & 1) - tok[nt][e & 1] * heads) * kLog2e * (float)(at_pos - key);
                            v -= m[nt][e & 1];
                            if (key > at_pos || (key < first_visible_key(at_pos, p.window) && key >= p.keep)) v = -INFINITY;
                            z[kt][nt][e] = v;
                            moves |= v > room + kLag;
                        }
            }
            if (!TILED) moves |= !all_seen;      // (every column sees the same keys: the first are the first of all)
            if (TILED && !all_seen)
#pragma unroll
                for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) moves |= !(seen >> (2 * nt + (e & 1)) & 1) && z[kt][nt][e] > -INFINITY;
            if (__any_sync(0xffffffffu, moves)) {
                float d = step;
#pragma unroll
                for (int x = 1; x < 32; x <<= 1) d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, x));
                d_max = fmaxf(d_max, d);
                const bool was_seen = all_seen;
                const float less = room - headroom(d_max);
                room -= less;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int kt = 0; kt < kTiles; ++kt) mx = fmaxf(mx, fmaxf(z[kt][nt][e], z[kt][nt][e + 2]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        // by how much the reference rises (the first time it may fall)
                        const bool unseen = TILED ? !(seen >> (2 * nt + e) & 1) : !was_seen;
                        float rise = unseen ? mx - room : fmaxf(less, mx - room);
                        if (mx == -INFINITY) rise = unseen ? 0.0f : less;
                        else if (TILED) seen |= 1u << (2 * nt + e);
                        const float corr = unseen ? 1.0f : fast_exp2(0.0f - rise);
                        m[nt][e] += rise;
                        od[nt][e] *= corr;
                        od[nt][e + 2] *= corr;
#pragma unroll
                        for (int kt = 0; kt < kTiles; ++kt) {
                            z[kt][nt][e] -= rise;
                            z[kt][nt][e + 2] -= rise;
                        }
#pragma unroll
                        for (int k = 0; k < 2 * NG; ++k) {
                            o[nt][k][e] *= corr;
                            o[nt][k][e + 2] *= corr;
                        }
                    }
                all_seen = !TILED || __all_sync(0xffffffffu, seen == (1u << (2 * NT)) - 1);
            }
            // -- values
#pragma unroll
            for (int kt = 0; kt < kTiles; ++kt) {
                uint32_t pb[NT][2];            // the weights as a right-hand operand: keys 2 c, 2 c + 1 (and + 8) of head r
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    pb[nt][0] = movmatrix_trans(pack_f16(fast_exp2(z[kt][nt][0]), fast_exp2(z[kt][nt][1])));
                    pb[nt][1] = movmatrix_trans(pack_f16(fast_exp2(z[kt][nt][2]), fast_exp2(z[kt][nt][3])));
                    mma_f16(od[nt], sd[kt][0], ones, sd[kt][1], ones, pb[nt][0], pb[nt][1]);
                }
                const uint8_t* vcode = at + kVCodes + kt * kCodes + (r * 4 + c) * 4 * NG;
                uint32_t vw[2][NG];
                lds_words<NG>(vw[0], vcode);
                lds_words<NG>(vw[1], vcode + 128 * NG);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t a[2][4] = {{centred_at<0>(vw[0][g]), centred_at<1>(vw[0][g]), centred_at<0>(vw[1][g]), centred_at<1>(vw[1][g])},
                                              {centred_at<2>(vw[0][g]), centred_at<3>(vw[0][g]), centred_at<2>(vw[1][g]), centred_at<3>(vw[1][g])}};
                    const uint32_t d0 = __shfl_sync(0xffffffffu, sd[kt][0], 8 * g + c), d1 = __shfl_sync(0xffffffffu, sd[kt][1], 8 * g + c);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t b0 = mul_f16x2(pb[nt][0], d0), b1 = mul_f16x2(pb[nt][1], d1);
                        mma_f16(o[nt][2 * g], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
                        mma_f16(o[nt][2 * g + 1], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
                    }
                }
            }
        }
        // -- on to the next pair: its queries come while this one's parts meet
        here.i += take;
        here.left -= take;
        const int left = here.left;
        if (!CLUSTER) {
            if (here.i == here.n) here.template next_pair<TILED>(p, st);
            ask_queries();
        }
        if (!CLUSTER && from == 0 && threadIdx.x == 0)      // the first block with a part of the pair, and the last
            st.parts[(size_t)t * st.pairs + y] =
                make_int2(blockIdx.x, whole ? (int)blockIdx.x : row.block_of(row.start(blockIdx.x + 1) - (left + take) + n_pages - 1));
        // -- the warps' parts meet: thread (r, c) holds lanes 32 g + 4 r to + 3 of heads 2 c and 2 c + 1.  Each warp leaves the other one's
        // head and finishes its own.
        __syncthreads();                 // (the last pair's part has been read)
        const int slot = 2 * blockIdx.x + (from > 0 ? 0 : 1);      // (a pair that began in an earlier block is this one's first)
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            if (pass == 1) __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if ((e == warp) != (pass == 1)) continue;
                    const int h = 8 * nt + 2 * c + e;
                    float* other = meet + h * (D + 4);
                    const float sum = __shfl_sync(0xffffffffu, od[nt][e + 2], c), ref = (TILED ? seen >> (2 * nt + e) & 1 : all_seen) ? m[nt][e] : -INFINITY;
                    float f0 = 1.0f, f1 = 0.0f, top = ref, total = sum;
                    if (pass == 1) {
                        top = fmaxf(ref, other[D]);
                        f0 = ref == -INFINITY ? 0.0f : exp2f(ref - top);
                        f1 = other[D] == -INFINITY ? 0.0f : exp2f(other[D] - top);
                        total = fmaf(other[D + 1], f1, sum * f0);
                        if (whole && h < nh) {
                            const float f = closing_factor(p, t0 + tok[nt][e], h0 + h - tok[nt][e] * heads, top / kLog2e, total);
                            f0 *= f;
                            f1 *= f;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float b = fmaf(8.0f, __shfl_sync(0xffffffffu, od[nt][e], 8 * g + c), __shfl_sync(0xffffffffu, od[nt][e], 8 * g + 4 + c));
                        const int d = 32 * g + 4 * r;
                        float4 v = make_float4(o[nt][2 * g][e] + b, o[nt][2 * g][e + 2] + b, o[nt][2 * g + 1][e] + b, o[nt][2 * g + 1][e + 2] + b);
                        if (pass == 0) {
                            *reinterpret_cast<float4*>(other + d) = v;
                            continue;
                        }
                        const float4 w = *reinterpret_cast<const float4*>(other + d);
                        v = make_float4(fmaf(w.x, f1, v.x * f0), fmaf(w.y, f1, v.y * f0), fmaf(w.z, f1, v.z * f0), fmaf(w.w, f1, v.w * f0));
                        if (h >= nh) continue;
                        if (CLUSTER) {
                            *reinterpret_cast<float4*>(other + d) = v;       // (this thread alone has read it)
                        } else if (whole) {
                            const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
                            const uint2 packed = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                            *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + ((size_t)(t0 + tok[nt][e]) * p.n_heads + h0 + h - tok[nt][e] * heads) * D + d) = packed;
                        } else {
                            *reinterpret_cast<float4*>(p.part + ((size_t)slot * COLS + h) * (D + 4) + d) = v;
                        }
                    }
                    if (r == 0 && pass == 0) {
                        other[D] = top;
                        other[D + 1] = total;
                    }
                    if (CLUSTER && r == 0 && pass == 1) {
                        other[D + 2] = top;
                        other[D + 3] = total;
                    }
                    if (!CLUSTER && r == 0 && pass == 1 && !whole && h < nh) {
                        float* part = p.part + ((size_t)slot * COLS + h) * (D + 4);
                        part[D] = top;
                        part[D + 1] = total;
                    }
                }
        }
    }
    cp_async_wait<0>();
    if constexpr (!CLUSTER) {
        zero_rows<D, TILED>(p, st);
    } else {
        // -- the blocks' parts meet: every block adds up its share of the lanes over all of them, in the order of their keys
        const int rank = blockIdx.x % st.cluster;
        if (here.n * rank / st.cluster == here.n * (rank + 1) / st.cluster) {         // (it had no page)
            if (threadIdx.x < COLS) {
                meet[threadIdx.x * (D + 4) + D + 2] = -INFINITY;
                meet[threadIdx.x * (D + 4) + D + 3] = 0.0f;
            }
        }
        cluster_barrier();
        const Tile tile = tile_of<TILED>(p, st, here.t);
        const int kvh = here.y / st.chunks, h0 = kvh * group + (here.y - kvh * st.chunks) * st.heads, heads = min(st.heads, (kvh + 1) * group - h0);
        const int count = TILED && st.cu != nullptr ? tile.count : 1;      // (a row of no sequence is zeros, see zero_rows)
        const int d0 = D * rank / st.cluster, lanes = D * (rank + 1) / st.cluster - d0;
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(meet);
        for (int x = threadIdx.x; x < heads * count * lanes; x += 32 * kStreamWarps) {
            const int h = x / lanes, d = d0 + x - h * lanes, tok = h / heads, head = h0 + h - tok * heads;
            const uint32_t col = at + h * (D + 4) * 4;
            float top = -INFINITY, sum = 0.0f, out = 0.0f;
#pragma unroll 8
            for (int k = 0; k < st.cluster; ++k) top = fmaxf(top, ld_cluster(col + (D + 2) * 4, k));
#pragma unroll 8
            for (int k = 0; k < st.cluster; ++k) {
                const float ref = ld_cluster(col + (D + 2) * 4, k), l = ld_cluster(col + (D + 3) * 4, k), v = ld_cluster(col + d * 4, k);
                if (ref == -INFINITY) continue;
                const float f = exp2f(ref - top);
                sum = fmaf(l, f, sum);
                out = fmaf(v, f, out);
            }
            const float f = here.n == 0 ? 0.0f : closing_factor(p, tile.t0 + tok, head, top / kLog2e, sum);
            reinterpret_cast<__nv_bfloat16*>(p.out)[((size_t)(tile.t0 + tok) * p.n_heads + head) * D + d] = __float2bfloat16_rn(here.n == 0 ? 0.0f : out * f);
        }
        cluster_barrier();          // a block's memory is read until every block is done
    }
}

// The parts of a pair that lies in several blocks, in the order of its keys.  grid = (tiles, pairs, columns of a pair), a thread a lane.
__global__ void __launch_bounds__(128) stream_merge_kernel(const AttnQ4 p, const Stream st, int cols) {
    const int y = blockIdx.y, h = blockIdx.z, D = p.D, d = threadIdx.x;
    wait_for_previous_kernels();
    let_next_kernel_start();
    const int2 b = st.parts[(size_t)blockIdx.x * st.pairs + y];
    if (b.x == b.y) return;              // that block has finished it
    const Tile tile = st.cu == nullptr ? Tile{(int)blockIdx.x, 1, 0, 0, 0} : tile_of<true>(p, st, blockIdx.x);
    const int group = p.n_heads / p.n_kv, kvh = y / st.chunks, h0 = kvh * group + y % st.chunks * st.heads;
    const int heads = min(st.heads, (kvh + 1) * group - h0), tok = h / heads, head = h0 + h - tok * heads;
    if (tok >= tile.count) return;       // no such column
    // the first part is its block's last, the others are their blocks' first
    const size_t step = (size_t)2 * cols * (D + 4);
    const float* first = p.part + ((size_t)(2 * b.x + 1) * cols + h) * (D + 4);
    const float* rest = p.part + ((size_t)(2 * b.x + 2) * cols + h) * (D + 4);
    const int n = b.y - b.x;
    // eight parts at a time, all asked for before any is needed
    float top = first[D], sum = first[D + 1], out = first[d];
    for (int i0 = 0; i0 < n; i0 += 8) {
        float ref[8], l[8], v[8], was = top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float* from = rest + min(i0 + i, n - 1) * step;
            ref[i] = i0 + i < n ? from[D] : -INFINITY;
            l[i] = from[D + 1];
            v[i] = from[d];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, ref[i]);
        float f = was == -INFINITY ? 0.0f : exp2f(was - top);
        sum *= f;
        out *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f = ref[i] == -INFINITY ? 0.0f : exp2f(ref[i] - top);
            sum = fmaf(l[i], f, sum);
            out = fmaf(v[i], f, out);
        }
    }
    const float f = closing_factor(p, tile.t0 + tok, head, top / kLog2e, sum);
    reinterpret_cast<__nv_bfloat16*>(p.out)[((size_t)(tile.t0 + tok) * p.n_heads + head) * D + d] = __float2bfloat16_rn(out * f);
}

// Pages of a token's walk that split s takes: [first, end).
__device__ __forceinline__ int2 split_pages(int n_walk, int n_splits, int s) {
    const int per = (n_walk + n_splits - 1) / n_splits;
    return make_int2(min(n_walk, s * per), min(n_walk, (s + 1) * per));
}

// A page at a time: keys as numbers to shared memory; scores, a thread a key and half of the heads; weights against the running
// maximum, a warp a head; values to shared memory; outputs, a thread a lane (two of heads of more than 128) and, of heads of 32 and 64 lanes,
// a part of the keys.  Bound by the latency of that chain (four sequences of up to 1 000 keys, 16 heads over 4 of 64 lanes: 11 us of which
// the bytes are worth 0.2; 25 with several pages a split), so a split is a page where there are blocks to spare.
template <int HEADS>
__global__ void __launch_bounds__(kAnyThreads) any_kernel(const AttnQ4 p) {
    extern __shared__ __align__(16) float any_smem[];
    constexpr int kHalf = HEADS >= 2 ? HEADS / 2 : 1;      // heads of a thread's scores
    const int D = p.D, NG = D / kGroup, ld = D + 4, tid = threadIdx.x;      // (rows 16 bytes further on than a multiple of all banks)
    float* tile = any_smem;                    // [64][D + 4]
    float* qs = tile + kPage * ld;             // [HEADS][D]
    float* ps = qs + HEADS * D;                // [64][HEADS] scores, then weights
    float* stat = ps + kPage * HEADS;          // [HEADS][3]: maximum, sum, correction
    const int t = blockIdx.x / p.n_splits, split = blockIdx.x % p.n_splits;
    const int group = p.n_heads / p.n_kv, chunks = (group + HEADS - 1) / HEADS;
    const int kvh = blockIdx.y / chunks, h0 = kvh * group + blockIdx.y % chunks * HEADS;
    const int nh = min(HEADS, (kvh + 1) * group - h0);
    const int seq = p.tok_seq[t], pos = p.tok_pos[t];
    const bool idle = seq < 0 || pos < 0 || seq >= p.bt_rows;
    const int first = idle ? 0 : first_visible_key(pos, p.window);
    const PageWalk walk(first, idle ? 0 : pos, p.keep);
    const int2 mine = idle ? make_int2(0, 0) : split_pages(walk.n, p.n_splits, split);
    for (int i = tid; i < HEADS * D; i += kAnyThreads)
        qs[i] = idle || i >= nh * D ? 0.0f : ld_f(p.q, ((size_t)t * p.n_heads + h0) * D + i, p.dt) * p.scale;
    if (tid < HEADS) {
        stat[tid * 3] = -INFINITY;
        stat[tid * 3 + 1] = 0.0f;
    }
    // the outputs' lanes and keys of this thread: lane d0 (and d0 + 128) of the keys from k0, every k_step-th
    const int parts = D <= 32 ? 4 : D <= 64 ? 2 : 1, wide = kAnyThreads / parts, d0 = tid % wide, k0 = tid / wide;
    float acc[HEADS][2];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) acc[h][0] = acc[h][1] = 0.0f;
    for (int i = mine.x; i < mine.y; ++i) {
        const int pi = walk.page(i), page = pi < p.bt_stride ? p.block_table[(size_t)seq * p.bt_stride + pi] : -1;
        if (page < 0 || page >= p.n_pages) continue;      // no such page: nothing is seen of it
        const int key0 = pi * kPage;
        const size_t at = ((size_t)page * p.n_kv + kvh) * q4_page_bytes(D);
        const uint8_t* kb = p.k_pages + at;
        const uint8_t* vb = p.v_pages + at;
        auto seen = [&](int key) { return key <= pos && (key >= first || key < p.keep); };
        __syncthreads();
#pragma unroll 4
        for (int w = tid; w < kPage * 4 * NG; w += kAnyThreads) {        // a word: eight lanes of one key
            const int row = w / (4 * NG), c = w % (4 * NG) / NG, g = w % NG;
            const uint32_t u = reinterpret_cast<const uint32_t*>(kb)[w];
            const float2 dm = __half22float2(reinterpret_cast<const __half2*>(kb + q4_scales_at(D))[row * NG + g]);
            float4* to = reinterpret_cast<float4*>(tile + row * ld + 32 * g + 8 * c);
            to[0] = make_float4(q4_number(u & 15, dm), q4_number(u >> 4 & 15, dm), q4_number(u >> 8 & 15, dm), q4_number(u >> 12 & 15, dm));
            to[1] = make_float4(q4_number(u >> 16 & 15, dm), q4_number(u >> 20 & 15, dm), q4_number(u >> 24 & 15, dm), q4_number(u >> 28, dm));
        }
        __syncthreads();
        {
            const int row = tid % kPage, hb = tid / kPage * kHalf;
            float z[kHalf];
#pragma unroll
            for (int h = 0; h < kHalf; ++h) z[h] = 0.0f;
            if (hb < HEADS) {
                for (int d = 0; d < D; d += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(tile + row * ld + d);
#pragma unroll
                    for (int h = 0; h < kHalf; ++h) {
                        const float4 q = *reinterpret_cast<const float4*>(qs + (hb + h) * D + d);
                        z[h] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, z[h]))));
                    }
                }
                const bool see = seen(key0 + row);
#pragma unroll
                for (int h = 0; h < kHalf; ++h) {
                    if (p.cap != 0.0f) z[h] = p.cap * tanhf(z[h] / p.cap);
                    z[h] -= slope_of(p, h0 + hb + h) * (float)(pos - key0 - row);
                    ps[row * HEADS + hb + h] = see ? z[h] : -INFINITY;
                }
            }
        }
        __syncthreads();
        // weights against the running maximum: a warp a head
        for (int h = tid >> 5; h < nh; h += kAnyThreads / 32) {
            const int lane = tid & 31;
            const float a = ps[lane * HEADS + h], b = ps[(32 + lane) * HEADS + h];
            const float m0 = stat[h * 3], m1 = fmaxf(m0, warp_max(fmaxf(a, b)));
            const float ea = m1 == -INFINITY ? 0.0f : expf(a - m1), eb = m1 == -INFINITY ? 0.0f : expf(b - m1);
            const float sum = warp_sum(ea + eb);
            ps[lane * HEADS + h] = ea;
            ps[(32 + lane) * HEADS + h] = eb;
            __syncwarp();
            if (lane == 0) {
                const float corr = m1 == -INFINITY ? 1.0f : expf(m0 - m1);
                stat[h * 3] = m1;
                stat[h * 3 + 1] = fmaf(stat[h * 3 + 1], corr, sum);
                stat[h * 3 + 2] = corr;
            }
        }
        // values: what no query may see counts as zero whatever lies there
#pragma unroll 4
        for (int w = tid; w < kPage * 4 * NG; w += kAnyThreads) {        // a word: four lanes of two positions
            const int g = w % NG, pr = w / NG % 4, r = w / (4 * NG) % 8, row = w / (32 * NG) * 8 + 2 * pr;
            const uint32_t u = reinterpret_cast<const uint32_t*>(vb)[w];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 dm = __half22float2(reinterpret_cast<const __half2*>(vb + q4_scales_at(D))[(row + k) * NG + g]);
                const uint32_t c = u >> (16 * k);
                float4 v = make_float4(q4_number(c & 15, dm), q4_number(c >> 4 & 15, dm), q4_number(c >> 8 & 15, dm), q4_number(c >> 12 & 15, dm));
                if (!seen(key0 + row + k)) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<float4*>(tile + (row + k) * ld + 32 * g + 4 * r) = v;
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = d0 + e * kAnyThreads;
            if (d >= D) continue;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) acc[h][e] *= h < nh ? stat[h * 3 + 2] : 0.0f;
#pragma unroll 8
            for (int row = k0; row < kPage; row += parts) {
                const float v = tile[row * ld + d];
#pragma unroll
                for (int h = 0; h < HEADS; ++h) acc[h][e] = fmaf(h < nh ? ps[row * HEADS + h] : 0.0f, v, acc[h][e]);
            }
        }
    }
    __syncthreads();
    if (parts > 1) {            // the keys' parts of heads of few lanes meet, in order
        float* sums = tile;     // [HEADS][128]
#pragma unroll
        for (int h = 0; h < HEADS; ++h) sums[h * kAnyThreads + tid] = acc[h][0];
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float s = sums[h * kAnyThreads + d0];
            for (int k = 1; k < parts; ++k) s += sums[h * kAnyThreads + k * wide + d0];
            acc[h][0] = s;
        }
    }
    if (k0 != 0) return;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= nh) break;
        const float m = stat[h * 3], l = stat[h * 3 + 1];
        const size_t row = (size_t)t * p.n_heads + h0 + h;
        if (p.n_splits == 1) {
            const float f = idle ? 0.0f : closing_factor(p, t, h0 + h, m, l);
            for (int e = 0; e < 2; ++e) {
                const int d = d0 + e * kAnyThreads;
                if (d < D) st_f(p.out, row * D + d, p.dt, acc[h][e] * f);
            }
        } else {
            float* o = p.part + (row * p.n_splits + split) * D;
            for (int e = 0; e < 2; ++e) {
                const int d = d0 + e * kAnyThreads;
                if (d < D) o[d] = acc[h][e];
            }
            if (d0 == 0) {
                float* ml = p.part + (size_t)p.n * p.n_heads * p.n_splits * D + (row * p.n_splits + split) * 2;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// grid = (n, n_heads): a block a row of a head, a warp of which makes the splits' factors.
__global__ void __launch_bounds__(kAnyThreads) merge_any_kernel(const AttnQ4 p) {
    __shared__ float factor[64];
    __shared__ float whole;
    const int h = blockIdx.y, t = blockIdx.x, lane = threadIdx.x;
    const size_t row = (size_t)t * p.n_heads + h;
    const float2* ml = reinterpret_cast<const float2*>(p.part + (size_t)p.n * p.n_heads * p.n_splits * p.D) + row * p.n_splits;
    if (lane < 32) {
        float2 a = make_float2(-INFINITY, 0.0f), b = a;
        if (lane < p.n_splits) a = ml[lane];
        if (lane + 32 < p.n_splits) b = ml[lane + 32];
        const float m = warp_max(fmaxf(a.x, b.x));
        const float fa = a.x == -INFINITY ? 0.0f : expf(a.x - m), fb = b.x == -INFINITY ? 0.0f : expf(b.x - m);
        factor[lane] = fa;
        factor[lane + 32] = fb;
        const float l = warp_sum(fmaf(a.y, fa, b.y * fb));
        if (lane == 0) whole = p.tok_seq[t] < 0 || p.tok_pos[t] < 0 || p.tok_seq[t] >= p.bt_rows ? 0.0f : closing_factor(p, t, h, m, l);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kAnyThreads) {
        float o = 0.0f;
#pragma unroll 8
        for (int s = 0; s < p.n_splits; ++s) o = fmaf(p.part[(row * p.n_splits + s) * p.D + d], factor[s], o);
        st_f(p.out, row * p.D + d, p.dt, o * whole);
    }
}

}  // namespace

// Heads of a block, and splits of a token's pages: enough blocks for the device, each with a page of the longest token at least.
static int any_heads(int group) { return group >= 8 ? 8 : group > 2 ? 4 : group; }
static int any_splits(int n, int n_heads, int n_kv, int longest) {
    const int group = n_heads / n_kv;
    const long blocks = (long)n * n_kv * ((group + any_heads(group) - 1) / any_heads(group));
    const long want = (4L * sm_count() + blocks - 1) / blocks, room = longest / kPage + 1;
    const long s = want < room ? want : room;
    return s < 1 ? 1 : (s > 64 ? 64 : (int)s);
}

static bool sizes_ok(int n, int n_heads, int n_kv, int D) {
    return n >= 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && D >= 32 && D <= 256 && D % 32 == 0;
}

// Whether the tensor-core kernel takes these sizes.  It has a capped score as a difference of two numbers of the cap's size: an error of
// some 1e-7 of the cap in the exponent, which beyond this one would show (a hundredth at 65 536, a tenth at 10^6).
constexpr float kMaxStreamCap = 4096.0f;
static bool streams(int dt, int D, float cap) { return dt == DT_BF16 && D <= 128 && cap <= kMaxStreamCap; }

// Blocks of a token's pages' row, all of which run at once, and how the heads of a key/value head are dealt with.
constexpr int kStreamMinPlaces = 4;
constexpr int kClusterKeys = 8 * kPage;      // see cluster_of
static int stream_tiles(int n_heads, int n_kv) { return n_heads / n_kv > 8 ? 2 : 1; }
static int stream_smem(int D, int tiles) {
    return kStreamWarps * kStreamStages * 40 * D + 8 * tiles * (D + 4) * (int)sizeof(float);
}
typedef void (*StreamKernel)(AttnQ4, Stream);
template <bool CLUSTER>
static StreamKernel stream_kernel_of(int D, int tiles) {
    switch (D / 32 * 2 + tiles - 1) {
        case 2: return stream_kernel<1, 1, CLUSTER>;
        case 3: return stream_kernel<1, 2, CLUSTER>;
        case 4: return stream_kernel<2, 1, CLUSTER>;
        case 5: return stream_kernel<2, 2, CLUSTER>;
        case 6: return stream_kernel<3, 1, CLUSTER>;
        case 7: return stream_kernel<3, 2, CLUSTER>;
        case 8: return stream_kernel<4, 1, CLUSTER>;
        default: return stream_kernel<4, 2, CLUSTER>;
    }
}
// Blocks of one kernel that the current device runs at once (asked once for each).
static int stream_blocks(int D, int tiles) {
    static int known[64][10] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count();
    int& n = known[dev][D / 32 * 2 + tiles - 1];
    if (n == 0) {
        const StreamKernel k = stream_kernel_of<false>(D, tiles);
        int per = 0;
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, stream_smem(D, tiles)) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, k, 32 * kStreamWarps, stream_smem(D, tiles)) != cudaSuccess || per < 1) {
            cudaGetLastError();
            per = 1;
        }
        n = per * sm_count();
    }
    return n;
}

// Blocks of a cluster that shares a pair, or 0: the row of pages.  Clusters, where they all run at once and either keep the device's blocks
// half busy or have at most eight pages a block (32 heads over 8, us, the row / clusters of 8 / of 16): one sequence of 300 keys 11.5 / 6.9 /
// 7.8, of 2 500 13.9 / 10.6 / 9.8, of 4 500 16.5 / 14.2 / 11.7; four of 2 500 15.7 / 11.3 / 13.3; twelve of 4 500 27.6 / 20.9 / -.
static int cluster_of(long pairs, int longest, int D, int tiles) {
    static int fit[64][10][2] = {};      // clusters of 8 and of 16 that the device runs at once (0: not asked yet)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    for (int i = 1; i >= 0; --i) {
        const int n = 8 << i;
        if (i == 1 && (longest <= 2048 || pairs * n > 2L * sm_count())) continue;
        int& f = fit[dev][D / 32 * 2 + tiles - 1][i];
        if (f == 0) {
            const StreamKernel k = stream_kernel_of<true>(D, tiles);
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)n;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3((unsigned)n);
            cfg.blockDim = dim3(32 * kStreamWarps);
            cfg.dynamicSmemBytes = stream_smem(D, tiles);
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, stream_smem(D, tiles)) != cudaSuccess ||
                cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
                cudaOccupancyMaxActiveClusters(&clusters, k, &cfg) != cudaSuccess) {
                cudaGetLastError();
                clusters = 0;
            }
            f = clusters > 0 ? clusters : -1;
        }
        if (pairs <= f && (longest <= n * kClusterKeys || 2 * pairs >= f)) return n;
    }
    return 0;
}

// Floats of scratch for a call of these sizes, `longest` the most keys that a token may see.
extern "C" long nncpu_attention_q4_scratch(int n, int n_heads, int n_kv, int D, int dt, int longest, float cap) {
    if (n <= 0 || !sizes_ok(n, n_heads, n_kv, D)) return 0;
    if (streams(dt, D, cap)) {
        // (enough for one column tile and for two, and for parts token by token)
        const int group = n_heads / n_kv, chunks = (group + 7) / 8;
        const long one = 8L * stream_blocks(D, 1), two = 16L * stream_blocks(D, 2);
        return 2L * (one > two ? one : two) * (D + 4) + 2L * n * n_kv * chunks;
    }
    const int s = any_splits(n, n_heads, n_kv, longest);
    return s > 1 ? (long)n * n_heads * s * (D + 2) : 0;
}

// one_seq (what the tensor-core kernel takes; the other one leaves it aside): the tokens are those of ONE sequence, at consecutive positions, from one_seq[0] to before
// one_seq[1] of the n; several of them then go through the pages together.
extern "C" int nncpu_attention_q4(const void* q, int dt, const uint8_t* k_pages, const uint8_t* v_pages, int n_pages,
                                  const int* block_table, int bt_rows, int bt_stride, const int* tok_seq, const int* tok_pos, void* out, float* part,
                                  long part_floats, int n, int n_heads, int n_kv, int D, float scale, int window, int keep,
                                  float slope_base, const float* sinks, float cap, const float* head_gate, int gate_ld, int longest,
                                  const int* one_seq, cudaStream_t stream) {
    NN_CHECK(sizes_ok(n, n_heads, n_kv, D), "attention_q4: %d tokens, %d heads over %d of %d lanes (whole groups of 32, at most 256)", n, n_heads, n_kv, D);
    NN_CHECK(cap >= 0.0f && keep >= 0 && (keep == 0 || window > 0) && (head_gate == nullptr || gate_ld >= n_heads),
             "attention_q4: cap %f, %d kept keys, gate rows of %d", cap, keep, gate_ld);
    NN_CHECK(bt_rows > 0 && bt_stride > 0 && n_pages > 0 && longest > 0, "attention_q4: %d pages, %d tables of %d, at most %d keys", n_pages, bt_rows,
             bt_stride, longest);
    const long need = nncpu_attention_q4_scratch(n, n_heads, n_kv, D, dt, longest, cap);
    NN_CHECK(need <= part_floats, "attention_q4: %ld floats of scratch, %ld are needed", part_floats, need);
    if (n == 0) return 0;
    AttnQ4 p{q, dt, k_pages, v_pages, n_pages, block_table, bt_rows, bt_stride, tok_seq, tok_pos, out, part, n, n_heads, n_kv, D, scale, window, keep,
             slope_base, sinks, cap, head_gate, gate_ld, any_splits(n, n_heads, n_kv, longest)};
    const int group = n_heads / n_kv;
    if (streams(dt, D, cap)) {
        NN_CHECK((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)part % 16 == 0,
                 "attention_q4: bfloat16 queries, output and scratch start on 16-byte boundaries");
        // several tokens of one sequence: in two column tiles, as many as have columns there
        const int tiles = one_seq != nullptr && n > 1 ? 2 : stream_tiles(n_heads, n_kv), chunks = (group + 8 * tiles - 1) / (8 * tiles);
        const int heads = (group + chunks - 1) / chunks, tile = one_seq != nullptr && n > 1 ? 16 / heads : 1;
        const int n_tiles = (n + tile - 1) / tile;
        const int cluster = cluster_of((long)n_tiles * n_kv * chunks, longest, D, tiles);
        NN_CHECK((long)n_tiles * n_kv * chunks * (bt_stride + 3L) < (1L << 31), "attention_q4: %d tokens of up to %d pages", n, bt_stride);
        NN_CHECK(n_kv <= 65535 / chunks, "attention_q4: %d key/value heads in %d parts", n_kv, chunks);
        Stream st{heads, chunks, n_kv * chunks, tile, n_tiles, one_seq, kStreamMinPlaces, stream_blocks(D, tiles), scale * kLog2e,
                  score_cap(scale, cap), cluster, nullptr};
        st.parts = reinterpret_cast<int2*>(part + 2L * st.blocks * 8 * tiles * (D + 4));
        // All blocks of the first kernel have to run at once, six to an SM, so it is not launched to start under the end of the one
        // before: beside blocks of that one an SM may find room for five, and the sixth, begun when those are done, doubles the time
        // (64 sequences of up to 8 000 keys: 84 us instead of 71).  The second one is.
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        cfg.blockDim = dim3(32 * kStreamWarps);
        cfg.dynamicSmemBytes = stream_smem(D, tiles);
        cfg.stream = stream;
        cfg.attrs = attr;
        cudaError_t e;
        if (cluster > 0) {
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)cluster;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3((unsigned)(n_tiles * st.pairs * cluster));
            cfg.numAttrs = 1 + overlap_attribute(attr + 1);
            e = cudaLaunchKernelEx(&cfg, stream_kernel_of<true>(D, tiles), p, st);
            NN_CHECK(e == cudaSuccess, "attention_q4: launch failed: %s", cudaGetErrorString(e));
            return 0;
        }
        cfg.gridDim = dim3((unsigned)st.blocks);
        cfg.numAttrs = 0;
        e = cudaLaunchKernelEx(&cfg, stream_kernel_of<false>(D, tiles), p, st);
        NN_CHECK(e == cudaSuccess, "attention_q4: launch failed: %s", cudaGetErrorString(e));
        cfg.gridDim = dim3((unsigned)n_tiles, (unsigned)st.pairs, (unsigned)(st.heads * tile));
        cfg.blockDim = dim3(D);
        cfg.dynamicSmemBytes = 0;
        cfg.numAttrs = overlap_attribute(attr);
        e = cudaLaunchKernelEx(&cfg, stream_merge_kernel, p, st, 8 * tiles);
        NN_CHECK(e == cudaSuccess, "attention_q4 (merge): launch failed: %s", cudaGetErrorString(e));
        return 0;
    }
    const int heads = any_heads(group), chunks = (group + heads - 1) / heads;
    const size_t smem = sizeof(float) * ((size_t)kPage * (D + 4) + (size_t)heads * (D + kPage + 3));
    NN_CHECK((uintptr_t)part % 16 == 0, "attention_q4: scratch starts on a 16-byte boundary");
    const auto any = heads == 8 ? any_kernel<8> : heads == 4 ? any_kernel<4> : heads == 2 ? any_kernel<2> : any_kernel<1>;
    NN_CHECK((long)n * p.n_splits < (1L << 31) && n_kv <= 65535 / chunks && n_heads <= 65535, "attention_q4: %d tokens in %d splits", n, p.n_splits);
    static bool done[4][64];
    if (first_use_on_this_device(done[heads == 8 ? 3 : heads / 2])) {
        const cudaError_t e = cudaFuncSetAttribute(any, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
        NN_CHECK(e == cudaSuccess, "attention_q4: shared memory: %s", cudaGetErrorString(e));
    }
    any<<<dim3((unsigned)(n * p.n_splits), (unsigned)(n_kv * chunks)), kAnyThreads, smem, stream>>>(p);
    NN_LAUNCH_OK("attention_q4");
    if (p.n_splits > 1) {
        merge_any_kernel<<<dim3((unsigned)n, (unsigned)n_heads), kAnyThreads, 0, stream>>>(p);
        NN_LAUNCH_OK("attention_q4 (merge)");
    }
    return 0;
}
