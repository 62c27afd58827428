// Keys and values in 4 bits: the append to the paged cache (with the heads' norms and rotation on the way), and the way back to
// numbers.  cache_q4.cuh says how the pages lie.
//
// The norm and the rotation are those of the 16- and 32-bit caches (crates/nncpu/src/model/forward.rs:278-351): q leaves as the
// attention reads it, a key is normed and rotated and a value taken as it is before they are cut to 4 bits.

#include <math.h>

#define NN_LIB cache_q4
#define NN_LAUNCH_OVERLAP
#include "common.cuh"
#include "cache_q4.cuh"

namespace {

struct Append {
    const void* qkv;        // [n, ld]: heads of q, then of k, then of v
    int qkv_dt, ld;
    const void* q_gamma;    // [D] or null
    const void* k_gamma;
    int g_dt;
    double eps;
    const float2* cs;       // [n, half] (cos, sin), or null: the pairs (i, i + half) of a head's first 2 half lanes turn
    int half;
    const int* tok_seq;
    const int* tok_pos;
    const int* block_table; // [bt_rows, bt_stride]
    int bt_rows, bt_stride;
    uint8_t* k_pages;       // [n_pages, n_kv, 40 D]
    uint8_t* v_pages;
    int n_pages;
    void* q_out;            // [n, n_heads D]
    int q_dt;
    int n, n_heads, n_kv, D;
    float temp_coef;        // c != 0: the query at position p times 1 + c ln(floor((p + 1) / temp_every) + 1)
    int temp_every;
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The page of a token's key, or -1 (a padding row, a position without a page).
__device__ __forceinline__ int page_of(const int* block_table, int bt_rows, int bt_stride, int n_pages, int seq, int pos) {
    if (seq < 0 || seq >= bt_rows || pos < 0 || pos / kPage >= bt_stride) return -1;
    const int p = block_table[(size_t)seq * bt_stride + pos / kPage];
    return p < n_pages ? p : -1;
}

// One head of one token, a warp's job; lane l holds lanes l, l + 32, ... of the head (one of every group).
template <int NG, typename F>
__device__ __forceinline__ void norm_rotate(F (&x)[NG], const void* gamma, int g_dt, F eps, const float2* cs, int half, F* row, int lane) {
    constexpr int D = 32 * NG;
    if (gamma != nullptr) {
        F s = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) s += x[g] * x[g];
        if constexpr (sizeof(F) == 8) s = warp_sum64(s);
        else s = warp_sum(s);
        const F r = F(1) / sqrt(s / F(D) + eps);
#pragma unroll
        for (int g = 0; g < NG; ++g) x[g] = x[g] * r * F(ld_f(gamma, 32 * g + lane, g_dt));
    }
    if (cs != nullptr) {
        __syncwarp();
#pragma unroll
        for (int g = 0; g < NG; ++g) row[32 * g + lane] = x[g];
        __syncwarp();
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int i = 32 * g + lane;
            if (i < 2 * half) {
                const bool second = i >= half;
                const float2 t = cs[second ? i - half : i];
                const F other = row[second ? i - half : i + half];
                x[g] = second ? x[g] * F(t.x) + other * F(t.y) : x[g] * F(t.x) - other * F(t.y);
            }
        }
    }
}

// A warp per (token, head of q, k or v): any sizes, types and strides.  Bound by instructions, its lanes' exchanges among them (2 048
// tokens of 32 heads over 8: 39 us with heads of 96 lanes, 71 of 256, whose bytes are worth 8 and 22; append_fast_kernel takes what
// models commonly have).
template <int NG>
__global__ void __launch_bounds__(256) append_kernel(const Append a) {
    constexpr int D = 32 * NG;
    __shared__ double rows[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_tok = a.n_heads + 2 * a.n_kv;
    const long item = (long)blockIdx.x * 8 + warp;
    if (item >= (long)a.n * per_tok) return;
    const int t = (int)(item / per_tok), h = (int)(item % per_tok);
    const int seq = a.tok_seq[t], pos = a.tok_pos[t];
    float x[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) x[g] = ld_f(a.qkv, (size_t)t * a.ld + (size_t)h * D + 32 * g + lane, a.qkv_dt);
    const float2* cs = a.cs == nullptr ? nullptr : a.cs + (size_t)t * a.half;
    if (h < a.n_heads) {
        norm_rotate<NG, float>(x, a.q_gamma, a.g_dt, (float)a.eps, cs, a.half, reinterpret_cast<float*>(rows[warp]), lane);
        float times = 1.0f;
        if (a.temp_coef != 0.0f) times = 1.0f + a.temp_coef * logf(floorf((float)(pos + 1) / (float)a.temp_every) + 1.0f);
#pragma unroll
        for (int g = 0; g < NG; ++g) st_f(a.q_out, ((size_t)t * a.n_heads + h) * D + 32 * g + lane, a.q_dt, x[g] * times);
        return;
    }
    const bool value = h >= a.n_heads + a.n_kv;
    const int kvh = (h - a.n_heads) - (value ? a.n_kv : 0);
    const int page = page_of(a.block_table, a.bt_rows, a.bt_stride, a.n_pages, seq, pos);
    if (page < 0) return;
    if (!value) {
        // In 64 bits: a key next to the border of two codes takes one or the other by its last bit.  B200's 64-bit rate is half of
        // its 32-bit one, and the kernel is bound by its loads and stores.
        double y[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) y[g] = x[g];
        norm_rotate<NG, double>(y, a.k_gamma, a.g_dt, a.eps, cs, a.half, rows[warp], lane);
#pragma unroll
        for (int g = 0; g < NG; ++g) x[g] = (float)y[g];
    }
    const int at = pos % kPage;
    uint8_t* base = (value ? a.v_pages : a.k_pages) + ((size_t)page * a.n_kv + kvh) * q4_page_bytes(D);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float v = q4_in_range(x[g]);
        const bool bad = __any_sync(0xffffffffu, v != v);
        float lo = v, hi = v;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        if (bad) lo = hi = __int_as_float(0x7FC00000);
        const Q4Scale s = q4_scale(lo, hi);
        uint32_t w = q4_code(v, s);
        if (value) {
            w <<= 4 * (lane & 3);
            w |= __shfl_xor_sync(0xffffffffu, w, 1);
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
            if ((lane & 3) == 0)
                reinterpret_cast<uint16_t*>(base)[2 * q4_value_word(at, lane >> 2, g, NG) + (at & 1)] = (uint16_t)w;
        } else {
            w <<= 4 * (lane & 7);
            w |= __shfl_xor_sync(0xffffffffu, w, 1);
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
            w |= __shfl_xor_sync(0xffffffffu, w, 4);
            if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(base)[q4_key_word(at, lane >> 3, g, NG)] = w;
        }
        if (lane == 0)
            reinterpret_cast<__half2*>(base + q4_scales_at(D))[at * NG + g] = __halves2half2(s.d, s.m);
    }
}

// ---------------------------------------------------------------------------
// Heads of 32, 64 and 128 lanes, rotated whole or not at all, in float32 rows of whole 16-byte pieces: T = D / 8 threads a head, each
// with four neighbouring lanes of either half, so that a rotation's partners are in one thread, a group is eight threads, and a
// thread's codes are two halves of words, which it stores.  A block takes a token and as many heads as it has rounds for, which share
// the token's angles.  grid = (n, blocks a token), 256 threads.
// Bound by instructions (62 % of the issue slots with four lanes a thread, whose rotation and norm took nine exchanges a head): 2 048
// tokens of 32 heads over 8 of 128 lanes, read back after, take 25.3 us; 31.8 with four lanes a thread; 32.5 and 27.2 in the registers
// of two and three blocks an SM.  Their bytes alone would take 12.1 us.
// ---------------------------------------------------------------------------
template <int D, typename F>
__device__ __forceinline__ void norm_rotate8(F (&x)[8], const float4* gamma, const float2 (&cs)[4], bool rotated, F eps, F times) {
    constexpr int T = D / 8;
    F r = times;
    if (gamma != nullptr) {
        F s = ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) + ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
#pragma unroll
        for (int o = T / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if constexpr (sizeof(F) == 8) r = rsqrt(s * (F(1) / D) + eps);
        else r = rsqrtf(s * (1.0f / D) + eps) * times;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[4 * i] *= r * F(gamma[i].x); x[4 * i + 1] *= r * F(gamma[i].y); x[4 * i + 2] *= r * F(gamma[i].z); x[4 * i + 3] *= r * F(gamma[i].w);
        }
    } else if (sizeof(F) == 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= r;
    }
    if (rotated) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const F a = x[e], b = x[e + 4];
            x[e] = a * F(cs[e].x) - b * F(cs[e].y);
            x[e + 4] = b * F(cs[e].x) + a * F(cs[e].y);
        }
    }
}

__device__ __forceinline__ float min_or_nan(float a, float b) {
    float m;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <int D>
__global__ void __launch_bounds__(256, 4) append_fast_kernel(const Append a) {
    constexpr int T = D / 8, NG = D / 32, kHeads = 256 / T;
    const int t = blockIdx.x, j = threadIdx.x % T, per_tok = a.n_heads + 2 * a.n_kv;
    wait_for_previous_kernels();
    let_next_kernel_start();
    const int seq = a.tok_seq[t], pos = a.tok_pos[t];
    const bool rotated = a.cs != nullptr;
    float2 cs[4] = {};
    if (rotated) {
        const float4* at = reinterpret_cast<const float4*>(a.cs + (size_t)t * (D / 2) + 4 * j);
        const float4 u = at[0], v = at[1];
        cs[0] = make_float2(u.x, u.y); cs[1] = make_float2(u.z, u.w); cs[2] = make_float2(v.x, v.y); cs[3] = make_float2(v.z, v.w);
    }
    float times = 1.0f;
    if (a.temp_coef != 0.0f) times = 1.0f + a.temp_coef * logf(floorf((float)(pos + 1) / (float)a.temp_every) + 1.0f);
    const int page = a.n_kv > 0 ? page_of(a.block_table, a.bt_rows, a.bt_stride, a.n_pages, seq, pos) : -1;
    const int at = page < 0 ? 0 : pos % kPage;
    const float* row = reinterpret_cast<const float*>(a.qkv) + (size_t)t * a.ld + 4 * j;
    // The next round's heads are asked for before a round's are worked on.  (All threads of a warp go round together: a round's last
    // heads may not be there.)
    const int stride = gridDim.y * kHeads, first = blockIdx.y * kHeads + threadIdx.x / T;
    auto ask = [&](int h, int half) {
        return h < per_tok ? *reinterpret_cast<const float4*>(row + (size_t)h * D + half * (D / 2)) : make_float4(0, 0, 0, 0);
    };
    float4 next0 = ask(first, 0), next1 = ask(first, 1);
    for (int h0 = blockIdx.y * kHeads; h0 < per_tok; h0 += stride) {
        const int h = h0 + threadIdx.x / T;
        const bool there = h < per_tok;
        const float4 v0 = next0, v1 = next1;
        next0 = ask(h + stride, 0);
        next1 = ask(h + stride, 1);
        float x[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        // a warp's heads are of one kind (all of q, all of k, ...) or take every branch that one of them takes
        const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
        float4 gamma[2] = {};
        if (const void* g = is_q ? a.q_gamma : is_v ? nullptr : a.k_gamma) {
            gamma[0] = ld_f4(g, 4 * j, a.g_dt);
            gamma[1] = ld_f4(g, D / 2 + 4 * j, a.g_dt);
        }
        if (__any_sync(0xffffffffu, there && is_q)) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e];
            norm_rotate8<D, float>(y, a.q_gamma != nullptr ? gamma : nullptr, cs, rotated, (float)a.eps, times);
            if (there && is_q) {
                const size_t to = ((size_t)t * a.n_heads + h) * D + 4 * j;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 z = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    if (a.q_dt == DT_F32) {
                        *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.q_out) + to + i * (D / 2)) = z;
                    } else {
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(z.x, z.y), hi = __floats2bfloat162_rn(z.z, z.w);
                        uint2 u;
                        u.x = *reinterpret_cast<const uint32_t*>(&lo);
                        u.y = *reinterpret_cast<const uint32_t*>(&hi);
                        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.q_out) + to + i * (D / 2)) = u;
                    }
                }
            }
        }
        if (!__any_sync(0xffffffffu, there && !is_q && page >= 0)) continue;
        if (__any_sync(0xffffffffu, there && !is_q && !is_v)) {
            // in 64 bits, see append_kernel
            double y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e];
            norm_rotate8<D, double>(y, a.k_gamma != nullptr ? gamma : nullptr, cs, rotated, a.eps, 1.0);
            if (!is_v)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
        }
        // A NaN stays in lo and hi.  (Limits of what is limited are limits of the limits: the lanes themselves only where one passes.)
        float lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo[i] = min_or_nan(min_or_nan(x[4 * i], x[4 * i + 1]), min_or_nan(x[4 * i + 2], x[4 * i + 3]));
            hi[i] = max_or_nan(max_or_nan(x[4 * i], x[4 * i + 1]), max_or_nan(x[4 * i + 2], x[4 * i + 3]));
        }
        if (D == 32) {          // (both halves are of one group, of four threads)
            lo[0] = lo[1] = min_or_nan(lo[0], lo[1]);
            hi[0] = hi[1] = max_or_nan(hi[0], hi[1]);
        }
        constexpr int kThreads = D == 32 ? 4 : 8;       // of a group
#pragma unroll
        for (int o = kThreads / 2; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                lo[i] = min_or_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
                hi[i] = max_or_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
            }
        if (fminf(lo[0], lo[1]) < -kHalfMax || fmaxf(hi[0], hi[1]) > kHalfMax) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = q4_in_range(x[e]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                lo[i] = q4_in_range(lo[i]);
                hi[i] = q4_in_range(hi[i]);
            }
        }
        const int kvh = h - a.n_heads - (is_v ? a.n_kv : 0), quad = j & 7;
        uint8_t* base = (is_v ? a.v_pages : a.k_pages) + ((size_t)max(page, 0) * a.n_kv + kvh) * q4_page_bytes(D);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Q4Scale s = q4_scale(lo[i], hi[i]);
            const uint16_t codes = (uint16_t)q4_codes(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], s);
            if (!there || is_q || page < 0) continue;
            const int g = D == 32 ? 0 : j / 8 + i * (NG / 2), four = D == 32 ? j + 4 * i : quad;     // the group, and the four of its eight
            const int half = is_v ? 2 * q4_value_word(at, four, g, NG) + (at & 1) : 2 * q4_key_word(at, four >> 1, g, NG) + (four & 1);
            reinterpret_cast<uint16_t*>(base)[half] = codes;
            if (four == 0) reinterpret_cast<__half2*>(base + q4_scales_at(D))[at * NG + g] = __halves2half2(s.d, s.m);
        }
    }
}

// What the cache holds of given tokens: a thread takes eight neighbouring lanes of a key and of a value.  (2 048 tokens of 8 heads of 128
// lanes to bfloat16: 6 us for 11 MB, most of it the latency of three loads one after another and the launch.)
__device__ __forceinline__ void put8(void* out, long i, int dt, const float (&x)[8]) {
    if (dt == DT_F32) {
        reinterpret_cast<float4*>(out)[2 * i] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(out)[2 * i + 1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
            u[e] = *reinterpret_cast<const uint32_t*>(&two);
        }
        reinterpret_cast<uint4*>(out)[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
__global__ void __launch_bounds__(256) read_kernel(const uint8_t* k_pages, const uint8_t* v_pages, int n_pages, const int* block_table,
                                                   int bt_rows, int bt_stride, const int* tok_seq, const int* tok_pos, void* k_out, void* v_out,
                                                   int out_dt, int n, int n_kv, int D) {
    wait_for_previous_kernels();
    let_next_kernel_start();
    const int per_tok = n_kv * D / 8, NG = D / kGroup;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)n * per_tok) return;
    const int t = (int)(i / per_tok), rest = (int)(i - (long)t * per_tok), h = rest / (D / 8), lane = (rest - h * (D / 8)) * 8;
    const int g = lane >> 5, c = (lane & 31) >> 3, pos = tok_pos[t];
    const int page = page_of(block_table, bt_rows, bt_stride, n_pages, tok_seq[t], pos), at = page < 0 ? 0 : pos % kPage;
    float k[8] = {}, v[8] = {};
    if (page >= 0) {
        const size_t base = ((size_t)page * n_kv + h) * q4_page_bytes(D);
        const uint8_t *kb = k_pages + base, *vb = v_pages + base;
        const uint32_t kw = reinterpret_cast<const uint32_t*>(kb)[q4_key_word(at, c, g, NG)];
        const uint16_t* vh = reinterpret_cast<const uint16_t*>(vb) + (at & 1);
        const uint32_t v0 = vh[2 * q4_value_word(at, 2 * c, g, NG)], v1 = vh[2 * q4_value_word(at, 2 * c + 1, g, NG)];
        const float2 ks = __half22float2(reinterpret_cast<const __half2*>(kb + q4_scales_at(D))[at * NG + g]);
        const float2 vs = __half22float2(reinterpret_cast<const __half2*>(vb + q4_scales_at(D))[at * NG + g]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            k[e] = q4_number(kw >> (4 * e) & 15, ks);
            v[e] = q4_number((e < 4 ? v0 : v1) >> (4 * (e & 3)) & 15, vs);
        }
    }
    put8(k_out, i, out_dt, k);
    put8(v_out, i, out_dt, v);
}

// The pages that a step's tokens see, as numbers in pages of their own: float16 or float32 rows of `lanes` >= D lanes, zeros behind a
// head's own and in rows behind the sequence's end (whatever the cache holds there).  Page i of sequence b goes to page b * width + i,
// and the table for the attention kernels is written too.  A block takes a page of keys or of values of one head, a thread eight
// neighbouring lanes of a row at a time: grid = (width, 2 n_kv, n_seqs).  (2 048 positions of 8 heads of 128 lanes to float16: 5.5 us
// for 2.6 MB read and 8.4 written; the attention over them takes 51.  To take the codes out inside the attention kernel would do it
// again for every tile of queries: 16 times here.)
struct Expand {
    const uint8_t* k_pages;
    const uint8_t* v_pages;
    int n_pages;
    const int* block_table;
    int bt_stride;
    const int* cu_seqlens;
    const int* tok_seq;
    const int* tok_pos;
    void* k_out;            // [n_seqs * width, n_kv, 64, lanes]
    void* v_out;
    int* table;             // [n_seqs, width]
    int* places;            // null, or [2, n_tok]: the tokens' sequences (-1: without a table) and positions (within it)
    int n_tok, n_kv, D, lanes, window, keep;
};

__device__ __forceinline__ void put8_row(float* row, const float (&x)[8]) {
    reinterpret_cast<float4*>(row)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(row)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void put8_row(__half* row, const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {       // (d c + m may pass the range by a rounding)
        const __half2 two = __floats2half2_rn(q4_in_range(x[2 * e]), q4_in_range(x[2 * e + 1]));
        u[e] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(row) = make_uint4(u[0], u[1], u[2], u[3]);
}

constexpr int kExpandThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const Expand p) {
    let_next_kernel_start();           // (which reads the step's metadata before it waits for this one)
    const int pi = blockIdx.x, b = blockIdx.z, row = b * gridDim.x + pi;
    const bool values = blockIdx.y >= p.n_kv;
    const int h = values ? blockIdx.y - p.n_kv : blockIdx.y;
    if (blockIdx.y == 0 && threadIdx.x == 0) p.table[row] = row;
    if (blockIdx.y == 1 && p.places != nullptr)
        for (int i = row * kExpandThreads + threadIdx.x; i < p.n_tok; i += gridDim.x * gridDim.z * kExpandThreads) {
            const int seq = p.tok_seq[i], pos = p.tok_pos[i];
            p.places[i] = pos < 0 || seq >= (int)gridDim.z ? -1 : seq;
            p.places[p.n_tok + i] = min(pos, (int)gridDim.x * kPage - 1);
        }
    int id = pi < p.bt_stride ? p.block_table[(size_t)b * p.bt_stride + pi] : -1;      // (asked for beside the next two)
    const int t0 = p.cu_seqlens[b], t1 = p.cu_seqlens[b + 1];
    if (t1 <= t0) return;
    const int first = first_visible_key(p.tok_pos[t0], p.window), last = p.tok_pos[t1 - 1];
    if (pi * kPage > last || (pi * kPage + kPage - 1 < first && pi * kPage >= p.keep)) return;      // no token sees the page
    if (id >= p.n_pages) id = -1;
    const int D = p.D, NG = D / kGroup, rows = id < 0 ? 0 : min(kPage, last + 1 - pi * kPage), per_row = p.lanes / 8;
    const uint8_t* base = (values ? p.v_pages : p.k_pages) + ((size_t)max(id, 0) * p.n_kv + h) * q4_page_bytes(D);
    const __half2* scales = reinterpret_cast<const __half2*>(base + q4_scales_at(D));
    T* out = reinterpret_cast<T*>(values ? p.v_out : p.k_out) + ((size_t)row * p.n_kv + h) * kPage * p.lanes;
#pragma unroll 4
    for (int i = threadIdx.x; i < kPage * per_row; i += kExpandThreads) {
        const int at = i / per_row, lane = (i - at * per_row) * 8, g = lane >> 5, c = (lane & 31) >> 3;
        float x[8] = {};
        if (at < rows && lane < D) {
            uint32_t u;
            if (values) {
                const uint16_t* half = reinterpret_cast<const uint16_t*>(base) + (at & 1);
                u = half[2 * q4_value_word(at, 2 * c, g, NG)] | (uint32_t)half[2 * q4_value_word(at, 2 * c + 1, g, NG)] << 16;
            } else {
                u = reinterpret_cast<const uint32_t*>(base)[q4_key_word(at, c, g, NG)];
            }
            const float2 dm = __half22float2(scales[at * NG + g]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = q4_number(u >> (4 * e) & 15, dm);
        }
        put8_row(out + (size_t)at * p.lanes + lane, x);
    }
}

// bfloat16 heads of D lanes in rows of `lanes`, zeros behind them.
__global__ void __launch_bounds__(256) longer_heads_kernel(const uint16_t* x, uint16_t* out, long rows, int D, int lanes) {
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= rows * lanes) return;
    const long row = i / lanes;
    const int lane = (int)(i % lanes);
    *reinterpret_cast<uint4*>(out + i) = lane < D ? *reinterpret_cast<const uint4*>(x + row * D + lane) : make_uint4(0, 0, 0, 0);
}

}  // namespace

static bool q4_lanes_ok(int D) { return D >= 32 && D <= 256 && D % 32 == 0; }

extern "C" int nncpu_qk_norm_rope_append_q4(const void* qkv, int qkv_dt, int ld, const void* q_gamma, const void* k_gamma, int g_dt,
                                            double eps, const float* cos_sin, int half, const int* tok_seq, const int* tok_pos,
                                            const int* block_table, int bt_rows, int bt_stride, uint8_t* k_pages, uint8_t* v_pages, int n_pages,
                                            void* q_out, int q_dt, int n, int n_heads, int n_kv, int D, float temp_coef,
                                            int temp_every, cudaStream_t stream) {
    NN_CHECK(q4_lanes_ok(D), "qk_norm_rope_append_q4: heads of %d lanes (whole groups of 32, at most 256)", D);
    NN_CHECK(n >= 0 && n_heads > 0 && n_kv >= 0 && ld >= (n_heads + 2 * n_kv) * D, "qk_norm_rope_append_q4: %d heads over %d in rows of %d", n_heads, n_kv, ld);
    NN_CHECK(half >= 0 && 2 * half <= D, "qk_norm_rope_append_q4: %d rotated pairs in a head of %d lanes", half, D);
    NN_CHECK(n_kv == 0 || (bt_stride > 0 && n_pages > 0 && k_pages != nullptr && v_pages != nullptr), "qk_norm_rope_append_q4: no pages to append to");
    NN_CHECK(temp_coef == 0.0f || temp_every > 0, "qk_norm_rope_append_q4: a temperature every %d positions", temp_every);
    if (n == 0) return 0;
    Append a{qkv, qkv_dt, ld, q_gamma, k_gamma, g_dt, eps, reinterpret_cast<const float2*>(cos_sin), half, tok_seq, tok_pos, block_table,
             bt_rows, bt_stride, k_pages, v_pages, n_pages, q_out, q_dt, n, n_heads, n_kv, D, temp_coef, temp_every};
    if ((D == 32 || D == 64 || D == 128) && qkv_dt == DT_F32 && ld % 4 == 0 && (cos_sin == nullptr || half == D / 2) && (uintptr_t)qkv % 16 == 0 &&
        (uintptr_t)q_out % 16 == 0 && (uintptr_t)cos_sin % 16 == 0 && (uintptr_t)q_gamma % 16 == 0 && (uintptr_t)k_gamma % 16 == 0) {
        const int rounds = (n_heads + 2 * n_kv + 2048 / D - 1) / (2048 / D);      // a block's rounds, were it alone with a token
        // as many blocks as eight on each SM ask for
        long per = (8L * sm_count() + n - 1) / n;
        per = per < rounds ? per : rounds;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)n, (unsigned)per);
        cfg.blockDim = dim3(256);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        cfg.attrs = attr;
        cfg.numAttrs = overlap_attribute(attr);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, D == 32 ? append_fast_kernel<32> : D == 64 ? append_fast_kernel<64> : append_fast_kernel<128>, a);
        NN_CHECK(e == cudaSuccess, "qk_norm_rope_append_q4: launch failed: %s", cudaGetErrorString(e));
        return 0;
    }
    const long items = (long)n * (n_heads + 2 * n_kv);
    const dim3 grid((unsigned)((items + 7) / 8));
    switch (D / 32) {
        case 1: append_kernel<1><<<grid, 256, 0, stream>>>(a); break;
        case 2: append_kernel<2><<<grid, 256, 0, stream>>>(a); break;
        case 3: append_kernel<3><<<grid, 256, 0, stream>>>(a); break;
        case 4: append_kernel<4><<<grid, 256, 0, stream>>>(a); break;
        case 5: append_kernel<5><<<grid, 256, 0, stream>>>(a); break;
        case 6: append_kernel<6><<<grid, 256, 0, stream>>>(a); break;
        case 7: append_kernel<7><<<grid, 256, 0, stream>>>(a); break;
        default: append_kernel<8><<<grid, 256, 0, stream>>>(a); break;
    }
    NN_LAUNCH_OK("qk_norm_rope_append_q4");
    return 0;
}

extern "C" int nncpu_q4_read(const uint8_t* k_pages, const uint8_t* v_pages, int n_pages, const int* block_table, int bt_rows, int bt_stride,
                             const int* tok_seq, const int* tok_pos, void* k_out, void* v_out, int out_dt, int n, int n_kv, int D,
                             cudaStream_t stream) {
    NN_CHECK(q4_lanes_ok(D), "q4_read: heads of %d lanes (whole groups of 32, at most 256)", D);
    NN_CHECK(n >= 0 && n_kv > 0 && bt_rows >= 0 && bt_stride > 0 && n_pages > 0, "q4_read: %d tokens, %d heads, %d pages", n, n_kv, n_pages);
    if (n == 0) return 0;
    NN_CHECK((uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0, "q4_read: outputs start on 16-byte boundaries");
    const long items = (long)n * n_kv * D / 8;
    NN_CHECK(items / 256 < (1L << 31), "q4_read: %d tokens", n);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((items + 255) / 256));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    cfg.attrs = attr;
    cfg.numAttrs = overlap_attribute(attr);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, read_kernel, k_pages, v_pages, n_pages, block_table, bt_rows, bt_stride, tok_seq, tok_pos, k_out, v_out,
                                             out_dt, n, n_kv, D);
    NN_CHECK(e == cudaSuccess, "q4_read: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

// half: float16, else float32.  places (or null): int32 [2, n_tok].  q (or null): bfloat16 [n_tok, n_heads * D] to q_out [n_tok, n_heads * lanes].
extern "C" int nncpu_q4_expand(const uint8_t* k_pages, const uint8_t* v_pages, int n_pages, const int* block_table, int bt_stride,
                               const int* cu_seqlens, const int* tok_seq, const int* tok_pos, int n_seqs, int width, int n_kv, int D,
                               int lanes, int window, int keep, int half, void* k_out, void* v_out, int* table, int* places, const void* q,
                               void* q_out, int n_tok, int n_heads,
                               cudaStream_t stream) {
    NN_CHECK(q4_lanes_ok(D) && lanes >= D && lanes % 8 == 0, "q4_expand: heads of %d lanes in rows of %d", D, lanes);
    NN_CHECK(n_seqs > 0 && n_seqs <= 65535 && width > 0 && n_kv > 0 && n_kv <= 32767 && n_pages > 0 && bt_stride > 0,
             "q4_expand: %d sequences of %d pages, %d heads", n_seqs, width, n_kv);
    if (q != nullptr && n_tok > 0) {
        const long pieces = (long)n_tok * n_heads * lanes / 8;
        longer_heads_kernel<<<(unsigned)((pieces + 255) / 256), 256, 0, stream>>>((const uint16_t*)q, (uint16_t*)q_out, (long)n_tok * n_heads, D, lanes);
        NN_LAUNCH_OK("q4_expand (queries)");
    }
    const Expand p{k_pages, v_pages, n_pages, block_table, bt_stride, cu_seqlens, tok_seq, tok_pos, k_out, v_out, table, places,
                   n_tok, n_kv, D, lanes, window, keep};
    // Not launched to start under the kernel before it: its blocks would wait in places that blocks of that one could take (a prompt of
    // 2 048 tokens with its append 83.6 us instead of 80.2).
    const dim3 grid((unsigned)width, (unsigned)(2 * n_kv), (unsigned)n_seqs);
    if (half) expand_kernel<__half><<<grid, kExpandThreads, 0, stream>>>(p);
    else expand_kernel<float><<<grid, kExpandThreads, 0, stream>>>(p);
    NN_LAUNCH_OK("q4_expand");
    return 0;
}
