// Per-head query/key RMS norm, position rotation and cache append in one pass, and the read-back of
// stored positions.
//
//   q' = R(p) (q / sqrt(mean q^2 + eps) * w_q),  k' = R(p) (k / sqrt(mean k^2 + eps) * w_k),  v' = v
//
// over each head's head_dim values; q' is written to q_out, k' and v' into the paged cache of any of
// its types. 4-bit blocks (32 dimensions, kv_layout.h): d = x_top / -8 with x_top the first value of
// the largest magnitude, code = min(15, trunc(x / d + 8.5)), stored scale fp16(d).
//
// Every product and sum is rounded on its own (no contraction) and the squares are summed in one
// fixed order, so a token's codes do not depend on which batch or prompt chunk it arrived in.
#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"
#include "kv_layout.h"
#include "launch.cuh"

namespace vsl {

constexpr int KA_THREADS = 128;

struct KvAppendParams {
    const float* qkv;
    long long stride;  // floats between rows
    int n_rows, n_heads, n_kv;
    const float* q_norm;
    const float* k_norm;
    float eps;
    const int32_t* seq;
    const int32_t* pos;
    int n_seq;
    const float* cos;
    const float* sin;
    int max_pos;
    int halves;  // rotation pairs (i, i + hd / 2) instead of (2 i, 2 i + 1)
    float* q_out;
    unsigned char* k_cache;
    unsigned char* v_cache;
    int n_pages;
    const int32_t* page_table;
    int max_pages, page_size;
    int* status;
};

// Page and slot of row r; page -1: padding (pos < 0) or refused (*bad set).
__device__ __forceinline__ void kv_locate(const int32_t* seq, const int32_t* pos, int n_seq,
                                          const int32_t* page_table, int max_pages, int page_size, int n_pages, int r,
                                          int& p, int& page, int& slot, bool& bad) {
    p = pos[r];
    page = -1;
    slot = 0;
    bad = false;
    if (p < 0) return;
    const int s = seq ? seq[r] : r;
    const int lp = p / page_size;
    bad = true;
    if (s < 0 || s >= n_seq || lp >= max_pages) return;
    const int pg = page_table[(size_t)s * max_pages + lp];
    if (pg < 0 || pg >= n_pages) return;
    bad = false;
    page = pg;
    slot = p - lp * page_size;
}

// Codes and scales of HEADS blocks of 32 values at once, four values per lane, a block per 8 lanes. A
// block that holds a NaN or an infinity becomes all NaN; a scale past fp16's range is cut to it.
template <int HEADS>
__device__ __forceinline__ void q4_codes(const float (*x)[4], uint32_t* codes, __half* d_out) {
    const uint32_t FULL = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    float d[HEADS], mine = 0.0f;
    bool wild[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        float top = x[i][0];
#pragma unroll
        for (int j = 1; j < 4; j++)
            if (fabsf(x[i][j]) > fabsf(top)) top = x[i][j];
        // as whole numbers the magnitudes order alike, NaN and infinities above all
        uint32_t own = 0, m;
#pragma unroll
        for (int j = 0; j < 4; j++) own = max(own, __float_as_uint(x[i][j]) & 0x7fffffffu);
        m = own;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(FULL, m, o));
        const uint32_t has = __ballot_sync(FULL, own == m) >> (lane & 24) & 0xffu;
        top = __shfl_sync(FULL, top, (lane & 24) + __ffs(has) - 1);
        wild[i] = m >= 0x7f800000u;
        d[i] = fminf(fmaxf(top * -0.125f, -65504.0f), 65504.0f);
        if ((lane & 7) == i || HEADS == 1) mine = d[i];
    }
    // a reciprocal per lane: lane i of the 8 for block i
    const float inv = fabsf(mine) >= 1.17549435e-38f ? __frcp_rn(mine) : 0.0f;
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const float r = HEADS == 1 ? inv : __shfl_sync(FULL, inv, (lane & 24) + i);
        uint32_t c = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)  // the conversion cuts at 0
            c |= __float2uint_rz(fminf(__fadd_rn(__fmul_rn(x[i][j], r), 8.5f), 15.0f)) << (4 * j);
        codes[i] = wild[i] ? 0x8888u : c;
        d_out[i] = wild[i] ? __ushort_as_half((unsigned short)0x7fff) : __float2half_rn(d[i]);
    }
}

// hd / 4 lanes per head, four consecutive dimensions per lane (one 16-byte load and store each). A
// lane group handles HEADS heads of one row: their loads are all requested first, beside the chain
// position -> page, and the row's rotation factors are read once.
// Measured on a B200: 8192 rows of 32 / 8 heads of 128 into the 4-bit cache 75 us (4.6 TB/s, 71 % of the
// measured copy rate; 213 us with one head per group and its load behind the page), fp16 65 us (5.7 TB/s),
// fp32 70 us (5.8 TB/s). Without norm and rotation 65, 61 and 66 us. So of the 4-bit cache's 75 us the codes
// take about 10 (against fp16, which stores 24 MB more), the norm 6, the rotation 4; the warps wait for their
// loads first (3.1 per issue), then for fixed latencies (2.1), with three quarters of the issue slots
// used. A decode step takes 2.8 us, which is the launch and the chain position -> page -> store.
template <int HD, int KVDT, int HEADS>
__global__ void __launch_bounds__(KA_THREADS) vsl_kv_append_kernel(KvAppendParams p) {
    constexpr int L = HD / 4, NB = HD / 32;
    pdl_wait();
    pdl_launch_dependents();
    const int r = (int)blockIdx.x, sl = threadIdx.x % L, lane = threadIdx.x & 31;
    const int H = p.n_heads + 2 * p.n_kv;
    // a lane group past the last head only takes part in the warp's shuffles
    const int h_first = ((int)blockIdx.y * (KA_THREADS / L) + (int)threadIdx.x / L) * HEADS;
    float x[HEADS][4];
    {
        const float4* src = reinterpret_cast<const float4*>(p.qkv + (size_t)r * p.stride + (size_t)h_first * HD) + sl;
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const float4 f = h_first + i < H ? __ldcs(src + i * L) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            x[i][0] = f.x; x[i][1] = f.y; x[i][2] = f.z; x[i][3] = f.w;
        }
    }
    int pos, page, slot;
    bool bad;
    kv_locate(p.seq, p.pos, p.n_seq, p.page_table, p.max_pages, p.page_size, p.n_pages, r, pos, page, slot, bad);
    if (page >= 0 && p.cos && pos >= p.max_pos) {
        page = -1;
        bad = true;
    }
    if (bad && threadIdx.x == 0) set_status(p.status, VSL_ERR_BOUNDS);
    if (page < 0) {  // the CTA's row: zeros as they are, for a norm or rotation may make NaN of them
#pragma unroll
        for (int i = 0; i < HEADS; i++)
            if (h_first + i < p.n_heads)
                __stcs(reinterpret_cast<float4*>(p.q_out + ((size_t)r * p.n_heads + h_first + i) * HD) + sl,
                       make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        return;
    }
    if (p.q_norm || p.k_norm) {
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            float s = __fadd_rn(__fadd_rn(__fmul_rn(x[i][0], x[i][0]), __fmul_rn(x[i][1], x[i][1])),
                                __fadd_rn(__fmul_rn(x[i][2], x[i][2]), __fmul_rn(x[i][3], x[i][3])));
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
            if (sl == i || HEADS == 1) mine = s;
        }
        // one root and reciprocal per lane: lane i of the group for its head i
        const float rn = __frcp_rn(__fsqrt_rn(__fadd_rn(mine * (1.0f / HD), p.eps)));
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const float t = HEADS == 1 ? rn : __shfl_sync(0xffffffffu, rn, (lane & ~(L - 1)) + i);
            const int h = h_first + i;
            const float* w = h < p.n_heads ? p.q_norm : h < p.n_heads + p.n_kv ? p.k_norm : nullptr;
            if (w) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(w) + sl);
                x[i][0] = __fmul_rn(__fmul_rn(x[i][0], t), f.x);
                x[i][1] = __fmul_rn(__fmul_rn(x[i][1], t), f.y);
                x[i][2] = __fmul_rn(__fmul_rn(x[i][2], t), f.z);
                x[i][3] = __fmul_rn(__fmul_rn(x[i][3], t), f.w);
            }
        }
    }
    if (p.cos) {
        const size_t row = (size_t)pos * (HD / 2);
        if (p.halves) {
            const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + row) + sl % (L / 2));
            const float4 d = __ldg(reinterpret_cast<const float4*>(p.sin + row) + sl % (L / 2));
            const float cs[4] = {c.x, c.y, c.z, c.w};
            // lower half: a c - b d; upper half: a d + b c
            const float sn[4] = {sl < L / 2 ? -d.x : d.x, sl < L / 2 ? -d.y : d.y, sl < L / 2 ? -d.z : d.z,
                                 sl < L / 2 ? -d.w : d.w};
#pragma unroll
            for (int i = 0; i < HEADS; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float o = __shfl_xor_sync(0xffffffffu, x[i][j], L / 2);
                    if (h_first + i < p.n_heads + p.n_kv)
                        x[i][j] = __fadd_rn(__fmul_rn(x[i][j], cs[j]), __fmul_rn(o, sn[j]));
                }
        } else {
            const float2 c = __ldg(reinterpret_cast<const float2*>(p.cos + row) + sl);
            const float2 d = __ldg(reinterpret_cast<const float2*>(p.sin + row) + sl);
#pragma unroll
            for (int i = 0; i < HEADS; i++) {
                if (h_first + i >= p.n_heads + p.n_kv) continue;
                const float a0 = x[i][0], b0 = x[i][1], a1 = x[i][2], b1 = x[i][3];
                x[i][0] = __fsub_rn(__fmul_rn(a0, c.x), __fmul_rn(b0, d.x));
                x[i][1] = __fadd_rn(__fmul_rn(a0, d.x), __fmul_rn(b0, c.x));
                x[i][2] = __fsub_rn(__fmul_rn(a1, c.y), __fmul_rn(b1, d.y));
                x[i][3] = __fadd_rn(__fmul_rn(a1, d.y), __fmul_rn(b1, c.y));
            }
        }
    }
    uint32_t codes[HEADS];
    __half d[HEADS];
    // by the whole warp, for it shuffles
    if (KVDT == VSL_Q4_0 && __any_sync(0xffffffffu, h_first + HEADS > p.n_heads)) q4_codes<HEADS>(x, codes, d);
    const size_t head_bytes = kv_head_page_bytes(KVDT, HD, p.page_size);
    // head 0 of K and of V in the row's page, and the lane's place in a head
    const size_t page_at = (size_t)page * p.n_kv * head_bytes;
    const int b = sl >> 3, u = sl & 7;
    const size_t k_at = page_at + (KVDT == VSL_Q4_0 ? kv_q4_k_piece(NB, slot, b, u) : ((size_t)slot * HD + 4 * sl) * (KVDT == VSL_F16 ? 2 : 4));
    const size_t v_at = KVDT == VSL_Q4_0 ? page_at + kv_q4_v_piece(NB, slot, b, u) : k_at;
    const size_t d_at = page_at + kv_q4_scales(HD, p.page_size) + (size_t)(slot * NB + b) * 2;
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const int h = h_first + i;
        if (h >= H) continue;
        if (h < p.n_heads) {
            __stcs(reinterpret_cast<float4*>(p.q_out + ((size_t)r * p.n_heads + h) * HD) + sl,
                   make_float4(x[i][0], x[i][1], x[i][2], x[i][3]));
            continue;
        }
        const bool is_v = h >= p.n_heads + p.n_kv;
        unsigned char* cache = (is_v ? p.v_cache : p.k_cache) + (size_t)(h - p.n_heads - (is_v ? p.n_kv : 0)) * head_bytes;
        unsigned char* dst = cache + (is_v ? v_at : k_at);
        if (KVDT == VSL_Q4_0) {
            *reinterpret_cast<unsigned short*>(dst) = (unsigned short)codes[i];
            if (u == 0) *reinterpret_cast<__half*>(cache + d_at) = d[i];
        } else if (KVDT == VSL_F16) {
            const __half2 lo = __floats2half2_rn(x[i][0], x[i][1]), hi = __floats2half2_rn(x[i][2], x[i][3]);
            uint2 v;
            v.x = *reinterpret_cast<const uint32_t*>(&lo);
            v.y = *reinterpret_cast<const uint32_t*>(&hi);
            *reinterpret_cast<uint2*>(dst) = v;
        } else {
            *reinterpret_cast<float4*>(dst) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
        }
    }
}

// Four stored values as fp32.
__device__ __forceinline__ void kv_widen(uint2 v, float x[4]) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    x[0] = a.x; x[1] = a.y; x[2] = c.x; x[3] = c.y;
}
__device__ __forceinline__ void kv_widen(float4 v, float x[4]) {
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void kv_store4(float* dst, const float x[4]) {
    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void kv_store4(__half* dst, const float x[4]) {
    const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
    uint2 v;
    v.x = *reinterpret_cast<const uint32_t*>(&lo);
    v.y = *reinterpret_cast<const uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(dst) = v;
}

struct KvReadParams {
    const unsigned char* k_cache;
    const unsigned char* v_cache;
    int n_pages;
    const int32_t* page_table;
    int max_pages, page_size, n_kv;
    const int32_t* seq;
    const int32_t* pos;
    int n_seq, n_rows;
    void* k_out;
    void* v_out;
    int* status;
};

// A lane group handles HEADS of a row's 2 n_kv K and V heads, all loads first. fp32 / fp16: four
// dimensions per lane. 4-bit: 8 lanes, head_dim / 16 bytes of codes each; a lane's run of K holds 8
// neighbouring dimensions of each of NB / 2 blocks, a run of V 4 of each of NB blocks. 8192 positions
// of 8 heads of 128 to fp16: 11 us (3.9 TB/s; 17 us with one 2-byte piece per lane; 16 rows take 2.1), of an
// fp16 cache 13.4 us (5.0 TB/s), of an fp32 cache to fp32 23.4 us (5.7 TB/s).
template <int HD, int KVDT, typename OT, int HEADS>
__global__ void __launch_bounds__(KA_THREADS) vsl_kv_read_kernel(KvReadParams p) {
    constexpr bool Q4 = KVDT == VSL_Q4_0;
    constexpr int L = Q4 ? 8 : HD / 4, NB = HD / 32;
    pdl_wait();
    pdl_launch_dependents();
    const unsigned id = (blockIdx.x * KA_THREADS + threadIdx.x) / L, groups = (2 * p.n_kv + HEADS - 1) / HEADS;
    const int sl = threadIdx.x % L;
    const int r = (int)(id / groups), h0 = (int)(id % groups) * HEADS;
    if (r >= p.n_rows) return;
    int pos, page, slot;
    bool bad;
    kv_locate(p.seq, p.pos, p.n_seq, p.page_table, p.max_pages, p.page_size, p.n_pages, r, pos, page, slot, bad);
    if (bad && sl == 0) set_status(p.status, VSL_ERR_BOUNDS);
    const size_t head_bytes = kv_head_page_bytes(KVDT, HD, p.page_size);
    const size_t page_at = page >= 0 ? (size_t)page * p.n_kv * head_bytes : 0;
    if constexpr (Q4) {
        using Run = typename std::conditional<NB == 4, uint2, uint32_t>::type;
        Run codes[HEADS], d[HEADS];  // K: scales of the lane's NB / 2 blocks, V: of all
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const int h = h0 + i;
            if (page < 0 || h >= 2 * p.n_kv) continue;
            const bool is_v = h >= p.n_kv;
            const unsigned char* head = (is_v ? p.v_cache : p.k_cache) + page_at + (size_t)(h - (is_v ? p.n_kv : 0)) * head_bytes;
            const unsigned char* scales = head + kv_q4_scales(HD, p.page_size) + (size_t)slot * NB * 2;
            codes[i] = *reinterpret_cast<const Run*>(head + (is_v ? kv_q4_v_piece(NB, slot, 0, sl)
                                                                   : kv_q4_k_piece(NB, slot, (sl & 1) * (NB / 2), sl & 6)));
            d[i] = *reinterpret_cast<const Run*>(scales);
        }
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const int h = h0 + i;
            if (h >= 2 * p.n_kv) continue;
            const bool is_v = h >= p.n_kv;
            OT* dst = static_cast<OT*>(is_v ? p.v_out : p.k_out) + ((size_t)r * p.n_kv + h - (is_v ? p.n_kv : 0)) * HD;
            const unsigned short* piece = reinterpret_cast<const unsigned short*>(&codes[i]);
            const __half* sc = reinterpret_cast<const __half*>(&d[i]);
#pragma unroll
            for (int k = 0; k < NB; k++) {
                // piece k: V block k, u = sl; K block (sl & 1) NB / 2 + k / 2, u = 2 (sl / 2) + k % 2
                const int blk = is_v ? k : (sl & 1) * (NB / 2) + k / 2, u = is_v ? sl : (sl & 6) + (k & 1);
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (page >= 0) {
                    const float s = __half2float(is_v ? sc[k] : sl & 1 ? sc[NB / 2 + k / 2] : sc[k / 2]);
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = (float)((int)((piece[k] >> (4 * j)) & 15u) - 8) * s;
                }
                kv_store4(dst + 32 * blk + 4 * u, x);
            }
        }
    } else {
        using Raw = typename std::conditional<KVDT == VSL_F16, uint2, float4>::type;
        Raw raw[HEADS];
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const int h = h0 + i;
            if (page < 0 || h >= 2 * p.n_kv) continue;
            const bool is_v = h >= p.n_kv;
            const unsigned char* head = (is_v ? p.v_cache : p.k_cache) + page_at + (size_t)(h - (is_v ? p.n_kv : 0)) * head_bytes;
            raw[i] = *(reinterpret_cast<const Raw*>(head) + (size_t)slot * L + sl);
        }
#pragma unroll
        for (int i = 0; i < HEADS; i++) {
            const int h = h0 + i;
            if (h >= 2 * p.n_kv) continue;
            const bool is_v = h >= p.n_kv;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (page >= 0) kv_widen(raw[i], x);
            kv_store4(static_cast<OT*>(is_v ? p.v_out : p.k_out) + ((size_t)r * p.n_kv + h - (is_v ? p.n_kv : 0)) * HD + 4 * sl, x);
        }
    }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Arguments the append and the read-back share.
static int kv_rows_check(const char* what, const void* k_cache, const void* v_cache, int kvdtype, int n_pages,
                         const int32_t* page_table, int max_pages, int page_size, int n_kv, int head_dim,
                         const int32_t* seq, const int32_t* pos, int n_seq, int n_rows) {
    if (!k_cache || !v_cache || !page_table || !pos) return set_error(VSL_ERR_INVALID, "%s: null pointer", what);
    if (n_rows < 0 || n_seq <= 0 || n_pages <= 0 || max_pages <= 0 || n_kv <= 0)
        return set_error(VSL_ERR_INVALID, "%s: %d rows, %d sequences of %d pages, pool of %d pages, %d KV heads", what,
                         n_rows, n_seq, max_pages, n_pages, n_kv);
    if (!seq && n_rows > n_seq)
        return set_error(VSL_ERR_INVALID, "%s: %d rows without a sequence index over %d sequences", what, n_rows, n_seq);
    if (head_dim != 64 && head_dim != 128)
        return set_error(VSL_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128 supported)", what, head_dim);
    if (!kv_dtype_ok(kvdtype)) return set_error(VSL_ERR_UNSUPPORTED, "%s: kv dtype %d", what, kvdtype);
    if (page_size <= 0 || page_size % 64)
        return set_error(VSL_ERR_INVALID, "%s: page_size %d must be a multiple of 64", what, page_size);
    if ((long long)max_pages * page_size > INT32_MAX)
        return set_error(VSL_ERR_INVALID, "%s: %d pages of %d positions pass the range of a position", what, max_pages,
                         page_size);
    if (!aligned16(k_cache) || !aligned16(v_cache))
        return set_error(VSL_ERR_INVALID, "%s: caches must be 16-byte aligned", what);
    return VSL_OK;
}

// Heads per lane group: one while that leaves threads to spare (a decode step: the shortest chain),
// else four (more loads in flight per thread than the threads of an SM can have with one). One / four, 32 / 8
// heads of 128 into the 4-bit cache, us: 16 rows 2.6 / 3.5, 96 rows 3.2 / 3.7, 200 rows 4.8 / 4.4, 1200 rows
// 18.5 / 13.3; read back 16 rows 2.1 / 3.6, 1200 rows 4.2 / 4.2.
constexpr int KA_HEADS = 4;
static bool few_heads(long long rows, int heads, int lanes) {
    return rows * heads * lanes <= (long long)sm_count() * 2048;
}

template <int HD, int KVDT, int HEADS>
static int launch_append_h(const KvAppendParams& p, cudaStream_t st) {
    constexpr int PER_BLOCK = KA_THREADS / (HD / 4) * HEADS;
    const dim3 grid((unsigned)p.n_rows, (unsigned)((p.n_heads + 2 * p.n_kv + PER_BLOCK - 1) / PER_BLOCK));
    return launch_status(launch_k(vsl_kv_append_kernel<HD, KVDT, HEADS>, grid, dim3(KA_THREADS), 0, st, p),
                         "qk_norm_rope_append launch");
}
template <int HD, int KVDT>
static int launch_append_t(const KvAppendParams& p, cudaStream_t st) {
    return few_heads(p.n_rows, p.n_heads + 2 * p.n_kv, HD / 4) ? launch_append_h<HD, KVDT, 1>(p, st)
                                                               : launch_append_h<HD, KVDT, KA_HEADS>(p, st);
}
template <int HD>
static int launch_append(const KvAppendParams& p, int kvdtype, cudaStream_t st) {
    return kvdtype == VSL_Q4_0  ? launch_append_t<HD, VSL_Q4_0>(p, st)
           : kvdtype == VSL_F16 ? launch_append_t<HD, VSL_F16>(p, st)
                                : launch_append_t<HD, VSL_F32>(p, st);
}

template <int HD, int KVDT, typename OT, int HEADS>
static int launch_read_h(const KvReadParams& p, cudaStream_t st) {
    const long long lanes = (long long)p.n_rows * ((2 * p.n_kv + HEADS - 1) / HEADS) * (KVDT == VSL_Q4_0 ? 8 : HD / 4);
    if (lanes > INT32_MAX) return set_error(VSL_ERR_UNSUPPORTED, "kv_read: %d rows are too many for one call", p.n_rows);
    return launch_status(launch_k(vsl_kv_read_kernel<HD, KVDT, OT, HEADS>, dim3((unsigned)((lanes + KA_THREADS - 1) / KA_THREADS)),
                                  dim3(KA_THREADS), 0, st, p),
                         "kv_read launch");
}
template <int HD, int KVDT, typename OT>
static int launch_read_t(const KvReadParams& p, cudaStream_t st) {
    return few_heads(p.n_rows, 2 * p.n_kv, KVDT == VSL_Q4_0 ? 8 : HD / 4) ? launch_read_h<HD, KVDT, OT, 1>(p, st)
                                                                          : launch_read_h<HD, KVDT, OT, KA_HEADS>(p, st);
}
template <int HD, typename OT>
static int launch_read(const KvReadParams& p, int kvdtype, cudaStream_t st) {
    return kvdtype == VSL_Q4_0  ? launch_read_t<HD, VSL_Q4_0, OT>(p, st)
           : kvdtype == VSL_F16 ? launch_read_t<HD, VSL_F16, OT>(p, st)
                                : launch_read_t<HD, VSL_F32, OT>(p, st);
}

}  // namespace vsl

using namespace vsl;

extern "C" int vsl_kv_page_bytes(int kvdtype, int n_kv, int head_dim, int page_size, size_t* bytes) {
    if (!bytes || n_kv <= 0 || page_size <= 0 || page_size % 64)
        return set_error(VSL_ERR_INVALID, "kv_page_bytes: %d KV heads, page_size %d (a multiple of 64)", n_kv, page_size);
    if (!kv_dtype_ok(kvdtype) || (head_dim != 64 && head_dim != 128))
        return set_error(VSL_ERR_UNSUPPORTED, "kv_page_bytes: head_dim %d / kv dtype %d", head_dim, kvdtype);
    *bytes = (size_t)n_kv * kv_head_page_bytes(kvdtype, head_dim, page_size);
    return VSL_OK;
}

extern "C" int vsl_qk_norm_rope_append(const float* qkv, long long qkv_stride, int n_rows, int n_heads, int n_kv,
                                       int head_dim, const float* q_norm_w, const float* k_norm_w, float eps,
                                       const int32_t* seq, const int32_t* pos, int n_seq, const float* rope_cos,
                                       const float* rope_sin, int max_pos, int rope_style, float* q_out, void* k_cache,
                                       void* v_cache, int kvdtype, int n_pages, const int32_t* page_table,
                                       int max_pages, int page_size, int* status, void* stream) {
    if (!qkv || !q_out) return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: null pointer");
    if (int rc = kv_rows_check("qk_norm_rope_append", k_cache, v_cache, kvdtype, n_pages, page_table, max_pages,
                               page_size, n_kv, head_dim, seq, pos, n_seq, n_rows))
        return rc;
    if (n_heads <= 0 || n_heads > 65536 || n_kv > 65536)
        return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: %d query heads, %d KV heads", n_heads, n_kv);
    if (qkv_stride < (long long)(n_heads + 2 * n_kv) * head_dim || qkv_stride % 4)
        return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: row stride %lld (at least %lld, a multiple of 4)",
                         qkv_stride, (long long)(n_heads + 2 * n_kv) * head_dim);
    if (!rope_cos != !rope_sin || (rope_cos && max_pos <= 0))
        return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: rotation tables need both cos and sin, and max_pos");
    if (rope_style != VSL_ROPE_ADJACENT && rope_style != VSL_ROPE_HALVES)
        return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: rope_style %d", rope_style);
    if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(rope_cos) ||
        !aligned16(rope_sin))
        return set_error(VSL_ERR_INVALID, "qk_norm_rope_append: float arrays must be 16-byte aligned");
    if (n_rows == 0) return VSL_OK;
    KvAppendParams p = {};
    p.qkv = qkv; p.stride = qkv_stride; p.n_rows = n_rows; p.n_heads = n_heads; p.n_kv = n_kv;
    p.q_norm = q_norm_w; p.k_norm = k_norm_w; p.eps = eps;
    p.seq = seq; p.pos = pos; p.n_seq = n_seq;
    p.cos = rope_cos; p.sin = rope_sin; p.max_pos = max_pos; p.halves = rope_style == VSL_ROPE_HALVES;
    p.q_out = q_out;
    p.k_cache = static_cast<unsigned char*>(k_cache);
    p.v_cache = static_cast<unsigned char*>(v_cache);
    p.n_pages = n_pages; p.page_table = page_table; p.max_pages = max_pages; p.page_size = page_size;
    p.status = status;
    return head_dim == 128 ? launch_append<128>(p, kvdtype, (cudaStream_t)stream)
                           : launch_append<64>(p, kvdtype, (cudaStream_t)stream);
}

extern "C" int vsl_kv_read(const void* k_cache, const void* v_cache, int kvdtype, int n_pages,
                           const int32_t* page_table, int max_pages, int page_size, int n_kv, int head_dim,
                           const int32_t* seq, const int32_t* pos, int n_seq, int n_rows, int out_dtype, void* k_out,
                           void* v_out, int* status, void* stream) {
    if (!k_out || !v_out) return set_error(VSL_ERR_INVALID, "kv_read: null pointer");
    if (int rc = kv_rows_check("kv_read", k_cache, v_cache, kvdtype, n_pages, page_table, max_pages, page_size, n_kv,
                               head_dim, seq, pos, n_seq, n_rows))
        return rc;
    if (out_dtype != VSL_F32 && out_dtype != VSL_F16)
        return set_error(VSL_ERR_UNSUPPORTED, "kv_read: output dtype %d", out_dtype);
    if (!aligned16(k_out) || !aligned16(v_out)) return set_error(VSL_ERR_INVALID, "kv_read: outputs must be 16-byte aligned");
    if (n_rows == 0) return VSL_OK;
    KvReadParams p = {};
    p.k_cache = static_cast<const unsigned char*>(k_cache);
    p.v_cache = static_cast<const unsigned char*>(v_cache);
    p.n_pages = n_pages; p.page_table = page_table; p.max_pages = max_pages; p.page_size = page_size; p.n_kv = n_kv;
    p.seq = seq; p.pos = pos; p.n_seq = n_seq; p.n_rows = n_rows; p.k_out = k_out; p.v_out = v_out; p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    if (out_dtype == VSL_F32)
        return head_dim == 128 ? launch_read<128, float>(p, kvdtype, st) : launch_read<64, float>(p, kvdtype, st);
    return head_dim == 128 ? launch_read<128, __half>(p, kvdtype, st) : launch_read<64, __half>(p, kvdtype, st);
}
