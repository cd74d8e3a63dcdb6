// Attention of many query rows per sequence (a prompt chunk) over the 4-bit paged cache: the form of
// vsl_flash_decode_q4 for tiles of 128 (row, head) columns, on tcgen05. Same results and rules as
// attention_q4.cu.
//
// With many rows the other form unpacks the codes again for every tile of 8 columns. Here a chunk of 64
// positions is unpacked once for 128 columns, into shared memory:
//   * K and V as two fp16 parts of (n - 8) d f each, f a power of two that brings the chunk's largest
//     scale below 2^16: the product has 14 bits, so the parts hold it exactly (to 2^-34 of the chunk's
//     largest value); q in two parts as well, divided by the power of two of its own row;
//   * S[128 columns][64 positions] = q k^T and O[128][head_dim] = p v, each as three products of parts
//     (low x high, high x low, high x high; low x low is below 2^-22), in TMEM. q and p are the operands
//     in TMEM, p in the place of its scores: from shared memory they cost the products' 128 rows of
//     reads again (7 % more time at 8192 positions);
//   * exponentials of up to 2^15, and p's low part times 2^11 (its product is scaled back in TMEM), so that
//     the parts reach down to 2^-50 of the largest; the factor 2^15 cancels in o / l. Rounding the exponent as
//     x + 15 costs up to 3e-7 of a weight, about what the 22 bits of its parts do;
//   * O of a chunk is taken out of TMEM and added in fp32 registers: no accumulation is longer than
//     12 (O) or 24 (S) matrix instructions, whose sums are cut, not rounded.
// Warps: 8 for the softmax (a TMEM lane each, half of the columns), 4 that unpack K and 4 that unpack V, of
// which one in turn issues the products (always the same one: 2.4 against 2.05 us per chunk). S, O, K and V
// have two buffers each: unpacking and scores of the next chunk run beside this one's exponentials, and O of
// the last chunk is added while this one's is being multiplied. The code is rolled up where it can be: three
// kinds of warps share the instruction caches, and straight code is slow the first time.
//
// A CTA has one tile of one KV head of one sequence and a part of its positions. Up to 8 parts are a
// cluster, which joins them through its shared memory, each CTA some of the rows. Where the tiles leave
// room for more, several clusters have parts of a tile, and the last to finish joins theirs, in order:
// results do not depend on the timing.
//
// Measured on a B200, 32 / 8 heads of 128, 128 rows: over 2048 positions 28.4 us (8 chunks per CTA), over 8192
// 77 us: 2 us per chunk and CTA and 12 us of set-up, first chunk, join and output. Of a chunk's 3700 cycles the
// softmax warps are busy for 2700 and the tensor cores for 2300 (a product of 64 columns takes as long as one
// of 128); the rest is waiting for one another.
//
// Every wait is bounded; one that runs out records VSL_ERR_TIMEOUT, and the CTA drains its products.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "../host/kernels.h"
#include "attention_q4.cuh"
#include "common.cuh"
#include "kv_layout.h"
#include "launch.cuh"

namespace vsl {

constexpr int FC_SM_WARPS = 8, FC_UN_WARPS = 4;  // softmax; unpacking K, and as many V
constexpr int FC_THREADS = 32 * (FC_SM_WARPS + 2 * FC_UN_WARPS);
constexpr int FC_CLUSTER = 8, FC_GROUPED = 4;    // CTAs of a cluster at most; at least, where several share a tile
constexpr int FC_CHUNK = 64;                     // positions
constexpr uint32_t FC_ATOM = FC_CHUNK * 128;      // 64 columns of 16 bits of a tile in shared memory
// TMEM columns: q high and low (pairs of 16-bit values), S[2], whose places p takes, O[2]
constexpr uint32_t FC_TMEM_COLS = 512, FC_TQ = 0, FC_TS = 128, FC_TO = FC_TS + 2 * FC_CHUNK;

template <int HD>
struct FcSmem {  // offsets from a 1024-byte boundary; two buffers of K and of V, parts high, low
    static constexpr uint32_t PART = HD / 64 * FC_ATOM, K = 0, V = 4 * PART, OUT_ROW = HD + 4;
    // then the rows of q, OUT_ROW floats apart; at the end those of the output, in the place of K and V
    static constexpr uint32_t Q = 8 * PART;
    static constexpr size_t BYTES = 1024 + Q + (size_t)FC_COLS * OUT_ROW * 4;
    static_assert(FC_COLS * OUT_ROW * 4 <= Q, "the output fits");
};
template <int HD>
__host__ __device__ constexpr int fc_part_floats() {
    return FC_COLS * (HD + 2);
}

// byte offset of 16-bit column `col` of row `r` in a K-major (or, for V, position-major) 128-byte-swizzled tile
__device__ __forceinline__ uint32_t fc_off(int r, int col, uint32_t atom) {
    return (uint32_t)(col >> 6) * atom + (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4));
}
// K-major operand, 128-byte swizzle: 8 rows of 128 bytes, 1024 bytes apart
__device__ __forceinline__ uint64_t fc_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// V as it is unpacked, MN-major: rows of positions, the next 64 dimensions an atom further
__device__ __forceinline__ uint64_t fc_desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(FC_ATOM >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D += A B, A in TMEM (a lane per row, pairs of 16-bit values along K in consecutive columns). The warp calls it
// as one, so that its operands stay in uniform registers; the lane with `leader` issues.
__device__ __forceinline__ void fc_mma(uint32_t leader, uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bd), "r"(idesc), "r"(acc), "r"(leader)
        : "memory");
}
// the same on top of D 2^-11
__device__ __forceinline__ void fc_mma_scaled(uint32_t leader, uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %4, 0;\n\tsetp.eq.b32 p, 0, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, 11;\n\t}" ::"r"(d),
        "r"(a), "l"(bd), "r"(idesc), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void fc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 consecutive fp32 columns of the warp's 32 TMEM lanes
__device__ __forceinline__ void fc_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void fc_ld16(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
// 8 columns of the warp's lanes; fc_st_wait before they are used
__device__ __forceinline__ void fc_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void fc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One chunk's share of an unpacking thread: two 16-byte runs of codes (8 bytes at head_dim 64), the scales of
// its two rows, and 16 bytes of all scales for the chunk's largest.
struct FcRaw {
    uint4 codes[2], top;
    uint2 scales[2];
    int page;  // < 0: nothing there
};
// Where the chunks of a tile are: pages in turn, read one chunk ahead.
struct FcPages {
    const int32_t* row;
    int n_pages, page_size, left, slot, page, slot_next;
    __device__ __forceinline__ FcPages(const FqParams& p, int b, int t, int n)
        : row(p.page_table + (size_t)b * p.max_pages + t / p.page_size), n_pages(p.n_pages), page_size(p.page_size), left(n),
          slot_next(t % p.page_size) {
        fetch();
    }
    __device__ __forceinline__ void fetch() { page = left-- > 0 ? __ldg(row) : -1; }
    // the next chunk's page (-1: none), with its slot; `missing` is set for a chunk that has no page
    __device__ __forceinline__ int next(bool& missing) {
        const bool there = left >= 0;
        const int r = page >= 0 && page < n_pages ? page : -1;
        missing |= there && r < 0;
        slot = slot_next;
        slot_next += FC_CHUNK;
        if (slot_next >= page_size) {
            slot_next = 0;
            row++;
        }
        fetch();
        return r;
    }
};
// K (row pair kr, kr + 8, quarter kt of each row) or V (rows 2 vp, + 1, eighths 2 vu, + 1) of a chunk. base: the
// cache at its KV head.
template <int HD, bool IS_V>
__device__ __forceinline__ void fc_load(const unsigned char* base, size_t page_stride, uint32_t scales_at, int page, int slot,
                                        int row, int col, int lane, FcRaw& r) {
    constexpr int NB = HD / 32;
    r.page = page;
    if (page < 0) return;
    const unsigned char* at = base + (size_t)page * page_stride;
    const unsigned char* sc = at + scales_at + slot * (2 * NB);
    const unsigned char* c0 = at + slot * (HD / 2) + (IS_V ? row * HD + col * (HD / 4) : row * (HD / 2) + col * (HD / 8));
    const unsigned char* c1 = c0 + (IS_V ? HD / 8 : 8 * (HD / 2));
    const int s0 = IS_V ? 2 * row : row, s1 = IS_V ? s0 + 1 : row + 8;
    if (HD == 128) {
        r.codes[0] = __ldcg(reinterpret_cast<const uint4*>(c0));
        r.codes[1] = __ldcg(reinterpret_cast<const uint4*>(c1));
        r.scales[0] = __ldcg(reinterpret_cast<const uint2*>(sc + s0 * 8));
        r.scales[1] = __ldcg(reinterpret_cast<const uint2*>(sc + s1 * 8));
    } else {
        const uint2 x = __ldcg(reinterpret_cast<const uint2*>(c0)), y = __ldcg(reinterpret_cast<const uint2*>(c1));
        r.codes[0] = IS_V ? make_uint4(x.x, 0, x.y, 0) : make_uint4(x.x, x.y, 0, 0);  // V: row 0 in x, row 1 in z
        r.codes[1] = IS_V ? make_uint4(y.x, 0, y.y, 0) : make_uint4(y.x, y.y, 0, 0);
        r.scales[0] = make_uint2(__ldcg(reinterpret_cast<const uint32_t*>(sc + s0 * 4)), 0);
        r.scales[1] = make_uint2(__ldcg(reinterpret_cast<const uint32_t*>(sc + s1 * 4)), 0);
    }
    r.top = make_uint4(0, 0, 0, 0);
    if (lane < FC_CHUNK * NB / 8) r.top = __ldcg(reinterpret_cast<const uint4*>(sc + lane * 16));
}
// Largest fp16 exponent field among the finite scales of the chunk's positions from `low` to `valid`, of which
// the lane holds eight scales.
template <int HD>
__device__ __forceinline__ uint32_t fc_top(const uint4& w, int lane, int low, int valid) {
    constexpr int NB = HD / 32, WORDS = NB / 2;  // words per position
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int at = lane * (4 / WORDS) + i / WORDS;
        if (at < low || at >= valid) continue;
        const uint32_t a = x[i] >> 10 & 31u, b = x[i] >> 26 & 31u;
        top = max(top, max(a == 31u ? 0u : a, b == 31u ? 0u : b));
    }
    return __reduce_max_sync(0xffffffffu, top);
}
__device__ __forceinline__ uint32_t hfms2(uint32_t a, uint32_t b, uint32_t c) {  // a b - c
    uint32_t r;
    asm("{.reg .b32 n;\n\tneg.f16x2 n, %3;\n\tfma.rn.f16x2 %0, %1, %2, n;}" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// A row's scales times 2^(30 - e), each in both halves of a word; zeros where `on` is false. The factor is
// more than fp16 holds: two steps, of which the first one loses nothing (e <= 30).
template <int NB>
__device__ __forceinline__ void fc_scales(const uint32_t (&words)[2], int e, bool on, uint32_t (&d2)[NB]) {
    const uint32_t up = (uint32_t)(30 - (e >> 1)) << 10, rest = (uint32_t)(30 - (e - (e >> 1))) << 10;  // 2^(15 - e / 2)
#pragma unroll
    for (int i = 0; i < NB / 2; i++) {
        const uint32_t w = on ? hmul2(hmul2(words[i], up | up << 16), rest | rest << 16) : 0u;
        d2[2 * i] = __byte_perm(w, w, 0x1010);
        d2[2 * i + 1] = __byte_perm(w, w, 0x3232);
    }
}
// Eight codes times d as two parts, in the order (0 4 1 5 2 6 3 7) in which the word holds their pairs.
__device__ __forceinline__ void fc_unpack(uint32_t w, uint32_t d2, uint4& hi, uint4& lo) {
    const uint32_t x = w >> 8;
    const uint32_t a = value_low(w), b = value_high(w), c = value_low(x), e = value_high(x);
    hi = make_uint4(hmul2(a, d2), hmul2(b, d2), hmul2(c, d2), hmul2(e, d2));
    lo = make_uint4(hfms2(a, d2, hi.x), hfms2(b, d2, hi.y), hfms2(c, d2, hi.z), hfms2(e, d2, hi.w));
}
__device__ __forceinline__ void fc_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same place in the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ uint32_t fc_remote(uint32_t saddr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ float fc_ld_remote(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 fc_ld_remote4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float fc_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

template <int HD>
__global__ void __launch_bounds__(FC_THREADS, 1) vsl_flash_chunk_q4_kernel(FqParams p, int most_groups, int cluster) {
    constexpr int NB = HD / 32, HALF = HD / 2;
    using L = FcSmem<HD>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_ready, k_full[2], v_full[2], s_full[2], p_ready, o_full[2];
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s, last_s;
    __shared__ float red[2][2][FC_COLS], weight[FC_CLUSTER][FC_COLS];
    __shared__ float k_mul[4], v_mul[2];  // k_mul 0: the chunk has no page
    __shared__ uint32_t v_bad[2][FC_UN_WARPS][1 + NB];  // any; per block the positions of non-finite scales
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
    volatile int* aborted = &abort_s;

    pdl_wait();
    // ---- the tile and this CTA's chunks of it ----
    const uint32_t id = blockIdx.x / (uint32_t)cluster, unit = id / (uint32_t)most_groups, bg = unit / (uint32_t)p.tiles;
    const int rank = (int)(blockIdx.x - id * cluster), group = (int)(id - unit * most_groups), c = (int)(unit - bg * p.tiles);
    const int b = (int)(bg / (uint32_t)p.n_kv), g = (int)bg - b * p.n_kv;
    const int cols = min(FC_COLS, p.rows * p.G - c * FC_COLS);
    const int pos = fq_pos(p, b);
    int t_lo, t_hi;
    fq_range(p, pos, c * FC_COLS / p.G, (c * FC_COLS + cols - 1) / p.G, 1, t_lo, t_hi);
    const int t_first = t_lo;  // positions before it hold nothing of the tile's: their scales do not count
    t_lo &= -FC_CHUNK;
    const int chunks = (t_hi - t_lo + FC_CHUNK - 1) / FC_CHUNK;
    // groups (clusters) that have a chunk for each of their CTAs; a group's CTAs all stay for its join
    const int groups = min(most_groups, max(1, (chunks + cluster - 1) / cluster));
    if (group >= groups) return;
    const int part = group * cluster + rank, parts = groups * cluster;
    const int first = (int)((long long)chunks * part / parts);
    const int n = (int)((long long)chunks * (part + 1) / parts) - first;
    t_lo += first * FC_CHUNK;

    if (threadIdx.x == 0) {
        mbar_init(&q_ready, FC_SM_WARPS);
        mbar_init(&p_ready, FC_SM_WARPS);
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], FC_UN_WARPS);
            mbar_init(&v_full[i], FC_UN_WARPS);
            mbar_init(&s_full[i], 1);
            mbar_init(&o_full[i], 1);
        }
        mbar_fence_init();
        abort_s = 0;
    }
    if (warp == FC_SM_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                     "r"(FC_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fc_fence_before();
    __syncthreads();
    fc_fence_after();
    constexpr uint32_t tmem = 0;  // all of it is this CTA's
    pdl_launch_dependents();

    // softmax threads: column t, half hc of the positions and of the dimensions
    const int t = threadIdx.x & (FC_COLS - 1), hc = (warp >> 2) & 1;
    alignas(8) float o[HALF];
    float m = -CUDART_INF_F, l = 0.0f;
    uint32_t nan_blocks = 0;  // blocks of V in which the column sees a scale that is not finite

    const size_t head_bytes = kv_head_page_bytes(VSL_Q4_0, HD, p.page_size), page_stride = p.n_kv * head_bytes;
    const uint32_t scales_at = (uint32_t)kv_q4_scales(HD, p.page_size);
    // fp32 accumulators (bits 4-5), fp16 operands; N / 8 from bit 17, M / 16 from bit 24; bit 16: B is MN-major
    constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(FC_CHUNK >> 3) << 17) | ((uint32_t)(FC_COLS >> 4) << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(FC_COLS >> 4) << 24) | (1u << 16);
    if (warp >= FC_SM_WARPS && warp < FC_SM_WARPS + FC_UN_WARPS) {
        // ================= K: unpacking, and (in turn) the scores =================
        const int w = warp - FC_SM_WARPS;
        const int kr = 16 * w + (lane & 7), kt = lane >> 3;  // rows kr, kr + 8
        const unsigned char* src = p.k_cache + g * head_bytes;
        FcPages pages(p, b, t_lo, n);
        FcRaw r;
        bool missing = false, ok = true;
        int last = -1;  // chunk whose product this warp issued last
        const int page0 = pages.next(missing);
        fc_load<HD, false>(src, page_stride, scales_at, page0, pages.slot, kr, kt, lane, r);
        for (int i = 0; i < n; i++) {
            const int t0 = t_lo + i * FC_CHUNK, low = t_first - t0, valid = r.page < 0 ? 0 : min(FC_CHUNK, t_hi - t0);
            // factor 2^(30 - e): the largest scale becomes less than 2^16, its products less than 2^10
            const int e = valid ? (int)fc_top<HD>(r.top, lane, low, valid) : 0;
            if (i >= 2) ok = mbar_wait(&s_full[i & 1], (uint32_t)(((i >> 1) - 1) & 1));  // S(i - 2) is there: K(i - 2) has been read
            ok = __all_sync(0xffffffffu, ok && !*aborted);  // the warp leaves as one
            if (!ok) break;
#pragma unroll 1
            for (int j = 0; j < 2; j++) {  // rolled: the code of three kinds of warps has to stay close to them
                const uint32_t words[4] = {r.codes[0].x, r.codes[0].y, r.codes[0].z, r.codes[0].w};
                const uint32_t sc[2] = {r.scales[0].x, r.scales[0].y};
                uint32_t d2[NB];
                fc_scales<NB>(sc, e, kr + 8 * j >= low && kr + 8 * j < valid, d2);
#pragma unroll
                for (int x = 0; x < NB; x++) {
                    uint4 hi, lo;
                    fc_unpack(valid ? words[x] : 0u, d2[x], hi, lo);
                    const uint32_t at = L::K + (uint32_t)(i & 1) * (2 * L::PART) + fc_off(kr + 8 * j, 32 * x + 8 * kt, FC_ATOM);
                    *reinterpret_cast<uint4*>(smem + at) = hi;
                    *reinterpret_cast<uint4*>(smem + at + L::PART) = lo;
                }
                r.codes[0] = r.codes[1];
                r.scales[0] = r.scales[1];
            }
            if (w == 0 && lane == 0) k_mul[i & 3] = valid ? fc_power(e - 21) : 0.0f;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[i & 1]);
            const int page = pages.next(missing);
            fc_load<HD, false>(src, page_stride, scales_at, page, pages.slot, kr, kt, lane, r);
            if (w == i % FC_UN_WARPS) {  // in turn: the issue holds a warp up
                if (i < FC_UN_WARPS) ok = mbar_wait(&q_ready, 0u);
                if (ok && i >= 2) ok = mbar_wait(&o_full[i & 1], (uint32_t)(((i >> 1) - 1) & 1));  // P(i - 2), in S(i)'s place, has been read
                ok = __all_sync(0xffffffffu, mbar_wait(&k_full[i & 1], (uint32_t)((i >> 1) & 1)) && ok && !*aborted);
                if (!ok) break;
                fc_fence_after();
#pragma unroll
                for (int x = 0; x < 3 * (HD / 64); x++) {  // low x high, high x low, high x high
                    const int part = x / (HD / 64), atom = x % (HD / 64);
                    const uint32_t a = tmem + FC_TQ + (part == 0 ? HD / 2 : 0) + atom * 32;
                    const uint64_t bd = fc_desc(base + L::K + (uint32_t)(i & 1) * (2 * L::PART)) + ((part == 1 ? L::PART : 0) + atom * FC_ATOM) / 16;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        fc_mma(lane == 0, tmem + FC_TS + (uint32_t)((i & 1) * FC_CHUNK), a + 8 * k, bd + (uint64_t)(2 * k), IDESC_S, x | k ? 1u : 0u);
                }
                if (lane == 0) fc_commit(&s_full[i & 1]);
                last = i;
                __syncwarp();
            }
        }
        if (missing) set_status(p.status, VSL_ERR_BOUNDS);
        if (!ok) {
            set_status(p.status, VSL_ERR_TIMEOUT);
            abort_s = 1;
        }
        // TMEM is not freed, nor shared memory used again, under a running product
        if (last >= 0 && (!ok || last == n - 1)) mbar_wait(&s_full[last & 1], (uint32_t)((last >> 1) & 1));
        __syncwarp();
    } else if (warp >= FC_SM_WARPS + FC_UN_WARPS) {
        // ================= V: unpacking, and (in turn) the products =================
        const int w = warp - FC_SM_WARPS - FC_UN_WARPS;
        const int vp = 8 * w + (lane & 3) + 4 * (lane >> 4), vu = (lane >> 2) & 3;  // rows 2 vp, + 1
        const unsigned char* src = p.v_cache + g * head_bytes;
        FcPages pages(p, b, t_lo, n);
        FcRaw r;
        bool missing = false, ok = true;
        int last = -1;  // chunk whose product this warp issued last
        const int page0 = pages.next(missing);
        fc_load<HD, true>(src, page_stride, scales_at, page0, pages.slot, vp, vu, lane, r);
        for (int i = 0; i < n; i++) {
            const int t0 = t_lo + i * FC_CHUNK, low = t_first - t0, valid = r.page < 0 ? 0 : min(FC_CHUNK, t_hi - t0);
            const int e = valid ? (int)fc_top<HD>(r.top, lane, low, valid) : 0;
            if (i >= 2) ok = mbar_wait(&o_full[i & 1], (uint32_t)(((i >> 1) - 1) & 1));  // the product with V(i - 2) is done
            ok = __all_sync(0xffffffffu, ok && !*aborted);
            if (!ok) break;
            uint32_t bad = 0;  // bit 4 j + x: row 2 vp + j, block x
#pragma unroll 1
            for (int j = 0; j < 2; j++) {
                uint32_t words[2] = {r.scales[0].x, r.scales[0].y}, d2[NB];
                const bool on = 2 * vp + j >= low && 2 * vp + j < valid;
#pragma unroll
                for (int x = 0; x < NB / 2; x++) {
                    if (on && (words[x] & 0x7c00u) == 0x7c00u) {
                        bad |= 1u << (4 * j + 2 * x);
                        words[x] &= 0xffff0000u;
                    }
                    if (on && (words[x] & 0x7c000000u) == 0x7c000000u) {
                        bad |= 2u << (4 * j + 2 * x);
                        words[x] &= 0xffffu;
                    }
                }
                fc_scales<NB>(words, e, on, d2);
#pragma unroll
                for (int x = 0; x < NB; x++) {
                    const uint32_t a = x < 2 ? r.codes[0].x : r.codes[0].y, c1 = x < 2 ? r.codes[1].x : r.codes[1].y;
                    uint4 hi, lo;
                    fc_unpack(valid ? __byte_perm(a, c1, x & 1 ? 0x7632u : 0x5410u) : 0u, d2[x], hi, lo);
                    const uint32_t at = L::V + (uint32_t)(i & 1) * (2 * L::PART) + fc_off(2 * vp + j, 32 * x + 8 * vu, FC_ATOM);
                    *reinterpret_cast<uint4*>(smem + at) = hi;
                    *reinterpret_cast<uint4*>(smem + at + L::PART) = lo;
                }
                r.codes[0].x = r.codes[0].z;
                r.codes[0].y = r.codes[0].w;
                r.codes[1].x = r.codes[1].z;
                r.codes[1].y = r.codes[1].w;
                r.scales[0] = r.scales[1];
            }
            const bool any = __any_sync(0xffffffffu, bad != 0);
            if (lane == 0) v_bad[i & 1][w][0] = any;
            if (any) {
#pragma unroll
                for (int x = 0; x < NB; x++) {
                    uint32_t rows = vu == 0 ? ((bad >> x & 1u) | (bad >> (4 + x) & 1u) << 1) << (2 * (vp & 7)) : 0u;
                    rows = __reduce_or_sync(0xffffffffu, rows);
                    if (lane == 0) v_bad[i & 1][w][1 + x] = rows;  // positions 16 w + bit
                }
            }
            if (w == 0 && lane == 0) v_mul[i & 1] = fc_power(e - 21);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[i & 1]);
            const int page = pages.next(missing);
            fc_load<HD, true>(src, page_stride, scales_at, page, pages.slot, vp, vu, lane, r);
            if (w == i % FC_UN_WARPS) {  // in turn: the issue holds a warp up
                ok = mbar_wait(&v_full[i & 1], (uint32_t)((i >> 1) & 1));
                ok = __all_sync(0xffffffffu, mbar_wait(&p_ready, (uint32_t)(i & 1)) && ok && !*aborted);
                if (!ok) break;
                fc_fence_after();
#pragma unroll
                for (int part = 0; part < 3; part++) {
                    const uint32_t a = tmem + FC_TS + (uint32_t)((i & 1) * FC_CHUNK) + (part == 0 ? 8 : 0);
                    const uint64_t bd = fc_desc_mn(base + L::V + (uint32_t)(i & 1) * (2 * L::PART)) + (part == 1 ? L::PART : 0) / 16;
#pragma unroll
                    for (int k = 0; k < FC_CHUNK / 16; k++) {
                        const uint32_t d = tmem + FC_TO + (uint32_t)((i & 1) * HD);
                        const uint64_t v = bd + (uint64_t)(k * (2048 >> 4));
                        if (part == 1 && k == 0) fc_mma_scaled(lane == 0, d, a, v, IDESC_O);  // p's low part is 2^11 times as large
                        else fc_mma(lane == 0, d, a + 16 * k, v, IDESC_O, part | k ? 1u : 0u);
                    }
                }
                if (lane == 0) fc_commit(&o_full[i & 1]);
                last = i;
                __syncwarp();
            }
        }
        if (missing) set_status(p.status, VSL_ERR_BOUNDS);
        if (!ok) {
            set_status(p.status, VSL_ERR_TIMEOUT);
            abort_s = 1;
        }
        if (last >= 0 && (!ok || last == n - 1)) mbar_wait(&o_full[last & 1], (uint32_t)((last >> 1) & 1));
        __syncwarp();
    } else {
        // ================= softmax =================
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        // ---- q: two parts of q log2(e) / sqrt(hd) 2^(16 - e), e from the row's largest magnitude, in the order of K.
        // The factor left for the scores is a power of two: the product is exact, no exponent can come out above
        // its row's maximum, however large the scores ----
        float q_mul;
        {
            // rows of q to shared memory, then a row half per thread
            constexpr int LANES = HD / 4, ROWS = FC_SM_WARPS * 32 / LANES;  // 16 bytes per lane
            const int d = threadIdx.x % LANES * 4;
            const int gc = c * FC_COLS + (int)threadIdx.x / LANES, row = gc / p.G;
            int h = gc - row * p.G;
            const float* from = p.q + (((size_t)b * p.rows + row) * p.n_heads + g * p.G + h) * HD + d;
            const size_t next_row = (size_t)(p.n_heads - p.G) * HD;
#pragma unroll 1
            for (int col = threadIdx.x / LANES; col < cols; col += ROWS) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + L::Q + (uint32_t)(col * L::OUT_ROW + d) * 4), "l"(from) : "memory");
                from += ROWS * HD;
                for (h += ROWS; h >= p.G; h -= p.G) from += next_row;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            named_barrier_sync(1, 32 * FC_SM_WARPS);
            const float4* src = reinterpret_cast<const float4*>(smem + L::Q + (size_t)(t * L::OUT_ROW + hc * HALF) * 4);
            float big = 0.0f;
            if (t < cols) {
#pragma unroll
                for (int j = 0; j < HALF / 4; j++) {
                    const float4 v = src[j];
                    big = fmaxf(fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                }
            }
            red[0][hc][t] = big;
            named_barrier_sync(2 + (warp & 3), 64);
            big = fmaxf(big, red[0][hc ^ 1][t]);
            // maxima below 2^-100, zero among them, take e = -100, so that no factor overflows
            const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253) - 127;
            const float down = p.scale * (1.4426950408889634f * 65536.0f) * fc_power(-e);
            q_mul = fc_power(e - 16);
#pragma unroll 1
            for (int k = 0; k < HALF / 16; k++) {  // rolled: straight code is slow the first time
                float x[16];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 v = t < cols ? src[4 * k + j] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
                }
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int d = 8 * (j / 4) + j % 4;  // pairs (d, d + 4)
                    const float a = x[d] * down, bb = x[d + 4] * down;
                    hi[j] = pack_rn(a, bb);
                    lo[j] = pack_rn(a - half_lo(hi[j]), bb - half_hi(hi[j]));
                }
                fc_st8(lanes + FC_TQ + hc * (HALF / 2) + 8 * k, hi);
                fc_st8(lanes + FC_TQ + HD / 2 + hc * (HALF / 2) + 8 * k, lo);
            }
            fc_st_wait();
            fc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready);
        }
        // positions the column sees; an unused one sees what the last one does, so that chunks stay whole
        const int pr = pos + (c * FC_COLS + min(t, cols - 1)) / p.G, c_hi = max(min(pr + 1, p.max_pages * p.page_size), 0);
        const int c_lo = c_hi > 0 ? min(sparse_first(p.sp, pr), c_hi - 1) : 0;
        if (pr >= c_hi && pr >= 0) set_status(p.status, VSL_ERR_BOUNDS);
#pragma unroll
        for (int j = 0; j < HALF; j++) o[j] = 0.0f;
        float alpha_last = 0.0f, v_last = 0.0f;
        bool ok = true;
        for (int i = 0; i <= n; i++) {  // a pass more, for the last chunk's output
            float mul = 0.0f, top = -CUDART_INF_F, m0 = 0.0f, alpha = 1.0f, v_next = 0.0f;
            const uint32_t s_at = lanes + FC_TS + (uint32_t)((i & 1) * FC_CHUNK + hc * 32);
            const int t0 = t_lo + i * FC_CHUNK + hc * 32;
            int lo = c_lo - t0, hi = c_hi - t0;  // of the 32 positions the column sees [lo, hi)
            if (i < n) {
                ok = __all_sync(0xffffffffu, ok && mbar_wait(&s_full[i & 1], (uint32_t)((i >> 1) & 1)) && !*aborted);
                if (ok) {
                    fc_fence_after();
                    float s[32];
                    fc_ld32(s_at, s);
                    mul = k_mul[i & 3];
                    if (mul == 0.0f) hi = 0;
                    mul = fmaxf(mul * q_mul, fc_power(-126));  // not zero: it meets infinities
                    if (__any_sync(0xffffffffu, lo > 0 || hi < 32)) {
#pragma unroll
                        for (int j = 0; j < 32; j++) s[j] = j >= lo && j < hi ? s[j] : -CUDART_INF_F;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) top = fmaxf(fmaxf(fmaxf(top, s[j]), fmaxf(s[j + 1], s[j + 2])), s[j + 3]);
                    top *= mul;
                    red[i & 1][hc][t] = top;
                }
                // the two warps of a column leave together
                if (named_barrier_or(2 + (warp & 3), 64, !ok)) {
                    ok = false;
                    break;
                }
                const float m_new = fmaxf(m, fmaxf(top, red[i & 1][hc ^ 1][t]));
                m0 = m_new == -CUDART_INF_F ? 0.0f : m_new;
                alpha = ex2(m - m0);
                m = m_new;
            }
            if (i > 0) ok = mbar_wait(&o_full[(i - 1) & 1], (uint32_t)(((i - 1) >> 1) & 1)) && !*aborted;
            ok = __all_sync(0xffffffffu, ok);
            if (i < n) {
                // exp2(s mul - m + 15); 15 - m rounded down, so that it is at most 2^15 and, -m being a float, at least 1
                // for the largest
                const float2 mul2x = make_float2(mul, mul), off = make_float2(__fsub_rd(15.0f, m0), __fsub_rd(15.0f, m0));
                float2 sum = make_float2(0.0f, 0.0f);
                const bool whole = __all_sync(0xffffffffu, lo <= 0 && hi >= 32);
#pragma unroll 1
                for (int j = 0; j < 32; j += 16) {  // the two parts of 16 p take the place of 16 scores
                    float y[16];
                    fc_ld16(s_at + j, y);
                    if (!whole) {
#pragma unroll
                        for (int k = 0; k < 16; k++) y[k] = j + k >= lo && j + k < hi ? y[k] : -CUDART_INF_F;
                    }
                    uint32_t ph[8], pl[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        float2 x = fma2(make_float2(y[2 * k], y[2 * k + 1]), mul2x, off);
                        x = make_float2(ex2(x.x), ex2(x.y));
                        sum = add2(sum, x);
                        ph[k] = pack_rn(x.x, x.y);
                        x = mul2(x, make_float2(2048.0f, 2048.0f));
                        const float2 z = fma2(make_float2(half_lo(ph[k]), half_hi(ph[k])), make_float2(-2048.0f, -2048.0f), x);
                        pl[k] = pack_rn(z.x, z.y);
                    }
                    fc_st8(s_at + j, ph);
                    fc_st8(s_at + j + 8, pl);
                }
                l = fmaf(l, alpha, sum.x + sum.y);
                ok = __all_sync(0xffffffffu, mbar_wait(&v_full[i & 1], (uint32_t)((i >> 1) & 1)) && ok);  // the scales of V(i) are there
                v_next = v_mul[i & 1];
                for (int w = 0; w < FC_UN_WARPS; w++) {
                    if (!v_bad[i & 1][w][0]) continue;
                    const int first_row = t_lo + i * FC_CHUNK + 16 * w;
                    const int a = min(max(c_lo - first_row, 0), 16), e = min(max(c_hi - first_row, a), 16);
                    const uint32_t seen = ((1u << e) - 1u) & ~((1u << a) - 1u);
                    for (int x = 0; x < NB; x++)
                        if (v_bad[i & 1][w][1 + x] & seen) nan_blocks |= 1u << x;
                }
                fc_st_wait();
                fc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready);
            }
            if (i > 0 && ok) {  // o = alpha o + O(i - 1)
                fc_fence_after();
                const bool same = __all_sync(0xffffffffu, alpha_last == 1.0f);  // no maximum had grown
#pragma unroll
                for (int x = 0; x < HALF / 32; x++) {
                    float v[32];
                    fc_ld32(lanes + FC_TO + (uint32_t)(((i - 1) & 1) * HD + hc * HALF + 32 * x), v);
                    float2* o2 = reinterpret_cast<float2*>(o) + 16 * x;
                    if (!same) {
#pragma unroll
                        for (int j = 0; j < 16; j++) o2[j] = mul2(o2[j], make_float2(alpha_last, alpha_last));
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) o2[j] = fma2(make_float2(v[2 * j], v[2 * j + 1]), make_float2(v_last, v_last), o2[j]);
                }
            }
            alpha_last = alpha;
            v_last = v_next;
        }
        fc_fence_before();
        if (!ok) {
            set_status(p.status, VSL_ERR_TIMEOUT);
            abort_s = 1;
        }
        red[0][hc][t] = l;
    }

    __syncthreads();
    if (warp == FC_SM_WARPS) {
        fc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(FC_TMEM_COLS) : "memory");
    }
    const bool has_row = warp < FC_SM_WARPS;
    if (has_row) {
        l = red[0][0][t] + red[0][1][t];
#pragma unroll
        for (int j = 0; j < HALF; j++)
            if (nan_blocks >> ((hc * HALF + j) / 32) & 1u) o[j] = CUDART_NAN_F;
    }

    // ---- output, through shared memory, with the join over the cluster: every CTA takes some rows of all ----
    float* rows = reinterpret_cast<float*>(smem);
    if (has_row) {
        float* dst = rows + t * L::OUT_ROW + hc * HALF;
#pragma unroll
        for (int j = 0; j < HALF; j += 8) {  // dimensions back in their order
            *reinterpret_cast<float4*>(dst + j) = make_float4(o[j], o[j + 2], o[j + 4], o[j + 6]);
            *reinterpret_cast<float4*>(dst + j + 4) = make_float4(o[j + 1], o[j + 3], o[j + 5], o[j + 7]);
        }
        if (hc == 0) {
            red[1][0][t] = m;
            red[1][1][t] = l;
        }
    }
    fc_cluster_sync();
    const int r0 = cols * rank / cluster, r1 = cols * (rank + 1) / cluster;
    float* mine = p.part + ((size_t)unit * most_groups + group) * fc_part_floats<HD>();
    for (int i = threadIdx.x; i < (r1 - r0 + 3) / 4 * 4 * FC_CLUSTER; i += FC_THREADS) {  // whole warps: 4 rows, 8 parts
        const int row = i / FC_CLUSTER, x = i % FC_CLUSTER;
        const bool there = x < cluster && row < r1 - r0;
        const float mx = there ? fc_ld_remote(fc_remote(smem_u32(&red[1][0][r0 + row]), x)) : -CUDART_INF_F;
        const float lx = there ? fc_ld_remote(fc_remote(smem_u32(&red[1][1][r0 + row]), x)) : 0.0f;
        float top = mx;
#pragma unroll
        for (int d = 1; d < FC_CLUSTER; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float w = ex2(mx - (top == -CUDART_INF_F ? 0.0f : top));
        float sum = lx * w;
#pragma unroll
        for (int d = 1; d < FC_CLUSTER; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (there) weight[x][row] = groups > 1 ? w : sum == 0.0f ? 0.0f : w / sum;  // a row that sees nothing gives zeros
        if (there && x == 0 && groups > 1) {
            __stcg(mine + FC_COLS * HD + r0 + row, top);
            __stcg(mine + FC_COLS * (HD + 1) + r0 + row, sum);
        }
    }
    __syncthreads();
    {
        constexpr int LANES = HD / 4, ROWS = FC_THREADS / LANES;
        const int d = threadIdx.x % LANES * 4;
        const int gc = c * FC_COLS + r0 + (int)threadIdx.x / LANES, q_row = gc / p.G;
        int h = gc - q_row * p.G;
        float* dst = p.out + (((size_t)b * p.rows + q_row) * p.n_heads + g * p.G + h) * HD + d;
        const size_t next_row = (size_t)(p.n_heads - p.G) * HD;
#pragma unroll 1
        for (int row = threadIdx.x / LANES; row < r1 - r0; row += ROWS) {
            const uint32_t at = base + (uint32_t)((r0 + row) * L::OUT_ROW + d) * 4;
            float4 v[FC_CLUSTER], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < FC_CLUSTER; x++)  // all of them on their way at once
                if (x < cluster) v[x] = fc_ld_remote4(fc_remote(at, x));
#pragma unroll
            for (int x = 0; x < FC_CLUSTER; x++)
                if (x < cluster) {
                    const float w = weight[x][row];
                    acc.x += v[x].x * w; acc.y += v[x].y * w; acc.z += v[x].z * w; acc.w += v[x].w * w;
                }
            __stcg(reinterpret_cast<float4*>(groups > 1 ? mine + (r0 + row) * HD + d : dst), acc);
            dst += ROWS * HD;
            for (h += ROWS; h >= p.G; h -= p.G) dst += next_row;
        }
    }
    if (cluster > 1) fc_cluster_sync();  // the others have read this CTA's rows
    if (groups == 1) return;
    // ---- the last of the groups joins their rows, in order ----
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* counter = p.counters + unit * FC_CLUSTER + rank;
        last_s = atomicAdd(counter, 1) == groups - 1;
        if (last_s) *counter = 0;
    }
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    const float* all = p.part + (size_t)unit * most_groups * fc_part_floats<HD>();
    for (int i = threadIdx.x; i < (r1 - r0) * (HD / 4); i += FC_THREADS) {
        const int row = r0 + i / (HD / 4), d = i % (HD / 4) * 4, gc = c * FC_COLS + row, q_row = gc / p.G;
        float top = -CUDART_INF_F, sum = 0.0f;
        for (int x = 0; x < groups; x++) top = fmaxf(top, __ldcg(all + (size_t)x * fc_part_floats<HD>() + FC_COLS * HD + row));
        if (top == -CUDART_INF_F) top = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int x = 0; x < groups; x++) {
            const float* from = all + (size_t)x * fc_part_floats<HD>();
            const float w = ex2(__ldcg(from + FC_COLS * HD + row) - top);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(from + row * HD + d));
            sum += __ldcg(from + FC_COLS * (HD + 1) + row) * w;
            acc.x += v.x * w; acc.y += v.y * w; acc.z += v.z * w; acc.w += v.w * w;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<float4*>(p.out + (((size_t)b * p.rows + q_row) * p.n_heads + g * p.G + gc - q_row * p.G) * HD + d) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

size_t fc_part_bytes() { return ((size_t)(sm_count() / FC_GROUPED) * fc_part_floats<128>() * sizeof(float) + 255) & ~(size_t)255; }

template <int HD>
static int fc_launch_t(const FqParams& p, long long units, cudaStream_t st) {
    auto kern = vsl_flash_chunk_q4_kernel<HD>;
    static thread_local int configured_dev = -1;
    static thread_local int active[FC_CLUSTER + 1];  // clusters of a size that run at once
    int dev = 0;
    cudaGetDevice(&dev);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(FC_THREADS);
    cfg.dynamicSmemBytes = FcSmem<HD>::BYTES;
    cfg.stream = st;
    cfg.attrs = attr;
    if (configured_dev != dev) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FcSmem<HD>::BYTES);
        cfg.numAttrs = 1;
        active[1] = sm_count();
        for (int n = 2; n <= FC_CLUSTER && e == cudaSuccess; n++) {
            attr[0].val.clusterDim.x = n;
            cfg.gridDim = dim3(n);
            e = cudaOccupancyMaxActiveClusters(&active[n], kern, &cfg);
        }
        if (e != cudaSuccess) return launch_status(e, "flash_decode_q4 set-up");
        configured_dev = dev;
    }
    // As many CTAs per tile as run at once, in clusters as large as that allows: 8 tiles over 60000 positions take
    // 132 us with 16 CTAs each, 243 with 8 (but 5 chunks 14 us in two clusters, 12 in one). Small clusters are not
    // grouped: FC_GROUPED bounds the workspace (2.4 MB).
    int cluster = 1, groups = 1;
    for (int n = 2; n <= FC_CLUSTER; n++) {
        const int fit = (int)std::min<long long>(std::min(active[n], sm_count() / n) / units, n < FC_GROUPED ? 1 : sm_count());
        if (fit >= 1 && fit * n >= groups * cluster) {
            cluster = n;
            groups = fit;
        }
    }
    attr[0].val.clusterDim.x = cluster;
    cfg.gridDim = dim3((unsigned)(units * groups * cluster));
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return launch_status(cudaLaunchKernelEx(&cfg, kern, p, groups, cluster), "flash_decode_q4 launch");
}

int fc_launch(FqParams p, int head_dim, cudaStream_t st) {
    p.tiles = (int)(((long long)p.rows * p.G + FC_COLS - 1) / FC_COLS);
    const long long units = (long long)p.B * p.n_kv * p.tiles;
    return head_dim == 128 ? fc_launch_t<128>(p, units, st) : fc_launch_t<64>(p, units, st);
}

}  // namespace vsl
