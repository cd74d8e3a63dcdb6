// Attention of one or several query rows per sequence over the 4-bit paged cache (kv_layout.h). Many rows:
// attention_q4_chunk.cu.
//
//   s_t = q . k_t / sqrt(hd),  p_t = exp(s_t - max s),  o = sum_t p_t v_t / sum_t p_t
//
// over the positions [first, pos] of each query row, K and V as blocks of 32 dimensions with codes
// n in 0..15 and a scale d: value (n - 8) d.
//
// What bounds it: the cache is read once (144 bytes per position and KV head at head_dim 128), and
// each of its codes has to become an operand: at the memory's rate an SM has about three instruction
// slots per 32 codes. So the codes go from registers into mma.sync (m16n8k16), whose fragments a warp
// can build itself; a tcgen05 operand would have to be written out to shared or tensor memory as
// 16-bit values first, four times the bytes the cache delivers.
//   - Both products have the exact integers n - 8 as the 16-row operand (rows: positions for the
//     scores, dimensions for the output): a shift, and a mask and a multiply-add per pair of codes, give
//     eight of them (the pairs sit in the words in the order the fragments want). Products of
//     codes alone (the offset subtracted from the sums) save the multiply-adds (3 % of the time), but
//     not the accuracy: errors 1.5 to 4 times those of a plain fp32 form.
//   - The scales stay in fp32: a block's partial scores are multiplied by its d, and p_t is multiplied
//     by d_t of each V block before the second product.
//   - The other operand, q (times log2(e) / sqrt(hd)) or p d, is split into two fp16 values (22 bits), the
//     low one of p d 2^11 times as large. With at most four (row, head) columns the parts are the two
//     halves of the eight operand columns, so that one instruction covers both; with up to eight they are
//     two instructions.
//   - Scores come out by (position, two columns) per lane, with a column's statistics in the lanes that
//     hold its outputs; movmatrix turns p d into the operand of the second product.
//
// Work is cut into stages of 32 positions of one item, that is one (sequence, KV head, tile of 8
// (row, head) columns). Every warp of the launch gets one contiguous part of an item: with at most q
// stages each, the parts of all items are as many as there are warps, whatever the lengths (with
// more items than warps, whole items in turn). A warp works through its part alone, with its own
// ring of 16-byte asynchronous copies (bulk copies of these 256 to 2048-byte runs held the issuing
// warp up for a fifth of its time). Parts (maximum, sum, output) of an item are joined per CTA in
// shared memory and, where the item crosses CTAs, by the last CTA to arrive, in the order of the
// positions: results do not depend on the timing.
//
// Twelve warps of 168 registers per SM: 16 of 128 take as long, 10 a sixth longer. Measured on a B200:
// 16 sequences of 8192 positions, 32 / 8 heads of 128: 44.5 us (3.4 TB/s, 53 % of the measured copy
// rate; 4.6 TB/s in the slope from 8192 to 24576 positions, so 12 us of start and joins); 131071 positions of
// one sequence 46.4 to 47.2 us; 384 positions of 32 heads 7.2 us. The loop issues 670 instructions
// per stage at two thirds of the SM's issue rate: that bounds it.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "../host/kernels.h"
#include "attention_q4.cuh"
#include "common.cuh"
#include "kv_layout.h"
#include "launch.cuh"

namespace vsl {

constexpr int FQ_WARPS = 12, FQ_THREADS = 32 * FQ_WARPS;
constexpr int FQ_STAGE = 32;                      // positions a warp stages and processes at once
constexpr int FQ_COLS = 8;                        // (row, head) columns per tile
constexpr int FQ_CTAS_PER_SM = 1;
constexpr int FQ_MAX_BATCH = 1024;

// Stages after which a warp's accumulators move to its place in the workspace. The matrix unit cuts
// its sums instead of rounding them, about 2^-26 of the sum per instruction and always towards zero, so a
// chain of instructions stays short whatever the length. Twice / four times as long (head_dim 128 / 64):
// 1 to 2 % faster, errors 1.4e-6 instead of 0.9e-6 / 0.7e-6 where a plain fp32 form has 1.2e-6 / 0.8e-6 (measured
// with a low part of p d that was cut; rounded, the errors are 0.6e-6 to 0.7e-6 at head_dim 128).
template <int HD, bool SPLIT_N>
__host__ __device__ constexpr int fq_chain() {
    return (SPLIT_N ? 16 : 8) / (HD == 64 ? 2 : 1);
}
// Stages a warp processes at once, of two such groups in its ring: two spread a group's fixed chain
// (wait, maxima, exponentials) over twice the positions (7 % faster in long runs); with eight columns of 128
// dimensions the registers hold one. Slopes in long runs of 32 heads over 8: 4.6 TB/s, 4.0 at head_dim 64; of 64
// heads 3.1 and 2.9 TB/s.
template <int HD, bool SPLIT_N>
__host__ __device__ constexpr int fq_group() {
    return SPLIT_N || HD == 64 ? 2 : 1;
}
template <int HD>
__host__ __device__ constexpr int fq_stage_bytes() {
    return FQ_STAGE * (HD + HD / 8);  // codes of K and V, scales of K and V
}
template <int HD>
__host__ __device__ constexpr int fq_col_stride() {
    return HD + 4;  // floats between the columns of a warp's partial: keeps 16-byte stores off one bank
}
template <int HD>
__host__ __device__ constexpr int fq_part_floats() {
    return FQ_COLS * (HD + 2);
}
// A warp's part of item `item` of sequence b, which the n warps from w0 on work on. w0 < 0: none.
struct FqTail {
    int w0, n, b, item;
};
template <int HD>
struct FqParts {  // the warps' parts of their items
    float o[FQ_WARPS][FQ_COLS][fq_col_stride<HD>()];
    float m[FQ_WARPS][FQ_COLS], l[FQ_WARPS][FQ_COLS];
};
template <int HD, bool SPLIT_N>
struct FqSmem {
    union {
        unsigned char ring[FQ_WARPS][2 * fq_group<HD, SPLIT_N>()][fq_stage_bytes<HD>()];
        FqParts<HD> parts;  // once every stage is consumed
    };
    FqTail tail[FQ_WARPS];
    uint32_t warp_sum[FQ_WARPS], warp_max[FQ_WARPS];
    int last[2];
};

__device__ __forceinline__ void mma16816(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// asynchronous copy of 16 bytes to shared memory, past L1
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// c = a b
__device__ __forceinline__ void mma16816_first(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// larger magnitude of each half (the signs are combined)
__device__ __forceinline__ uint32_t hmax_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// the two halves of h times k (fp16), plus c, in fp32
__device__ __forceinline__ float2 fma_half(uint32_t h, unsigned short k, float2 c) {
    float2 r;
    asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tfma.rn.f32.f16 %0, a, %3, %4;\n\tfma.rn.f32.f16 %1, b, %3, %5;}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(h), "h"(k), "f"(c.x), "f"(c.y));
    return r;
}
// transpose of an 8x8 matrix of fp16 (row lane / 4, columns 2 (lane % 4) and + 1)
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

// Stages of each of the sequence's items with its first row at pos.
__device__ __forceinline__ uint32_t fq_units(const FqParams& p, int pos) {
    int lo, hi;
    fq_range(p, pos, 0, p.rows - 1, FQ_STAGE, lo, hi);
    return max(1, (hi - lo + FQ_STAGE - 1) / FQ_STAGE);  // an empty sequence keeps one: its output is set to zero
}
__device__ __forceinline__ float* fq_out(const FqParams& p, int b, int g, int c, int col, int hd) {
    const int gc = c * FQ_COLS + col, row = gc / p.G, h = g * p.G + gc % p.G;
    return p.out + (((size_t)b * p.rows + row) * p.n_heads + h) * hd;
}

// Join n partial results of an item, in order, into its output: the first at `first`, the following
// CTAs' at rest + 2 i * (floats of a partial), by half of the CTA's threads. The loads of eight parts
// are in flight at once.
template <int HD>
__device__ __forceinline__ void fq_join(const FqParams& p, int b, int g, int c, int cols, int n, const float* first,
                                        const float* rest) {
    constexpr int PF = fq_part_floats<HD>(), CHUNK = 8;
    for (int i = threadIdx.x % (FQ_THREADS / 2); i < cols * (HD / 4); i += FQ_THREADS / 2) {
        const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
        float M = -CUDART_INF_F, L = 0.0f;
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = 0; k0 < n; k0 += CHUNK) {
            float m[CHUNK], l[CHUNK];
            float4 v[CHUNK];
            float top = M;
#pragma unroll
            for (int k = 0; k < CHUNK; k++) {
                m[k] = -CUDART_INF_F;
                if (k0 + k >= n) continue;
                const float* q = k0 + k == 0 ? first : rest + (size_t)(2 * (k0 + k)) * PF;
                m[k] = __ldcg(q + FQ_COLS * HD + col);
                l[k] = __ldcg(q + FQ_COLS * HD + FQ_COLS + col);
                v[k] = __ldcg(reinterpret_cast<const float4*>(q + col * HD + d));
            }
#pragma unroll
            for (int k = 0; k < CHUNK; k++) top = fmaxf(top, m[k]);
            const float top0 = top == -CUDART_INF_F ? 0.0f : top, a = ex2(M - top0);
            M = top;
            L *= a;
            r.x *= a; r.y *= a; r.z *= a; r.w *= a;
#pragma unroll
            for (int k = 0; k < CHUNK; k++) {
                if (k0 + k >= n) continue;
                const float w = ex2(m[k] - top0);
                L += l[k] * w;
                r.x += v[k].x * w; r.y += v[k].y * w; r.z += v[k].z * w; r.w += v[k].w * w;
            }
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees nothing gives zeros
        *reinterpret_cast<float4*>(fq_out(p, b, g, c, col, HD) + d) =
            make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
    }
}

// SPLIT_N: at most four columns; the two parts of p d are the halves of the eight operand columns.
template <int HD, bool SPLIT_N>
__global__ void __launch_bounds__(FQ_THREADS, FQ_CTAS_PER_SM) vsl_flash_decode_q4_kernel(FqParams p) {
    constexpr int NB = HD / 32, PF = fq_part_floats<HD>(), GROUP = fq_group<HD, SPLIT_N>(), FQ_RING = 2 * GROUP;
    constexpr uint32_t CODE_BYTES = FQ_STAGE * HD / 2, SCALE_BYTES = FQ_STAGE * NB * 2, STAGE_BYTES = fq_stage_bytes<HD>();
    extern __shared__ __align__(16) unsigned char smem_raw[];
    FqSmem<HD, SPLIT_N>& sm = *reinterpret_cast<FqSmem<HD, SPLIT_N>*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g4 = lane >> 2, t4 = lane & 3;  // fragment group and quad lane
    pdl_wait();

    // ---- this warp's part: stages [part * q, ..) of item `item` of sequence b ----
    const uint32_t items_per_seq = (uint32_t)(p.n_kv * p.tiles), workers = gridDim.x * FQ_WARPS;
    const uint32_t worker = blockIdx.x * FQ_WARPS + warp, items = (uint32_t)p.B * items_per_seq;
    const bool many = items >= workers;  // whole items in turn
    int b = -1, item = 0, pos = 0;       // b < 0: nothing (left) to do
    FqTail tail = {-1, 1, 0, 0};
    uint32_t part = 0, q = 0x40000000u;
    // Stages per part from the stages of all items and of the longest: ceil(s / q) parts of each item
    // of s stages are at most as many as there are workers. A CTA per item needs no join between CTAs,
    // which costs about as much as a stage: with q + 4 instead of q + 1 below, 4 x 2048 positions of 8 KV heads
    // took 15.4 us against 11.8, 8 x 2048 15.5 against 14.0; with q + 2, 16 x 8192 took 1 % more.
    auto plan = [&](uint32_t total, uint32_t most, bool& cta_items) {
        const unsigned long long all = (unsigned long long)total * items_per_seq;
        const uint32_t room = workers - items;
        q = all <= 0xffffffffull ? ((uint32_t)all + room - 1) / room : (uint32_t)((all + room - 1) / room);
        const uint32_t q_cta = (most + FQ_WARPS - 1) / FQ_WARPS;
        cta_items = items <= gridDim.x && q_cta <= q + 1;
        if (cta_items) q = q_cta;
    };
    if (many) {
        b = (int)(worker / items_per_seq);
        item = (int)(worker % items_per_seq);
    } else if (p.B <= 32) {  // a sequence per lane, every warp for itself
        const int mine = lane < p.B ? fq_pos(p, lane) : 0;
        const uint32_t st = lane < p.B ? fq_units(p, mine) : 0;
        bool cta_items;
        plan(__reduce_add_sync(0xffffffffu, st), __reduce_max_sync(0xffffffffu, st), cta_items);
        const uint32_t n = (st + q - 1) / q, width = cta_items && st ? FQ_WARPS : n;
        uint32_t end = width * items_per_seq;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += v;
        }
        const uint32_t who = __ballot_sync(0xffffffffu, worker < end);
        if (who) {
            const int src = __ffs(who) - 1;
            const uint32_t wide = __shfl_sync(0xffffffffu, width, src);
            const uint32_t at = worker - __shfl_sync(0xffffffffu, end - width * items_per_seq, src);
            tail.n = (int)__shfl_sync(0xffffffffu, n, src);
            pos = __shfl_sync(0xffffffffu, mine, src);
            item = (int)(at / wide);
            part = at - (uint32_t)item * wide;
            tail.w0 = (int)(worker - part);
            if (part < (uint32_t)tail.n) b = src;
        }
    } else {  // up to FQ_MAX_BATCH sequences: some per thread, the CTA together
        constexpr int PER = (FQ_MAX_BATCH + FQ_THREADS - 1) / FQ_THREADS;
        const int per = (p.B + FQ_THREADS - 1) / FQ_THREADS;
        uint32_t st[PER], total = 0, most = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int s = tid * per + i;
            st[i] = i < per && s < p.B ? fq_units(p, fq_pos(p, s)) : 0;
            total += st[i];
            most = max(most, st[i]);
        }
        total = __reduce_add_sync(0xffffffffu, total);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) {
            sm.warp_sum[warp] = total;
            sm.warp_max[warp] = most;
        }
        if (tid < FQ_WARPS) sm.tail[tid].w0 = -1;
        __syncthreads();
        total = most = 0;
        for (int w = 0; w < FQ_WARPS; w++) {
            total += sm.warp_sum[w];
            most = max(most, sm.warp_max[w]);
        }
        bool cta_items;
        plan(total, most, cta_items);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) n += (cta_items && st[i] ? FQ_WARPS : (st[i] + q - 1) / q) * items_per_seq;
        uint32_t end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += v;
        }
        __syncthreads();
        if (lane == 31) sm.warp_sum[warp] = end;
        __syncthreads();
        for (int w = 0; w < warp; w++) end += sm.warp_sum[w];
        // the thread whose sequences a warp's number falls into describes the warp's part
        uint32_t base = end - n;
        for (int i = 0; i < PER; i++) {
            const uint32_t parts = (st[i] + q - 1) / q, width = cta_items && st[i] ? FQ_WARPS : parts;
            for (uint32_t w = max(base, blockIdx.x * FQ_WARPS); w < min(base + width * items_per_seq, (blockIdx.x + 1) * FQ_WARPS); w++) {
                const uint32_t it = (w - base) / width;
                sm.tail[w % FQ_WARPS] = FqTail{(int)(base + it * width), (int)parts, tid * per + i, (int)it};
            }
            base += width * items_per_seq;
        }
        __syncthreads();
        tail = sm.tail[warp];
        __syncthreads();
        if (tail.w0 >= 0) {
            part = worker - (uint32_t)tail.w0;
            item = tail.item;
            if (part < (uint32_t)tail.n) {
                b = tail.b;
                pos = fq_pos(p, b);
            }
        }
    }
    tail.b = b;
    tail.item = item;
    const uint32_t head_bytes = (uint32_t)kv_head_page_bytes(VSL_Q4_0, HD, p.page_size), page_stride = p.n_kv * head_bytes;
    const uint32_t scales_at = (uint32_t)kv_q4_scales(HD, p.page_size);
    const uint32_t ring0 = smem_u32(sm.ring[warp]) + lane * 16;
    constexpr int SCALE_LANES = SCALE_BYTES / 16;

    float o[NB][2][4];
    float2 mc = make_float2(0.0f, 0.0f), l = mc;
    float f = 1.0f;

    while (b >= 0 && b < p.B) {
        if (many) pos = fq_pos(p, b);
        int g = item, c = 0;
        if (p.tiles > 1) {
            g = item / p.tiles;
            c = item % p.tiles;
        }
        const int cols = min(FQ_COLS, p.rows * p.G - c * FQ_COLS);
        int t_first, t_end;
        fq_range(p, pos, 0, p.rows - 1, FQ_STAGE, t_first, t_end);
        const uint32_t s0 = part * q;
        const int n = (int)min(q, (uint32_t)max(1, (t_end - t_first + FQ_STAGE - 1) / FQ_STAGE) - s0);
        int tile_lo = t_first, tile_hi = t_end;
        if (p.tiles > 1) fq_range(p, pos, c * FQ_COLS / p.G, (c * FQ_COLS + cols - 1) / p.G, FQ_STAGE, tile_lo, tile_hi);
        t_first += (int)s0 * FQ_STAGE;

        // ---- the lane's query column g4 (SPLIT_N: columns 4-7 are the low parts of 0-3) ----
        float x[NB][8];
        {
            const int col = SPLIT_N ? (g4 & 3) : g4;
            const int gc = c * FQ_COLS + col, row = p.G == 1 ? gc : gc / p.G, h = g * p.G + gc - row * p.G;
            const float4* src = reinterpret_cast<const float4*>(p.q + (((size_t)b * p.rows + row) * p.n_heads + h) * HD) + 2 * t4;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const float4 a = col < cols ? __ldcg(src + 8 * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float4 d = col < cols ? __ldcg(src + 8 * i + 1) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
                x[i][4] = d.x; x[i][5] = d.y; x[i][6] = d.z; x[i][7] = d.w;
            }
        }

        // page ids of the next 32 stages, one per lane; -1: not staged (outside the tile's range, or no page)
        int pages = -1;
        auto load_pages = [&](int k0) {
            const int t0 = t_first + (k0 + lane) * FQ_STAGE;
            pages = -1;
            if (k0 + lane < n && t0 >= tile_lo && t0 < tile_hi) {
                const int pg = p.page_table[(size_t)b * p.max_pages + t0 / p.page_size];
                if (pg >= 0 && pg < p.n_pages) pages = pg;
                else set_status(p.status, VSL_ERR_BOUNDS);
            }
        };
        uint32_t staged = 0;               // ring buffers that hold a stage
        int slot = t_first % p.page_size;  // of the next stage to issue
        // stages k .. k + GROUP - 1 into ring buffers buf ..: 16 bytes per lane and copy; the scales of K by
        // the first lanes, of V by the next ones. Every call closes one copy group.
        const unsigned char* k_src = p.k_cache + (size_t)g * head_bytes + lane * 16;
        const unsigned char* v_src = p.v_cache + (size_t)g * head_bytes + lane * 16;
        const unsigned char* s_src = (lane < SCALE_LANES ? k_src : v_src - SCALE_LANES * 16) + scales_at;
        auto issue = [&](int k, int buf) {
#pragma unroll
            for (int j = 0; j < GROUP; j++) {
                if (k + j >= n) break;
                if (((k + j) & 31) == 0) load_pages(k + j);
                const int page = __shfl_sync(0xffffffffu, pages, (k + j) & 31);
                if (page >= 0) {
                    staged |= 1u << (buf + j);
                    const size_t at = (uint64_t)(uint32_t)page * page_stride + (uint32_t)(slot * (HD / 2));
                    const uint32_t dst = ring0 + (buf + j) * STAGE_BYTES;
#pragma unroll
                    for (int i = 0; i < (int)CODE_BYTES / 512; i++) {
                        cp16(dst + i * 512, k_src + at + i * 512);
                        cp16(dst + CODE_BYTES + i * 512, v_src + at + i * 512);
                    }
                    if (lane < 2 * SCALE_LANES)
                        cp16(dst + 2 * CODE_BYTES, s_src + (uint64_t)(uint32_t)page * page_stride + (uint32_t)(slot * (NB * 2)));
                }
                slot += FQ_STAGE;
                if (slot >= p.page_size) slot = 0;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        issue(0, 0);

        // ---- q fragments: two fp16 parts of q / 2^e, e from the column's largest magnitude ----
        uint32_t qh[NB][4], ql[SPLIT_N ? 1 : NB][4];  // k steps 2 i, 2 i + 1 of block i, two registers each
        float2 q_mul;   // score accumulator -> base-2 exponent
        {
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(x[i][j]));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // The parts hold q log2(e) / sqrt(hd) 2^(16 - e), below 2^15, with big * 2^-e in [1, 2). Maxima below 2^-100,
            // zero among them, take e = -100, so that no factor overflows. What is left for the scores is a power
            // of two (the codes' unit is 2^-9): score times q_mul is exact, and so no weight can come out above 1,
            // and the largest as exactly 1, however large the scores.
            const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253) - 127;
            const float up = __uint_as_float((uint32_t)(127 + e - 7) << 23);
            q_mul = make_float2(__shfl_sync(0xffffffffu, up, 8 * t4), __shfl_sync(0xffffffffu, up, 8 * t4 + 4));
            const float scale = p.scale * (1.4426950408889634f * 65536.0f) * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {  // the pairs (j, j + 4) of the lane's word
                    const float v0 = x[i][j] * scale, v1 = x[i][j + 4] * scale;
                    const uint32_t hi = pack_rn(v0, v1), lo = pack_rn(v0 - half_lo(hi), v1 - half_hi(hi));
                    qh[i][j] = SPLIT_N && g4 >= 4 ? lo : hi;
                    ql[i % (SPLIT_N ? 1 : NB)][j] = lo;
                }
        }
        issue(GROUP, GROUP);  // not before: every warp's first stages come first

        // positions the lane's columns 2 t4, + 1 see (SPLIT_N: of the column whose part they are)
        int c_lo[2], c_hi[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int col = (SPLIT_N ? 2 * (t4 & 1) : 2 * t4) + j, gc = c * FQ_COLS + col;
            c_lo[j] = c_hi[j] = 0;
            if (col < cols) {
                const int pr = pos + (p.G == 1 ? gc : gc / p.G);
                c_hi[j] = max(min(pr + 1, p.max_pages * p.page_size), 0);
                if (c_hi[j] > 0) c_lo[j] = min(sparse_first(p.sp, pr), c_hi[j] - 1);
                if (pr >= c_hi[j] && pr >= 0) set_status(p.status, VSL_ERR_BOUNDS);
            } else {  // an unused column: seen like the tile's first row
                c_hi[j] = -1;
            }
        }
        // positions seen by every / by any column
        const int full_lo = __reduce_max_sync(0xffffffffu, max(c_lo[0], c_lo[1]));
        const int full_hi = __reduce_min_sync(0xffffffffu, min(c_hi[0] < 0 ? INT32_MAX : c_hi[0], c_hi[1] < 0 ? INT32_MAX : c_hi[1]));
        const int any_lo = __reduce_min_sync(0xffffffffu, min(c_hi[0] < 0 ? INT32_MAX : c_lo[0], c_hi[1] < 0 ? INT32_MAX : c_lo[1]));
        const int any_hi = __reduce_max_sync(0xffffffffu, max(c_hi[0], c_hi[1]));

#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[i][j][k] = 0.0f;
        mc = make_float2(-CUDART_INF_F, -CUDART_INF_F);  // running maxima (base-2 exponents) of columns 2 t4, + 1
        l = make_float2(0.0f, 0.0f);                     // sums over this lane's positions
        uint32_t d_exp = 103;                            // largest exponent of a V scale so far (2^-24 at least)
        f = __uint_as_float((127u + 16u + 24u) << 23);   // 2^16 / 2^(d_exp - 127): d f is at most 65504
        // SPLIT_N: columns 0-3 take p d rounded to fp16, columns 4-7 the rest, 2^11 times as large, as without the
        // factor it would end at fp16's 2^-24, a part of 2^-40 of the largest
        const float2 low_scale = t4 >= 2 ? make_float2(2048.0f, 2048.0f) : make_float2(1.0f, 1.0f);
        const unsigned short low_take = t4 >= 2 ? 0xe800 : 0;  // -2048, 0

        // adds the earlier chains' sums to the accumulators
        float2 chain_m = mc;   // mc and f at the end of the last chain
        float chain_f = 0.0f;  // 0: none yet
        float4* chain = p.chains + ((size_t)blockIdx.x * FQ_WARPS + warp) * (HD / 16) * 32 + lane;
        auto add_chains = [&]() {
            if (chain_f == 0.0f) return;
            const float ratio = f / chain_f;  // powers of two
            const float ax = chain_m.x == -CUDART_INF_F ? 0.0f : ex2(chain_m.x - mc.x) * ratio;
            const float ay = chain_m.y == -CUDART_INF_F ? 0.0f : ex2(chain_m.y - mc.y) * ratio;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                const float4 v = chain[i * 32];
                float* c = o[i / 2][i & 1];
                c[0] += v.x * ax;
                c[1] += v.y * ay;
                c[2] += v.z * ax;
                c[3] += v.w * ay;
            }
        };
        // T stages from position t0 on in ring buffers buf ..; WHOLE: every column sees all of them.
        auto stage = [&](int t0, int buf, auto t_tag, auto whole_tag) {
            constexpr int T = decltype(t_tag)::value;
            constexpr bool WHOLE = decltype(whole_tag)::value;
            const unsigned char* ring = sm.ring[warp][buf];
            // ---- scores: lane (g4, t4) gets columns 2 t4, + 1 of positions 8 i + g4 ----
            float2 s[4 * T];
#pragma unroll
            for (int j = 0; j < 2 * T; j++) {
                const unsigned char* kc = ring + (j >> 1) * STAGE_BYTES;
                const unsigned char* ks = kc + 2 * CODE_BYTES;
                uint32_t w[2][NB], ds[2][NB / 2];  // codes and scales of positions 16 j + g4 and + 8
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int row = 16 * (j & 1) + 8 * hf + g4;
                    if (NB == 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(kc + row * 64 + t4 * 16);
                        const uint2 y = *reinterpret_cast<const uint2*>(ks + row * 8);
                        w[hf][0] = v.x; w[hf][1] = v.y; w[hf][2 % NB] = v.z; w[hf][3 % NB] = v.w;
                        ds[hf][0] = y.x; ds[hf][1 % (NB / 2)] = y.y;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(kc + row * 32 + t4 * 8);
                        w[hf][0] = v.x; w[hf][1] = v.y;
                        ds[hf][0] = *reinterpret_cast<const uint32_t*>(ks + row * 4);
                    }
                }
                float2 a = make_float2(0.0f, 0.0f), c8 = a;
#pragma unroll
                for (int blk = 0; blk < NB; blk++) {
                    const uint32_t w0 = w[0][blk], w1 = w[1][blk], x0 = w0 >> 8, x1 = w1 >> 8;
                    const uint32_t a0 = value_low(w0), a1 = value_low(w1), a2 = value_high(w0), a3 = value_high(w1);
                    const uint32_t e0 = value_low(x0), e1 = value_low(x1), e2 = value_high(x0), e3 = value_high(x1);
                    float cc[4];
                    mma16816_first(cc, a0, a1, a2, a3, qh[blk][0], qh[blk][1]);
                    mma16816(cc, e0, e1, e2, e3, qh[blk][2], qh[blk][3]);
                    if (!SPLIT_N) {
                        const uint32_t* lo = ql[blk % (SPLIT_N ? 1 : NB)];
                        mma16816(cc, a0, a1, a2, a3, lo[0], lo[1]);
                        mma16816(cc, e0, e1, e2, e3, lo[2], lo[3]);
                    }
                    const float d0 = blk & 1 ? half_hi(ds[0][blk / 2]) : half_lo(ds[0][blk / 2]);
                    const float d1 = blk & 1 ? half_hi(ds[1][blk / 2]) : half_lo(ds[1][blk / 2]);
                    a = fma2(make_float2(d0, d0), make_float2(cc[0], cc[1]), a);
                    c8 = fma2(make_float2(d1, d1), make_float2(cc[2], cc[3]), c8);
                }
                s[2 * j] = a;
                s[2 * j + 1] = c8;
            }
            uint32_t top = 0;  // magnitude bits of the V scales of the positions `lane` of the stages
#pragma unroll
            for (int i = 0; i < T; i++) {
                const unsigned char* vs = ring + i * STAGE_BYTES + 2 * CODE_BYTES + SCALE_BYTES;
                uint32_t v;
                if (NB == 4) {
                    const uint2 y = *reinterpret_cast<const uint2*>(vs + lane * 8);
                    v = hmax_abs2(y.x, y.y);
                } else {
                    v = *reinterpret_cast<const uint32_t*>(vs + lane * 4);
                }
                if (!WHOLE && (t0 + lane < any_lo || t0 + lane >= any_hi)) v = 0;  // what no column sees may hold anything
                top = hmax_abs2(top, v);
            }
            top &= 0x7fff7fffu;
            top = max(top >> 16, top & 0xffffu);
#pragma unroll
            for (int i = 0; i < 4 * T; i++) {
                if (SPLIT_N) {  // q's two parts
                    s[i].x += __shfl_xor_sync(0xffffffffu, s[i].x, 2);
                    s[i].y += __shfl_xor_sync(0xffffffffu, s[i].y, 2);
                }
                if (!WHOLE) {
                    const int t = t0 + 8 * i + g4;
                    if (t < c_lo[0] || t >= c_hi[0]) s[i].x = -CUDART_INF_F;
                    if (t < c_lo[1] || t >= c_hi[1]) s[i].y = -CUDART_INF_F;
                }
            }
            // ---- running maxima and V scale exponent ----
            // Once no lane has a larger score, as in most stages, nothing has to be reduced over the lanes.
            float2 m_new = s[0];
#pragma unroll
            for (int i = 1; i < 4 * T; i++) m_new = make_float2(fmaxf(m_new.x, s[i].x), fmaxf(m_new.y, s[i].y));
            // fp16 exponent field e: scales below 2^(e - 14); e = 0 for zeros and subnormals
            uint32_t need = (top >> 10) + 113u;  // 127 - 14
            if (__any_sync(0xffffffffu, m_new.x * q_mul.x > mc.x || m_new.y * q_mul.y > mc.y ||
                                            need > d_exp)) {
                // A scale that is not finite does not count, or the other blocks would lose digits with it. Lanes whose
                // position no column sees have top = 0.
                if (__any_sync(0xffffffffu, top >= 0x7c00u)) {
                    uint32_t finite = 113u;
#pragma unroll
                    for (int i = 0; i < T; i++)
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            const unsigned char* vs = ring + i * STAGE_BYTES + 2 * CODE_BYTES + SCALE_BYTES;
                            const uint32_t e = *reinterpret_cast<const uint16_t*>(vs + lane * (2 * NB) + 2 * j) >> 10 & 31u;
                            finite = max(finite, e < 31u ? e + 113u : 0u);
                        }
                    if (top >= 0x7c00u) need = finite;
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    m_new.x = fmaxf(m_new.x, __shfl_xor_sync(0xffffffffu, m_new.x, d));
                    m_new.y = fmaxf(m_new.y, __shfl_xor_sync(0xffffffffu, m_new.y, d));
                }
                m_new = make_float2(fmaxf(mc.x, m_new.x * q_mul.x), fmaxf(mc.y, m_new.y * q_mul.y));
                float2 alpha = make_float2(ex2(mc.x - (m_new.x == -CUDART_INF_F ? 0.0f : m_new.x)),
                                           ex2(mc.y - (m_new.y == -CUDART_INF_F ? 0.0f : m_new.y)));
                mc = m_new;
                l = mul2(l, alpha);
                const uint32_t e_new = max(d_exp, (uint32_t)__reduce_max_sync(0xffffffffu, need));
                const float f_new = __uint_as_float((127u + 16u + 127u - e_new) << 23);
                const float ratio = __uint_as_float((127u + d_exp - e_new) << 23);  // a power of two: f_new / f
                d_exp = e_new;
                f = f_new;
                alpha = mul2(alpha, make_float2(ratio, ratio));
#pragma unroll
                for (int i = 0; i < NB; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        o[i][j][0] *= alpha.x;
                        o[i][j][1] *= alpha.y;
                        o[i][j][2] *= alpha.x;
                        o[i][j][3] *= alpha.y;
                    }
            }
            const float2 m_neg = make_float2(mc.x == -CUDART_INF_F ? 0.0f : -mc.x, mc.y == -CUDART_INF_F ? 0.0f : -mc.y);
#pragma unroll
            for (int i = 0; i < 4 * T; i++) {
                s[i] = fma2(s[i], q_mul, m_neg);
                s[i] = make_float2(ex2(s[i].x), ex2(s[i].y));
                l = add2(l, s[i]);
            }
            // ---- output: 16 positions at a time ----
#pragma unroll
            for (int j = 0; j < 2 * T; j++) {
                const unsigned char* vc = ring + (j >> 1) * STAGE_BYTES + CODE_BYTES;
                const unsigned char* vs = vc + CODE_BYTES + SCALE_BYTES;
                uint32_t wa[2][NB];  // [positions 2 t4, + 1 / 8 + 2 t4, + 1][codes of the first, of the second]
                uint32_t ds[2][NB / 2];  // scales of positions 16 j + g4 and + 8
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int pair = 8 * (j & 1) + 4 * hf + t4, row = 16 * (j & 1) + 8 * hf + g4;
                    if (NB == 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(vc + pair * 128 + g4 * 16);
                        const uint2 y = *reinterpret_cast<const uint2*>(vs + row * 8);
                        wa[hf][0] = v.x; wa[hf][1] = v.y; wa[hf][2 % NB] = v.z; wa[hf][3 % NB] = v.w;
                        ds[hf][0] = y.x; ds[hf][1 % (NB / 2)] = y.y;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(vc + pair * 64 + g4 * 8);
                        wa[hf][0] = v.x; wa[hf][1] = v.y;
                        ds[hf][0] = *reinterpret_cast<const uint32_t*>(vs + row * 4);
                    }
                }
                float2 pf[2];
#pragma unroll
                for (int hf = 0; hf < 2; hf++) pf[hf] = make_float2(s[2 * j + hf].x * f, s[2 * j + hf].y * f);
#pragma unroll
                for (int blk = 0; blk < NB; blk++) {
                    uint32_t bh[2], bl[2];
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const float d = blk & 1 ? half_hi(ds[hf][blk / 2]) : half_lo(ds[hf][blk / 2]);
                        float2 pd = make_float2(pf[hf].x * d, pf[hf].y * d);
                        if (!WHOLE) {  // a position the column does not see adds nothing, were its scale NaN
                            if (pf[hf].x == 0.0f) pd.x = 0.0f;
                            if (pf[hf].y == 0.0f) pd.y = 0.0f;
                        }
                        if (SPLIT_N) {
                            const uint32_t hi = pack_rn(pd.x, pd.y);
                            const float2 r = fma_half(hi, low_take, mul2(pd, low_scale));
                            bh[hf] = transpose8(pack_rn(r.x, r.y));
                        } else {
                            const uint32_t hi = pack_rn(pd.x, pd.y);
                            const float2 t = make_float2(half_lo(hi), half_hi(hi));
                            const float2 r = mul2(fma2(t, make_float2(-1.0f, -1.0f), pd), make_float2(2048.0f, 2048.0f));
                            bh[hf] = transpose8(hi);
                            bl[hf] = transpose8(pack_rn(r.x, r.y));
                        }
                    }
                    const uint32_t sel = blk & 1 ? 0x7632u : 0x5410u;
                    const uint32_t x = __byte_perm(wa[0][blk / 2], wa[0][NB / 2 + blk / 2], sel);
                    const uint32_t y = __byte_perm(wa[1][blk / 2], wa[1][NB / 2 + blk / 2], sel);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t xs = e ? x >> 8 : x, ys = e ? y >> 8 : y;
                        const uint32_t a0 = value_low(xs), a1 = value_high(xs), a2 = value_low(ys), a3 = value_high(ys);
                        mma16816(o[blk][e], a0, a1, a2, a3, bh[0], bh[1]);
                        if (!SPLIT_N) {  // the low part is 2^11 times as large against codes 2^-11 as large
                            constexpr uint32_t S = 0x10001000u;
                            mma16816(o[blk][e], hmul2(a0, S), hmul2(a1, S), hmul2(a2, S), hmul2(a3, S), bl[0], bl[1]);
                        }
                    }
                }
            }
        };

        for (int k = 0, buf = 0; k < n; k += GROUP) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();  // every lane's copies are there
            const int t0 = t_first + k * FQ_STAGE;
            const bool whole = t0 >= full_lo && t0 + GROUP * FQ_STAGE <= full_hi && (staged >> buf & (1u << GROUP) - 1) == (1u << GROUP) - 1;
            if (whole) {
                stage(t0, buf, std::integral_constant<int, GROUP>{}, std::true_type{});
            } else {
#pragma unroll 1
                for (int i = 0; i < GROUP; i++)
                    if (staged >> (buf + i) & 1u)
                        stage(t0 + i * FQ_STAGE, buf + i, std::integral_constant<int, 1>{}, std::false_type{});
            }
            staged &= ~(((1u << GROUP) - 1) << buf);
            __syncwarp();  // the buffers' reads are done in every lane
            issue(k + FQ_RING, buf);
            buf = buf ? 0 : GROUP;
            if ((k + GROUP) % fq_chain<HD, SPLIT_N>() == 0 && k + GROUP < n) {
                add_chains();
#pragma unroll
                for (int i = 0; i < 2 * NB; i++) {
                    float* c = o[i / 2][i & 1];
                    chain[i * 32] = make_float4(c[0], c[1], c[2], c[3]);
                    c[0] = c[1] = c[2] = c[3] = 0.0f;
                }
                chain_m = mc;
                chain_f = f;
            }
        }
        add_chains();

        // ---- the segment's result: lane (g4, t4) holds columns 2 t4, + 1, dimensions 32 i + 4 g4 .. + 3 ----
        if (SPLIT_N) {  // columns 4-7 hold the low parts of 0-3, times 2^11
            const float unit = t4 >= 2 ? 1.0f / 2048.0f : 1.0f;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        o[i][j][k] *= unit;
                        o[i][j][k] += __shfl_xor_sync(0xffffffffu, o[i][j][k], 2);
                    }
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l.x += __shfl_xor_sync(0xffffffffu, l.x, d);
            l.y += __shfl_xor_sync(0xffffffffu, l.y, d);
        }
        f = 512.0f / f;  // the codes' unit is 2^-9
        if (tail.n > 1) break;  // joined below
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int col = 2 * t4 + j;
            if (col >= cols) continue;
            // a row that sees nothing gives zeros; without weights because its scores overflowed, NaN
            const float lj = j ? l.y : l.x, w = lj == 0.0f && (j ? mc.y : mc.x) == -CUDART_INF_F ? 0.0f : f / lj;
            float* dst = fq_out(p, b, g, c, col, HD);
#pragma unroll
            for (int i = 0; i < NB; i++)
                *reinterpret_cast<float4*>(dst + 32 * i + 4 * g4) =
                    make_float4(o[i][0][j] * w, o[i][0][2 + j] * w, o[i][1][j] * w, o[i][1][2 + j] * w);
        }
        if (!many) break;
        item += (int)workers;
        b += item / (int)items_per_seq;
        item %= (int)items_per_seq;
    }
    pdl_launch_dependents();  // the next kernel's CTAs may take the SMs as they empty

    // ---- join the CTA's parts ----
    const bool joins = b >= 0 && tail.n > 1;
    if (lane == 0) sm.tail[warp] = joins ? tail : FqTail{-1, 0, 0, 0};
    __syncthreads();
    FqParts<HD>& pt = sm.parts;  // every stage is consumed: the ring's space takes the parts
    if (joins) {
        if (g4 == 0) {
            *reinterpret_cast<float2*>(&pt.m[warp][2 * t4]) = mc;
            *reinterpret_cast<float2*>(&pt.l[warp][2 * t4]) = l;
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < NB; i++)
                *reinterpret_cast<float4*>(&pt.o[warp][2 * t4 + j][32 * i + 4 * g4]) =
                    make_float4(o[i][0][j] * f, o[i][0][2 + j] * f, o[i][1][j] * f, o[i][1][2 + j] * f);
    }
    __syncthreads();
    // the items that other CTAs have a part in: 0 begins in an earlier CTA, 1 ends in a later one
    FqTail shared_tail[2];
    shared_tail[0].w0 = shared_tail[1].w0 = -1;
    const int key = lane < FQ_WARPS ? sm.tail[lane].w0 : -1;
    for (uint32_t left = __ballot_sync(0xffffffffu, key >= 0); left;) {  // an item of the CTA's at a time
        const int e0 = __ffs(left) - 1;
        const uint32_t set = __ballot_sync(0xffffffffu, key == __shfl_sync(0xffffffffu, key, e0));
        const int e1 = e0 + __popc(set);
        left &= ~set;
        const FqTail t = sm.tail[e0];
        int g = t.item, c = 0;
        if (p.tiles > 1) {
            g = t.item / p.tiles;
            c = t.item % p.tiles;
        }
        const int cols = min(FQ_COLS, p.rows * p.G - c * FQ_COLS);
        const bool before = t.w0 < (int)blockIdx.x * FQ_WARPS, after = t.w0 + t.n > ((int)blockIdx.x + 1) * FQ_WARPS;
        if (before) shared_tail[0] = t;
        else if (after) shared_tail[1] = t;
        float* dst = p.part + ((size_t)2 * blockIdx.x + (before ? 0 : 1)) * PF;
        for (int i = tid; i < cols * (HD / 4); i += FQ_THREADS) {
            const int col = i / (HD / 4), d = 4 * (i % (HD / 4));
            float M = -CUDART_INF_F;
            for (int e = e0; e < e1; e++) M = fmaxf(M, pt.m[e][col]);
            const float M0 = M == -CUDART_INF_F ? 0.0f : M;
            float L = 0.0f;
            float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int e = e0; e < e1; e++) {
                const float w = ex2(pt.m[e][col] - M0);
                const float4 v = *reinterpret_cast<const float4*>(&pt.o[e][col][d]);
                L += pt.l[e][col] * w;
                r.x += v.x * w; r.y += v.y * w; r.z += v.z * w; r.w += v.w * w;
            }
            if (!before && !after) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                *reinterpret_cast<float4*>(fq_out(p, t.b, g, c, col, HD) + d) =
                    make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
            } else {
                *reinterpret_cast<float4*>(dst + col * HD + d) = r;
                if (d == 0) {
                    dst[FQ_COLS * HD + col] = M;
                    dst[FQ_COLS * HD + FQ_COLS + col] = L;
                }
            }
        }
    }
    if (shared_tail[0].w0 < 0 && shared_tail[1].w0 < 0) return;
    // ---- the last CTA to arrive with a part of an item joins all of them ----
    __threadfence();
    __syncthreads();
    if (tid < 2) {
        const FqTail t = tid ? shared_tail[1] : shared_tail[0];
        int last = 0;
        if (t.w0 >= 0) {
            int* counter = p.counters + (size_t)t.b * items_per_seq + t.item;
            last = atomicAdd(counter, 1) == (t.w0 + t.n - 1) / FQ_WARPS - t.w0 / FQ_WARPS;
            if (last) *counter = 0;
        }
        sm.last[tid] = last;
    }
    __syncthreads();
    // half of the threads for each of the two items
    const int half = tid >= FQ_THREADS / 2;
    if (!sm.last[half]) return;
    __threadfence();
    const FqTail t = half ? shared_tail[1] : shared_tail[0];
    int g = t.item, c = 0;
    if (p.tiles > 1) {
        g = t.item / p.tiles;
        c = t.item % p.tiles;
    }
    const int c_first = t.w0 / FQ_WARPS, c_last = (t.w0 + t.n - 1) / FQ_WARPS;
    fq_join<HD>(p, t.b, g, c, min(FQ_COLS, p.rows * p.G - c * FQ_COLS), c_last - c_first + 1,
                p.part + ((size_t)2 * c_first + 1) * PF, p.part + (size_t)2 * c_first * PF);
}

static int fq_grid(long long max_units) {
    return (int)std::min<long long>((max_units + FQ_WARPS - 1) / FQ_WARPS, (long long)sm_count() * FQ_CTAS_PER_SM);
}

template <int HD, bool SPLIT_N>
static int launch_fq(const FqParams& p, int grid, cudaStream_t st) {
    auto kern = vsl_flash_decode_q4_kernel<HD, SPLIT_N>;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(FqSmem<HD, SPLIT_N>));
        if (e != cudaSuccess) return launch_status(e, "flash_decode_q4 smem attribute");
        configured_dev = dev;
    }
    return launch_status(launch_k(kern, dim3(grid), dim3(FQ_THREADS), sizeof(FqSmem<HD, SPLIT_N>), st, p), "flash_decode_q4 launch");
}

// Workspace: the partial results and chains (sizes that depend on the device alone), then the counters, so
// calls of different shapes find every counter that another shape left at zero.
static size_t fq_part_bytes() {
    return ((size_t)2 * sm_count() * FQ_CTAS_PER_SM * fq_part_floats<128>() * sizeof(float) + 255) & ~(size_t)255;
}
static size_t fq_chain_bytes() { return (size_t)sm_count() * FQ_CTAS_PER_SM * FQ_WARPS * (128 / 16) * 32 * sizeof(float4); }
static int fq_tiles(int rows, int n_heads, int n_kv) {
    return (int)(((long long)rows * (n_heads / n_kv) + FQ_COLS - 1) / FQ_COLS);
}
static size_t fq_scratch_bytes() { return std::max(fq_part_bytes() + fq_chain_bytes(), fc_part_bytes()); }
static size_t fq_workspace(int B, int rows, int n_heads, int n_kv) {
    const size_t counters = std::max((size_t)B * n_kv * fq_tiles(rows, n_heads, n_kv), (size_t)sm_count());
    return fq_scratch_bytes() + ((counters * sizeof(int) + 255) & ~(size_t)255);
}
static int fq_check_shape(const char* what, int B, int rows, int n_heads, int n_kv, int head_dim) {
    if (B <= 0 || rows <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv)
        return set_error(VSL_ERR_INVALID, "%s: %d sequences of %d rows, %d heads over %d KV heads", what, B, rows, n_heads,
                         n_kv);
    if (B > FQ_MAX_BATCH || rows > 65536 || n_heads > 4096)
        return set_error(VSL_ERR_UNSUPPORTED, "%s: %d sequences of %d rows, %d heads (at most %d, 65536, 4096)", what, B,
                         rows, n_heads, FQ_MAX_BATCH);
    if (head_dim != 64 && head_dim != 128)
        return set_error(VSL_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128 supported)", what, head_dim);
    return VSL_OK;
}

int flash_decode_q4_impl(const float* q, const void* k_cache, const void* v_cache, int n_pages,
                         const int32_t* page_table, int max_pages, int page_size, const int32_t* pos, int B, int rows,
                         int n_heads, int n_kv, int head_dim, float* out, void* workspace, size_t workspace_bytes,
                         const SparseMask* sparse, int* status, cudaStream_t st) {
    if (!q || !k_cache || !v_cache || !page_table || !pos || !out || !workspace)
        return set_error(VSL_ERR_INVALID, "flash_decode_q4: null pointer");
    if (int rc = fq_check_shape("flash_decode_q4", B, rows, n_heads, n_kv, head_dim)) return rc;
    if (n_pages <= 0 || max_pages <= 0 || page_size <= 0 || page_size % 64)
        return set_error(VSL_ERR_INVALID, "flash_decode_q4: %d pages, %d per sequence, page_size %d (a multiple of 64)",
                         n_pages, max_pages, page_size);
    if ((long long)max_pages * page_size > (1 << 30))
        return set_error(VSL_ERR_UNSUPPORTED, "flash_decode_q4: %d pages of %d positions (at most 2^30 positions)",
                         max_pages, page_size);
    if (sparse && sparse->min_len > 0 && (sparse->window < 0 || sparse->global_tokens < 0 || sparse->block <= 0))
        return set_error(VSL_ERR_INVALID, "flash_decode_q4: sparse mask window %d, global %d, block %d", sparse->window,
                         sparse->global_tokens, sparse->block);
    for (const void* a : {(const void*)q, k_cache, v_cache, (const void*)out, (const void*)workspace})
        if ((uintptr_t)a & 15) return set_error(VSL_ERR_INVALID, "flash_decode_q4: arrays must be 16-byte aligned");
    if (n_kv * kv_head_page_bytes(VSL_Q4_0, head_dim, page_size) >= ((size_t)1 << 31))
        return set_error(VSL_ERR_UNSUPPORTED, "flash_decode_q4: pages of %d positions and %d KV heads pass 2 GiB", page_size,
                         n_kv);
    const size_t need = fq_workspace(B, rows, n_heads, n_kv);
    if (workspace_bytes < need)
        return set_error(VSL_ERR_INVALID, "flash_decode_q4: workspace %zu bytes < %zu", workspace_bytes, need);
    FqParams p = {};
    p.q = q;
    p.k_cache = static_cast<const unsigned char*>(k_cache);
    p.v_cache = static_cast<const unsigned char*>(v_cache);
    p.n_pages = n_pages; p.page_table = page_table; p.max_pages = max_pages; p.page_size = page_size;
    p.pos = pos; p.B = B; p.rows = rows; p.n_heads = n_heads; p.n_kv = n_kv; p.G = n_heads / n_kv;
    p.tiles = fq_tiles(rows, n_heads, n_kv);
    p.scale = 1.0f / sqrtf((float)head_dim);
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.chains = reinterpret_cast<float4*>(static_cast<char*>(workspace) + fq_part_bytes());
    p.counters = reinterpret_cast<int*>(static_cast<char*>(workspace) + fq_scratch_bytes());
    p.status = status;
    if (sparse) p.sp = *sparse;
    const long long units = ((long long)max_pages * page_size + FQ_STAGE - 1) / FQ_STAGE;
    if ((double)B * n_kv * p.tiles * units > 2e9)
        return set_error(VSL_ERR_UNSUPPORTED, "flash_decode_q4: %d sequences x %d KV heads x %d column tiles over %lld "
                         "positions is too much for one call", B, n_kv, p.tiles, (long long)max_pages * page_size);
    // From 48 columns per KV head on (80 at head_dim 64) the form for many rows, which unpacks once for all of them,
    // is faster. Few rows / many rows, in us, by columns: 32 / 8 heads of 128, 16 x 2048 positions: 32: 65.6 / 83,
    // 48: 128 / 75, 128: 315 / 80; 1 x 2048: 32: 15.4 / 18.5, 48: 16.0 / 16.0, 128: 22.1 / 19.8, 512: 63 / 28.5;
    // head_dim 64, 4 x 4000: 64: 36.2 / 40, 96: 53 / 35.7.
    if ((long long)rows * p.G >= (head_dim == 128 ? 48 : 80)) return fc_launch(p, head_dim, st);
    const int grid = fq_grid((long long)B * n_kv * p.tiles * units);
    const bool few = rows * p.G <= FQ_COLS / 2;
    if (head_dim == 128) return few ? launch_fq<128, true>(p, grid, st) : launch_fq<128, false>(p, grid, st);
    return few ? launch_fq<64, true>(p, grid, st) : launch_fq<64, false>(p, grid, st);
}

}  // namespace vsl

extern "C" int vsl_flash_decode_q4_workspace_size(int B, int rows, int n_heads, int n_kv, int head_dim, size_t* bytes) {
    if (!bytes) return vsl::set_error(VSL_ERR_INVALID, "flash_decode_q4_workspace_size: null pointer");
    if (int rc = vsl::fq_check_shape("flash_decode_q4_workspace_size", B, rows, n_heads, n_kv, head_dim)) return rc;
    *bytes = vsl::fq_workspace(B, rows, n_heads, n_kv);
    return VSL_OK;
}

extern "C" int vsl_flash_decode_q4(const float* q, const void* k_cache, const void* v_cache, int n_pages,
                                   const int32_t* page_table, int max_pages, int page_size, const int32_t* pos, int B,
                                   int rows, int n_heads, int n_kv, int head_dim, float* out, void* workspace,
                                   size_t workspace_bytes, const vsl_sparse_mask* mask, int* status, void* stream) {
    vsl::SparseMask m = {};
    if (mask && mask->min_len > 0) m = vsl::SparseMask{mask->min_len, mask->window, mask->global_tokens, mask->block};
    return vsl::flash_decode_q4_impl(q, k_cache, v_cache, n_pages, page_table, max_pages, page_size, pos, B, rows,
                                     n_heads, n_kv, head_dim, out, workspace, workspace_bytes, &m, status,
                                     (cudaStream_t)stream);
}
