// Key / value cache of 8 bits: rotary table, filling it from a prompt, and the attention of single tokens against it.
//
// Format (k44_decoder.cuh): blocks of 64 tokens of one column and head, e4m3 codes with one FP32 scale per block for keys and
// one for values,  scale = max(amax, 2^-24) / 448,  code = e4m3(x / scale);  infinities count as the largest FP16 number, a NaN
// stays a NaN of its own value. The open block is kept as FP16 rows, so that a scale is chosen once, with all 64 tokens known.
// A block is brought to 8 bits by the step that appends its last token and read in 8 bits from the next block on.
#include "k44_decoder.cuh"
#include "k44_ptx.cuh"

namespace k44b {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- rotary table ---------------------------------------------------------------------------------------------------------
__global__ void k44_rope_table_kernel(float2 *table, uint32_t positions, uint32_t half, double theta, int llama3) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (uint64_t)positions * half) return;
    const uint32_t pos = (uint32_t)(i / half), p = (uint32_t)(i % half);
    double f = exp((double)p * (-2.0 * log(theta) / (double)(2u * half)));
    if (llama3) {       // Llama-3 long-context frequency scaling, as in the other rotary commands
        const double ratio = 1303.7972938088068 * f;
        const double smooth = fmin(1.0, fmax(0.0, (ratio - 1.0) / 3.0));
        f = (1.0 - smooth) * (f * 0.03125) + smooth * f;
    }
    double s, c;
    sincos((double)pos * f, &s, &c);
    table[i] = make_float2((float)c, (float)s);
}

// one rotation, each product and sum rounded by itself: the same bits wherever a key is rotated
__device__ __forceinline__ void rotate(float &a, float &b, float2 cs) {
    const float x = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
    b = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
    a = x;
}

// ---- 8 bits -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float finite_abs(float x) { return fminf(fabsf(x), 65504.0f); }     // NaN -> 65504: see amax_of
// largest magnitude of the numbers among (m, x); a NaN does not count
__device__ __forceinline__ float amax_of(float m, float x) { return x != x ? m : fmaxf(m, finite_abs(x)); }
__device__ __forceinline__ float scale_of(float amax) { return __fdiv_rn(fmaxf(amax, 5.9604644775390625e-8f), 448.0f); }
// four values -> four codes, the first in the lowest byte; the conversion saturates at +-448
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * inv), "f"(a * inv));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * inv), "f"(c * inv));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// two codes (low 16 bits) -> two FP16 numbers, exactly: every e4m3 number is an FP16 number
__device__ __forceinline__ uint32_t from_codes(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
__device__ __forceinline__ float2 half2_of(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// ---- filling the cache from a prompt ----------------------------------------------------------------------------------------
// CTA = one block of 64 tokens of one sequence and head. Keys are rotated and rounded to FP16 first, then treated as the step
// by step path treats them. HBM-bound: 4 bytes read and 2 written per pair of key and value elements.
template <int D>
__global__ void __launch_bounds__(256) k44_kv8_fill_kernel(const Kv8FillArgs a) {
    dep_enter();
    constexpr int ROW = 64 + 8;                                      // padded row of 64 tokens (halves)
    __shared__ __align__(16) __half ks[D * ROW];
    __shared__ __align__(16) __half vs[D * ROW];
    __shared__ float red[2][8];
    const uint32_t block = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
    const int2 sl = a.sequences[seq];
    if (sl.x < 0) return;
    const uint32_t len = (uint32_t)sl.y;
    // a plan's tables are checked by the host; the cache's own limits are checked here as well
    if ((uint32_t)sl.x >= a.cache.columns || sl.y < 0 || len > a.cache.max_seq || len > a.seq_len || (uint64_t)seq * a.seq_len + len > a.columns) {
        if (tid == 0u) atomicOr(a.status, (uint32_t)ST_BAD_INDEX);
        return;
    }
    const uint64_t ch = (uint64_t)sl.x * a.cache.h_kv + h;
    if (block == 0u && tid == 0u) a.cache.tail_block[ch] = (len % kKv8Block) ? (int)(len / kKv8Block) : -1;
    const uint32_t t0 = block * kKv8Block;
    if (t0 >= len) return;
    const uint32_t n = min(kKv8Block, len - t0), col0 = seq * a.seq_len + t0;
    const __half *kg = a.k + (uint64_t)h * D * a.pitch + col0, *vg = a.v + (uint64_t)h * D * a.pitch + col0;
    if ((col0 & 7u) == 0u) {
        for (uint32_t e = tid; e < D * 8u; e += 256u) {              // 16-byte pieces; a piece that starts inside the row ends inside it
            const uint32_t d = e >> 3, c = (e & 7u) * 8u;
            uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
            if (c < n) {
                kk = __ldg(reinterpret_cast<const uint4 *>(kg + (uint64_t)d * a.pitch + c));
                vv = __ldg(reinterpret_cast<const uint4 *>(vg + (uint64_t)d * a.pitch + c));
            }
            *reinterpret_cast<uint4 *>(ks + d * ROW + c) = kk;
            *reinterpret_cast<uint4 *>(vs + d * ROW + c) = vv;
        }
    } else {                                                         // sequences that do not start on a 16-byte boundary
        for (uint32_t e = tid; e < D * 64u; e += 256u) {
            const uint32_t d = e >> 6, c = e & 63u;
            ks[d * ROW + c] = c < n ? kg[(uint64_t)d * a.pitch + c] : __half(0.f);
            vs[d * ROW + c] = c < n ? vg[(uint64_t)d * a.pitch + c] : __half(0.f);
        }
    }
    __syncthreads();
    // rotate: a thread owns one token and every fourth pair
    const uint32_t tok = tid & 63u, part = tid >> 6;
    float kmax = 0.f, vmax = 0.f;
    if (tok < n) {
        const float2 *cs = a.rope + (uint64_t)(t0 + tok) * (D / 2);
#pragma unroll 4
        for (uint32_t p = part; p < D / 2; p += 4u) {
            float x = __half2float(ks[p * ROW + tok]), y = __half2float(ks[(p + D / 2) * ROW + tok]);
            rotate(x, y, __ldg(cs + p));
            const __half hx = __float2half_rn(x), hy = __float2half_rn(y);
            ks[p * ROW + tok] = hx;
            ks[(p + D / 2) * ROW + tok] = hy;
            kmax = amax_of(amax_of(kmax, __half2float(hx)), __half2float(hy));
            vmax = amax_of(amax_of(vmax, __half2float(vs[p * ROW + tok])), __half2float(vs[(p + D / 2) * ROW + tok]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
    }
    if ((tid & 31u) == 0u) { red[0][tid >> 5] = kmax; red[1][tid >> 5] = vmax; }
    __syncthreads();
    if (n == kKv8Block) {                                            // a whole block: 8 bits
#pragma unroll
        for (int w = 0; w < 8; ++w) { kmax = fmaxf(kmax, red[0][w]); vmax = fmaxf(vmax, red[1][w]); }
        const float ksc = scale_of(kmax), vsc = scale_of(vmax), ki = 1.0f / ksc, vi = 1.0f / vsc;
        uint8_t *codes = a.cache.codes + (ch * a.cache.blocks + block) * (2u * kKv8Block * D);
        if (tid == 0u) a.cache.scales[ch * a.cache.blocks + block] = make_float2(ksc, vsc);
        for (uint32_t e = tid; e < 64u * D / 16u; e += 256u) {        // 16 codes of a key: 16 dimensions of one token
            const uint32_t t = e & 63u, d0 = (e >> 6) * 16u;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half *x = ks + (d0 + 4 * i) * ROW + t;
                w[i] = codes4(__half2float(x[0]), __half2float(x[ROW]), __half2float(x[2 * ROW]), __half2float(x[3 * ROW]), ki);
            }
            *reinterpret_cast<uint4 *>(codes + (d0 >> 6) * 4096u + t * 64u + (d0 & 63u)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        for (uint32_t e = tid; e < 64u * D / 16u; e += 256u) {        // 16 codes of a value: 16 tokens of one dimension
            const uint32_t d = e >> 2, c = (e & 3u) * 16u;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = half2_of(*reinterpret_cast<const uint32_t *>(vs + d * ROW + c + 4 * i)), y = half2_of(*reinterpret_cast<const uint32_t *>(vs + d * ROW + c + 4 * i + 2));
                w[i] = codes4(x.x, x.y, y.x, y.y, vi);
            }
            *reinterpret_cast<uint4 *>(codes + kKv8Block * D + d * 64u + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {                                                         // the open block: FP16 rows; rows behind the last token stay as they were
        __half *kt = a.cache.k_tail + ch * (kKv8Block * D), *vt = a.cache.v_tail + ch * (kKv8Block * D);
        for (uint32_t e = tid; e < n * D; e += 256u) { const uint32_t t = e / D, d = e % D; kt[t * D + d] = ks[d * ROW + t]; }
        for (uint32_t e = tid; e < 64u * D; e += 256u) { const uint32_t d = e >> 6, c = e & 63u; if (c < n) vt[d * 64u + c] = vs[d * ROW + c]; }
    }
}

// ---- single tokens against the cache -------------------------------------------------------------------------------------------
// o = sum_t softmax_t(q . k_t / sqrt(D)) v_t over the visible positions t of a column, for the group of query heads that share
// one key / value head, so that every code is read once. Memory-bound: 2 D bytes per position and key / value head.
//
// Work: a unit is one visible 8-bit block of one (column, head), or its open block with the new token. All units in a row
// (column, head, block) are cut into equal shares, one per warp of the grid, whatever the columns' lengths; a warp that holds
// a (column, head) whole writes its output, the others leave (accumulator, maximum, sum) and the last one to arrive adds the
// parts in the order of the warps, so that the result does not depend on the order of arrival.
// Loads: a block is 2 * 64 * D contiguous bytes; each warp keeps a ring of them in flight with bulk copies.
// Products on mma.sync: 8 (or 16) query heads are the rows of m16n8k16 — tcgen05 would need 64 rows and its operands as FP16
// in shared memory, for a kernel that waits for HBM. Keys: a lane takes 16 consecutive dimensions of one token (16 bytes),
// values: 16 consecutive tokens of one dimension; which logical k index they stand for is free as long as the other operand
// agrees, so codes go from shared memory to the operand registers without a shuffle: token of score tile i, column 2 j + e =
// 16 j + 2 i + e, and the scores' accumulator layout is the second product's A operand as it stands.
// The values' scale is folded into the exponent (p' = p * scale): p' <= 1 is what is rounded to FP16, and the sum uses p' / scale.
// q is split into two FP16 numbers (high and low part): with exact codes the scores are then as good as in 32 bits.
constexpr uint32_t kWarps64 = 8, kWarps128 = 4, kStages = 3;

__device__ __forceinline__ void mma16816(float &c0, float &c1, float &c2, float &c3, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c0), "+f"(c1), "+f"(c2), "+f"(c3) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// what a column's token sees: 8-bit blocks [0, sink_blocks) and [from, open), and the open block
struct Seen {
    uint32_t sink_blocks, from, open, units;
};
__device__ __forceinline__ Seen seen_of(int pos, uint32_t window, uint32_t sinks) {
    Seen s;
    s.open = (uint32_t)pos / kKv8Block;
    s.from = 0u; s.sink_blocks = 0u;
    if (window && (uint32_t)pos >= window) {
        s.from = ((uint32_t)pos - window + 1u) / kKv8Block;
        s.sink_blocks = min(s.from, (uint32_t)(((uint64_t)sinks + kKv8Block - 1u) / kKv8Block));
    }
    s.units = s.sink_blocks + (s.open - s.from) + 1u;
    return s;
}

template <int D, int WARPS, bool WIDE>           // WIDE: 9 to 16 query heads per key / value head
__global__ void __launch_bounds__(WARPS * 32, 1) k44_kv8_attn_kernel(const Kv8AttnArgs a) {
    constexpr int DT = D / 8, KS = D / 16, HF = D / 64, R = WIDE ? 2 : 1;      // dimension tiles, k steps, halves, row sets
    constexpr uint32_t BLK = 2u * kKv8Block * D, GP = 8u * R, PROW = D + 2u;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[WARPS * kStages];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, j = lane & 3u;
    const uint32_t H = a.cache.h_kv, G = a.h_q / H, C = a.columns;
    uint32_t *prefix = reinterpret_cast<uint32_t *>(smem_raw + WARPS * kStages * BLK);      // [C + 1] units before a column
    const uint32_t ring = ptx::smem_addr(smem_raw) + warp * kStages * BLK;
    const uint32_t bar0 = ptx::smem_addr(bars) + warp * kStages * 8u;
    if (lane == 0u) {
        for (uint32_t s = 0; s < kStages; ++s) ptx::mbar_init(bar0 + 8u * s, 1);
        ptx::fence_mbar_init();
    }
    dep_enter();
    // ---- units before each column ----
    auto pos_of = [&](uint32_t c) -> int {
        const int p = a.positions[c];
        return p >= 0 && (uint32_t)p < a.cache.max_seq ? p : -1;
    };
    for (uint32_t c = threadIdx.x; c < C; c += WARPS * 32u) {
        const int p = pos_of(c);
        if (p < 0 && a.positions[c] >= 0 && blockIdx.x == 0u) atomicOr(a.status, (uint32_t)ST_BAD_INDEX);
        prefix[c + 1u] = H * (p < 0 ? 1u : seen_of(p, a.window, a.sinks).units);
    }
    __syncthreads();
    if (warp == 0u) {
        uint32_t base = 0;
        for (uint32_t c0 = 0; c0 < C; c0 += 32u) {
            uint32_t v = c0 + lane < C ? prefix[c0 + lane + 1u] : 0u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const uint32_t n = __shfl_up_sync(0xffffffffu, v, o); if (lane >= (uint32_t)o) v += n; }
            if (c0 + lane < C) prefix[c0 + lane + 1u] = base + v;
            base += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0u) prefix[0] = 0u;
    }
    __syncthreads();
    const uint32_t total = prefix[C];
    const uint32_t workers = min(gridDim.x * WARPS, total), me = warp * gridDim.x + blockIdx.x;       // neighbours sit on different SMs
    if (me >= workers) return;
    auto share = [&](uint32_t w) -> uint32_t { return (uint32_t)((uint64_t)w * total / workers); };
    auto worker_of = [&](uint32_t u) -> uint32_t { return (uint32_t)((((uint64_t)u + 1u) * workers - 1u) / total); };
    const uint32_t u_begin = share(me), u_end = share(me + 1u);
    uint32_t col = 0;                                                        // the column that holds u_begin
    {
        uint32_t lo = 0, hi = C - 1u;
        while (lo < hi) { const uint32_t mid = (lo + hi + 1u) >> 1; if (prefix[mid] <= u_begin) lo = mid; else hi = mid - 1u; }
        col = lo;
    }
    // ---- the ring's own walk over this warp's 8-bit blocks, ahead of the one below ----
    uint32_t iu = u_begin, icol = col, ihead = 0, iper = 1, iat = 0, issued = 0;
    Seen iseen = {};
    int ipos = -1;
    auto enter_issue = [&]() {
        ipos = pos_of(icol);
        iseen = ipos < 0 ? Seen{0u, 0u, 0u, 1u} : seen_of(ipos, a.window, a.sinks);
        iper = iseen.units;
    };
    enter_issue();
    { const uint32_t rem = iu - prefix[icol]; ihead = rem / iper; iat = rem % iper; }
    const uint64_t policy = ptx::policy_evict_first();
    auto issue_next = [&]() {                                                 // lane 0 only; next 8-bit block into the next stage
        while (iu < u_end) {
            const bool block8 = iat + 1u < iper;
            const uint32_t b = iat < iseen.sink_blocks ? iat : iseen.from + (iat - iseen.sink_blocks);
            const uint64_t ch = (uint64_t)icol * H + ihead;
            ++iu; ++iat;
            const bool wrap = iat == iper;
            if (block8) {
                const uint32_t st = issued % kStages;
                ptx::mbar_arrive_expect_tx(bar0 + 8u * st, BLK);
                ptx::bulk_g2s(ring + st * BLK, a.cache.codes + (ch * a.cache.blocks + b) * BLK, BLK, bar0 + 8u * st, policy);
                ++issued;
            }
            if (wrap) {
                iat = 0;
                if (++ihead == H) { ihead = 0; ++icol; if (iu < u_end) enter_issue(); }
            }
            if (block8) return;
        }
    };
    if (lane == 0u)
        for (uint32_t s = 0; s < kStages; ++s) issue_next();
    __syncwarp();

    const float sm = rsqrtf((float)D) * kLog2e;
    uint32_t u = u_begin, consumed = 0;
    bool ok = true;
    while (u < u_end && ok) {
        while (prefix[col + 1u] <= u) ++col;
        const int pos = pos_of(col);
        const Seen sn = pos < 0 ? Seen{0u, 0u, 0u, 1u} : seen_of(pos, a.window, a.sinks);
        const uint32_t rem = u - prefix[col], head = rem / sn.units, at0 = rem % sn.units;
        const uint32_t n_units = min(sn.units - at0, u_end - u);               // this warp's part of the (column, head)
        const uint32_t seg0 = prefix[col] + head * sn.units;
        const uint64_t ch = (uint64_t)col * H + head;
        if (pos < 0) {                                                          // idle column: zeros
            for (uint32_t e = lane; e < G * D; e += 32u) a.out[((uint64_t)head * G * D + e) * a.pitch + col] = __half(0.f);
            u += 1u;
            continue;
        }
        // ---- q of the group, rotated, as two FP16 operands ----
        uint32_t qh[R][KS][2], ql[R][KS][2];
        const float2 *cs = a.rope + (uint64_t)pos * (D / 2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t row = g + 8u * r;
            float x[HF][16];
#pragma unroll
            for (int f = 0; f < HF; ++f)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    x[f][e] = row < G ? __half2float(a.q[((uint64_t)(head * G + row) * D + 64u * f + 16u * j + e) * a.pitch + col]) : 0.f;
            if (HF == 2) {                                                      // pairs (d, d + 64): both halves of this lane
#pragma unroll
                for (int e = 0; e < 16; ++e) rotate(x[0][e], x[HF - 1][e], __ldg(cs + 16u * j + e));
            } else {                                                            // pairs (d, d + 32): lane j and lane j ^ 2
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float other = __shfl_xor_sync(0xffffffffu, x[0][e], 2);
                    float lo = j < 2u ? x[0][e] : other, hi = j < 2u ? other : x[0][e];
                    rotate(lo, hi, __ldg(cs + 16u * (j & 1u) + e));
                    x[0][e] = j < 2u ? lo : hi;
                }
            }
#pragma unroll
            for (int f = 0; f < HF; ++f)
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float x0 = x[f][4 * s + 2 * t], x1 = x[f][4 * s + 2 * t + 1];
                        const uint32_t hi = pack2(x0, x1);
                        const float2 hf = half2_of(hi);
                        qh[r][4 * f + s][t] = hi;
                        ql[r][4 * f + s][t] = pack2(x0 - hf.x, x1 - hf.y);
                    }
        }
        float acc[DT][2 * R], m[R], l[R];
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 2 * R; ++e) acc[t][e] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.f; }

        // scores -> weights of one block: masked, scaled, running maximum; p (FP16 operand) and l
        auto soften = [&](float (&s)[8][2 * R], uint32_t t_base, uint32_t t_end, float kscale, float vscale, bool edge, uint32_t (&p)[R][8]) {
            const float mul = kscale * sm, lv = log2f(vscale), rv = 1.0f / vscale;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = s[i][2 * r + e] * mul;
                        if (edge) {
                            const uint32_t t = t_base + 16u * j + 2u * i + e;
                            const bool vis = t < t_end && (a.window == 0u || t + a.window > (uint32_t)pos || t < a.sinks);
                            v = vis ? v : -INFINITY;
                        }
                        v += lv;
                        s[i][2 * r + e] = v;
                        mx = fmaxf(mx, v);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.f : mn, back = exp2f(m[r] - base);
                m[r] = mn;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p0 = exp2f(s[i][2 * r] - base), p1 = exp2f(s[i][2 * r + 1] - base);
                    sum += p0 + p1;
                    p[r][i] = pack2(p0, p1);
                }
                l[r] = fmaf(l[r], back, sum * rv);
#pragma unroll
                for (int t = 0; t < DT; ++t) { acc[t][2 * r] *= back; acc[t][2 * r + 1] *= back; }
            }
        };

        for (uint32_t i0 = 0; i0 < n_units && ok; ++i0) {
            const uint32_t at = at0 + i0;
            if (at + 1u < sn.units) {
                // ---- an 8-bit block ----
                const uint32_t b = at < sn.sink_blocks ? at : sn.from + (at - sn.sink_blocks);
                const float2 sc = __ldg(a.cache.scales + ch * a.cache.blocks + b);
                const uint32_t st = consumed % kStages, ph = (consumed / kStages) & 1u, src = ring + st * BLK;
                if (!ptx::mbar_try_wait(bar0 + 8u * st, ph)) {
                    const long long t0 = clock64();
                    while (ok && !ptx::mbar_try_wait(bar0 + 8u * st, ph)) ok = (unsigned long long)(clock64() - t0) < a.wait_cycles;
                }
                ok = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
                if (!ok) break;
                float s[8][2 * R];
                const uint32_t tok_row = 16u * (g >> 1) + (g & 1u);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float c0 = 0.f, c1 = 0.f, c2 = 0.f, c3 = 0.f;
#pragma unroll
                    for (int f = 0; f < HF; ++f) {
                        const uint4 kk = lds16(src + f * 4096u + (tok_row + 2u * i) * 64u + j * 16u);
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const uint32_t w = word(kk, t), b0 = from_codes(w), b1 = from_codes(w >> 16);
                            mma16816(c0, c1, c2, c3, qh[0][4 * f + t][0], WIDE ? qh[R - 1][4 * f + t][0] : 0u, qh[0][4 * f + t][1], WIDE ? qh[R - 1][4 * f + t][1] : 0u, b0, b1);
                            mma16816(c0, c1, c2, c3, ql[0][4 * f + t][0], WIDE ? ql[R - 1][4 * f + t][0] : 0u, ql[0][4 * f + t][1], WIDE ? ql[R - 1][4 * f + t][1] : 0u, b0, b1);
                        }
                    }
                    s[i][0] = c0; s[i][1] = c1;
                    if (WIDE) { s[i][2 * R - 2] = c2; s[i][2 * R - 1] = c3; }
                }
                const uint32_t t_base = b * kKv8Block;
                const bool edge = a.window != 0u && !(t_base + a.window > (uint32_t)pos || t_base + kKv8Block <= a.sinks);
                uint32_t p[R][8];
                soften(s, t_base, t_base + kKv8Block, sc.x, sc.y, edge, p);
                uint4 keep = make_uint4(~0u, ~0u, ~0u, ~0u);                     // a hidden token's codes become 0: its NaN must not count
                if (edge) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = 0u;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t t = t_base + 16u * j + 4u * i + e;
                            if (t + a.window > (uint32_t)pos || t < a.sinks) w[i] |= 0xffu << (8 * e);
                        }
                    }
                    keep = make_uint4(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    uint4 vv = lds16(src + kKv8Block * D + (8u * t + g) * 64u + j * 16u);
                    vv.x &= keep.x; vv.y &= keep.y; vv.z &= keep.z; vv.w &= keep.w;
                    float c2 = WIDE ? acc[t][2 * R - 2] : 0.f, c3 = WIDE ? acc[t][2 * R - 1] : 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t w = word(vv, k);
                        mma16816(acc[t][0], acc[t][1], c2, c3, p[0][2 * k], WIDE ? p[R - 1][2 * k] : 0u, p[0][2 * k + 1], WIDE ? p[R - 1][2 * k + 1] : 0u, from_codes(w), from_codes(w >> 16));
                    }
                    if (WIDE) { acc[t][2 * R - 2] = c2; acc[t][2 * R - 1] = c3; }
                }
                __syncwarp();
                ++consumed;
                if (lane == 0u) issue_next();
            } else {
                // ---- the open block: append the new token, then attend to its FP16 rows ----
                const uint32_t b = sn.open, slot = (uint32_t)pos % kKv8Block;
                __half *kt = a.cache.k_tail + ch * (kKv8Block * D), *vt = a.cache.v_tail + ch * (kKv8Block * D);
                uint8_t *codes = a.cache.codes + (ch * a.cache.blocks + b) * BLK;
                const bool other = a.cache.tail_block[ch] != (int)b;
                __syncwarp();
                if (other) {
                    if (slot != 0u) {                                            // back inside a block already in 8 bits: its rows start from those
                        const float2 sc = a.cache.scales[ch * a.cache.blocks + b];
                        for (uint32_t e = lane; e < 64u * D / 2u; e += 32u) {
                            const uint32_t k2 = e * 2u, t = (k2 >> 6) & 63u, d = (k2 >> 12) * 64u + (k2 & 63u);
                            const float2 x = half2_of(from_codes(*reinterpret_cast<const uint16_t *>(codes + k2)));
                            if (t < slot) *reinterpret_cast<uint32_t *>(kt + t * D + d) = pack2(x.x * sc.x, x.y * sc.x);
                            const float2 y = half2_of(from_codes(*reinterpret_cast<const uint16_t *>(codes + kKv8Block * D + k2)));
                            *reinterpret_cast<uint32_t *>(vt + k2) = pack2(y.x * sc.y, y.y * sc.y);
                        }
                    }
                    if (lane == 0u) a.cache.tail_block[ch] = (int)b;
                    __syncwarp();
                }
#pragma unroll
                for (uint32_t p0 = 0; p0 < D / 2; p0 += 32u) {
                    const uint32_t p = p0 + lane;
                    float x = __half2float(a.k[((uint64_t)head * D + p) * a.pitch + col]), y = __half2float(a.k[((uint64_t)head * D + p + D / 2) * a.pitch + col]);
                    rotate(x, y, __ldg(cs + p));
                    kt[slot * D + p] = __float2half_rn(x);
                    kt[slot * D + p + D / 2] = __float2half_rn(y);
                    vt[p * 64u + slot] = a.v[((uint64_t)head * D + p) * a.pitch + col];
                    vt[(p + D / 2) * 64u + slot] = a.v[((uint64_t)head * D + p + D / 2) * a.pitch + col];
                }
                __syncwarp();
                float s[8][2 * R];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float c0 = 0.f, c1 = 0.f, c2 = 0.f, c3 = 0.f;
                    const uint32_t tok = 16u * (g >> 1) + (g & 1u) + 2u * i;
#pragma unroll
                    for (int f = 0; f < HF; ++f) {
                        uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0;
                        if (tok <= slot) {
                            const uint4 *row = reinterpret_cast<const uint4 *>(kt + tok * D + 64u * f + 16u * j);
                            k0 = row[0]; k1 = row[1];
                        }
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const uint4 &kk = t < 2 ? k0 : k1;
                            const uint32_t b0 = word(kk, 2 * (t & 1)), b1 = word(kk, 2 * (t & 1) + 1);
                            mma16816(c0, c1, c2, c3, qh[0][4 * f + t][0], WIDE ? qh[R - 1][4 * f + t][0] : 0u, qh[0][4 * f + t][1], WIDE ? qh[R - 1][4 * f + t][1] : 0u, b0, b1);
                            mma16816(c0, c1, c2, c3, ql[0][4 * f + t][0], WIDE ? ql[R - 1][4 * f + t][0] : 0u, ql[0][4 * f + t][1], WIDE ? ql[R - 1][4 * f + t][1] : 0u, b0, b1);
                        }
                    }
                    s[i][0] = c0; s[i][1] = c1;
                    if (WIDE) { s[i][2 * R - 2] = c2; s[i][2 * R - 1] = c3; }
                }
                uint32_t p[R][8];
                soften(s, b * kKv8Block, (uint32_t)pos + 1u, 1.0f, 1.0f, true, p);
                uint32_t keep[8];                                                // pairs of tokens: rows behind the last token and hidden ones become 0
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    keep[i] = 0u;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t t = b * kKv8Block + 16u * j + 2u * i + e;
                        if (t <= (uint32_t)pos && (a.window == 0u || t + a.window > (uint32_t)pos || t < a.sinks)) keep[i] |= 0xffffu << (16 * e);
                    }
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
                    if (16u * j <= slot) {
                        const uint4 *row = reinterpret_cast<const uint4 *>(vt + (8u * t + g) * 64u + 16u * j);
                        v0 = row[0]; v1 = row[1];
                    }
                    float c2 = WIDE ? acc[t][2 * R - 2] : 0.f, c3 = WIDE ? acc[t][2 * R - 1] : 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 &vv = k < 2 ? v0 : v1;
                        const uint32_t b0 = word(vv, 2 * (k & 1)) & keep[2 * k], b1 = word(vv, 2 * (k & 1) + 1) & keep[2 * k + 1];
                        mma16816(acc[t][0], acc[t][1], c2, c3, p[0][2 * k], WIDE ? p[R - 1][2 * k] : 0u, p[0][2 * k + 1], WIDE ? p[R - 1][2 * k + 1] : 0u, b0, b1);
                    }
                    if (WIDE) { acc[t][2 * R - 2] = c2; acc[t][2 * R - 1] = c3; }
                }
                if (slot == kKv8Block - 1u) {                                    // the block is whole: bring it to 8 bits
                    float kmax = 0.f, vmax = 0.f;
                    for (uint32_t e = lane; e < 64u * D / 8u; e += 32u) {
                        const uint4 x = reinterpret_cast<const uint4 *>(kt)[e], y = reinterpret_cast<const uint4 *>(vt)[e];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 xf = half2_of(word(x, i)), yf = half2_of(word(y, i));
                            kmax = amax_of(amax_of(kmax, xf.x), xf.y);
                            vmax = amax_of(amax_of(vmax, yf.x), yf.y);
                        }
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
                        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
                    }
                    const float ksc = scale_of(kmax), vsc = scale_of(vmax), ki = 1.0f / ksc, vi = 1.0f / vsc;
                    for (uint32_t e = lane; e < 64u * D / 8u; e += 32u) {
                        const uint4 x = reinterpret_cast<const uint4 *>(kt)[e], y = reinterpret_cast<const uint4 *>(vt)[e];
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float2 x0 = half2_of(word(x, 2 * i)), x1 = half2_of(word(x, 2 * i + 1)), y0 = half2_of(word(y, 2 * i)), y1 = half2_of(word(y, 2 * i + 1));
                            w[i] = codes4(x0.x, x0.y, x1.x, x1.y, ki);
                            w[2 + i] = codes4(y0.x, y0.y, y1.x, y1.y, vi);
                        }
                        const uint32_t t = e * 8u / D, d = e * 8u % D;
                        *reinterpret_cast<uint2 *>(codes + (d >> 6) * 4096u + t * 64u + (d & 63u)) = make_uint2(w[0], w[1]);
                        *reinterpret_cast<uint2 *>(codes + kKv8Block * D + e * 8u) = make_uint2(w[2], w[3]);
                    }
                    if (lane == 0u) a.cache.scales[ch * a.cache.blocks + b] = make_float2(ksc, vsc);
                }
            }
        }
        if (!ok) break;
        // ---- this part is done: the output, or a part of it ----
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        bool write = n_units == sn.units;
        if (!write) {
            // slot 0 belongs to the (column, head) that holds this warp's first unit, slot 1 to the other one it may share
            float *mine = a.partial + ((uint64_t)me * 2u + (u == u_begin ? 0u : 1u)) * (GP * PROW);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float *row = mine + (g + 8u * r) * PROW;
                if (g + 8u * r < G) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) __stcg(reinterpret_cast<float2 *>(row + 8u * t + 2u * j), make_float2(acc[t][2 * r], acc[t][2 * r + 1]));
                    if (j == 0u) __stcg(reinterpret_cast<float2 *>(row + D), make_float2(m[r], l[r]));
                }
            }
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0u) before = atomicAdd(a.counters + ch, n_units);
            before = __shfl_sync(0xffffffffu, before, 0);
            if (before + n_units == sn.units) {                                  // all parts are there
                __threadfence();
                if (lane == 0u) a.counters[ch] = 0u;
                const uint32_t w0 = worker_of(seg0), w1 = worker_of(seg0 + sn.units - 1u);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
                    for (int t = 0; t < DT; ++t) { acc[t][2 * r] = 0.f; acc[t][2 * r + 1] = 0.f; }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t row = g + 8u * r;
                    for (uint32_t w = w0 + j; w <= w1 && row < G; w += 4u) {
                        const float *src = a.partial + ((uint64_t)w * 2u + (share(w) >= seg0 ? 0u : 1u)) * (GP * PROW) + row * PROW;
                        m[r] = fmaxf(m[r], __ldcg(src + D));
                    }
                    m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
                    m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
                    const float base = m[r] == -INFINITY ? 0.f : m[r];
                    if (row < G) {
                        for (uint32_t w = w0; w <= w1; ++w) {
                            const float *src = a.partial + ((uint64_t)w * 2u + (share(w) >= seg0 ? 0u : 1u)) * (GP * PROW) + row * PROW;
                            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(src + D));
                            const float f = exp2f(ml.x - base);
                            l[r] = fmaf(ml.y, f, l[r]);
#pragma unroll
                            for (int t = 0; t < DT; ++t) {
                                const float2 x = __ldcg(reinterpret_cast<const float2 *>(src + 8u * t + 2u * j));
                                acc[t][2 * r] = fmaf(x.x, f, acc[t][2 * r]);
                                acc[t][2 * r + 1] = fmaf(x.y, f, acc[t][2 * r + 1]);
                            }
                        }
                    }
                }
                write = true;
            }
        }
        if (write) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t row = g + 8u * r;
                if (row < G) {
                    const float inv = 1.0f / l[r];
                    __half *dst = a.out + ((uint64_t)(head * G + row) * D + 2u * j) * a.pitch + col;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        dst[(uint64_t)(8u * t) * a.pitch] = __float2half_rn(acc[t][2 * r] * inv);
                        dst[(uint64_t)(8u * t + 1u) * a.pitch] = __float2half_rn(acc[t][2 * r + 1] * inv);
                    }
                }
            }
        }
        u += n_units;
    }
    if (!ok) {                                                                    // gave up: report, wait (bounded) for own copies, leave
        if (lane == 0u) {
            atomicOr(a.status, (uint32_t)ST_TIMEOUT_PRODUCER);
            for (uint32_t i = consumed; i < issued; ++i) {
                const long long t0 = clock64();
                bool done = false;
                while (!done && (unsigned long long)(clock64() - t0) < a.wait_cycles) done = ptx::mbar_try_wait(bar0 + 8u * (i % kStages), (i / kStages) & 1u);
                if (!done) atomicOr(a.status, (uint32_t)ST_TIMEOUT_DRAIN);
            }
        }
        __syncwarp();
    }
}

template <int D, int WARPS>
constexpr uint32_t attn_smem(uint32_t columns) { return WARPS * kStages * 2u * kKv8Block * D + (columns + 1u) * 4u; }

}  // namespace

cudaError_t launch_rope_table(float2 *table, uint32_t positions, uint32_t head_dim, double theta, bool llama3, cudaStream_t s) {
    const uint64_t n = (uint64_t)positions * (head_dim / 2u);
    k44_rope_table_kernel<<<(uint32_t)((n + 255u) / 256u), 256, 0, s>>>(table, positions, head_dim / 2u, theta, llama3 ? 1 : 0);
    return cudaGetLastError();
}

cudaError_t launch_kv8_fill(const Kv8FillArgs &a, bool pdl, cudaStream_t s) {
    const dim3 grid((a.seq_len + kKv8Block - 1u) / kKv8Block, a.cache.h_kv, (a.columns + a.seq_len - 1u) / a.seq_len);
    return a.cache.head_dim == 64u ? launch_dep(k44_kv8_fill_kernel<64>, grid, dim3(256), 0, pdl, s, a)
                                   : launch_dep(k44_kv8_fill_kernel<128>, grid, dim3(256), 0, pdl, s, a);
}

cudaError_t kv8_attn_setup() {
    cudaError_t e = cudaFuncSetAttribute(k44_kv8_attn_kernel<64, kWarps64, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_smem<64, kWarps64>(kKv8MaxColumns));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k44_kv8_attn_kernel<64, kWarps64, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_smem<64, kWarps64>(kKv8MaxColumns));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k44_kv8_attn_kernel<128, kWarps128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_smem<128, kWarps128>(kKv8MaxColumns));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k44_kv8_attn_kernel<128, kWarps128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_smem<128, kWarps128>(kKv8MaxColumns));
    return e;
}

uint64_t kv8_attn_partial_bytes(uint32_t num_sms, uint32_t group, uint32_t head_dim) {
    return (uint64_t)num_sms * (head_dim == 64u ? kWarps64 : kWarps128) * 2u * (group > 8u ? 16u : 8u) * (head_dim + 2u) * sizeof(float);
}

cudaError_t launch_kv8_attn(const Kv8AttnArgs &a, uint32_t num_sms, bool pdl, cudaStream_t s) {
    const bool wide = a.h_q / a.cache.h_kv > 8u;
    const dim3 grid(num_sms);
    if (a.cache.head_dim == 64u)
        return wide ? launch_dep(k44_kv8_attn_kernel<64, kWarps64, true>, grid, dim3(kWarps64 * 32u), attn_smem<64, kWarps64>(a.columns), pdl, s, a)
                    : launch_dep(k44_kv8_attn_kernel<64, kWarps64, false>, grid, dim3(kWarps64 * 32u), attn_smem<64, kWarps64>(a.columns), pdl, s, a);
    return wide ? launch_dep(k44_kv8_attn_kernel<128, kWarps128, true>, grid, dim3(kWarps128 * 32u), attn_smem<128, kWarps128>(a.columns), pdl, s, a)
                : launch_dep(k44_kv8_attn_kernel<128, kWarps128, false>, grid, dim3(kWarps128 * 32u), attn_smem<128, kWarps128>(a.columns), pdl, s, a);
}

}  // namespace k44b
