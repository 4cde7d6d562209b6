// Key / value cache of 8 bits: rotary table, filling it from a prompt, and the attention of single tokens against it.
//
// Format (k44_decoder.cuh): blocks of 64 tokens of one column and head, e4m3 codes with one FP32 scale per block for keys and
// one for values,  scale = max(amax, 2^-24) / 448,  code = e4m3(x / scale);  infinities count as the largest FP16 number, a NaN
// stays a NaN of its own value; keys are rotated, and rounded to FP16, where finite ones end at the largest number. The open block is kept
// as FP16 rows, so that a scale is chosen once, with all 64 tokens known.
// A block is brought to 8 bits by the step that appends its last token and read in 8 bits from the next block on.
#include "k44_decoder.cuh"
#include "k44_ptx.cuh"

#include <algorithm>
#include <numeric>

namespace k44b {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- rotary table ---------------------------------------------------------------------------------------------------------
__global__ void k44_rope_table_kernel(float2 *table, uint32_t positions, uint32_t half, double theta, int llama3, int pairs_first) {
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
    const float size = pairs_first ? kWindowHeld : 1.0f;
    table[pairs_first ? (uint64_t)p * positions + pos : i] = make_float2(size * (float)c, size * (float)s);
}

// one rotation, each product and sum rounded by itself: the same bits wherever a key is rotated
__device__ __forceinline__ void rotate(float &a, float &b, float2 cs) {
    const float x = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
    b = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
    a = x;
}

// A rotated pair of FP16 numbers may be sqrt(2) longer than the largest one; in the cache such a key is the largest number. Infinities
// and NaN stay what they are.
__device__ __forceinline__ float held(float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x; }

// ---- 8 bits -------------------------------------------------------------------------------------------------------------------
// largest magnitudes so far, two at a time; the maximum of a number and a NaN is the number
__device__ __forceinline__ __half2 amax_of(__half2 m, uint32_t two) { return __hmax2(m, __habs2(*reinterpret_cast<const __half2 *>(&two))); }
__device__ __forceinline__ float amax_of(__half2 m) { const float2 f = __half22float2(m); return fminf(fmaxf(f.x, f.y), 65504.0f); }
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
// the same, and what is beyond the largest number becomes that; a NaN stays one
__device__ __forceinline__ uint32_t pack2_finite(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// ---- filling the cache from a prompt ----------------------------------------------------------------------------------------
// CTA = the keys or the values of one block of 64 tokens of one sequence, some of its heads one after the other. Keys are rotated and
// rounded to FP16 first, then treated as the step by step path treats them. What it cannot do without is HBM: 4 bytes read and 2 written
// per pair of key and value elements. Keys pass through shared memory once, to be turned from channel rows to token rows: a thread owns one token and 8
// rotation pairs, neighbours the next pairs, so that table and codes are read and written in whole sectors and a token's elements stay
// in registers from the rotation to the code. Values need no turning: a thread takes 8 tokens of a channel from the canvas to their
// codes. The next head's rows load meanwhile. Columns are read from the 16-byte boundary below a sequence's first one.
// 64 prompts of up to 512 tokens, 8 heads of 64: 17.5 us for 50 MB. Keys and values in one CTA 20.7 (123 registers, half as many
// CTAs); without heads in a row 25 (each CTA waits for its length, rows and angles in turn), with 2 or 3 18 to 19, with 8 20 (too
// few CTAs). With 128 dimensions 32.8 for 100 MB. What bounds it is those waits of the first CTAs, CTAs of the grid that a short sequence
// leaves without work, and the last ones' uneven end; HBM is at a fifth while it runs.
template <int D>
__global__ void __launch_bounds__(256, D == 64 ? 4 : 2) k44_kv8_fill_kernel(const Kv8FillArgs a, uint32_t heads) {
    dep_enter();
    constexpr uint32_t PER = D / 16, TOKENS = 256u / PER, ROUNDS = 64u / TOKENS, N = D / 32;   // N pieces of 8 elements per thread
    constexpr uint32_t ROW = 64 + 10;                                // 37 words: rows 8 apart, and pieces of neighbouring rows, on different banks
    __shared__ __align__(16) __half xs[D * ROW];
    __shared__ float red[8];
    const uint32_t block = blockIdx.x, seq = blockIdx.z, tid = threadIdx.x, H = a.cache.h_kv;
    const uint32_t t0 = block * kKv8Block, part = tid % PER, p0 = part * 8u, tok0 = tid / PER, groups = gridDim.y / 2u;
    const bool is_k = blockIdx.y < groups;
    const int2 sl = a.sequences[seq];
    if (sl.x < 0) return;
    const uint32_t len = (uint32_t)sl.y;
    // a plan's tables are checked by the host; the cache's own limits are checked here as well
    if ((uint32_t)sl.x >= a.cache.columns || sl.y < 0 || len > a.cache.max_seq || len > a.seq_len || (uint64_t)seq * a.seq_len + len > a.columns) {
        if (tid == 0u) atomicOr(a.status, (uint32_t)ST_BAD_INDEX);
        return;
    }
    const uint32_t h0 = (is_k ? blockIdx.y : blockIdx.y - groups) * heads, h1 = min(h0 + heads, H);
    if (is_k && block == 0u && tid < h1 - h0) a.cache.tail_block[(uint64_t)sl.x * H + h0 + tid] = (len % kKv8Block) ? (int)(len / kKv8Block) : -1;
    if (t0 >= len) return;
    const uint32_t n = min(kKv8Block, len - t0), col0 = seq * a.seq_len + t0, shift = col0 & 7u, base = col0 - shift, end = shift + n;
    const __half *rows = (is_k ? a.k : a.v) + base;
    // piece e of a head: 8 columns of row e >> 3; with a shift, a ninth piece per row. Pieces start before column `columns`, and rows
    // are whole multiples of 64 columns, so a piece that starts inside a row ends inside it.
    uint4 next[N], ninth = make_uint4(0, 0, 0, 0);
    auto fetch = [&](uint32_t h) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t e = 256u * i + tid, c = (e & 7u) * 8u;
            next[i] = c < end ? __ldcg(reinterpret_cast<const uint4 *>(rows + ((uint64_t)h * D + (e >> 3)) * a.pitch + c)) : make_uint4(0, 0, 0, 0);
        }
        if (end > 64u && tid < D) ninth = __ldcg(reinterpret_cast<const uint4 *>(rows + ((uint64_t)h * D + tid) * a.pitch + 64u));
    };
    auto stage = [&](uint32_t row, uint32_t c, uint4 x) {
        uint32_t *to = reinterpret_cast<uint32_t *>(xs + row * ROW + c);
        to[0] = x.x; to[1] = x.y; to[2] = x.z; to[3] = x.w;
    };
    auto stage_all = [&] {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) { const uint32_t e = 256u * i + tid; stage(e >> 3, (e & 7u) * 8u, next[i]); }
        if (end > 64u && tid < D) stage(tid, 64u, ninth);
        __syncthreads();
    };
    auto whole_max = [&](float m) {                                  // of the CTA; its barrier also ends all reading of xs
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((tid & 31u) == 0u) red[tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
        return m;
    };
    auto eight = [](const uint32_t *w, float inv) {
        const float2 x = half2_of(w[0]), y = half2_of(w[1]), z = half2_of(w[2]), q = half2_of(w[3]);
        return make_uint2(codes4(x.x, x.y, y.x, y.y, inv), codes4(z.x, z.y, q.x, q.y, inv));
    };
    fetch(h0);
    if (is_k) {
        float2 cs[ROUNDS][8];
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r) {
            const uint32_t t = t0 + r * TOKENS + tok0;
            const float4 *from = reinterpret_cast<const float4 *>(a.rope + (uint64_t)t * (D / 2) + p0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = t < len ? __ldg(from + i) : make_float4(0.f, 0.f, 0.f, 0.f);       // the table may end with the cache
                cs[r][2 * i] = make_float2(v.x, v.y);
                cs[r][2 * i + 1] = make_float2(v.z, v.w);
            }
        }
        for (uint32_t h = h0; h < h1; ++h) {
            const uint64_t ch = (uint64_t)sl.x * H + h;
            if (h != h0) __syncthreads();
            stage_all();
            if (h + 1u < h1) fetch(h + 1u);
            // a round's token: its 8 pairs, rotated and rounded by `pack`
            auto turn = [&](uint32_t r, uint32_t (&lo)[4], uint32_t (&hi)[4], auto pack) {
                const __half *x = xs + p0 * ROW + shift + r * TOKENS + tok0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    float u[2], v[2];
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        u[e] = __half2float(x[(2 * i + e) * ROW]);
                        v[e] = __half2float(x[(2 * i + e + D / 2) * ROW]);
                        rotate(u[e], v[e], cs[r][2 * i + e]);
                    }
                    lo[i] = pack(u[0], u[1]);
                    hi[i] = pack(v[0], v[1]);
                }
            };
            if (n == kKv8Block) {                                    // a whole block: 8 bits, where infinities too count as the largest number
                __half2 amax = __float2half2_rn(0.f);
                uint32_t lo[ROUNDS][4], hi[ROUNDS][4];
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; ++r) {
                    turn(r, lo[r], hi[r], [](float x, float y) { return pack2_finite(x, y); });
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) amax = amax_of(amax_of(amax, lo[r][i]), hi[r][i]);
                }
                const float scale = scale_of(whole_max(amax_of(amax))), inv = 1.0f / scale;
                uint8_t *codes = a.cache.codes + (ch * a.cache.blocks + block) * (2u * kKv8Block * D);
                if (tid == 0u) a.cache.scales[ch * a.cache.blocks + block].x = scale;
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; ++r) {
                    uint8_t *row = codes + (r * TOKENS + tok0) * 64u;
                    const uint32_t p1 = p0 + D / 2;
                    *reinterpret_cast<uint2 *>(row + p0) = eight(lo[r], inv);
                    *reinterpret_cast<uint2 *>(row + (p1 >> 6) * 4096u + (p1 & 63u)) = eight(hi[r], inv);
                }
            } else {                                                 // the open block: FP16 rows; rows behind the last token stay as they were
                __half *tail = a.cache.k_tail + ch * (kKv8Block * D);
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; ++r) {
                    const uint32_t t = r * TOKENS + tok0;
                    if (t >= n) continue;
                    uint32_t lo[4], hi[4];
                    turn(r, lo, hi, [](float x, float y) { return pack2(held(x), held(y)); });
                    *reinterpret_cast<uint4 *>(tail + t * D + p0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    *reinterpret_cast<uint4 *>(tail + t * D + p0 + D / 2) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                }
            }
        }
        return;
    }
    for (uint32_t h = h0; h < h1; ++h) {
        const uint64_t ch = (uint64_t)sl.x * H + h;
        uint4 x[N];
        if (h != h0) __syncthreads();
        if (shift) stage_all();
        __half2 amax = __float2half2_rn(0.f);
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            uint32_t *w = reinterpret_cast<uint32_t *>(&x[i]);
            x[i] = next[i];
            if (shift) {
                const uint32_t e = 256u * i + tid;
                const unsigned short *from = reinterpret_cast<const unsigned short *>(xs + (e >> 3) * ROW + (e & 7u) * 8u + shift);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (uint32_t)from[2 * j] | ((uint32_t)from[2 * j + 1] << 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = amax_of(amax, w[j]);
        }
        if (h + 1u < h1) fetch(h + 1u);
        if (n == kKv8Block) {
            const float scale = scale_of(whole_max(amax_of(amax))), inv = 1.0f / scale;
            uint8_t *codes = a.cache.codes + (ch * a.cache.blocks + block) * (2u * kKv8Block * D) + kKv8Block * D;
            if (tid == 0u) a.cache.scales[ch * a.cache.blocks + block].y = scale;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) *reinterpret_cast<uint2 *>(codes + (256u * i + tid) * 8u) = eight(reinterpret_cast<const uint32_t *>(&x[i]), inv);
        } else {
            __half *tail = a.cache.v_tail + ch * (kKv8Block * D);
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const uint32_t e = 256u * i + tid, c = (e & 7u) * 8u;
                if (c + 8u <= n) *reinterpret_cast<uint4 *>(tail + e * 8u) = x[i];
                else {
                    const __half *one = reinterpret_cast<const __half *>(&x[i]);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) if (c + j < n) tail[e * 8u + j] = one[j];
                }
            }
        }
    }
}

// ---- single tokens against the cache -------------------------------------------------------------------------------------------
// o = sum_t softmax_t(q . k_t / sqrt(D)) v_t over the visible positions t of a column, for the group of query heads that share
// one key / value head, so that every code is read once. Memory-bound: 2 D bytes per position and key / value head.
//
// Two launches. The first rotates q and k, leaves q in the order in which the second loads it, appends the new tokens to the open
// blocks and brings completed blocks to 8 bits: on the canvas a column's channels are `pitch` elements apart, and warps that each
// gather theirs cost 6 to 8 us of a step of 64 columns (11 000 to 16 000 cycles per warp, 32 sectors per load), a transposing
// pass over 8 columns at a time 2 to 3.
//
// Work of the second: a unit is one visible 8-bit block of one (column, head), or its open block. All units in a row
// (column, head, block), each with a weight, are cut into equal shares, one per warp of the grid, whatever the columns' lengths; a
// warp that holds a (column, head) whole writes its output, the others leave (accumulator, maximum, sum) and the last one to
// arrive adds the parts in the order of the warps, so that the result does not depend on the order of arrival.
// Loads: each warp keeps a ring of granules of 64 * D bytes in flight with bulk copies: the keys of an 8-bit block are one
// granule, its values another, the FP16 keys of the open block two, its values two. Nothing in the walk over the blocks waits for
// a global load of its own; scales are fetched 32 blocks at a time.
// Products on mma.sync: 8 (or 16) query heads are the rows of m16n8k16 — tcgen05 would need 64 rows and its operands as FP16
// in shared memory, for a kernel that waits for HBM. Keys: a lane takes 16 consecutive dimensions of one token (16 bytes),
// values: 16 consecutive tokens of one dimension; which logical k index they stand for is free as long as the other operand
// agrees, so codes go from shared memory to the operand registers without a shuffle: token of score tile i, column 2 j + e =
// 16 j + 2 i + e, and the scores' accumulator layout is the second product's A operand as it stands.
// The values' scale is 2^e times a number between 1 and 2. That number is folded into the exponent (p' = p * number, and the sum uses
// p' / number), while the accumulator is kept in units of 2^e and moves by a power of two, exactly, where a block has another e: what is
// rounded to FP16 is a weight relative to the largest one, not to that times its block's scale, or one loud block (a value of
// 6e4 next to values of 1) would leave nothing of the weights behind it. p' <= 1 is held as 2^15 p', so that FP16 has whole
// precision down to 2^-29 and something down to 2^-40 of the largest weight. The rounding is the tensor cores' type, 2^-11 of a weight, of
// the order of the output's own (2.4e-4 relative to 64 bits; with weights in 32 bits 2.0e-4).
// Half of q (a rotated pair of FP16 numbers may be sqrt(2) longer than the largest one) is split into two FP16 numbers (high and low
// part): with exact codes the scores are then as good as in 32 bits. With up to 8 heads the low parts are rows 8 to 15 of the operand,
// which would be empty, and cost nothing.
// Measured, both launches: 48 columns at up to 8190 positions, 32 heads on 8 of 128 dimensions: 79 us for the 350 to 400 MB
// of the lengths drawn (4.4 to 4.9 TB/s; the same without the products; 192 KB in flight per SM are 4 us of HBM's full rate, so what is
// lost is the start and the last warps' uneven end); 64 columns at 511, D = 64, each completing a block: 24 us; 64 columns at up to 16000 with a
// window of 1024: 28; one column at 1500: 15, a chain of latencies. 16 query heads on one: 27 us for 64 columns at 511 (32 heads on 2 of
// 64), 95 for 48 columns at up to 8190 (32 on 2 of 128, 82 MB): few (column, head) pairs, long chains of products in each warp.
constexpr float kWeightBits = 15.f;
constexpr uint32_t kOpenWeight = 4;                              // an open block: one and a half times the bytes, and the work around it
// warps per SM and granules per warp (192 KB of an SM's shared memory in all): as many warps as the registers allow
template <int D, bool WIDE> constexpr uint32_t kWarps = WIDE || D == 128 ? 8u : 12u;
template <int D, bool WIDE> constexpr uint32_t kRing = 192u * 1024u / (kWarps<D, WIDE> * kKv8Block * D);

__device__ __forceinline__ void mma16816(float &c0, float &c1, float &c2, float &c3, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c0), "+f"(c1), "+f"(c2), "+f"(c3) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }       // -126 .. 127
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// what a column's token sees: 8-bit blocks [0, sink_blocks) and [from, open), and the open block
struct Seen {
    uint32_t sink_blocks, from, open, units;            // units: those 8-bit blocks and the open one
    __device__ uint32_t weight() const { return units - 1u + kOpenWeight; }
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

// A column's position where it is inside the cache, -1 (idle) otherwise.
__device__ __forceinline__ int position_of(const Kv8AttnArgs &a, uint32_t c) {
    const int p = a.positions[c];
    return p >= 0 && (uint32_t)p < a.cache.max_seq ? p : -1;
}

// First launch. Grid (8 columns, key / value head, role): role 0 q, 1 keys, 2 values, a warp per column. It lets the second launch start
// once its own predecessors are done: what that one does before it waits in turn (cutting up the work, copies of 8-bit blocks) needs
// nothing of this one's, so the two overlap.
// Roles 1 and 2 read a block that is about to be complete before they wait for the new token's row, and patch that in.
template <int D, bool WIDE>           // WIDE: 9 to 16 query heads per key / value head
__global__ void __launch_bounds__(256) k44_kv8_prepare_kernel(const Kv8AttnArgs a) {
    constexpr int KS = D / 16, HF = D / 64, R = WIDE ? 2 : 1, TILE = kKv8Block * D, ROWS = 8 * R * D, PAD = ROWS + 8;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, j = lane & 3u;
    const uint32_t H = a.cache.h_kv, G = a.h_q / H, C = a.columns;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- rows of the head for 8 columns, turned: [column][row] ----
    __half *xs = reinterpret_cast<__half *>(smem_raw);
    const uint32_t head = blockIdx.y, c0 = blockIdx.x * 8u, col = c0 + warp;
    const bool is_q = blockIdx.z == 0u, is_k = blockIdx.z == 1u;
    const int pos = col < C ? position_of(a, col) : -1;
    const uint64_t ch = (uint64_t)col * H + head;
    const uint32_t b = (uint32_t)pos / kKv8Block, slot = (uint32_t)pos % kKv8Block;
    constexpr int N = TILE / 8 / 32;                                           // 16-byte pieces of a block per lane
    __half *tail = (is_k ? a.cache.k_tail : a.cache.v_tail) + ch * TILE;
    uint8_t *codes = a.cache.codes + (ch * a.cache.blocks + b) * (2u * TILE) + (is_k ? 0u : TILE);
    uint4 piece[N];
    const bool whole = !is_q && pos >= 0 && slot == kKv8Block - 1u;
    int tag = 0;
    if (!is_q && pos >= 0) tag = a.cache.tail_block[ch];
    if (whole)
#pragma unroll
        for (int i = 0; i < N; ++i) piece[i] = reinterpret_cast<const uint4 *>(tail)[32 * i + lane];
    const uint32_t rows = is_q ? G * D : (uint32_t)D;
    const __half *rows_of = is_q ? a.q + (uint64_t)head * G * D * a.pitch : (is_k ? a.k : a.v) + (uint64_t)head * D * a.pitch;
    for (uint32_t r = tid; r < rows; r += 256u) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(rows_of + (uint64_t)r * a.pitch + c0));
        const __half *h = reinterpret_cast<const __half *>(&v);
#pragma unroll
        for (int c = 0; c < 8; ++c) xs[c * PAD + r] = h[c];
    }
    if (is_q) for (uint32_t r = rows + tid; r < (uint32_t)ROWS; r += 256u)      // rows of the operand without a head
#pragma unroll
        for (int c = 0; c < 8; ++c) xs[c * PAD + r] = __half(0.f);
    if (is_q && lane == 0u && col < C) a.counters[ch] = 0u;                    // of the parts that have arrived; a run that gave up leaves some
    if (is_q && head == 0u && lane == 0u && col < C && pos < 0 && a.positions[col] >= 0) atomicOr(a.status, (uint32_t)ST_BAD_INDEX);
    __syncthreads();
    if (pos < 0) return;
    const float2 *cs = a.rope + (uint64_t)pos * (D / 2);
    __half *x = xs + warp * PAD;
    if (is_q) {
        // ---- operand words of lane (g, j): row g (+ 8), dimensions 64 f + 16 j + 4 s + 2 t, + 1; high parts, then low parts ----
        uint4 *frag = a.q_frag + ch * (R * KS * 32u) + lane;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int f = 0; f < HF; ++f) {
                const uint32_t d0 = 64u * f + 16u * j, p0 = d0 % (D / 2);
                const __half *lo16 = x + (g + 8u * r) * D + p0;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float y[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int i = 4 * s + 2 * t + e;
                            float u = __half2float(lo16[i]), v = __half2float(lo16[i + D / 2]);
                            rotate(u, v, __ldg(cs + p0 + i));
                            y[e] = 0.5f * (d0 < D / 2 ? u : v);
                        }
                        hi[t] = pack2(y[0], y[1]);
                        const float2 hf = half2_of(hi[t]);
                        lo[t] = pack2(y[0] - hf.x, y[1] - hf.y);
                    }
                    frag[(r * KS + 4 * f + s) * 32] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
                }
            }
        }
        return;
    }
    // ---- append the new token to the open block (whose number the second launch writes down) ----
    const bool rebuild = tag != (int)b && slot != 0u;                          // back inside a block that was complete: its rows start from its 8 bits
    if (rebuild) {
        const float2 both = a.cache.scales[ch * a.cache.blocks + b];
        const float old = is_k ? both.x : both.y;
        for (uint32_t e = lane; e < TILE / 2u; e += 32u) {
            const uint32_t c2 = 2u * e, t = (c2 >> 6) & 63u, d = (c2 >> 12) * 64u + (c2 & 63u);
            const float2 f = half2_of(from_codes(*reinterpret_cast<const uint16_t *>(codes + c2)));
            const uint32_t v = pack2(f.x * old, f.y * old);
            if (!is_k) *reinterpret_cast<uint32_t *>(tail + c2) = v;
            else if (t < slot) *reinterpret_cast<uint32_t *>(tail + t * D + d) = v;
        }
        __syncwarp();
    }
#pragma unroll
    for (int f = 0; f < HF; ++f) {
        const uint32_t p = 32u * f + lane;
        if (is_k) {
            float u = __half2float(x[p]), v = __half2float(x[p + D / 2]);
            rotate(u, v, __ldg(cs + p));
            const __half hu = __float2half_rn(held(u)), hv = __float2half_rn(held(v));
            tail[slot * D + p] = hu; tail[slot * D + p + D / 2] = hv;
            x[p] = hu; x[p + D / 2] = hv;
        } else {
            tail[p * 64u + slot] = x[p];
            tail[(p + D / 2) * 64u + slot] = x[p + D / 2];
        }
    }
    if (!whole) return;
    // ---- the block is complete: bring it to 8 bits ----
    __syncwarp();
    if (rebuild)
#pragma unroll
        for (int i = 0; i < N; ++i) piece[i] = reinterpret_cast<const uint4 *>(tail)[32 * i + lane];
    __half2 amax = __float2half2_rn(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {                                              // the new token's row (keys) or column (values)
        const uint32_t at = (32u * i + lane) * 8u;
        if (is_k) { if (at / D == kKv8Block - 1u) piece[i] = *reinterpret_cast<const uint4 *>(x + at % D); }
        else if ((at & 63u) == 56u) piece[i].w = (piece[i].w & 0xffffu) | ((uint32_t)__half_as_ushort(x[at >> 6]) << 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = amax_of(amax, word(piece[i], e));
    }
    float mx = amax_of(amax);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float scale = scale_of(mx), inv = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 x0 = half2_of(piece[i].x), x1 = half2_of(piece[i].y), x2 = half2_of(piece[i].z), x3 = half2_of(piece[i].w);
        const uint32_t at = (32u * i + lane) * 8u, t = at / D, d = at % D;
        *reinterpret_cast<uint2 *>(codes + (is_k ? (d >> 6) * 4096u + t * 64u + (d & 63u) : at)) = make_uint2(codes4(x0.x, x0.y, x1.x, x1.y, inv), codes4(x2.x, x2.y, x3.x, x3.y, inv));
    }
    if (lane == 0u) reinterpret_cast<float *>(a.cache.scales + ch * a.cache.blocks + b)[is_k ? 0 : 1] = scale;
}

template <int D, bool WIDE>
__global__ void __launch_bounds__(kWarps<D, WIDE> * 32, 1) k44_kv8_attn_kernel(const Kv8AttnArgs a) {
    constexpr int DT = D / 8, KS = D / 16, HF = D / 64, R = WIDE ? 2 : 1;      // dimension tiles, k steps, halves, row sets
    constexpr uint32_t GRAN = kKv8Block * D, WARPS = kWarps<D, WIDE>, RING = kRing<D, WIDE>, GP = 8u * R, PROW = D + 2u;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[WARPS * RING];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, j = lane & 3u;
    const uint32_t H = a.cache.h_kv, G = a.h_q / H, C = a.columns;
    uint8_t *const ring_ptr = smem_raw + warp * RING * GRAN;
    const uint32_t ring = ptx::smem_addr(ring_ptr);
    const uint32_t bar0 = ptx::smem_addr(bars) + warp * RING * 8u;
    if (lane == 0u) {
        for (uint32_t s = 0; s < RING; ++s) ptx::mbar_init(bar0 + 8u * s, 1);
        ptx::fence_mbar_init();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- cut up the work: weight before each column ----
    uint32_t *prefix = reinterpret_cast<uint32_t *>(smem_raw + WARPS * RING * GRAN);       // [C + 1]
    for (uint32_t c = threadIdx.x; c < C; c += WARPS * 32u) {
        const int p = position_of(a, c);
        prefix[c + 1u] = H * (p < 0 ? 1u : seen_of(p, a.window, a.sinks).weight());
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
    // Which share a warp takes: its number times a step that shares no factor with the number of warps. Shares that cost more than
    // they weigh (open blocks) come at a regular distance; in the order of the warps they would meet on the same few SMs where that
    // distance divides the SMs (64 columns x 8 heads did), with a step near the golden ratio an SM's shares lie all over the row.
    const uint32_t me = (blockIdx.x * WARPS + warp) * a.spread % a.workers, total = prefix[C];
    const uint32_t workers = min(a.workers, total), each = total / workers, more = total % workers;       // the first `more` shares weigh one more
    if (me >= workers) return;
    auto share = [&](uint32_t w) -> uint32_t { return w * each + min(w, more); };
    auto worker_of = [&](uint32_t x) -> uint32_t { return x < more * (each + 1u) ? x / (each + 1u) : more + (x - more * (each + 1u)) / each; };
    const uint32_t x_begin = share(me), x_end = share(me + 1u);             // this warp's units are those that start in here
    // a place in the row of units
    struct At {
        uint32_t col, head, unit, x;                                        // x: where the unit starts
        int pos;
        Seen seen;
    };
    auto enter = [&](At &t) {
        t.pos = position_of(a, t.col);
        t.seen = t.pos < 0 ? Seen{0u, 0u, 0u, 1u} : seen_of(t.pos, a.window, a.sinks);
    };
    auto per_head = [&](const At &t) -> uint32_t { return t.pos < 0 ? 1u : t.seen.weight(); };
    auto next_head = [&](At &t) {                                           // to the first unit of the next (column, head)
        t.x += per_head(t) - t.unit;
        t.unit = 0u;
        if (++t.head == H) { t.head = 0u; ++t.col; if (t.col < C) enter(t); }
    };
    auto block_of = [&](const Seen &s, uint32_t unit) -> uint32_t { return unit < s.sink_blocks ? unit : s.from + (unit - s.sink_blocks); };
    At at;
    {
        uint32_t lo = 0, hi = C - 1u;
        while (lo < hi) { const uint32_t mid = (lo + hi + 1u) >> 1; if (prefix[mid] <= x_begin) lo = mid; else hi = mid - 1u; }
        at.col = lo;
        enter(at);
        const uint32_t rem = x_begin - prefix[lo], per = per_head(at);
        at.head = rem / per; at.unit = rem % per; at.x = x_begin;
    }
    if (at.unit >= at.seen.units) next_head(at);                            // the share begins inside an open block's weight
    // ---- q of a (column, head) as operands, and the scales of 32 of its blocks: a lane holds those of one ----
    const float sm = 2.0f * rsqrtf((float)D) * kLog2e;                      // of halves of q
    uint32_t qh[R][KS][2], ql[R][KS][2];
    float sc_mul = 0.f, sc_log = 0.f, sc_inv = 0.f;
    int sc_exp = 0;
    auto fetch_scales = [&](uint32_t first) {
        const uint32_t unit = first + lane;
        if (at.pos >= 0 && unit + 1u < at.seen.units) {
            const float2 sc = __ldg(a.cache.scales + ((uint64_t)at.col * H + at.head) * a.cache.blocks + block_of(at.seen, unit));
            // The cache's own scales lie between 2^-33 and 2^8. Larger ones are left for the number, whose range is that of 32 bits; one below
            // 2^-60, such as the 0 of a block that nobody has written, counts as that: its values come out below 2^-51, and a hidden score
            // of -inf times a key's scale stays -inf.
            const float key = sc.x < pow2(-60) ? pow2(-60) : sc.x, scale = sc.y < pow2(-60) ? pow2(-60) : sc.y;
            sc_exp = min(60, (int)(__float_as_uint(scale) >> 23 & 255u) - 127);
            const float number = scale * pow2(-sc_exp);
            sc_mul = key * sm; sc_log = log2f(number); sc_inv = 1.0f / number;
        }
    };
    auto fetch_head = [&]() {
        const uint4 *frag = a.q_frag + ((uint64_t)at.col * H + at.head) * (R * KS * 32u) + lane;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint4 w = __ldcg(frag + (r * KS + k) * 32);
                qh[r][k][0] = w.x; qh[r][k][1] = w.y; ql[r][k][0] = w.z; ql[r][k][1] = w.w;
            }
        fetch_scales(at.unit);
    };
    // ---- the ring's own walk, one granule per call, lane 0 only: runs of contiguous granules ----
    At ahead = at;
    uint32_t issued = 0, left = 0, rem = 0;                                  // granules left in the run, bytes left in it
    bool values = false;                                                     // the open block's keys are out, its values are next
    const uint8_t *src = nullptr;
    const uint64_t policy = ptx::policy_evict_first();
    bool early = true;                                                       // the first launch may still be at work: only what was there before it
    auto next_run = [&]() -> bool {
        while (ahead.x < x_end && ahead.col < C) {
            if (ahead.pos < 0) { next_head(ahead); continue; }
            if (early && ahead.unit + 1u >= ahead.seen.units) return false;
            const Seen &n = ahead.seen;
            const uint64_t ch = (uint64_t)ahead.col * H + ahead.head;
            if (ahead.unit + 1u < n.units) {
                const uint32_t run = min(min((ahead.unit < n.sink_blocks ? n.sink_blocks : n.units - 1u) - ahead.unit, x_end - ahead.x), 65536u);
                src = a.cache.codes + (ch * a.cache.blocks + block_of(n, ahead.unit)) * (2u * GRAN);
                left = 2u * run; rem = left * GRAN;
                ahead.unit += run; ahead.x += run;
            } else if (!values) {                                            // only the rows that are there
                src = reinterpret_cast<const uint8_t *>(a.cache.k_tail) + ch * (2u * GRAN);
                left = 2u; rem = ((uint32_t)ahead.pos % kKv8Block + 1u) * (2u * D);
                values = true;
            } else {
                src = reinterpret_cast<const uint8_t *>(a.cache.v_tail) + ch * (2u * GRAN);
                left = 2u; rem = 2u * GRAN;
                values = false;
                next_head(ahead);
            }
            return true;
        }
        return false;
    };
    auto issue = [&]() {
        if (left == 0u && !next_run()) return;
        const uint32_t bar = bar0 + 8u * (issued % RING), bytes = min(rem, GRAN);
        if (bytes) {
            ptx::mbar_arrive_expect_tx(bar, bytes);
            ptx::bulk_g2s(ring + issued % RING * GRAN, src, bytes, bar, policy);
        } else ptx::mbar_arrive(bar);
        src += bytes; rem -= bytes;
        --left; ++issued;
    };
    if (lane == 0u)
        for (uint32_t s = 0; s < RING; ++s) issue();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    early = false;
    if (lane == 0u)
        while (issued < RING && (left || next_run())) issue();
    __syncwarp();
    if (at.x < x_end && at.col < C) fetch_head();

    uint32_t consumed = 0;
    bool ok = true;
    auto granule = [&](uint32_t i) -> uint8_t * { return ring_ptr + ((consumed + i) % RING) * GRAN; };
    auto arrived = [&](uint32_t i) -> bool {                                  // whole warp; bounded
        const uint32_t n = consumed + i, bar = bar0 + 8u * (n % RING), ph = (n / RING) & 1u;
        bool here = ptx::mbar_try_wait(bar, ph);
        if (!here) {
            const long long t0 = clock64();
            while (!(here = ptx::mbar_try_wait(bar, ph)) && (unsigned long long)(clock64() - t0) < a.wait_cycles) {}
        }
        return __all_sync(0xffffffffu, here ? 1 : 0) != 0;
    };
    auto release = [&](uint32_t n) {                                          // n granules have been read by every lane
        __syncwarp();
        consumed += n;
        if (lane == 0u) for (uint32_t i = 0; i < n; ++i) issue();
    };

    for (bool first = true; at.x < x_end && at.col < C && ok; first = false) {
        const uint32_t col = at.col, head = at.head;
        const int pos = at.pos;
        const Seen sn = at.seen;
        const uint64_t ch = (uint64_t)col * H + head;
        if (pos < 0) {                                                          // idle column: zeros
            for (uint32_t e = lane; e < G * D; e += 32u) a.out[((uint64_t)head * G * D + e) * a.pitch + col] = __half(0.f);
            next_head(at);
            continue;
        }
        if (!first) fetch_head();
        const uint32_t seg0 = at.x - at.unit, unit0 = at.unit;
        const uint32_t n_units = min(sn.units - unit0, x_end - at.x);            // this warp's part of the (column, head): units start one after the other
        const bool has_open = unit0 + n_units == sn.units;
        float acc[DT][2 * R], m[R], l[R];
        int unit = 0;                                                            // acc counts in 2^unit
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 2 * R; ++e) acc[t][e] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.f; }

        // scores of 8 tokens more: k step 4 f + t of tile i
        auto score = [&](float (&c)[4], int k, uint32_t b0, uint32_t b1) {
            if (WIDE) {
                mma16816(c[0], c[1], c[2], c[3], qh[0][k][0], qh[R - 1][k][0], qh[0][k][1], qh[R - 1][k][1], b0, b1);
                mma16816(c[0], c[1], c[2], c[3], ql[0][k][0], ql[R - 1][k][0], ql[0][k][1], ql[R - 1][k][1], b0, b1);
            } else mma16816(c[0], c[1], c[2], c[3], qh[0][k][0], ql[0][k][0], qh[0][k][1], ql[0][k][1], b0, b1);
        };
        // scores -> weights of one block: masked, scaled, running maximum; p (FP16 operand) and l
        auto soften = [&](float (&s)[8][4], uint32_t t_base, uint32_t t_end, float mul, float lv, float rv, int ev, bool edge, uint32_t (&p)[R][8]) {
            const float moved = pow2(unit - ev);                                 // both within +-60
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (!WIDE) s[i][e] += s[i][2 + e];
                        if (edge) {
                            const uint32_t t = t_base + 16u * j + 2u * i + e;
                            const bool vis = t < t_end && (a.window == 0u || t + a.window > (uint32_t)pos || t < a.sinks);
                            if (!vis) s[i][2 * r + e] = -INFINITY;
                        }
                        mx = fmaxf(mx, s[i][2 * r + e]);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)), mul, lv);
                const float mn = fmaxf(m[r], mx), shift = mn == -INFINITY ? 0.f : (lv - mn) + kWeightBits;
                if (__any_sync(0xffffffffu, mn != m[r] || unit != ev)) {          // a new maximum: what is summed so far shrinks
                    float back = mn == -INFINITY ? 1.f : fast_exp2(m[r] - mn);
                    m[r] = mn;
                    l[r] *= back;
                    back *= moved;
#pragma unroll
                    for (int t = 0; t < DT; ++t) { acc[t][2 * r] *= back; acc[t][2 * r + 1] *= back; }
                }
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p0 = fast_exp2(fmaf(s[i][2 * r], mul, shift)), p1 = fast_exp2(fmaf(s[i][2 * r + 1], mul, shift));
                    sum += p0 + p1;
                    p[r][i] = pack2(p0, p1);
                }
                l[r] = fmaf(sum, rv, l[r]);
            }
            unit = ev;
        };
        auto weigh = [&](int t, uint32_t (&p)[R][8], int k, uint32_t b0, uint32_t b1) {
            float c2 = WIDE ? acc[t][2 * R - 2] : 0.f, c3 = WIDE ? acc[t][2 * R - 1] : 0.f;
            mma16816(acc[t][0], acc[t][1], c2, c3, p[0][2 * k], WIDE ? p[R - 1][2 * k] : 0u, p[0][2 * k + 1], WIDE ? p[R - 1][2 * k + 1] : 0u, b0, b1);
            if (WIDE) { acc[t][2 * R - 2] = c2; acc[t][2 * R - 1] = c3; }
        };

        const uint32_t n8 = has_open ? n_units - 1u : n_units;
        for (uint32_t i0 = 0; i0 < n8; ++i0) {
            // ---- an 8-bit block ----
            if (i0 && (i0 & 31u) == 0u) fetch_scales(unit0 + i0);
            const float mul = __shfl_sync(0xffffffffu, sc_mul, i0 & 31u), lv = __shfl_sync(0xffffffffu, sc_log, i0 & 31u), rv = __shfl_sync(0xffffffffu, sc_inv, i0 & 31u);
            const int ev = __shfl_sync(0xffffffffu, sc_exp, i0 & 31u);
            const uint32_t t_base = block_of(sn, unit0 + i0) * kKv8Block;
            const bool edge = a.window != 0u && !(t_base + a.window > (uint32_t)pos || t_base + kKv8Block <= a.sinks);
            if (!(ok = arrived(0))) break;
            float s[8][4];
            const uint8_t *const k_row = granule(0) + (16u * (g >> 1) + (g & 1u)) * 64u + j * 16u;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
            for (int f = 0; f < HF; ++f) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 kk[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) kk[i] = *reinterpret_cast<const uint4 *>(k_row + f * 4096u + (4 * h + i) * 128u);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {                            // the tiles' chains are independent of one another
                            const uint32_t w = word(kk[i], t);
                            score(s[4 * h + i], 4 * f + t, from_codes(w), from_codes(w >> 16));
                        }
                }
            }
            uint32_t p[R][8];
            soften(s, t_base, t_base + kKv8Block, mul, lv, rv, ev, edge, p);
            release(1);
            uint4 keep = make_uint4(~0u, ~0u, ~0u, ~0u);                         // a hidden token's codes become 0: its NaN must not count
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
            if (!(ok = arrived(0))) break;
            const uint8_t *const v_row = granule(0) + g * 64u + j * 16u;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                uint4 vv = *reinterpret_cast<const uint4 *>(v_row + t * 512u);
                vv.x &= keep.x; vv.y &= keep.y; vv.z &= keep.z; vv.w &= keep.w;
#pragma unroll
                for (int k = 0; k < 4; ++k) { const uint32_t w = word(vv, k); weigh(t, p, k, from_codes(w), from_codes(w >> 16)); }
            }
            release(1);
        }
        if (ok && has_open) {
            // ---- the open block: FP16 rows ----
            const uint32_t b = sn.open;
            if (lane == 0u) a.cache.tail_block[ch] = (int)b;
            ok = arrived(0) && arrived(1);
            if (!ok) break;
            const __half *g0 = reinterpret_cast<const __half *>(granule(0)), *g1 = reinterpret_cast<const __half *>(granule(1));       // keys: tokens 0 .. 31, 32 .. 63
            float s[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
            const __half *k_row = (g < 4u ? g0 : g1) + (16u * ((g >> 1) & 1u) + (g & 1u)) * D + 16u * j;      // token 16 (g / 2) + g % 2 + 2 i
#pragma unroll
            for (int f = 0; f < HF; ++f)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 k0 = *reinterpret_cast<const uint4 *>(k_row + 64 * f + 2 * i * D), k1 = *reinterpret_cast<const uint4 *>(k_row + 64 * f + 2 * i * D + 8);
#pragma unroll
                    for (int t = 0; t < 4; ++t) { const uint4 &kk = t < 2 ? k0 : k1; score(s[i], 4 * f + t, word(kk, 2 * (t & 1)), word(kk, 2 * (t & 1) + 1)); }
                }
            uint32_t p[R][8];
            soften(s, b * kKv8Block, (uint32_t)pos + 1u, sm, 0.f, 1.0f, 0, true, p);
            release(2);
            ok = arrived(0) && arrived(1);
            if (!ok) break;
            g0 = reinterpret_cast<const __half *>(granule(0)); g1 = reinterpret_cast<const __half *>(granule(1));      // values: the first and the second half of the dimensions
            uint32_t keep[8];                                                    // pairs of tokens: rows behind the last token and hidden ones become 0
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
                const uint4 *row = reinterpret_cast<const uint4 *>((t < DT / 2 ? g0 : g1) + (8u * (t % (DT / 2)) + g) * 64u + 16u * j);
                const uint4 v0 = row[0], v1 = row[1];
#pragma unroll
                for (int k = 0; k < 4; ++k) { const uint4 &vv = k < 2 ? v0 : v1; weigh(t, p, k, word(vv, 2 * (k & 1)) & keep[2 * k], word(vv, 2 * (k & 1) + 1) & keep[2 * k + 1]); }
            }
            release(2);
        }
        if (!ok) break;
        // ---- this part is done: the output, or a part of it ----
        const float counts = pow2(unit);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        if (n_units == sn.units) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t row = g + 8u * r;
                if (row < G) {
                    const float inv = counts / l[r];
                    __half *dst = a.out + ((uint64_t)(head * G + row) * D + 2u * j) * a.pitch + col;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        dst[(uint64_t)(8u * t) * a.pitch] = __float2half_rn(acc[t][2 * r] * inv);
                        dst[(uint64_t)(8u * t + 1u) * a.pitch] = __float2half_rn(acc[t][2 * r + 1] * inv);
                    }
                }
            }
        } else {
            // slot 0 belongs to the (column, head) in which this warp's share begins, slot 1 to the other one it may split with a neighbour
            float *own = a.partial + ((uint64_t)me * 2u + (x_begin >= seg0 ? 0u : 1u)) * (GP * PROW);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t row = g + 8u * r;
                if (row < G) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) __stcg(reinterpret_cast<float2 *>(own + row * D + 8u * t + 2u * j), make_float2(acc[t][2 * r] * counts, acc[t][2 * r + 1] * counts));
                    if (j == 0u) __stcg(reinterpret_cast<float2 *>(own + GP * D + 2u * row), make_float2(m[r], l[r]));
                }
            }
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0u) before = atomicAdd(a.counters + ch, n_units);
            before = __shfl_sync(0xffffffffu, before, 0);
            if (before + n_units == sn.units) {                                  // all parts are there
                __threadfence();
                const uint32_t w0 = worker_of(seg0), n = worker_of(seg0 + sn.units - 1u) - w0 + 1u;
                auto part = [&](uint32_t i) -> const float * { return a.partial + ((uint64_t)(w0 + i) * 2u + (share(w0 + i) >= seg0 ? 0u : 1u)) * (GP * PROW); };
                // a lane takes four dimensions of a row, the parts in their order, four of them in flight (short code: it is fetched cold)
                for (uint32_t e = lane * 4u; e < G * D; e += 128u) {
                    const uint32_t row = e / D;
                    float M = -INFINITY, L = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (uint32_t i0 = 0; i0 < n; i0 += 4u) {
                        float2 ml[4];
                        float4 x[4];
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i) {
                            ml[i] = make_float2(-INFINITY, 0.f);
                            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (i0 + i < n) {
                                const float *src = part(i0 + i);
                                ml[i] = __ldcg(reinterpret_cast<const float2 *>(src + GP * D + 2u * row));
                                x[i] = __ldcg(reinterpret_cast<const float4 *>(src + e));
                            }
                        }
                        const float mn = fmaxf(fmaxf(M, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x)), to = mn == -INFINITY ? 0.f : mn, back = fast_exp2(M - to);
                        M = mn;
                        L *= back; o.x *= back; o.y *= back; o.z *= back; o.w *= back;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i) {
                            const float f = fast_exp2(ml[i].x - to);
                            L = fmaf(ml[i].y, f, L);
                            o.x = fmaf(x[i].x, f, o.x); o.y = fmaf(x[i].y, f, o.y); o.z = fmaf(x[i].z, f, o.z); o.w = fmaf(x[i].w, f, o.w);
                        }
                    }
                    const float inv = 1.0f / L;
                    __half *dst = a.out + ((uint64_t)head * G * D + e) * a.pitch + col;
                    dst[0] = __float2half_rn(o.x * inv);
                    dst[a.pitch] = __float2half_rn(o.y * inv);
                    dst[2ull * a.pitch] = __float2half_rn(o.z * inv);
                    dst[3ull * a.pitch] = __float2half_rn(o.w * inv);
                }
            }
        }
        if (has_open) next_head(at);
        else { at.unit += n_units; at.x += n_units; }
    }
    if (!ok) {                                                                    // gave up: report, wait (bounded) for own copies, leave
        if (lane == 0u) {
            atomicOr(a.status, (uint32_t)ST_TIMEOUT_PRODUCER);
            for (uint32_t i = consumed; i < issued; ++i) {
                const long long t0 = clock64();
                bool done = false;
                while (!done && (unsigned long long)(clock64() - t0) < a.wait_cycles) done = ptx::mbar_try_wait(bar0 + 8u * (i % RING), (i / RING) & 1u);
                if (!done) atomicOr(a.status, (uint32_t)ST_TIMEOUT_DRAIN);
            }
        }
        __syncwarp();
    }
}

template <int D, bool WIDE> constexpr uint32_t attn_smem(uint32_t columns) { return kWarps<D, WIDE> * kRing<D, WIDE> * kKv8Block * D + (columns + 1u) * 4u; }
template <int D, bool WIDE> constexpr uint32_t kPrepareSmem = 8u * (8u * (WIDE ? 2u : 1u) * D + 8u) * 2u;
template <int D, bool WIDE> cudaError_t attn_setup() {
    return cudaFuncSetAttribute(k44_kv8_attn_kernel<D, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, attn_smem<D, WIDE>(kKv8MaxColumns));
}
template <int D, bool WIDE> cudaError_t attn_launch(const Kv8AttnArgs &a, uint32_t num_sms, bool pdl, cudaStream_t s) {
    Kv8AttnArgs b = a;
    b.workers = num_sms * kWarps<D, WIDE>;
    b.spread = (uint32_t)(0.6180339887 * b.workers);
    while (std::gcd(b.spread, b.workers) != 1u) ++b.spread;
    const cudaError_t e = launch_dep(k44_kv8_prepare_kernel<D, WIDE>, dim3((a.columns + 7u) / 8u, a.cache.h_kv, 3), dim3(256), kPrepareSmem<D, WIDE>, pdl, s, b);
    if (e != cudaSuccess) return e;
    return launch_dep(k44_kv8_attn_kernel<D, WIDE>, dim3(num_sms), dim3(kWarps<D, WIDE> * 32u), attn_smem<D, WIDE>(a.columns), pdl, s, b);
}

}  // namespace

cudaError_t launch_rope_table(float2 *table, uint32_t positions, uint32_t head_dim, double theta, bool llama3, bool pairs_first, cudaStream_t s) {
    const uint64_t n = (uint64_t)positions * (head_dim / 2u);
    k44_rope_table_kernel<<<(uint32_t)((n + 255u) / 256u), 256, 0, s>>>(table, positions, head_dim / 2u, theta, llama3 ? 1 : 0, pairs_first ? 1 : 0);
    return cudaGetLastError();
}

cudaError_t launch_kv8_fill(const Kv8FillArgs &a, bool pdl, cudaStream_t s) {
    // no sequence is longer than any of these
    const uint32_t longest = std::min(a.seq_len, std::min(a.columns, a.cache.max_seq)), H = a.cache.h_kv;
    const uint32_t blocks = (longest + kKv8Block - 1u) / kKv8Block, seqs = (a.columns - 1u) / a.seq_len + 1u;
    // as many heads in a row as leave eight CTAs for each of 148 SMs, up to four
    const uint32_t heads = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>(4u, 2ull * blocks * seqs * H / 1184u));
    const dim3 grid(blocks, 2u * ((H + heads - 1u) / heads), seqs);
    return a.cache.head_dim == 64u ? launch_dep(k44_kv8_fill_kernel<64>, grid, dim3(256), 0, pdl, s, a, heads)
                                   : launch_dep(k44_kv8_fill_kernel<128>, grid, dim3(256), 0, pdl, s, a, heads);
}

cudaError_t kv8_attn_setup() {
    for (cudaError_t e : {attn_setup<64, false>(), attn_setup<64, true>(), attn_setup<128, false>(), attn_setup<128, true>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

uint64_t kv8_attn_frag_bytes(uint32_t columns, uint32_t h_kv, uint32_t group, uint32_t head_dim) {
    return (uint64_t)columns * h_kv * (group > 8u ? 2u : 1u) * (head_dim / 16u) * 32u * sizeof(uint4);
}

uint64_t kv8_attn_partial_bytes(uint32_t num_sms, uint32_t group, uint32_t head_dim) {
    const bool wide = group > 8u;
    const uint32_t warps = head_dim == 64u ? (wide ? kWarps<64, true> : kWarps<64, false>) : (wide ? kWarps<128, true> : kWarps<128, false>);
    return (uint64_t)num_sms * warps * 2u * (wide ? 16u : 8u) * (head_dim + 2u) * sizeof(float);
}

cudaError_t launch_kv8_attn(const Kv8AttnArgs &a, uint32_t num_sms, bool pdl, cudaStream_t s) {
    const bool wide = a.h_q / a.cache.h_kv > 8u;
    if (a.cache.head_dim == 64u) return wide ? attn_launch<64, true>(a, num_sms, pdl, s) : attn_launch<64, false>(a, num_sms, pdl, s);
    return wide ? attn_launch<128, true>(a, num_sms, pdl, s) : attn_launch<128, false>(a, num_sms, pdl, s);
}

}  // namespace k44b
