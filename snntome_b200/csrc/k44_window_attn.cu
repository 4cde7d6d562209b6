// Prompt attention with a sliding window and sinks: rotary embedding and causal grouped-query attention of every sequence of a
// prompt plan (blocks of seq_len columns, any length), on the fifth-generation tensor cores.
//
//   visible(t, c):  s0 <= c <= t  and  (window == 0  or  c > t - window  or  c < s0 + sinks),   s0 = first column of t's sequence
//   o_t = sum_c softmax_c(q_t . k_c / sqrt(D)) v_c
//
// Two launches. The first rotates k and lays it out token by token (the rows a tensor-core operand wants), and copies v; q, k and v
// on the canvas stay as they are. The second is the attention: a CTA owns 128 columns of one query head, rotates its q on the way
// into shared memory (in the first launch, written and read again, q cost 2 us more for four prompts of 1000) and walks the tiles
// of 64 keys that any of its columns sees — hidden tiles are never read. Tiles are cut at multiples of 64 canvas
// columns whatever the sequences' lengths, so that every copy is aligned; sequences that end inside a tile cost a mask.
#include "k44_decoder.cuh"
#include "k44_ptx.cuh"

namespace k44b {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ bool finite_bits(uint32_t h) { return (h & 0x7c00u) != 0x7c00u; }

// ---- operands ---------------------------------------------------------------------------------------------------------------
// CTA = 64 columns of a few heads of k, or of one head of v. Columns behind the plan's last one become zero. Values of v that are
// not finite become zero too, and their tile is flagged: a hidden column has weight 0, but 0 * inf is not 0, so such values must not reach the
// tensor cores; the attention adds them to the columns that do see them, whatever their weight. A flagged tile leaves a word of 64 bits per dimension for the
// columns that hold +inf (or NaN) and one for -inf (or NaN): a column of the output needs an AND with what it sees, not the values
// (2048 columns, 8 heads on 2 of 64, one infinity for all to see: 47 us without, 1867 with the values read, 61 with the words). The rotated q and k, and the weights, are rounded to FP16, the
// tensor cores' type: 2^-11 of each, so some 4e-4 of the output's size, of the order of its own rounding to FP16. q and k are held at
// half their size there: a pair of FP16 numbers may be sqrt(2) longer than the largest one, and halves are exact down to 2^-13.
template <int D>
__global__ void __launch_bounds__(256) k44_window_operands_kernel(const WindowAttnArgs a, uint32_t heads) {
    asm volatile("griddepcontrol.wait;" ::: "memory");              // in this order: the attention reads q before it waits itself
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int ROW = 64 + 2;                                     // 33 words: pairs 8 rows apart fall on different banks
    __shared__ __align__(16) __half xs[D * ROW];
    const uint32_t tile = blockIdx.x, tid = threadIdx.x, col0 = tile * 64u, turned = (a.h_kv + heads - 1u) / heads;
    uint32_t h = blockIdx.y * heads;
    if (blockIdx.y >= turned) {
        h = blockIdx.y - turned;
        const __half *src = a.v + (uint64_t)h * D * a.pitch + col0;
        __half *dst = a.v_rows + (uint64_t)h * D * a.pitch + col0;
        uint32_t bad = 0;
        for (uint32_t e = tid; e < D * 8u; e += 256u) {
            const uint32_t d = e >> 3, c = (e & 7u) * 8u;
            uint4 x = __ldcg(reinterpret_cast<const uint4 *>(src + (uint64_t)d * a.pitch + c));
            uint32_t *w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c0 = col0 + c + 2u * i;
                uint32_t keep = (c0 < a.columns ? 0xffffu : 0u) | (c0 + 1u < a.columns ? 0xffff0000u : 0u);
                w[i] &= keep;
                if (!finite_bits(w[i])) { bad = 1u; w[i] &= 0xffff0000u; }
                if (!finite_bits(w[i] >> 16)) { bad = 1u; w[i] &= 0xffffu; }
            }
            *reinterpret_cast<uint4 *>(dst + (uint64_t)d * a.pitch + c) = x;
        }
        const int any = __syncthreads_or((int)bad);
        if (tid == 0u) a.v_flags[h * (a.pitch / 64u) + tile] = any ? 1u : 0u;
        if (!any) return;
        uint4 *marks = a.v_marks + ((uint64_t)h * (a.pitch / 64u) + tile) * D;
        for (uint32_t e = tid; e < D * 8u; e += 256u) {                      // eight neighbours hold a dimension
            const uint32_t d = e >> 3, c = (e & 7u) * 8u;
            const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(src + (uint64_t)d * a.pitch + c));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t up = 0, down = 0;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                const uint32_t v = w[i >> 1] >> (16u * (i & 1u)) & 0xffffu;
                if (finite_bits(v) || col0 + c + i >= a.columns) continue;
                if (v != 0xfc00u) up |= 1u << i;
                if (v != 0x7c00u) down |= 1u << i;
            }
            up <<= c & 31u; down <<= c & 31u;
            uint32_t m[4] = {c < 32u ? up : 0u, c < 32u ? 0u : up, c < 32u ? down : 0u, c < 32u ? 0u : down};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) m[i] |= __shfl_xor_sync(0xffffffffu, m[i], o);
            if ((e & 7u) == 0u) marks[d] = make_uint4(m[0], m[1], m[2], m[3]);
        }
        return;
    }
    // A thread owns one token and 8 rotation pairs (16 bytes of either half of the token's row); neighbours own the next pairs, so that
    // table and rows are read and written in whole lines. Its angles serve every head of the CTA.
    constexpr uint32_t PER = D / 16, TOKENS = 256u / PER, ROUNDS = 64u / TOKENS;
    const uint32_t part = tid % PER, p0 = part * 8u;
    float2 cs[ROUNDS][8];
#pragma unroll
    for (uint32_t n = 0; n < ROUNDS; ++n) {
        const uint32_t col = col0 + n * TOKENS + tid / PER;
        const float4 *from = reinterpret_cast<const float4 *>(a.rope + (uint64_t)(col % a.seq_len) * (D / 2) + p0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = col < a.columns ? __ldg(from + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            cs[n][2 * i] = make_float2(kWindowHeld * v.x, kWindowHeld * v.y);
            cs[n][2 * i + 1] = make_float2(kWindowHeld * v.z, kWindowHeld * v.w);
        }
    }
    const uint32_t h0 = h, h1 = min(h0 + heads, a.h_kv);
    uint4 next[D / 32];                                                      // the rows of the head after this one
    auto fetch = [&](uint32_t i) {
        const __half *src = a.k + (uint64_t)i * D * a.pitch + col0;
#pragma unroll
        for (int n = 0; n < D / 32; ++n) { const uint32_t e = 256u * n + tid; next[n] = __ldcg(reinterpret_cast<const uint4 *>(src + (uint64_t)(e >> 3) * a.pitch + (e & 7u) * 8u)); }
    };
    fetch(h0);
    for (h = h0; h < h1; ++h) {
        __half *dst = a.k_rows + ((uint64_t)h * a.pitch + col0) * D;
        if (h != h0) __syncthreads();
#pragma unroll
        for (int n = 0; n < D / 32; ++n) {
            const uint32_t e = 256u * n + tid;
            uint32_t *to = reinterpret_cast<uint32_t *>(xs + (e >> 3) * ROW + (e & 7u) * 8u);
            to[0] = next[n].x; to[1] = next[n].y; to[2] = next[n].z; to[3] = next[n].w;
        }
        __syncthreads();
        if (h + 1u < h1) fetch(h + 1u);
#pragma unroll
        for (uint32_t n = 0; n < ROUNDS; ++n) {
            const uint32_t tok = n * TOKENS + tid / PER;
            const bool live = col0 + tok < a.columns;
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u[2], v[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = __half2float(xs[(p0 + 2 * i + e) * ROW + tok]), y = __half2float(xs[(p0 + 2 * i + e + D / 2) * ROW + tok]);
                    const float2 r = cs[n][2 * i + e];
                    u[e] = live ? x * r.x - y * r.y : 0.f;
                    v[e] = live ? x * r.y + y * r.x : 0.f;
                }
                const __half2 l2 = __floats2half2_rn(u[0], u[1]), h2 = __floats2half2_rn(v[0], v[1]);
                lo[i] = *reinterpret_cast<const uint32_t *>(&l2);
                hi[i] = *reinterpret_cast<const uint32_t *>(&h2);
            }
            *reinterpret_cast<uint4 *>(dst + (uint64_t)tok * D + p0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            *reinterpret_cast<uint4 *>(dst + (uint64_t)tok * D + p0 + D / 2) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        }
    }
}

// ---- attention -----------------------------------------------------------------------------------------------------------------
// Warp 0 copies (TMA), one thread of warp 1 issues the MMAs, warps 2-5 are the softmax: a thread owns one column (= TMEM lane).
// Tensor memory: a buffer of 64 columns of scores, over whose first half the weights are written as FP16 pairs once the scores are
// read (the A operand of the second product), and D columns of output. 128 x 64 exponentials take 512 cycles of the SM's 16 per
// cycle, the two products of a tile 256 (D = 64) or 512 at 4096 multiplications a cycle: at D = 128 the tensor cores have as much to do
// as the exponential unit (28 and 25 % busy), at D = 64 half as much (25 and 45 %). Nothing of it overlaps within one column's chain (scores, maximum, weights, output), so
// what counts is how many chains an SM holds: D = 64 runs four CTAs per SM (128 columns of tensor memory each, 80 registers, the
// second half of the scores read twice, one stage of keys and values), D = 128 two, each with a second buffer in which the next
// scores are made meanwhile. Both launches, 8192 tokens, 32 heads on 8, window 1024, D = 64: 154 to 157 us (with two stages 160, three CTAs
// of more registers 172, two CTAs with two buffers 164, two warps to a row 180); four prompts of 1000, 32 heads on 8, D = 128: 87 us
// (with one buffer 107). Without its exponentials the former still takes 142, without exponentials and products 128: in this kernel the
// chain's waits and reads of tensor memory bound it. Scores four times as large as these unit normal queries and keys give, whose maxima
// keep growing, take 179 and 119 us: the output is read and written back at every rescale.
// The output is rescaled only when a column's maximum has grown by more than 2^8 since the last time: weights up to 256 are as
// exact in FP16 as weights up to 1, and the sum is kept against the same maximum. Weights are held times 2^7 (up to 2^15), so that FP16
// has whole precision down to 2^-21 and something down to 2^-32 of the maximum: thousands of keys far below a first one still add up.
template <int D> struct Shape {
    static constexpr uint32_t HF = D / 64;
    static constexpr uint32_t Q_BYTES = 128u * D * 2u, K_BYTES = 64u * D * 2u, V_BYTES = K_BYTES;
    static constexpr uint32_t STAGES = D == 64 ? 1u : 2u, CTAS = D == 64 ? 4u : 2u, BUFFERS = D == 64 ? 1u : 2u;
    static constexpr bool HOLD = D != 64;                        // registers for all 64 scores
    static constexpr uint32_t O_COL = BUFFERS * 64u, TMEM_COLS = O_COL + D > 128u ? 256u : 128u;
    static constexpr uint32_t SMEM = Q_BYTES + STAGES * (K_BYTES + V_BYTES) + 1024u + 256u;
};
constexpr uint32_t kThreads = 192, kKeys = 64;
constexpr float kWeightBits = 7.f;

__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    // K-major rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)1u << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the largest of three
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// bits from .. to of a word (either may lie outside it)
__device__ __forceinline__ uint32_t bits(int from, int to) {
    if (to < 0 || from > 31 || from > to) return 0u;
    return (0xffffffffu >> (31 - min(to, 31))) & (0xffffffffu << max(from, 0));
}

// what column t sees: [lo, t] and [s0, s0 + sk)
struct Sight {
    uint32_t t, s0, lo, sk;
    __device__ __forceinline__ Sight(const WindowAttnArgs &a, uint32_t column) : t(column) {
        s0 = t / a.seq_len * a.seq_len;
        lo = a.window && t - s0 >= a.window ? t - a.window + 1u : s0;
        sk = lo > s0 ? min(a.sinks, lo - s0) : 0u;
    }
    __device__ __forceinline__ uint32_t seen(uint32_t c0) const {           // of the 32 keys from c0
        const int at = (int)c0;
        return bits((int)lo - at, (int)t - at) | bits((int)s0 - at, (int)(s0 + sk) - 1 - at);
    }
};

template <int D>
__global__ void __launch_bounds__(kThreads, Shape<D>::CTAS)
k44_window_attn_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __grid_constant__ CUtensorMap o_map, const WindowAttnArgs a) {
    using S = Shape<D>;
    constexpr uint32_t HF = S::HF, ST = S::STAGES, NB = S::BUFFERS, kOCol = S::O_COL, kTmemCols = S::TMEM_COLS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = q_smem + S::Q_BYTES, v_smem = k_smem + ST * S::K_BYTES, ctl = v_smem + ST * S::V_BYTES;
    const uint32_t q_full = ctl, k_full = ctl + 8u, k_empty = k_full + 8u * ST, v_full = k_empty + 8u * ST, v_empty = v_full + 8u * ST;
    const uint32_t s_full = v_empty + 8u * ST, p_full = s_full + 16u, pv_done = p_full + 16u;
    uint8_t *ctl_ptr = smem_raw + (ctl - ptx::smem_addr(smem_raw));
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(ctl_ptr + 192), *abort_word = tmem_slot + 1, *flagged = tmem_slot + 2;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 128);
        for (uint32_t s = 0; s < ST; ++s) {
            ptx::mbar_init(k_full + 8u * s, 1); ptx::mbar_init(k_empty + 8u * s, 1);
            ptx::mbar_init(v_full + 8u * s, 1); ptx::mbar_init(v_empty + 8u * s, 1);
        }
        for (uint32_t b = 0; b < 2u; ++b) { ptx::mbar_init(s_full + 8u * b, 1); ptx::mbar_init(p_full + 8u * b, 128); ptx::mbar_init(pv_done + 8u * b, 1); }
        *abort_word = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_addr(const_cast<uint32_t *>(tmem_slot)), kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait_for(bar, parity, 20000u)) {
            if (*abort_word != 0u) return false;
            if ((unsigned long long)(clock64() - t0) > a.wait_cycles) return false;
        }
        return true;
    };
    const uint32_t hq = blockIdx.x, qt = gridDim.y - 1u - blockIdx.y, hk = hq / (a.h_q / a.h_kv);      // the longest rows first
    const uint32_t t_first = qt * 128u;
    // ---- q, rotated, as the rows of the first product's A operand ----
    // A thread owns two neighbouring columns and every other group of 8 rotation pairs, so that a warp reads whole lines of the canvas.
    // The table's cosines and sines are half their size, and so is q (multiplied here instead, it cost 2 us of four prompts of 1000).
    // The launch of the operands starts this one once what came before it is done, so q is there before the wait below.
    if (warp >= 2u) {
        const uint32_t row = (warp & 1u) * 64u + 2u * lane, t = t_first + row;
        const bool live0 = t < a.columns, live1 = t + 1u < a.columns;
        const __half *q = a.q + (uint64_t)hq * D * a.pitch + t;
        const float2 *r0 = a.rope_pairs + (live0 ? t % a.seq_len : 0u), *r1 = a.rope_pairs + (live1 ? (t + 1u) % a.seq_len : 0u);
#pragma unroll
        for (uint32_t p0 = (warp & 2u) * 4u; p0 < D / 2u; p0 += 16u) {
            uint32_t x[8], y[8];
            float2 c0[8], c1[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = live0 ? __ldg(reinterpret_cast<const uint32_t *>(q + (uint64_t)(p0 + i) * a.pitch)) : 0u;
                y[i] = live0 ? __ldg(reinterpret_cast<const uint32_t *>(q + (uint64_t)(p0 + i + D / 2u) * a.pitch)) : 0u;
                c0[i] = __ldg(r0 + (uint64_t)(p0 + i) * a.positions);
                c1[i] = __ldg(r1 + (uint64_t)(p0 + i) * a.positions);
            }
            uint32_t w[4][4];                                               // [column, half][pairs]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 u[2], v[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[2 * i + e])), g = __half22float2(*reinterpret_cast<const __half2 *>(&y[2 * i + e]));
                    const float2 a0 = c0[2 * i + e], a1 = c1[2 * i + e];
                    u[e] = make_float2(f.x * a0.x - g.x * a0.y, f.y * a1.x - g.y * a1.y);
                    v[e] = make_float2(f.x * a0.y + g.x * a0.x, f.y * a1.y + g.y * a1.x);
                }
                const __half2 h[4] = {__floats2half2_rn(u[0].x, u[1].x), __floats2half2_rn(v[0].x, v[1].x), __floats2half2_rn(u[0].y, u[1].y), __floats2half2_rn(v[0].y, v[1].y)};
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k][i] = k < 2 || live1 ? *reinterpret_cast<const uint32_t *>(&h[k]) : 0u;
            }
            uint8_t *rows = smem_raw + (q_smem - ptx::smem_addr(smem_raw));
#pragma unroll
            for (int k = 0; k < 4; ++k) {                                   // 16 bytes each, in the 128-byte swizzle
                const uint32_t n = row + (k >> 1), d = p0 + (k & 1) * (D / 2u);
                *reinterpret_cast<uint4 *>(rows + (d >> 6) * 16384u + n * 128u + ((((d & 63u) >> 3) ^ (n & 7u)) << 4)) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
            }
        }
        ptx::fence_proxy_async();
        ptx::mbar_arrive(q_full);
    }
    dep_enter();
    // ---- which tiles of keys ----
    const uint32_t t_last = min(t_first + 127u, a.columns - 1u);
    const uint32_t s_first = t_first / a.seq_len * a.seq_len;                       // start of the first column's sequence
    const bool one_seq = t_last - s_first < a.seq_len;
    uint32_t lo_first = s_first;
    if (a.window && t_first - s_first >= a.window) lo_first = t_first - a.window + 1u;
    const uint32_t w_tile = lo_first / kKeys, sink_tile = s_first / kKeys;
    uint32_t n_sink = 0;
    if (a.window && a.sinks && sink_tile < w_tile) n_sink = min(w_tile, (s_first + min(a.sinks, a.seq_len) - 1u) / kKeys + 1u) - sink_tile;
    const uint32_t n = n_sink + (t_last / kKeys - w_tile + 1u);
    auto key_tile = [&](uint32_t j) -> uint32_t { return j < n_sink ? sink_tile + j : w_tile + (j - n_sink); };

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            const uint64_t keep = ptx::policy_evict_last();
            uint32_t k_issued = 0, v_issued = 0;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t s = j % ST, ph = (j / ST) & 1u, c0 = key_tile(j) * kKeys;
                if (!(ok = wait(k_empty + 8u * s, ph ^ 1u))) break;
                ptx::mbar_arrive_expect_tx(k_full + 8u * s, S::K_BYTES);
                for (uint32_t f = 0; f < HF; ++f) ptx::tma_load_2d(k_smem + s * S::K_BYTES + f * 8192u, &k_map, (int32_t)(64u * f), (int32_t)(hk * a.pitch + c0), k_full + 8u * s, keep);
                ++k_issued;
                if (!(ok = wait(v_empty + 8u * s, ph ^ 1u))) break;
                ptx::mbar_arrive_expect_tx(v_full + 8u * s, S::V_BYTES);
                ptx::tma_load_2d(v_smem + s * S::V_BYTES, &v_map, (int32_t)c0, (int32_t)(hk * D), v_full + 8u * s, keep);
                ++v_issued;
            }
            if (!ok) {
                if (*abort_word == 0u) atomicOr(a.status, (uint32_t)ST_TIMEOUT_PRODUCER);
                *abort_word = 1u;
                // wait (bounded) for this CTA's copies in flight before its shared memory goes away
                auto drain = [&](uint32_t bar, uint32_t parity) {
                    const long long t0 = clock64();
                    bool done = false;
                    while (!done && (unsigned long long)(clock64() - t0) < a.wait_cycles) done = ptx::mbar_try_wait(bar, parity);
                    if (!done) atomicOr(a.status, (uint32_t)ST_TIMEOUT_DRAIN);
                };
                for (uint32_t i = k_issued > ST ? k_issued - ST : 0u; i < k_issued; ++i) drain(k_full + 8u * (i % ST), (i / ST) & 1u);
                for (uint32_t i = v_issued > ST ? v_issued - ST : 0u; i < v_issued; ++i) drain(v_full + 8u * (i % ST), (i / ST) & 1u);
            }
        }
        __syncwarp();
        bool any = false;                                                       // of this CTA's tiles with values that are not finite
        for (uint32_t j = lane; j < n; j += 32u) any |= a.v_flags[hk * (a.pitch / 64u) + key_tile(j)] != 0u;
        any = __any_sync(0xffffffffu, any) != 0;
        if (lane == 0) *flagged = any ? 1u : 0u;
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc_s = (1u << 4) | ((kKeys >> 3) << 17) | ((128u >> 4) << 24), idesc_o = (1u << 4) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
            auto scores = [&](uint32_t j) -> bool {
                const uint32_t s = j % ST, to = tmem + j % NB * kKeys;
                if (!wait(k_full + 8u * s, (j / ST) & 1u)) return false;
                ptx::tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < D / 16u; ++k)
                    ptx::umma_f16(to, desc_sw128(q_smem + (k >> 2) * 16384u) + (k & 3u) * 2u, desc_sw128(k_smem + s * S::K_BYTES + (k >> 2) * 8192u) + (k & 3u) * 2u, idesc_s, k != 0u ? 1u : 0u);
                ptx::umma_commit(k_empty + 8u * s);
                ptx::umma_commit(s_full + 8u * (j % NB));
                return true;
            };
            ok = wait(q_full, 0u) && scores(0u) && (NB == 1u || n < 2u || scores(1u));
            for (uint32_t j = 0; j < n && ok; ++j) {
                const uint32_t s = j % ST;
                if (!(ok = wait(v_full + 8u * s, (j / ST) & 1u) && wait(p_full + 8u * (j % NB), (j / NB) & 1u))) break;
                ptx::tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < kKeys / 16u; ++k)
                    ptx::umma_f16_a_tmem(tmem + kOCol, tmem + j % NB * kKeys + 8u * k, desc_sw128(v_smem + s * S::V_BYTES) + k * 2u, idesc_o, (j != 0u || k != 0u) ? 1u : 0u);
                ptx::umma_commit(v_empty + 8u * s);
                ptx::umma_commit(pv_done + 8u * (j & 1u));
                if (j + NB < n) ok = scores(j + NB);                        // over the weights that the product before it has read
            }
            if (!ok) {
                if (*abort_word == 0u) atomicOr(a.status, (uint32_t)ST_TIMEOUT_MMA);
                *abort_word = 1u;
            }
        }
        __syncwarp();
    } else {
        const uint32_t quarter = warp & 3u, row = quarter * 32u + lane, t = t_first + row;
        const uint32_t lane_base = tmem + ((quarter * 32u) << 16);
        const float mul = rsqrtf((float)D) * kLog2e / (kWindowHeld * kWindowHeld);
        const Sight sight(a, t);
        // Scores j are made after the product j - BUFFERS, so a warp that has seen them knows of the products up to j - 2 at least. A parity tells
        // two phases apart: with one barrier for all products, a warp ahead of the others would take the end of product j - 3 for
        // that of j - 1. So odd and even products have a barrier each.
        auto product_done = [&](uint32_t j) -> bool { return wait(pv_done + 8u * (j & 1u), (j >> 1) & 1u); };
        float m = -INFINITY, l = 0.f;                                     // maximum that the weights are kept against (scaled), their sum
        for (uint32_t j = 0; j < n && ok; ++j) {
            const uint32_t c0 = key_tile(j) * kKeys, from = lane_base + j % NB * kKeys;
            // nothing to hide: all keys before all columns, inside every column's window (or among the sinks), one sequence
            const bool whole = one_seq && c0 + kKeys - 1u <= t_first && c0 >= s_first &&
                               (a.window == 0u || t_first + 127u < c0 + a.window || c0 + kKeys <= s_first + a.sinks);
            ok = __all_sync(0xffffffffu, wait(s_full + 8u * (j % NB), (j / NB) & 1u) ? 1 : 0) != 0;
            if (!ok) break;
            ptx::tc_fence_after();
            uint32_t r[32], r2[S::HOLD ? 32 : 1];                              // scores of the first 32 keys, and, where registers allow, of the others
            // Of 32 columns and 32 keys on an edge most see all or nothing: those need no mask, these no exponentials.
            const uint32_t see0 = whole ? ~0u : sight.seen(c0), see1 = whole ? ~0u : sight.seen(c0 + 32u);
            const bool any0 = whole || __any_sync(0xffffffffu, see0 != 0u), any1 = whole || __any_sync(0xffffffffu, see1 != 0u);
            const bool all0 = whole || __all_sync(0xffffffffu, see0 == ~0u), all1 = whole || __all_sync(0xffffffffu, see1 == ~0u);
            auto hide = [&](uint32_t (&x)[32], uint32_t see) {
#pragma unroll
                for (int i = 0; i < 32; ++i) if (!(see & (1u << i))) x[i] = 0xff800000u;
            };
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // short chains
            auto largest = [&](const uint32_t (&x)[32]) {
#pragma unroll
                for (int i = 0; i < 16; ++i) top[i & 3] = max3(top[i & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 16]));
            };
            if constexpr (!S::HOLD) {
                if (any1) {
                    ptx::tmem_ld_32x32(from + 32u, r);
                    ptx::tmem_ld_wait();
                    if (!all1) hide(r, see1);
                    largest(r);
                }
                if (any0) {
                    ptx::tmem_ld_32x32(from, r);
                    ptx::tmem_ld_wait();
                }
            } else {
                ptx::tmem_ld_32x32(from, r);
                ptx::tmem_ld_32x32(from + 32u, r2);
                ptx::tmem_ld_wait();
                if (!all1) hide(r2, see1);
                if (any1) largest(r2);
            }
            if (any0) {
                if (!all0) hide(r, see0);
                largest(r);
            }
            const float mx = max3(fmaxf(top[0], top[1]), top[2], top[3]) * mul;
            if (__any_sync(0xffffffffu, mx > m + 8.0f || (m == -INFINITY && mx != -INFINITY))) {
                const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : fast_exp2(m - mn);
                m = mn;
                l *= f;
                if (j != 0u) {
                    ok = __all_sync(0xffffffffu, product_done(j - 1u) ? 1 : 0) != 0;       // the product before this one still adds to the output
                    if (!ok) break;
                    ptx::tc_fence_after();
#pragma unroll 1
                    for (uint32_t d0 = 0; d0 < D; d0 += 32u) {
                        uint32_t o[32];
                        ptx::tmem_ld_32x32(lane_base + kOCol + d0, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        ptx::tmem_st_32x32(lane_base + kOCol + d0, o);
                    }
                }
            }
            const float shift = m == -INFINITY ? 0.f : m - kWeightBits;
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            auto weights = [&](const uint32_t (&x)[32], bool any, uint32_t to) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = 0u;
                if (any) {
                    const float2 mul2 = make_float2(mul, mul), shift2 = make_float2(-shift, -shift);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 e = ptx::fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), mul2, shift2);
                        e.x = fast_exp2(e.x); e.y = fast_exp2(e.y);
                        sum[i & 1] = ptx::add2(sum[i & 1], e);
                        const __half2 h = __floats2half2_rn(e.x, e.y);
                        p[i] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                }
                ptx::tmem_st_32x16(to, p);
            };
            weights(r, any0, from);                                        // over scores that have been read: those of 32 .. 63 are still there
            if constexpr (!S::HOLD) {
                if (any1) {
                    ptx::tmem_ld_32x32(from + 32u, r);
                    ptx::tmem_ld_wait();
                    if (!all1) hide(r, see1);
                }
                weights(r, any1, from + 16u);
            } else weights(r2, any1, from + 16u);
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(p_full + 8u * (j % NB));
        }
        if (ok) ok = __all_sync(0xffffffffu, product_done(n - 1u) ? 1 : 0) != 0;
        const bool tile = t_first + 128u <= a.columns;
        if (ok) {
            ptx::tc_fence_after();
            const float inv = 1.0f / l;
            // Rows of the output are columns of the canvas: 2 bytes per lane and dimension, 128 stores of 64 bytes each per warp, which took
            // 4500 cycles per item (D = 128). Whole tiles go through the shared memory that held q and out with tensor copies instead.
            __half *const out_s = reinterpret_cast<__half *>(smem_raw + (q_smem - ptx::smem_addr(smem_raw)));      // [half of the columns][dimension][64]
            __half *dst = tile ? out_s + (row >> 6) * (D * 64u) + (row & 63u) : a.out + (uint64_t)hq * D * a.pitch + t;
            const uint64_t step = tile ? 64u : a.pitch;
#pragma unroll 1
            for (uint32_t d0 = 0; d0 < D; d0 += 32u) {
                uint32_t o[32];
                ptx::tmem_ld_32x32(lane_base + kOCol + d0, o);
                ptx::tmem_ld_wait();
                if (t < a.columns) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) dst[(uint64_t)(d0 + i) * step] = __float2half_rn(__uint_as_float(o[i]) * inv);
                }
            }
            if (tile) {
                ptx::fence_proxy_async();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (threadIdx.x == 64u && *abort_word == 0u) {
                    for (uint32_t f = 0; f < 2u; ++f) ptx::tma_store_2d(&o_map, (int32_t)(t_first + 64u * f), (int32_t)(hq * D), q_smem + f * (D * 128u));
                    ptx::bulk_commit_group();
                    ptx::bulk_wait_group<0>();
                }
            }
        } else {
            if (lane == 0) {
                if (*abort_word == 0u) atomicOr(a.status, (uint32_t)ST_TIMEOUT_EPILOGUE);
                *abort_word = 1u;
            }
            __syncwarp();
            if (tile) asm volatile("bar.arrive 1, 128;" ::: "memory");         // a warp that came through may wait for this one
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 1) ptx::tmem_dealloc(tmem, kTmemCols);
    // Values that were kept from the tensor cores: a column that sees one gets it, on the canvas, where the output is by now. Here, because it
    // hardly ever runs and took registers from the softmax (4 us of four prompts of 1000, 5 of 8192 tokens; here 1 and nothing).
    if (*flagged == 0u || *abort_word != 0u || threadIdx.x >= 128u || t_first + threadIdx.x >= a.columns) return;
    ptx::fence_proxy_async();
    const Sight sight(a, t_first + threadIdx.x);
#pragma unroll 1
    for (uint32_t j = 0; j < n; ++j) {
        const uint32_t kt = key_tile(j);
        if (a.v_flags[hk * (a.pitch / 64u) + kt] == 0u) continue;
        const uint32_t see0 = sight.seen(kt * kKeys), see1 = sight.seen(kt * kKeys + 32u);
        const uint4 *marks = a.v_marks + ((uint64_t)hk * (a.pitch / 64u) + kt) * D;
        __half *dst = a.out + (uint64_t)hq * D * a.pitch + sight.t;
#pragma unroll 4
        for (uint32_t d = 0; d < D; ++d, dst += a.pitch) {
            const uint4 w = marks[d];
            const bool up = ((w.x & see0) | (w.y & see1)) != 0u, down = ((w.z & see0) | (w.w & see1)) != 0u;
            if (up || down) *dst = __float2half_rn(__half2float(*dst) + (up ? INFINITY : 0.f) + (down ? -INFINITY : 0.f));
        }
    }
}

}  // namespace

uint64_t window_attn_scratch_bytes(uint32_t pitch, uint32_t h_kv, uint32_t head_dim) {
    const uint64_t row = (uint64_t)pitch * head_dim * 2u;
    return 2u * kv8_align(h_kv * row) + kv8_align((uint64_t)h_kv * (pitch / 64u) * 4u) + (uint64_t)h_kv * (pitch / 64u) * head_dim * sizeof(uint4);
}

void window_attn_place(WindowAttnArgs &a, void *scratch) {
    const uint64_t row = (uint64_t)a.pitch * a.head_dim * 2u;
    uint8_t *p = (uint8_t *)scratch;
    a.k_rows = (__half *)p; p += kv8_align(a.h_kv * row);
    a.v_rows = (__half *)p; p += kv8_align(a.h_kv * row);
    a.v_flags = (uint32_t *)p; p += kv8_align((uint64_t)a.h_kv * (a.pitch / 64u) * 4u);
    a.v_marks = (uint4 *)p;
}

cudaError_t window_attn_setup() {
    cudaError_t e = cudaFuncSetAttribute(k44_window_attn_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<64>::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k44_window_attn_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<128>::SMEM);
    return e;
}

cudaError_t launch_window_attn(const WindowAttnArgs &a, const WindowAttnMaps &m, bool pdl, cudaStream_t s) {
    // operands for whole tiles of 128 columns (what lies behind the last column is zero, not whatever the scratch held)
    const uint32_t tiles = (a.columns + 127u) / 128u;
    const uint32_t wide = std::min(2u * tiles, a.pitch / 64u), turned = a.h_kv;
    // several heads per CTA (they share the angles, and one head's rows load while another's are turned) where that leaves CTAs enough:
    // 8192 tokens, 32 heads on 32: 175 us for both launches, with one head per CTA 180. Enough: four for each of 148 SMs.
    const uint32_t heads = std::max(1u, std::min(8u, wide * turned / 592u));
    const dim3 g1(wide, (turned + heads - 1u) / heads + a.h_kv), g2(a.h_q, tiles);
    cudaError_t e;
    if (a.head_dim == 64u) {
        e = launch_dep(k44_window_operands_kernel<64>, g1, dim3(256), 0, pdl, s, a, heads);
        if (e == cudaSuccess) e = launch_dep(k44_window_attn_kernel<64>, g2, dim3(kThreads), Shape<64>::SMEM, pdl, s, m.k, m.v, m.out, a);
    } else {
        e = launch_dep(k44_window_operands_kernel<128>, g1, dim3(256), 0, pdl, s, a, heads);
        if (e == cudaSuccess) e = launch_dep(k44_window_attn_kernel<128>, g2, dim3(kThreads), Shape<128>::SMEM, pdl, s, m.k, m.v, m.out, a);
    }
    return e;
}

}  // namespace k44b
