// Probabilities of an answer: per column of a logits tensor [rows][pitch] the log probability of a given row, the entropy of
// the distribution, and the `top` most probable rows (largest value first, the lowest row first among equals).
//
//   M = max_r x_r log2 e,  t_r = x_r log2 e - M,  L = sum_r 2^t_r,  W = sum_r 2^t_r t_r
//   log p_r = ln 2 (t_r - log2 L),   entropy = ln 2 (log2 L - W / L)
//
// t_r is one fused multiply-add; that log2 e is a 32-bit number moves x_r by 1.3e-8 of itself, a quarter of its 32-bit rounding.
//
// Two launches. The first reads the logits once. A warp owns groups of 64 rows. HBM-bound for many columns: the exponentials, 16 per
// cycle and SM, take two thirds of the time of the bytes, so that every other instruction per value counts. The group's maximum is
// taken on packed FP16 pairs, then every value costs one exponential against the largest value so far, without a rescale of its
// own, and half a 32-bit operation each on packed pairs. It leaves (M, L, W) per chunk of rows and the maximum of every group. The
// second launch, one CTA per column, joins the chunks and finds the alternatives exactly: ordered by (maximum, lower rows first), the first `top` of any division of the rows
// into groups hold the `top` largest values, because the best row of each of those groups comes before every row of any other
// group. So it goes from blocks of 512 rows to groups of 64 to rows, and reads only `top` * 64 values again.
//
// FP32 sums over groups, then chunks, then the column (a tree: rounding error grows with its depth, not with the rows). Exponentials are
// the special-function unit's, 2^-22 of each: 7e-8 relative to 64 bits, as much as 32-bit results are rounded.
// 262144 rows, 64 columns, 20 alternatives: 27 us (128256 rows: 16.8); maxima of groups past the 2048th are read twice by the second launch.
#include "k44_decoder.cuh"
#include "k44_ptx.cuh"

namespace k44b {
namespace {

// FP16 bits -> 16-bit order: NaN 1, then -inf .. +inf; both zeros are equal. 0 is left for "no row".
__device__ __forceinline__ uint32_t order_of(uint32_t u) {
    const uint32_t mag = u & 0x7fffu;
    if (mag > 0x7c00u) return 1u;
    return (u & 0x8000u) ? 0x8000u - mag : 0x8000u + mag;
}

__device__ __forceinline__ float value_of(uint32_t order) {
    return __half2float(__ushort_as_half((unsigned short)(order == 1u ? 0x7e00u : order < 0x8000u ? 0x8000u | (0x8000u - order) : order - 0x8000u)));
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// (M, L, W) of two sets of rows together. An empty set, or one without a value above -inf, has M = -inf, L = 0, W = 0.
constexpr float kLeast = -200000.0f;                         // below every finite M, and finite: 0 * t stays 0
__device__ __forceinline__ void join(float &m0, float &l0, float &w0, float m1, float l1, float w1) {
    const float m = fmaxf(m0, m1), base = m == -INFINITY ? 0.f : m;
    const float t0 = fmaxf(m0, kLeast) - base, t1 = fmaxf(m1, kLeast) - base, f0 = fast_exp2(t0), f1 = fast_exp2(t1);
    w0 = fmaf(fmaf(l0, t0, w0), f0, fmaf(l1, t1, w1) * f1);
    l0 = fmaf(l0, f0, l1 * f1);
    m0 = m;
}

// 8 values of a row against the maxima of their columns: l += 2^t, w += 2^t t.
// CLAMP: -inf becomes -65504 on the packed pairs, where that changes nothing (0 * -inf would not be 0; a NaN stays one).
template <bool CLAMP>
__device__ __forceinline__ void add_row(const uint4 &v, const float (&base)[8], float (&l)[8], float (&w)[8]) {
    const __half2 least = __halves2half2(__ushort_as_half((unsigned short)0xfbffu), __ushort_as_half((unsigned short)0xfbffu));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __half2 h = reinterpret_cast<const __half2 *>(&v)[k];
        if (CLAMP) h = __hmax2_nan(h, least);
        const float2 x = __half22float2(h);
        float2 t = ptx::fma2(x, make_float2(kLog2e, kLog2e), make_float2(-base[2 * k], -base[2 * k + 1]));
        const float2 p = make_float2(fast_exp2(t.x), fast_exp2(t.y));
        if (!CLAMP) t = make_float2(fmaxf(t.x, kLeast), fmaxf(t.y, kLeast));
        const float2 l2 = ptx::add2(make_float2(l[2 * k], l[2 * k + 1]), p), w2 = ptx::fma2(p, t, make_float2(w[2 * k], w[2 * k + 1]));
        l[2 * k] = l2.x; l[2 * k + 1] = l2.y;
        w[2 * k] = w2.x; w[2 * k + 1] = w2.y;
    }
}

// A warp's group of 64 rows: `row(i)` gives the lane's 8 values of its i-th row. Adds to (M, L, W) and returns the packed maxima.
template <int CG, typename Row>
__device__ __forceinline__ void add_group(Row row, __half2 (&mx)[4], float (&m)[8], float (&base)[8], bool &low, float (&L)[8], float (&W)[8]) {
    constexpr int I = 2 * CG;
#pragma unroll
    for (int i = 0; i < I; ++i) {                          // of numbers; NaN where a group has nothing else
        const uint4 v = row(i);
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = i ? __hmax2(mx[k], h[k]) : h[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int o = CG; o < 32; o <<= 1) mx[k] = __hmax2(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
    // a column's sums are kept against the largest value so far, which soon stays the same
    bool grown = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 x = __half22float2(mx[k]);
        grown |= x.x * kLog2e > m[2 * k] || x.y * kLog2e > m[2 * k + 1];
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            join(m[k], L[k], W[k], __half2float((k & 1) ? __high2half(mx[k >> 1]) : __low2half(mx[k >> 1])) * kLog2e, 0.f, 0.f);
            base[k] = m[k] == -INFINITY ? 0.f : m[k];
        }
        bool l = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) l |= base[k] < -86000.0f;
        low = __any_sync(0xffffffffu, l);                  // there -65504 is not as good as -inf
    }
    constexpr int U = CG == 8 ? 4 : I, V = CG == 8 ? 1 : I;       // rows in registers are indexed by constants only
    if (!low) {
#pragma unroll U
        for (int i = 0; i < I; ++i) add_row<true>(row(i), base, L, W);
    } else {
#pragma unroll V
        for (int i = 0; i < I; ++i) add_row<false>(row(i), base, L, W);
    }
}

// What a CTA's warps have: one (M, L, W) per column and chunk.
template <int CG, int WARPS>
__device__ __forceinline__ void leave_parts(const LogprobArgs &a, float (&m)[8], float (&L)[8], float (&W)[8]) {
    __shared__ float4 part_s[WARPS][8 * CG];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, cg = lane % CG, rl = lane / CG;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int o = CG; o < 32; o <<= 1) {                            // the lanes of a column have the same maximum
            L[k] += __shfl_xor_sync(0xffffffffu, L[k], o);
            W[k] += __shfl_xor_sync(0xffffffffu, W[k], o);
        }
        if (rl == 0u) part_s[warp][cg * 8u + k] = make_float4(m[k], L[k], W[k], 0.f);
    }
    __syncthreads();
    const uint32_t c = threadIdx.x, col = blockIdx.x * CG * 8u + c;
    if (c < 8u * CG && col < a.columns) {
        float M = part_s[0][c].x, l = part_s[0][c].y, w = part_s[0][c].z;
#pragma unroll 1
        for (int i = 1; i < WARPS; ++i) join(M, l, w, part_s[i][c].x, part_s[i][c].y, part_s[i][c].z);
        a.parts[(uint64_t)col * a.chunks + blockIdx.y] = make_float4(M, l, w, 0.f);
    }
}

// The maxima of a group's 8 columns are in all lanes: lane row rl writes those of its share of them (short: it is once per 64 rows)
template <int CG>
__device__ __forceinline__ void leave_maxima(const LogprobArgs &a, const __half2 (&mx)[4], uint32_t col0, uint32_t rl, uint32_t group) {
    if (rl >= 4u) return;
    const __half2 p = rl < 2u ? (rl == 0u ? mx[0] : mx[1]) : (rl == 2u ? mx[2] : mx[3]);
    const uint32_t u = *reinterpret_cast<const uint32_t *>(&p), col = col0 + 2u * rl;
    uint16_t *to = a.group_max + (uint64_t)col * a.group_stride + group;
    if (col < a.columns) to[0] = (uint16_t)order_of(u & 0xffffu);
    if (col + 1u < a.columns) to[a.group_stride] = (uint16_t)order_of(u >> 16);
}

// Up to 16 columns: CG groups of 8 columns (a lane reads 16 bytes of a row), 32 / CG rows per warp load. A group's rows stay in
// registers between its maximum and its exponentials. Warp w of a chunk takes its groups w, w + 8, ...
template <int CG>
__global__ void __launch_bounds__(256) k44_logprob_parts_kernel(const LogprobArgs a) {
    dep_enter();
    constexpr int I = 2 * CG, RL = 32 / CG;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, cg = lane % CG, rl = lane / CG;
    const uint32_t col0 = (blockIdx.x * CG + cg) * 8u, g_end = min((blockIdx.y + 1u) * a.chunk_groups, a.groups);
    float m[8], base[8], L[8], W[8];
    bool low = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) { m[k] = -INFINITY; base[k] = 0.f; L[k] = 0.f; W[k] = 0.f; }
    for (uint32_t group = blockIdx.y * a.chunk_groups + warp; group < g_end; group += 8u) {
        uint4 v[I];
        const __half *src = a.x + (uint64_t)(group * kLogprobGroup + rl) * a.pitch + col0;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            v[i] = make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);         // rows past the end: probability 0
            if (col0 < a.columns && group * kLogprobGroup + rl + RL * i < a.rows) v[i] = __ldcg(reinterpret_cast<const uint4 *>(src + (uint64_t)(RL * i) * a.pitch));
        }
        __half2 mx[4];
        add_group<CG>([&](int i) -> uint4 { return v[i]; }, mx, m, base, low, L, W);
        leave_maxima<CG>(a, mx, col0, rl, group);
    }
    leave_parts<CG, 8>(a, m, L, W);
}

// More columns: tiles of 64. A warp's groups come as tensor copies of 64 rows x 64 columns (8 KB) and are read from shared memory
// twice (maxima, exponentials). 16 warps with one group each in flight (128256 x 1000 logits, both launches: 65 to 70 us) beat 12 with two
// (70) and 24 with one (73); held in registers, two groups per warp, the compiler spilled 600 bytes a thread (136 us).
constexpr int kTileWarps = 16, kTileStages = 1;
constexpr uint32_t kTileBytes = kLogprobGroup * 64u * 2u, kTileSmem = kTileWarps * kTileStages * kTileBytes + 1024u;

__global__ void __launch_bounds__(kTileWarps * 32, 1) k44_logprob_tiles_kernel(const __grid_constant__ CUtensorMap map, const LogprobArgs a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kTileWarps * kTileStages];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, cg = lane & 7u, rl = lane >> 3;
    const uint32_t col0 = (blockIdx.x * 8u + cg) * 8u, g_end = min((blockIdx.y + 1u) * a.chunk_groups, a.groups);
    uint8_t *ring = smem_raw + ((1024u - (ptx::smem_addr(smem_raw) & 1023u)) & 1023u) + warp * kTileStages * kTileBytes;
    const uint32_t bar0 = ptx::smem_addr(bars) + warp * kTileStages * 8u;
    if (lane == 0u) {
        for (int s = 0; s < kTileStages; ++s) ptx::mbar_init(bar0 + 8u * s, 1);
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&map);
    }
    __syncwarp();
    dep_enter();
    const uint64_t policy = ptx::policy_evict_first();
    uint32_t group = blockIdx.y * a.chunk_groups + warp, ahead = group, issued = 0;
    auto issue = [&]() {                                             // lane 0
        if (ahead >= g_end) return;
        const uint32_t s = issued++ % kTileStages;
        ptx::mbar_arrive_expect_tx(bar0 + 8u * s, kTileBytes);
        ptx::tma_load_2d(ptx::smem_addr(ring) + s * kTileBytes, &map, (int32_t)(blockIdx.x * 64u), (int32_t)(ahead * kLogprobGroup), bar0 + 8u * s, policy);
        ahead += kTileWarps;
    };
    if (lane == 0u)
        for (int s = 0; s < kTileStages; ++s) issue();
    float m[8], base[8], L[8], W[8];
    bool low = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) { m[k] = -INFINITY; base[k] = 0.f; L[k] = 0.f; W[k] = 0.f; }
    bool ok = true;
    for (uint32_t n = 0; group < g_end; group += kTileWarps, ++n) {
        const uint32_t s = n % kTileStages, ph = (n / kTileStages) & 1u;
        bool here = ptx::mbar_try_wait(bar0 + 8u * s, ph);
        if (!here) {
            const long long t0 = clock64();
            while (!(here = ptx::mbar_try_wait(bar0 + 8u * s, ph)) && (unsigned long long)(clock64() - t0) < a.wait_cycles) {}
        }
        ok = __all_sync(0xffffffffu, here ? 1 : 0) != 0;
        if (!ok) break;
        const uint4 *tile = reinterpret_cast<const uint4 *>(ring + s * kTileBytes) + rl * 8u + cg;
        const uint32_t left = a.rows - group * kLogprobGroup;
        __half2 mx[4];
        if (left >= kLogprobGroup) add_group<8>([&](int i) -> uint4 { return tile[32 * i]; }, mx, m, base, low, L, W);
        else add_group<8>([&](int i) -> uint4 { return rl + 4u * i < left ? tile[32 * i] : make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }, mx, m, base, low, L, W);
        __syncwarp();
        if (lane == 0u) issue();
        leave_maxima<8>(a, mx, col0, rl, group);
    }
    if (!ok && lane == 0u) {                                          // gave up: report, wait (bounded) for own copies
        atomicOr(a.status, (uint32_t)ST_TIMEOUT_PRODUCER);
        for (uint32_t i = issued > (uint32_t)kTileStages ? issued - kTileStages : 0u; i < issued; ++i) {
            const long long t0 = clock64();
            bool done = false;
            while (!done && (unsigned long long)(clock64() - t0) < a.wait_cycles) done = ptx::mbar_try_wait(bar0 + 8u * (i % kTileStages), (i / kTileStages) & 1u);
            if (!done) atomicOr(a.status, (uint32_t)ST_TIMEOUT_DRAIN);
        }
    }
    __syncwarp();
    leave_parts<8, kTileWarps>(a, m, L, W);
}

// The `top` largest of the keys that a warp holds, K per lane: lane i gets the i-th. Keys are distinct, or 0 for none. Each lane
// keeps its keys in order, so that a round costs one warp-wide maximum and a shift in the lane that had it.
template <int K>
__device__ __forceinline__ uint32_t warp_top(uint32_t (&key)[K], uint32_t top, uint32_t lane) {
#pragma unroll
    for (int i = 1; i < K; ++i)
#pragma unroll
        for (int j = i; j > 0; --j) {
            const uint32_t hi = max(key[j - 1], key[j]), lo = min(key[j - 1], key[j]);
            key[j - 1] = hi; key[j] = lo;
        }
    uint32_t got = 0;
    for (uint32_t t = 0; t < top; ++t) {
        const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
        if (best == 0u) break;
        if (lane == t) got = best;
        const bool mine = key[0] == best;
#pragma unroll
        for (int i = 0; i + 1 < K; ++i) key[i] = mine ? key[i + 1] : key[i];
        key[K - 1] = mine ? 0u : key[K - 1];
    }
    return got;
}

constexpr int kFinalThreads = 256, kFinalWarps = kFinalThreads / 32, kListGroups = 128, kListRows = 1024;

__global__ void __launch_bounds__(kFinalThreads) k44_logprob_final_kernel(const LogprobArgs a) {
    dep_enter();
    __shared__ float4 red_s[kFinalWarps];
    __shared__ uint32_t list_s[kFinalWarps][kLogprobTop], group_s[kFinalWarps][kLogprobTop], count_s[2], least_s;
    __shared__ __align__(16) uint32_t key_s[kFinalThreads];
    __shared__ unsigned long long row_s[kListRows];
    const uint32_t col = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    // ---- join the chunks ----
    const float4 *parts = a.parts + (uint64_t)col * a.chunks;
    float M = -INFINITY, L = 0.f, W = 0.f, target = 0.f;
    int t = -1;
    if (a.logprobs) t = a.targets[col];
    const bool known = t >= 0 && (uint32_t)t < a.rows;
    if (known && tid == 0u) target = __half2float(a.x[(uint64_t)t * a.pitch + col]);
    for (uint32_t c = tid; c < a.chunks; c += kFinalThreads) {
        const float4 p = __ldcg(parts + c);
        join(M, L, W, p.x, p.y, p.z);
    }
    if (warp * 32u < a.chunks) {
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) {
            const float m1 = __shfl_xor_sync(0xffffffffu, M, o), l1 = __shfl_xor_sync(0xffffffffu, L, o), w1 = __shfl_xor_sync(0xffffffffu, W, o);
            join(M, L, W, m1, l1, w1);
        }
    }
    if (lane == 0u) red_s[warp] = make_float4(M, L, W, 0.f);
    // ---- alternatives: a value that at least `top` rows reach ----
    // Four threads take every 64th group; the top-th largest of the 64 maxima is such a value (where there are as many), and hardly
    // more groups reach it than are needed. Their rows that reach it are listed and ranked by counting.
    const uint16_t *gm = a.group_max + (uint64_t)col * a.group_stride;
    auto key_of = [&](uint32_t g) -> uint32_t { return g < a.groups ? ((uint32_t)__ldcg(gm + g) << 16) | (65535u - g) : 0u; };
    bool listed = false;
    if (a.top) {
        uint32_t mine = 0, key[8];                                      // the first 2048 groups stay in registers
#pragma unroll
        for (int i = 0; i < 8; ++i) key[i] = key_of(i * kFinalThreads + tid);
#pragma unroll
        for (int i = 0; i < 8; ++i) mine = max(mine, key[i]);
        for (uint32_t g = 8u * kFinalThreads + tid; g < a.groups; g += kFinalThreads) mine = max(mine, key_of(g));
        uint32_t bin = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
        bin = max(bin, __shfl_xor_sync(0xffffffffu, bin, 2));
        if (tid == 0u) { count_s[0] = 0u; count_s[1] = 0u; least_s = 1u; }
        if ((tid & 3u) == 0u) key_s[tid >> 2] = bin;
        __syncthreads();
        uint32_t rank = 0;
#pragma unroll
        for (uint32_t i = 0; i < kFinalThreads / 16; ++i) {
            const uint4 o = reinterpret_cast<const uint4 *>(key_s)[i];
            rank += (o.x > bin) + (o.y > bin) + (o.z > bin) + (o.w > bin);
        }
        if (bin && rank == a.top - 1u) least_s = bin;
        __syncthreads();
        const uint32_t least = least_s;
        auto list = [&](uint32_t k) {
            if (k < least) return;
            const uint32_t at = atomicAdd(&count_s[0], 1u);
            if (at < kListGroups) key_s[at] = 65535u - (k & 0xffffu);
        };
        if (mine >= least) {
#pragma unroll
            for (int i = 0; i < 8; ++i) list(key[i]);
            for (uint32_t g = 8u * kFinalThreads + tid; g < a.groups; g += kFinalThreads) list(key_of(g));
        }
        __syncthreads();
        const uint32_t n_groups = count_s[0];
        if (n_groups <= kListGroups) {
#pragma unroll 4
            for (uint32_t place = tid; place < n_groups * kLogprobGroup; place += kFinalThreads) {
                const uint32_t r = key_s[place / kLogprobGroup] * kLogprobGroup + place % kLogprobGroup;
                if (r < a.rows) {
                    const uint32_t o = order_of(__half_as_ushort(a.x[(uint64_t)r * a.pitch + col]));
                    if (o >= least >> 16) {
                        const uint32_t at = atomicAdd(&count_s[1], 1u);
                        if (at < kListRows) row_s[at] = ((unsigned long long)o << 32) | (0xffffffffu - r);
                    }
                }
            }
            __syncthreads();
            listed = count_s[1] <= kListRows;
        }
    }
    if (a.top && !listed) {
        // ---- too many equal values: go down from blocks of 512 rows (8 groups: 16 bytes of the table) to groups to rows, each time
        // taking the first `top` by (maximum, lower rows first); every warp for itself down to the groups ----
        uint32_t best = 0;
        const uint32_t blocks = (a.groups + 7u) / 8u;
        for (uint32_t b0 = 0; b0 < blocks; b0 += 256u) {
            uint32_t key[9];
            key[8] = best;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = b0 + 32u * i + lane;
                key[i] = 0u;
                if (b < blocks) {
                    const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(gm + 8u * b));
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t mx = 0;
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) if (8u * b + e < a.groups) mx = max(mx, (w[e >> 1] >> (16u * (e & 1u))) & 0xffffu);
                    key[i] = (mx << 16) | (65535u - b);
                }
            }
            best = warp_top<9>(key, a.top, lane);
        }
        uint32_t key[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t place = 32u * i + lane, from = __shfl_sync(0xffffffffu, best, place >> 3), g = (65535u - (from & 0xffffu)) * 8u + (place & 7u);
            key[i] = from && g < a.groups ? ((uint32_t)__ldcg(gm + g) << 16) | (65535u - g) : 0u;
        }
        best = warp_top<8>(key, a.top, lane);
        // in the order of their rows, so that a place in the list orders rows too
        const uint32_t g = best ? 65535u - (best & 0xffffu) : 0xffffffffu;
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < 32u; ++i) {
            const uint32_t o = __shfl_sync(0xffffffffu, g, i);
            rank += (o < g || (o == g && i < lane)) ? 1u : 0u;
        }
        group_s[warp][rank] = g;
        __syncwarp();
        // ---- the alternatives: up to 32 groups of 64 rows, 8 per thread ----
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t place = i * kFinalThreads + tid, q = group_s[warp][place / kLogprobGroup], r = q * kLogprobGroup + place % kLogprobGroup;
            key[i] = 0u;
            if (q != 0xffffffffu && r < a.rows) key[i] = (order_of(__half_as_ushort(a.x[(uint64_t)r * a.pitch + col])) << 16) | (65535u - place);
        }
        list_s[warp][lane] = warp_top<8>(key, a.top, lane);
    }
    __syncthreads();
    M = red_s[0].x; L = red_s[0].y; W = red_s[0].z;
#pragma unroll 1
    for (int w = 1; w < kFinalWarps; ++w) join(M, L, W, red_s[w].x, red_s[w].y, red_s[w].z);
    const float log2_l = log2f(L);
    constexpr float kLn2 = 0.69314718055994531f;
    if (tid == 0u) {
        if (a.entropy) a.entropy[col] = (log2_l - W / L) * kLn2;
        if (a.logprobs) a.logprobs[col] = known ? (fmaf(target, kLog2e, -M) - log2_l) * kLn2 : __int_as_float(0x7fc00000);      // no such row: NaN
    }
    if (a.top == 0u) return;
    auto write = [&](uint32_t rank, uint32_t r, uint32_t order) {
        a.top_rows[(uint64_t)rank * a.columns + col] = (int)r;
        a.top_logprobs[(uint64_t)rank * a.columns + col] = (fmaf(value_of(order), kLog2e, -M) - log2_l) * kLn2;
    };
    if (listed) {
        const uint32_t n = count_s[1];
        for (uint32_t i = tid; i < n; i += kFinalThreads) {
            const unsigned long long mine = row_s[i];
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t o = 0; o < n; ++o) rank += row_s[o] > mine ? 1u : 0u;
            if (rank < a.top) write(rank, 0xffffffffu - (uint32_t)mine, (uint32_t)(mine >> 32));
        }
        return;
    }
    if (warp != 0u) return;
    uint32_t key[kFinalWarps];
#pragma unroll
    for (int w = 0; w < kFinalWarps; ++w) key[w] = list_s[w][lane];
    const uint32_t best = warp_top<kFinalWarps>(key, a.top, lane);
    if (lane < a.top) {
        const uint32_t place = 65535u - (best & 0xffffu);
        write(lane, group_s[0][place / kLogprobGroup] * kLogprobGroup + place % kLogprobGroup, best >> 16);
    }
}

}  // namespace

// Chunks: one wave of CTAs, each with at least a group per warp. Up to 16 columns four CTAs of 8 warps fit an SM, wider tensors have
// one of 16 warps.
static uint32_t chunk_groups_of(uint32_t groups, uint32_t columns, uint32_t num_sms) {
    const bool tiles = columns > 16u;
    const uint32_t warps = tiles ? kTileWarps : 8u, ctas = tiles ? std::max(1u, num_sms / ((columns + 63u) / 64u)) : 4u * num_sms;
    return std::max(warps, (groups + ctas - 1u) / ctas);
}

uint64_t logprob_scratch_bytes(uint32_t rows, uint32_t columns, uint32_t num_sms) {
    LogprobArgs a;
    a.rows = rows; a.columns = columns;
    logprob_place(a, nullptr, num_sms);
    return kv8_align((uint64_t)columns * a.chunks * sizeof(float4)) + (uint64_t)columns * a.group_stride * sizeof(uint16_t);
}

void logprob_place(LogprobArgs &a, void *scratch, uint32_t num_sms) {
    a.groups = (a.rows + kLogprobGroup - 1u) / kLogprobGroup;
    a.group_stride = (a.groups + 7u) / 8u * 8u;                           // 16-byte rows
    a.chunk_groups = chunk_groups_of(a.groups, a.columns, num_sms);
    a.chunks = (a.groups + a.chunk_groups - 1u) / a.chunk_groups;
    a.parts = (float4 *)scratch;
    a.group_max = (uint16_t *)((uint8_t *)scratch + kv8_align((uint64_t)a.columns * a.chunks * sizeof(float4)));
}

cudaError_t logprob_setup() { return cudaFuncSetAttribute(k44_logprob_tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem); }

cudaError_t launch_logprobs(const LogprobArgs &a, const CUtensorMap &map, bool pdl, cudaStream_t s) {
    // Few columns: those beyond the plan's are not read, a lane's 16 bytes are 8 columns and most lanes are left to rows. 128256 rows, 20
    // alternatives: 16 columns 14.5 us (tiles 15.2), 32 columns 17.8 (tiles 15.1), so more than 16 take tiles.
    const uint32_t cg = (a.columns + 7u) / 8u;
    cudaError_t e;
    if (cg == 1u) e = launch_dep(k44_logprob_parts_kernel<1>, dim3(1, a.chunks), dim3(256), 0, pdl, s, a);
    else if (cg == 2u) e = launch_dep(k44_logprob_parts_kernel<2>, dim3(1, a.chunks), dim3(256), 0, pdl, s, a);
    else e = launch_dep(k44_logprob_tiles_kernel, dim3((a.columns + 63u) / 64u, a.chunks), dim3(kTileWarps * 32), kTileSmem, pdl, s, map, a);
    if (e == cudaSuccess) e = launch_dep(k44_logprob_final_kernel, dim3(a.columns), dim3(kFinalThreads), 0, pdl, s, a);
    return e;
}

}  // namespace k44b
