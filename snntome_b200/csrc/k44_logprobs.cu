// Probabilities of an answer: per column of a logits tensor [rows][pitch] the log probability of a given row, the entropy of
// the distribution, and the `top` most probable rows (largest value first, the lowest row first among equals).
//
//   m = max_r x_r,  L = sum_r e^(x_r - m),  W = sum_r e^(x_r - m) (x_r - m)
//   log p_r = x_r - m - ln L,   entropy = ln L - W / L
//
// Two launches. The first reads the logits once: a warp owns groups of 64 rows; the group's maximum is taken on packed FP16
// pairs, then every value costs one exponential against that maximum, so no running rescale is needed. It leaves (m, L, W) per
// 512 rows and the maximum of every group of 64 rows. The second launch, one CTA per column, joins the parts and finds the
// alternatives exactly: ordered by (maximum, lower group first), the first `top` groups hold the `top` largest values, because
// the best row of each of those groups comes before every row of any other group. So only `top` * 64 values are read again.
//
// FP32 sums over groups, then chunks, then the column (a tree: rounding error grows with its depth, not with the rows).
#include "k44_decoder.cuh"

namespace k44b {
namespace {

// FP16 bits -> 16-bit order: NaN 1, then -inf .. +inf; both zeros are equal. 0 is left for "no row".
__device__ __forceinline__ uint32_t order_of(uint32_t u) {
    const uint32_t mag = u & 0x7fffu;
    if (mag > 0x7c00u) return 1u;
    return (u & 0x8000u) ? 0x8000u - mag : 0x8000u + mag;
}

// CG: groups of 8 columns per CTA (a lane reads 16 bytes = 8 columns of a row); 32 / CG rows per warp load, 2 * CG loads
template <int CG>
__global__ void __launch_bounds__(256) k44_logprob_parts_kernel(const LogprobArgs a) {
    dep_enter();
    constexpr int I = 2 * CG, RL = 32 / CG;
    __shared__ float4 part_s[8][8 * CG];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, cg = lane % CG, rl = lane / CG;
    const uint32_t col0 = (blockIdx.x * CG + cg) * 8u, chunk = blockIdx.y;
    const uint32_t group = chunk * 8u + warp, r0 = group * kLogprobGroup + rl;
    const bool live_cols = col0 < a.columns;
    uint4 v[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const uint32_t r = r0 + RL * i;
        v[i] = make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);      // rows past the end: probability 0
        if (live_cols && r < a.rows) v[i] = __ldg(reinterpret_cast<const uint4 *>(a.x + (uint64_t)r * a.pitch + col0));
    }
    __half2 mx[4];                                     // of numbers; NaN where a group has nothing else
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = i ? __hmax2(mx[k], h[k]) : h[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int o = CG; o < 32; o <<= 1) mx[k] = __hmax2(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
    }
    float m[8], L[8], W[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(mx[k]);
        m[2 * k] = f.x; m[2 * k + 1] = f.y;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) { L[k] = 0.f; W[k] = 0.f; }
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float x = (k & 1) ? __high2float(h[k >> 1]) : __low2float(h[k >> 1]);
            const float mm = m[k] == -INFINITY ? 0.f : m[k];
            const float z = x - mm, e = exp2f(z * 1.4426950408889634f);
            L[k] += e;                                         // NaN goes through here
            W[k] = fmaf(e, fmaxf(z, -65504.0f), W[k]);          // 0 * -inf would not be 0
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int o = CG; o < 32; o <<= 1) {
            L[k] += __shfl_xor_sync(0xffffffffu, L[k], o);
            W[k] += __shfl_xor_sync(0xffffffffu, W[k], o);
        }
    }
    if (rl == 0u) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            part_s[warp][cg * 8u + k] = make_float4(m[k], L[k], W[k], 0.f);
            if (col0 + k < a.columns && group < a.groups)
                a.group_max[(uint64_t)(col0 + k) * a.groups + group] = (uint16_t)order_of(__half_as_ushort((k & 1) ? __high2half(mx[k >> 1]) : __low2half(mx[k >> 1])));
        }
    }
    __syncthreads();
    const uint32_t c = threadIdx.x, col = blockIdx.x * CG * 8u + c;
    if (c < 8u * CG && col < a.columns) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 8; ++w) M = fmaxf(M, part_s[w][c].x);
        const float base = M == -INFINITY ? 0.f : M;
        float sl = 0.f, sw = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float4 p = part_s[w][c];
            const float d = fmaxf(p.x, -131008.0f) - base, f = exp2f(d * 1.4426950408889634f);      // a part without a finite value: 0
            sl = fmaf(p.y, f, sl);
            sw = fmaf(fmaf(p.y, d, p.z), f, sw);
        }
        a.parts[(uint64_t)col * a.chunks + chunk] = make_float4(M, sl, sw, 0.f);
    }
}

// The `top` largest of the keys that a warp holds, K per lane, largest first: lane i gets the i-th. Keys are distinct or 0.
template <int K>
__device__ __forceinline__ uint32_t warp_top(uint32_t (&key)[K], uint32_t top, uint32_t lane) {
    uint32_t mine = 0, got = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) mine = max(mine, key[i]);
    for (uint32_t t = 0; t < top; ++t) {
        const uint32_t best = __reduce_max_sync(0xffffffffu, mine);
        if (best == 0u) break;
        if (lane == t) got = best;
        if (mine == best) {
            mine = 0;
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if (key[i] == best) key[i] = 0u;
                mine = max(mine, key[i]);
            }
        }
    }
    return got;
}

constexpr int kFinalThreads = 128, kFinalWarps = kFinalThreads / 32, kHeld = 16;     // new keys per lane and round

__global__ void __launch_bounds__(kFinalThreads) k44_logprob_final_kernel(const LogprobArgs a) {
    dep_enter();
    __shared__ float4 red_s[kFinalWarps];
    __shared__ uint32_t list_s[kFinalWarps][kLogprobTop], group_s[kLogprobTop];
    const uint32_t col = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    // ---- join the parts ----
    const float4 *parts = a.parts + (uint64_t)col * a.chunks;
    float M = -INFINITY, L = 0.f, W = 0.f;
    auto join = [](float &m0, float &l0, float &w0, float m1, float l1, float w1) {
        const float m = fmaxf(m0, m1), base = m == -INFINITY ? 0.f : m;
        const float d0 = fmaxf(m0, -131008.0f) - base, d1 = fmaxf(m1, -131008.0f) - base;
        const float f0 = exp2f(d0 * 1.4426950408889634f), f1 = exp2f(d1 * 1.4426950408889634f);
        w0 = fmaf(fmaf(l0, d0, w0), f0, fmaf(l1, d1, w1) * f1);
        l0 = fmaf(l0, f0, l1 * f1);
        m0 = m;
    };
    for (uint32_t c = tid; c < a.chunks; c += kFinalThreads) {
        const float4 p = __ldg(parts + c);
        join(M, L, W, p.x, p.y, p.z);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m1 = __shfl_xor_sync(0xffffffffu, M, o), l1 = __shfl_xor_sync(0xffffffffu, L, o), w1 = __shfl_xor_sync(0xffffffffu, W, o);
        join(M, L, W, m1, l1, w1);
    }
    if (lane == 0u) red_s[warp] = make_float4(M, L, W, 0.f);
    __syncthreads();
    M = red_s[0].x; L = red_s[0].y; W = red_s[0].z;
#pragma unroll
    for (int w = 1; w < kFinalWarps; ++w) join(M, L, W, red_s[w].x, red_s[w].y, red_s[w].z);
    const float ln = logf(L);
    if (tid == 0u) {
        if (a.entropy) a.entropy[col] = ln - W / L;
        if (a.logprobs) {
            const int t = a.targets[col];
            float lp = __int_as_float(0x7fc00000);                     // no such row: NaN
            if (t >= 0 && (uint32_t)t < a.rows) lp = (__half2float(a.x[(uint64_t)t * a.pitch + col]) - M) - ln;
            a.logprobs[col] = lp;
        }
    }
    if (a.top == 0u) return;
    // ---- the groups that hold the alternatives ----
    const uint16_t *gm = a.group_max + (uint64_t)col * a.groups;
    uint32_t best = 0;                                                 // this warp's list so far, one key per lane
    for (uint32_t g0 = 0; g0 < a.groups; g0 += kFinalThreads * kHeld) {
        uint32_t key[kHeld + 1];
        key[kHeld] = best;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t g = g0 + i * kFinalThreads + tid;
            key[i] = g < a.groups ? ((uint32_t)__ldg(gm + g) << 16) | (65535u - g) : 0u;
        }
        best = warp_top<kHeld + 1>(key, a.top, lane);
    }
    list_s[warp][lane] = best;
    __syncthreads();
    if (warp == 0u) {
        uint32_t key[kFinalWarps];
#pragma unroll
        for (int w = 0; w < kFinalWarps; ++w) key[w] = list_s[w][lane];
        best = warp_top<kFinalWarps>(key, a.top, lane);
        // in the order of their rows, so that a place in the list orders rows too
        const uint32_t g = best ? 65535u - (best & 0xffffu) : 0xffffffffu;
        uint32_t rank = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t o = __shfl_sync(0xffffffffu, g, i);
            rank += (o < g || (o == g && (uint32_t)i < lane)) ? 1u : 0u;
        }
        group_s[rank] = g;
    }
    __syncthreads();
    // ---- the alternatives themselves: up to 32 groups of 64 rows = 16 per thread ----
    uint32_t key[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const uint32_t place = i * kFinalThreads + tid, g = group_s[place / kLogprobGroup];
        const uint32_t r = g * kLogprobGroup + place % kLogprobGroup;
        key[i] = 0u;
        if (g != 0xffffffffu && r < a.rows) key[i] = (order_of(__half_as_ushort(a.x[(uint64_t)r * a.pitch + col])) << 16) | (65535u - place);
    }
    best = warp_top<kHeld>(key, a.top, lane);
    list_s[warp][lane] = best;
    __syncthreads();
    if (warp == 0u) {
        uint32_t k4[kFinalWarps];
#pragma unroll
        for (int w = 0; w < kFinalWarps; ++w) k4[w] = list_s[w][lane];
        best = warp_top<kFinalWarps>(k4, a.top, lane);
        if (lane < a.top) {
            const uint32_t place = 65535u - (best & 0xffffu);
            const uint32_t r = group_s[place / kLogprobGroup] * kLogprobGroup + place % kLogprobGroup;
            a.top_rows[(uint64_t)lane * a.columns + col] = (int)r;
            a.top_logprobs[(uint64_t)lane * a.columns + col] = (__half2float(a.x[(uint64_t)r * a.pitch + col]) - M) - ln;
        }
    }
}

}  // namespace

static uint32_t chunks_of(uint32_t rows) { return (rows + kLogprobChunk - 1u) / kLogprobChunk; }
static uint32_t groups_of(uint32_t rows) { return (rows + kLogprobGroup - 1u) / kLogprobGroup; }

uint64_t logprob_scratch_bytes(uint32_t rows, uint32_t columns) {
    return kv8_align((uint64_t)columns * chunks_of(rows) * sizeof(float4)) + (uint64_t)columns * groups_of(rows) * sizeof(uint16_t);
}

void logprob_place(LogprobArgs &a, void *scratch) {
    a.chunks = chunks_of(a.rows); a.groups = groups_of(a.rows);
    a.parts = (float4 *)scratch;
    a.group_max = (uint16_t *)((uint8_t *)scratch + kv8_align((uint64_t)a.columns * a.chunks * sizeof(float4)));
}

cudaError_t launch_logprobs(const LogprobArgs &a, bool pdl, cudaStream_t s) {
    // columns beyond the plan's are not read: a lane's 16 bytes are 8 columns, and few columns leave most lanes to rows
    const uint32_t cg = (a.columns + 7u) / 8u;
    cudaError_t e;
    if (cg == 1u) e = launch_dep(k44_logprob_parts_kernel<1>, dim3(1, a.chunks), dim3(256), 0, pdl, s, a);
    else if (cg == 2u) e = launch_dep(k44_logprob_parts_kernel<2>, dim3(1, a.chunks), dim3(256), 0, pdl, s, a);
    else if (cg <= 4u) e = launch_dep(k44_logprob_parts_kernel<4>, dim3(1, a.chunks), dim3(256), 0, pdl, s, a);
    else e = launch_dep(k44_logprob_parts_kernel<8>, dim3((cg + 7u) / 8u, a.chunks), dim3(256), 0, pdl, s, a);
    if (e == cudaSuccess) e = launch_dep(k44_logprob_final_kernel, dim3(a.columns), dim3(kFinalThreads), 0, pdl, s, a);
    return e;
}

}  // namespace k44b
