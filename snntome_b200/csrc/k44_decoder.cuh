// Decoder operators beyond the reference's commands: prompt attention with a sliding window and sinks, a key / value cache
// of 8 bits with the attention that reads it, and the probabilities of an answer. Arguments and launchers; the kernels are in
// k44_window_attn.cu, k44_kv8.cu and k44_logprobs.cu.
#pragma once
#include "k44_kernels.cuh"

namespace k44b {

enum DecoderKind : int { AUX_WINDOW_ATTN = 13, AUX_KV8_FILL = 14, AUX_KV8_ATTN = 15, AUX_LOGPROBS = 16 };

// ---- rotary table ------------------------------------------------------------------------------------------------------
// (cos, sin) of position * frequency for every position and rotation pair, [positions][head_dim / 2]. Angles are formed and
// reduced in 64 bits: a 32-bit angle at position 16000 is off by up to 1e-3, more than the rounding of an FP16 result.
// pairs_first: [pair][position], and both times kWindowHeld: what the prompt attention's q is rotated by.
constexpr float kWindowHeld = 0.5f;                  // the size at which the prompt attention holds rotated q and k
cudaError_t launch_rope_table(float2 *table, uint32_t positions, uint32_t head_dim, double theta, bool llama3, bool pairs_first, cudaStream_t s);

// ---- 8-bit cache ---------------------------------------------------------------------------------------------------------
// Blocks of 64 tokens of one column (sequence) and head. Keys and values of a block lie side by side as e4m3 codes, each with
// one FP32 scale; the block that is still open is kept as FP16 rows:
//   codes       [column][head][block][ K: dim / 64 | token | 64 dims ][ V: dim | 64 tokens ]    (2 * 64 * dim bytes per block)
//   scales      [column][head][block][K, V] FP32
//   k_tail      [column][head][64 tokens][dim] FP16        v_tail  [column][head][dim][64 tokens] FP16
//   tail_block  [column][head] int32: number of the open block, -1 none
// every part starting on a 256-byte boundary. Values run along tokens because tokens are what their product sums over.
constexpr uint32_t kKv8Block = 64;
struct Kv8Cache {
    uint8_t *codes = nullptr;
    float2 *scales = nullptr;
    __half *k_tail = nullptr, *v_tail = nullptr;
    int *tail_block = nullptr;
    uint32_t columns = 0, h_kv = 0, head_dim = 0, max_seq = 0, blocks = 0;
};
inline uint64_t kv8_align(uint64_t n) { return (n + 255u) / 256u * 256u; }
// lays the parts out behind `data`; returns the bytes they take
inline uint64_t kv8_layout(Kv8Cache &c, uint8_t *data, uint32_t columns, uint32_t h_kv, uint32_t head_dim, uint32_t max_seq) {
    c.columns = columns; c.h_kv = h_kv; c.head_dim = head_dim; c.max_seq = max_seq;
    c.blocks = (max_seq + kKv8Block - 1u) / kKv8Block;
    const uint64_t ch = (uint64_t)columns * h_kv;
    uint64_t at = 0;
    c.codes = data; at += kv8_align(ch * c.blocks * 2u * kKv8Block * head_dim);
    c.scales = (float2 *)(data + at); at += kv8_align(ch * c.blocks * sizeof(float2));
    c.k_tail = (__half *)(data + at); at += kv8_align(ch * kKv8Block * head_dim * 2u);
    c.v_tail = (__half *)(data + at); at += kv8_align(ch * kKv8Block * head_dim * 2u);
    c.tail_block = (int *)(data + at); at += kv8_align(ch * sizeof(int));
    return at;
}

struct Kv8FillArgs {
    Kv8Cache cache;
    const __half *k = nullptr, *v = nullptr;         // canvas tensors, channel-major
    const int2 *sequences = nullptr;                 // per sequence of the plan: (cache column or -1, length)
    const float2 *rope = nullptr;
    uint32_t *status = nullptr;
    uint32_t pitch = 0, columns = 0, seq_len = 0;
};
cudaError_t launch_kv8_fill(const Kv8FillArgs &a, bool pdl, cudaStream_t s);

struct Kv8AttnArgs {
    Kv8Cache cache;
    const __half *q = nullptr, *k = nullptr, *v = nullptr;
    __half *out = nullptr;
    const int *positions = nullptr;                  // per column: position of its new token, -1 idle
    const float2 *rope = nullptr;
    uint32_t *status = nullptr;
    uint4 *q_frag = nullptr;                         // [column][head]: the group's rotated q as operand words
    float *partial = nullptr;                        // [worker][2][8 or 16 heads][head_dim + 2]
    uint32_t *counters = nullptr;                    // [column][head]: units of it that have arrived; every run clears them first
    uint32_t pitch = 0, columns = 0, h_q = 0, window = 0, sinks = 0;
    uint32_t workers = 0, spread = 1;                // warps, and their step over the shares (set by the launcher)
    unsigned long long wait_cycles = 0;
};
constexpr uint32_t kKv8MaxColumns = 4096;
cudaError_t launch_kv8_attn(const Kv8AttnArgs &a, uint32_t num_sms, bool pdl, cudaStream_t s);
cudaError_t kv8_attn_setup();                        // opt in to large dynamic shared memory (once per device)
uint64_t kv8_attn_frag_bytes(uint32_t columns, uint32_t h_kv, uint32_t group, uint32_t head_dim);
uint64_t kv8_attn_partial_bytes(uint32_t num_sms, uint32_t group, uint32_t head_dim);

// ---- prompt attention with a window and sinks ---------------------------------------------------------------------------
struct WindowAttnArgs {
    const __half *q = nullptr, *k = nullptr, *v = nullptr;
    __half *out = nullptr;
    // re-laid operands: rotated k [h_kv][pitch][head_dim], v [h_kv * head_dim][pitch] with
    // non-finite values replaced by zero, per (head, 64 columns) whether there were any, and which: [h_kv][64 columns][head_dim]
    __half *k_rows = nullptr, *v_rows = nullptr;
    uint32_t *v_flags = nullptr;
    uint4 *v_marks = nullptr;
    const float2 *rope = nullptr, *rope_pairs = nullptr;       // [position][pair], [pair][position]: `positions` of them
    uint32_t *status = nullptr;
    uint32_t pitch = 0, columns = 0, h_q = 0, h_kv = 0, head_dim = 0, seq_len = 0, window = 0, sinks = 0, positions = 0;
    unsigned long long wait_cycles = 0;
};
struct WindowAttnMaps { CUtensorMap k, v, out; };
uint64_t window_attn_scratch_bytes(uint32_t pitch, uint32_t h_kv, uint32_t head_dim);
void window_attn_place(WindowAttnArgs &a, void *scratch);
cudaError_t launch_window_attn(const WindowAttnArgs &a, const WindowAttnMaps &m, bool pdl, cudaStream_t s);
cudaError_t window_attn_setup();

// ---- answer probabilities --------------------------------------------------------------------------------------------------
struct LogprobArgs {
    const __half *x = nullptr;                       // logits [rows][pitch]
    const int *targets = nullptr;
    float *logprobs = nullptr, *entropy = nullptr, *top_logprobs = nullptr;
    int *top_rows = nullptr;
    float4 *parts = nullptr;                         // [column][chunk]: M, L and W of k44_logprobs.cu, in powers of 2
    uint16_t *group_max = nullptr;                   // [column][group]: order of the largest value of 64 rows
    uint32_t *status = nullptr;
    unsigned long long wait_cycles = 0;
    uint32_t rows = 0, pitch = 0, columns = 0, top = 0, chunks = 0, groups = 0, chunk_groups = 0, group_stride = 0;
};
constexpr uint32_t kLogprobGroup = 64, kLogprobTop = 32;
constexpr uint32_t kLogprobMaxRows = 65528u * kLogprobGroup;           // a group's number in 16 bits
uint64_t logprob_scratch_bytes(uint32_t rows, uint32_t columns, uint32_t num_sms);
void logprob_place(LogprobArgs &a, void *scratch, uint32_t num_sms);
cudaError_t logprob_setup();
cudaError_t launch_logprobs(const LogprobArgs &a, const CUtensorMap &map, bool pdl, cudaStream_t s);      // map: the logits as rows of `pitch`, boxes of 64 x 64

// programmatic dependent launch, as in k44_valu.cu. A grid may start while the one before it still writes: what that one leaves (canvas
// rows, operands, parts) is read by ordinary loads (`__ldcg`) after the wait, and only what nobody writes while the grid exists by `__ldg`.
__device__ __forceinline__ void dep_enter() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... KArgs, typename... Args>
inline cudaError_t launch_dep(void (*kernel)(KArgs...), dim3 grid, dim3 block, uint32_t smem, bool pdl, cudaStream_t s, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = pdl ? 1u : 0u;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace k44b
