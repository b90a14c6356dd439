// The gated delta rule over the tokens of a ragged batch of chunks, on the slots' int8 state.
//
// Per token and value head, S [128 x 128] (rows: value dims, columns: key dims):
//   S <- alpha S;  u = beta (v - S k);  S <- S + u k^T;  o = S q
// (the recurrence of cuda/delta_net.cu:99-119 without the requantisation after every token: the state is read from its
// eight bits once per call, carried in fp32, and written back once, with the rounding of cuda/delta_net.cu:137-175).
//
// The rows of S are independent of one another: four lanes share a row and hold it in registers, a CTA has 32 rows of one
// head of one chunk and walks through its tokens, 16 at a time in shared memory.

#include "chunk.cuh"

namespace qwc {
namespace {

constexpr int kDim = kDeltaHeadDim;
constexpr int kRowsPerCta = 32;
constexpr int kRecurrentThreads = 128;
constexpr int kBlockTokens = 16;

__global__ void __launch_bounds__(kRecurrentThreads) delta_recurrent_kernel(
    int8_t* __restrict__ state, float* __restrict__ state_scales, const uint32_t* __restrict__ state_slots,
    const uint32_t* __restrict__ continues, const uint32_t* __restrict__ begins, const __nv_bfloat16* __restrict__ qkv,
    const float* __restrict__ alpha, const float* __restrict__ beta, __nv_bfloat16* __restrict__ out, int tokens,
    int v_heads, int state_capacity, int* status) {
    pdl_launch_dependents();
    __shared__ float k_rows[kBlockTokens][kDim];
    __shared__ float q_rows[kBlockTokens][kDim];
    __shared__ float v_rows[kBlockTokens][kRowsPerCta];
    __shared__ float2 gates[kBlockTokens];
    const int row_begin = blockIdx.x * kRowsPerCta;
    const int head = blockIdx.y;
    const int key_head = head / (v_heads / kDeltaKeyHeads);
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDim;
    const int local = threadIdx.x >> 2;
    const int sub = threadIdx.x & 3;
    pdl_wait();
    const ChunkSpan span = chunk_span(begins, blockIdx.z, tokens);
    if (span.length == 0) {
        return;
    }
    const uint32_t slot = __ldcg(state_slots + blockIdx.z);
    if (slot >= static_cast<uint32_t>(state_capacity)) {
        if (threadIdx.x == 0) {
            atomicCAS(status, 0, kStatusStateSlotRange);
        }
        return;
    }
    const size_t state_row = (static_cast<size_t>(slot) * v_heads + head) * kDim + row_begin + local;
    // columns 16 i + 4 sub .. + 3
    float s[32];
    const bool holds = continues == nullptr || __ldcg(continues + blockIdx.z) != 0;
    const float scale = holds ? state_scales[state_row] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const char4 codes = holds ? *reinterpret_cast<const char4*>(state + state_row * kDim + 16 * i + 4 * sub) : make_char4(0, 0, 0, 0);
        s[4 * i] = codes.x * scale;
        s[4 * i + 1] = codes.y * scale;
        s[4 * i + 2] = codes.z * scale;
        s[4 * i + 3] = codes.w * scale;
    }
    for (int first = 0; first < span.length; first += kBlockTokens) {
        const int count = min(kBlockTokens, span.length - first);
        __syncthreads();
        for (int t = 0; t < count; ++t) {
            const size_t token = static_cast<size_t>(span.begin) + first + t;
            const __nv_bfloat16* row = qkv + token * channels;
            q_rows[t][threadIdx.x] = __bfloat162float(row[key_head * kDim + threadIdx.x]);
            k_rows[t][threadIdx.x] = __bfloat162float(row[(kDeltaKeyHeads + key_head) * kDim + threadIdx.x]);
            if (threadIdx.x < kRowsPerCta) {
                v_rows[t][threadIdx.x] =
                    __bfloat162float(row[(2 * kDeltaKeyHeads + head) * kDim + row_begin + threadIdx.x]);
            }
            if (threadIdx.x == 0) {
                gates[t] = make_float2(alpha[token * v_heads + head], beta[token * v_heads + head]);
            }
        }
        __syncthreads();
        for (int t = 0; t < count; ++t) {
            const float2 gate = gates[t];
            float dot = 0.0f;
            float k[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 part = *reinterpret_cast<const float4*>(&k_rows[t][16 * i + 4 * sub]);
                k[4 * i] = part.x;
                k[4 * i + 1] = part.y;
                k[4 * i + 2] = part.z;
                k[4 * i + 3] = part.w;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                s[i] *= gate.x;
                dot = fmaf(s[i], k[i], dot);
            }
            dot += __shfl_xor_sync(0xffffffffu, dot, 1);
            dot += __shfl_xor_sync(0xffffffffu, dot, 2);
            const float u = gate.y * (v_rows[t][local] - dot);
            float result = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 q = *reinterpret_cast<const float4*>(&q_rows[t][16 * i + 4 * sub]);
                const float part[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[4 * i + j] = fmaf(u, k[4 * i + j], s[4 * i + j]);
                    result = fmaf(s[4 * i + j], part[j], result);
                }
            }
            result += __shfl_xor_sync(0xffffffffu, result, 1);
            result += __shfl_xor_sync(0xffffffffu, result, 2);
            if (sub == 0) {
                const size_t token = static_cast<size_t>(span.begin) + first + t;
                out[(token * v_heads + head) * kDim + row_begin + local] = __float2bfloat16(result);
            }
        }
    }
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        peak = fmaxf(peak, fabsf(s[i]));
    }
    peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
    const float inverse = peak == 0.0f ? 0.0f : __fdiv_rn(127.0f, peak);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        *reinterpret_cast<char4*>(state + state_row * kDim + 16 * i + 4 * sub) =
            make_char4(static_cast<char>(__float2int_rn(s[4 * i] * inverse)), static_cast<char>(__float2int_rn(s[4 * i + 1] * inverse)),
                       static_cast<char>(__float2int_rn(s[4 * i + 2] * inverse)), static_cast<char>(__float2int_rn(s[4 * i + 3] * inverse)));
    }
    if (sub == 0) {
        state_scales[state_row] = __fmul_rn(peak, 1.0f / 127.0f);
    }
}

// RMSNorm over the 128 dims of a value head, times weight, times silu(gate): in place on the bf16 rows of the batch's
// chunks.  A warp per token and head, four dims per lane; one rounding.
constexpr int kNormWarps = 8;

__global__ void __launch_bounds__(kNormWarps * 32) delta_norm_rows_kernel(
    __nv_bfloat16* __restrict__ rows, const __nv_bfloat16* __restrict__ gate, const __nv_bfloat16* __restrict__ weight,
    const uint32_t* __restrict__ begins, int sequences, int tokens, int v_heads, int gate_stride, float epsilon) {
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const size_t item = static_cast<size_t>(blockIdx.x) * kNormWarps + (threadIdx.x >> 5);
    const size_t token = item / v_heads;
    const int head = static_cast<int>(item % v_heads);
    pdl_wait();
    const uint32_t low = __ldcg(begins), high = __ldcg(begins + sequences);
    if (token < low || token >= high || token >= tokens) {
        return;
    }
    uint2* at = reinterpret_cast<uint2*>(rows + (token * v_heads + head) * kDim) + lane;
    const uint2 raw = *at;
    const uint2 gates = *(reinterpret_cast<const uint2*>(gate + token * gate_stride + head * kDim) + lane);
    const uint2 gains = *(reinterpret_cast<const uint2*>(weight) + lane);
    const auto unpack = [](const uint2& words, float (&x)[4]) {
        x[0] = __uint_as_float(words.x << 16);
        x[1] = __uint_as_float(words.x & 0xffff0000u);
        x[2] = __uint_as_float(words.y << 16);
        x[3] = __uint_as_float(words.y & 0xffff0000u);
    };
    float x[4], z[4], w[4];
    unpack(raw, x);
    unpack(gates, z);
    unpack(gains, w);
    const float sum = warp_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
    const float inverse = rsqrtf(sum / static_cast<float>(kDim) + epsilon);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] *= inverse * w[i] * (z[i] / (1.0f + __expf(-z[i])));
    }
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    *at = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

}  // namespace
}  // namespace qwc

extern "C" size_t qwc_delta_chunk_workspace_bytes(int tokens, int sequences) {
    (void)tokens;
    (void)sequences;
    return 0;
}

extern "C" int qwc_delta_chunk_int8(void* state, float* state_scales, const void* state_slots, const void* continues,
                                    const void* chunk_begins, const void* qkv, const void* alpha, const void* beta,
                                    void* out, int state_capacity, int tokens, int sequences, const void* gate,
                                    int gate_stride, const void* norm_weight, float epsilon, void* workspace,
                                    size_t workspace_bytes, cudaStream_t stream) {
    using namespace qwc;
    const int v_heads = current_shape().delta_value_heads;
    const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (gate_stride == 0) {
        gate_stride = v_heads * kDim;
    }
    if (state == nullptr || state_scales == nullptr || state_slots == nullptr || chunk_begins == nullptr ||
        qkv == nullptr || alpha == nullptr || beta == nullptr || out == nullptr || tokens <= 0 ||
        tokens > kMaxChunkTokens || sequences <= 0 || sequences > kMaxChunkSequences || state_capacity < sequences ||
        (gate == nullptr) != (norm_weight == nullptr) || !aligned(state) || !aligned(state_scales) || !aligned(qkv) ||
        !aligned(out) || workspace_bytes < qwc_delta_chunk_workspace_bytes(tokens, sequences)) {
        return cudaErrorInvalidValue;
    }
    if (gate != nullptr && (gate_stride < v_heads * kDim || gate_stride % 8 != 0 || !aligned(gate) ||
                            !aligned(norm_weight) || !isfinite(epsilon) || epsilon <= 0.0f)) {
        return cudaErrorInvalidValue;
    }
    int* status = status_ptr();
    if (status == nullptr) {
        return cudaErrorInvalidValue;
    }
    const cudaError_t launched = launch_chained(
        delta_recurrent_kernel, dim3(kDim / kRowsPerCta, v_heads, sequences), dim3(kRecurrentThreads), 0, stream,
        static_cast<int8_t*>(state), state_scales, static_cast<const uint32_t*>(state_slots),
        static_cast<const uint32_t*>(continues), static_cast<const uint32_t*>(chunk_begins),
        static_cast<const __nv_bfloat16*>(qkv), static_cast<const float*>(alpha), static_cast<const float*>(beta),
        static_cast<__nv_bfloat16*>(out), tokens, v_heads, state_capacity, status);
    if (launched != cudaSuccess || gate == nullptr) {
        return launched;
    }
    const int items = tokens * v_heads;  // at most 65536 * 48
    return launch_chained(delta_norm_rows_kernel, dim3((items + kNormWarps - 1) / kNormWarps), dim3(kNormWarps * 32), 0,
                          stream, static_cast<__nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(gate),
                          static_cast<const __nv_bfloat16*>(norm_weight), static_cast<const uint32_t*>(chunk_begins),
                          sequences, tokens, v_heads, gate_stride, epsilon);
}
