// In front of the gated delta rule, for the tokens of a ragged batch of chunks: causal convolution over the tokens,
// SiLU, L2 normalisation of q and k, decay and write strength.  What qwc_delta_prepare_decode does for one token of each
// sequence (cuda/delta_prepare.cu:44-86,168-245), with the convolution running through the chunk: token i of a channel is
//   silu(w0 x[i-3] + w1 x[i-2] + w2 x[i-1] + w3 x[i]),
// rows before the chunk come from the slot's history (or are zeros where a sequence begins), and the last three rows
// become the history.
//
// Bound by memory: every projected row is read once and every prepared row written once.  A thread owns eight
// channels (16 bytes of a row) and walks along the tokens of a tile with the last three rows in registers; sixteen
// lanes hold a head, so a norm is four shuffles.  Tiles start at their chunk's first row, so that the history of a slot
// is read and replaced by the same threads (a tile holds the first three tokens of its chunk or all of it).
//
// q, k and v leave as bf16, rounded once: they are operands of matrix products in the delta rule.  Everything between
// is fp32 (the decode form rounds the SiLU's result to bf16 in between).

#include "chunk.cuh"

namespace qwc {
namespace {

constexpr int kPrepareThreads = 256;
constexpr int kChannels = 8;                                  // of a thread
constexpr int kGroupChannels = kPrepareThreads * kChannels;   // of a CTA: 16 heads
constexpr int kTileTokens = 8;
constexpr int kTaps = 4;
static_assert(kTileTokens >= kTaps - 1, "the first tile of a chunk reads the whole history");
static_assert(kGroupChannels == kDeltaKeyHeads * kDeltaHeadDim, "a CTA's channels are q, k or values");

__device__ __forceinline__ void unpack8(const uint4& raw, float (&out)[kChannels]) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[2 * i] = __uint_as_float(words[i] << 16);
        out[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ uint4 pack8(const float (&in)[kChannels]) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(in[2 * i], in[2 * i + 1]);
        words[i] = *reinterpret_cast<const uint32_t*>(&pair);
    }
    return make_uint4(words[0], words[1], words[2], words[3]);
}

// log(1 + e^x) to fp32's accuracy.
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

__global__ void __launch_bounds__(kPrepareThreads) delta_prepare_chunk_kernel(
    const __nv_bfloat16* __restrict__ mixed, const __nv_bfloat16* __restrict__ a_projection,
    const __nv_bfloat16* __restrict__ b_projection, const __nv_bfloat16* __restrict__ conv_weight,
    const __nv_bfloat16* __restrict__ a_log, const __nv_bfloat16* __restrict__ dt_bias, float* __restrict__ conv_state,
    const uint32_t* __restrict__ state_slots, const uint32_t* __restrict__ continues,
    const uint32_t* __restrict__ begins, __nv_bfloat16* __restrict__ qkv, float* __restrict__ alpha,
    float* __restrict__ beta, int tokens, int sequences, int mixed_stride, int gate_stride, int v_heads,
    int state_capacity, int* status) {
    pdl_launch_dependents();
    const int groups = 2 + v_heads / kDeltaKeyHeads;
    const int channels = groups * kGroupChannels;
    const int group = blockIdx.x;  // q, k, the values, and last the gates
    const int channel = group * kGroupChannels + threadIdx.x * kChannels;
    float taps[kTaps][kChannels];
    if (group < groups) {
        // never written during a step: fetched before the wait
        const uint4* at = reinterpret_cast<const uint4*>(conv_weight + static_cast<size_t>(channel) * kTaps);
#pragma unroll
        for (int i = 0; i < kChannels / 2; ++i) {
            float pair[8];
            unpack8(at[i], pair);
#pragma unroll
            for (int j = 0; j < kTaps; ++j) {
                taps[j][2 * i] = pair[j];
                taps[j][2 * i + 1] = pair[kTaps + j];
            }
        }
    }
    pdl_wait();
    const ChunkTile tile = find_chunk_tile(begins, sequences, tokens, kTileTokens, blockIdx.y);
    if (tile.sequence < 0) {
        return;
    }
    const uint32_t slot = __ldcg(state_slots + tile.sequence);
    if (slot >= static_cast<uint32_t>(state_capacity)) {
        // a slot beyond the pool: nothing of this chunk is read or written, the host learns of it through the status
        // word (the whole CTA takes this branch)
        if (threadIdx.x == 0) {
            atomicCAS(status, 0, kStatusStateSlotRange);
        }
        return;
    }
    const int first = tile.index * kTileTokens;  // in the chunk
    const int count = min(kTileTokens, tile.span.length - first);
    const size_t row = static_cast<size_t>(tile.span.begin) + first;
    if (group == groups) {
        for (int i = threadIdx.x; i < count * v_heads; i += kPrepareThreads) {
            const size_t at = row + i / v_heads;
            const int head = i % v_heads;
            const float a = __bfloat162float(a_projection[at * gate_stride + head]) + __bfloat162float(dt_bias[head]);
            const float b = __bfloat162float(b_projection[at * gate_stride + head]);
            alpha[at * v_heads + head] = expf(-expf(__bfloat162float(a_log[head])) * softplus(a));
            beta[at * v_heads + head] = 1.0f / (1.0f + expf(-b));
        }
        return;
    }

    const __nv_bfloat16* source = mixed + row * mixed_stride + channel;
    float window[kTaps][kChannels];  // the last three rows and this one
    if (first == 0) {
        float* history = conv_state + (static_cast<size_t>(slot) * channels + channel) * (kTaps - 1);
        const bool holds = continues == nullptr || __ldcg(continues + tile.sequence) != 0;
        float held[kChannels * (kTaps - 1)];
#pragma unroll
        for (int i = 0; i < kChannels * (kTaps - 1); ++i) {
            held[i] = holds ? history[i] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < kChannels; ++c) {
#pragma unroll
            for (int j = 0; j < kTaps - 1; ++j) {
                window[j][c] = held[c * (kTaps - 1) + j];
            }
        }
        // the history that this chunk leaves: its last three rows, behind what a shorter one keeps of the old
#pragma unroll
        for (int j = 0; j < kTaps - 1; ++j) {
            const int from = tile.span.length - (kTaps - 1) + j;  // in the chunk; negative: old history
            float value[kChannels];
            if (from >= 0) {
                unpack8(*reinterpret_cast<const uint4*>(source + static_cast<size_t>(from) * mixed_stride), value);
            }
#pragma unroll
            for (int c = 0; c < kChannels; ++c) {
                const float old = from == -1 ? held[c * 3 + 2] : from == -2 ? held[c * 3 + 1] : held[c * 3];
                history[c * (kTaps - 1) + j] = from >= 0 ? value[c] : old;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTaps - 1; ++j) {
            unpack8(*reinterpret_cast<const uint4*>(source - static_cast<size_t>(kTaps - 1 - j) * mixed_stride), window[j]);
        }
    }
    uint4 raw[kTileTokens];
#pragma unroll
    for (int t = 0; t < kTileTokens; ++t) {
        if (t < count) {
            raw[t] = *reinterpret_cast<const uint4*>(source + static_cast<size_t>(t) * mixed_stride);
        }
    }
    __nv_bfloat16* target = qkv + row * channels + channel;
#pragma unroll
    for (int t = 0; t < kTileTokens; ++t) {
        if (t < count) {  // (uniform over the CTA)
            unpack8(raw[t], window[kTaps - 1]);
            float value[kChannels];
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < kChannels; ++c) {
                float convolved = taps[0][c] * window[0][c];
                convolved = fmaf(taps[1][c], window[1][c], convolved);
                convolved = fmaf(taps[2][c], window[2][c], convolved);
                convolved = fmaf(taps[3][c], window[3][c], convolved);
                value[c] = convolved / (1.0f + __expf(-convolved));
                sum = fmaf(value[c], value[c], sum);
                window[0][c] = window[1][c];
                window[1][c] = window[2][c];
                window[2][c] = window[3][c];
            }
            if (group < 2) {
#pragma unroll
                for (int offset = 1; offset < kDeltaHeadDim / kChannels; offset <<= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, offset);
                }
                const float inverse = rsqrtf(sum + 1e-6f) * (group == 0 ? 0.08838834764831845f : 1.0f);  // 128^-1/2
#pragma unroll
                for (int c = 0; c < kChannels; ++c) {
                    value[c] *= inverse;
                }
            }
            *reinterpret_cast<uint4*>(target + static_cast<size_t>(t) * channels) = pack8(value);
        }
    }
}

}  // namespace
}  // namespace qwc

extern "C" int qwc_delta_prepare_chunk(const void* mixed_qkv, const void* a_projection, const void* b_projection,
                                       const void* conv_weight, const void* a_log, const void* dt_bias,
                                       void* conv_state, const void* state_slots, const void* continues,
                                       const void* chunk_begins, void* qkv, void* alpha, void* beta,
                                       int state_capacity, int tokens, int sequences, int mixed_stride,
                                       int gate_stride, cudaStream_t stream) {
    using namespace qwc;
    const int v_heads = current_shape().delta_value_heads;
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDeltaHeadDim;
    const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (mixed_qkv == nullptr || a_projection == nullptr || b_projection == nullptr || conv_weight == nullptr ||
        a_log == nullptr || dt_bias == nullptr || conv_state == nullptr || state_slots == nullptr ||
        chunk_begins == nullptr || qkv == nullptr || alpha == nullptr || beta == nullptr || tokens <= 0 ||
        tokens > kMaxChunkTokens || sequences <= 0 || sequences > kMaxChunkSequences || state_capacity < sequences ||
        mixed_stride < channels || mixed_stride % 8 != 0 || gate_stride < v_heads || !aligned(mixed_qkv) ||
        !aligned(conv_weight) || !aligned(qkv)) {
        return cudaErrorInvalidValue;
    }
    int* status = status_ptr();
    if (status == nullptr) {
        return cudaErrorInvalidValue;
    }
    const dim3 grid(2 + v_heads / kDeltaKeyHeads + 1, most_chunk_tiles(tokens, sequences, kTileTokens));
    return launch_chained(delta_prepare_chunk_kernel, grid, dim3(kPrepareThreads), 0, stream,
                          static_cast<const __nv_bfloat16*>(mixed_qkv), static_cast<const __nv_bfloat16*>(a_projection),
                          static_cast<const __nv_bfloat16*>(b_projection), static_cast<const __nv_bfloat16*>(conv_weight),
                          static_cast<const __nv_bfloat16*>(a_log), static_cast<const __nv_bfloat16*>(dt_bias),
                          static_cast<float*>(conv_state), static_cast<const uint32_t*>(state_slots),
                          static_cast<const uint32_t*>(continues), static_cast<const uint32_t*>(chunk_begins),
                          static_cast<__nv_bfloat16*>(qkv), static_cast<float*>(alpha), static_cast<float*>(beta),
                          tokens, sequences, mixed_stride, gate_stride, v_heads, state_capacity, status);
}
