// In front of the gated delta rule, for the tokens of a ragged batch of chunks: causal convolution over the tokens,
// SiLU, L2 normalisation of q and k, decay and write strength.  What qwc_delta_prepare_decode does for one token of each
// sequence (cuda/delta_prepare.cu:44-86,168-245), with the convolution running through the chunk: token i of a channel is
//   silu(w0 x[i-3] + w1 x[i-2] + w2 x[i-1] + w3 x[i]),
// rows before the chunk come from the slot's history (or are zeros where a sequence begins), and the last three rows
// become the history.
//
// Bound by memory: every projected row is read once and every prepared row written once.  A warp has a head, four channels
// (8 bytes of a row) to a lane, and walks along the tokens of a tile with the last three rows in registers; a norm is five
// shuffles.  Tiles start at their chunk's first row, so that the history of a slot is read and replaced by the same threads
// (a tile holds the first three tokens of its chunk or all of it).
//
// q, k and v leave as bf16, rounded once: they are operands of matrix products in the delta rule.  Everything between
// is fp32 (the decode form rounds the SiLU's result to bf16 in between).

#include "chunk.cuh"

namespace qwc {
namespace {

constexpr int kPrepareWarps = 8;   // heads of a CTA
constexpr int kStepTokens = 8;    // in flight
constexpr int kTaps = 4;
static_assert(kStepTokens >= kTaps - 1, "the first tile of a chunk reads the whole history");

// Channels in pairs: the multiplications and additions of two take one instruction.
struct Channels {
    float2 lo, hi;
};

__device__ __forceinline__ Channels unpack4(const uint2& raw) {
    return {make_float2(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u)),
            make_float2(__uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u))};
}

__device__ __forceinline__ Channels multiply(const Channels& a, const Channels& b) {
    return {__fmul2_rn(a.lo, b.lo), __fmul2_rn(a.hi, b.hi)};
}

__device__ __forceinline__ Channels multiply_add(const Channels& a, const Channels& b, const Channels& c) {
    return {__ffma2_rn(a.lo, b.lo, c.lo), __ffma2_rn(a.hi, b.hi, c.hi)};
}

// log(1 + e^x) to fp32's accuracy.
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// `kTileTokens`: of a CTA.  A longer tile reads the three rows before it and its channels' taps, and looks for its chunk,
// less often; a shorter one leaves more CTAs (see the launch).
template <int kTileTokens>
__global__ void __launch_bounds__(kPrepareWarps * 32) delta_prepare_chunk_kernel(
    const __nv_bfloat16* __restrict__ mixed, const __nv_bfloat16* __restrict__ a_projection,
    const __nv_bfloat16* __restrict__ b_projection, const __nv_bfloat16* __restrict__ conv_weight,
    const __nv_bfloat16* __restrict__ a_log, const __nv_bfloat16* __restrict__ dt_bias, float* __restrict__ conv_state,
    const uint32_t* __restrict__ state_slots, const uint32_t* __restrict__ continues,
    const uint32_t* __restrict__ begins, __nv_bfloat16* __restrict__ qkv, float* __restrict__ alpha,
    float* __restrict__ beta, int tokens, int sequences, int mixed_stride, int gate_stride, int v_heads,
    int state_capacity, int* status) {
    pdl_launch_dependents();
    const int heads = 2 * kDeltaKeyHeads + v_heads;  // q, k, the values
    const int channels = heads * kDeltaHeadDim;
    const int head = blockIdx.x * kPrepareWarps + (threadIdx.x >> 5);
    const int channel = head * kDeltaHeadDim + (threadIdx.x & 31) * 4;
    const bool gates = blockIdx.x * kPrepareWarps >= heads;  // the last CTA of a tile
    pdl_wait();
    Channels taps[kTaps];
    if (!gates) {
        // (on its way while the tile is looked for)
        const uint4* at = reinterpret_cast<const uint4*>(conv_weight + static_cast<size_t>(channel) * kTaps);
        const uint4 raw[2] = {at[0], at[1]};  // four taps of a channel are 8 bytes
        const Channels c0 = unpack4(make_uint2(raw[0].x, raw[0].y)), c1 = unpack4(make_uint2(raw[0].z, raw[0].w));
        const Channels c2 = unpack4(make_uint2(raw[1].x, raw[1].y)), c3 = unpack4(make_uint2(raw[1].z, raw[1].w));
        taps[0] = {make_float2(c0.lo.x, c1.lo.x), make_float2(c2.lo.x, c3.lo.x)};
        taps[1] = {make_float2(c0.lo.y, c1.lo.y), make_float2(c2.lo.y, c3.lo.y)};
        taps[2] = {make_float2(c0.hi.x, c1.hi.x), make_float2(c2.hi.x, c3.hi.x)};
        taps[3] = {make_float2(c0.hi.y, c1.hi.y), make_float2(c2.hi.y, c3.hi.y)};
    }
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
    if (gates) {
        for (int i = threadIdx.x; i < count * v_heads; i += kPrepareWarps * 32) {
            const size_t at = row + i / v_heads;
            const int of = i % v_heads;
            const float a = __bfloat162float(a_projection[at * gate_stride + of]) + __bfloat162float(dt_bias[of]);
            const float b = __bfloat162float(b_projection[at * gate_stride + of]);
            alpha[at * v_heads + of] = expf(-expf(__bfloat162float(a_log[of])) * softplus(a));
            beta[at * v_heads + of] = 1.0f / (1.0f + expf(-b));
        }
        return;
    }

    const __nv_bfloat16* source = mixed + row * mixed_stride + channel;
    // eight rows ahead of the one at hand (behind the tile's last: that one again, and not stored)
    uint2 raw[kStepTokens];
    const auto fetch = [&](int t) {
        const uint32_t offset = static_cast<uint32_t>(min(t, count - 1)) * static_cast<uint32_t>(mixed_stride);
        return *reinterpret_cast<const uint2*>(source + offset);
    };
#pragma unroll
    for (int t = 0; t < kStepTokens; ++t) {
        raw[t] = fetch(t);
    }
    Channels window[kTaps];  // the last three rows and this one
    if (first == 0) {
        // twelve numbers: three of each channel
        float4* history = reinterpret_cast<float4*>(conv_state + (static_cast<size_t>(slot) * channels + channel) * (kTaps - 1));
        float held[12] = {};
        if (continues == nullptr || __ldcg(continues + tile.sequence) != 0) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const float4 part = history[i];
                held[4 * i] = part.x;
                held[4 * i + 1] = part.y;
                held[4 * i + 2] = part.z;
                held[4 * i + 3] = part.w;
            }
        }
        // the history that this chunk leaves: its last three rows, behind what a shorter one keeps of the old
        float left[12];
#pragma unroll
        for (int j = 0; j < kTaps - 1; ++j) {
            window[j] = {make_float2(held[j], held[3 + j]), make_float2(held[6 + j], held[9 + j])};
            const int from = tile.span.length - (kTaps - 1) + j;  // in the chunk; negative: old history
            Channels row = {};
            if (from >= 0) {
                row = unpack4(*reinterpret_cast<const uint2*>(source + static_cast<size_t>(from) * mixed_stride));
            }
            const float value[4] = {row.lo.x, row.lo.y, row.hi.x, row.hi.y};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float old = from == -1 ? held[c * 3 + 2] : from == -2 ? held[c * 3 + 1] : held[c * 3];
                left[c * 3 + j] = from >= 0 ? value[c] : old;
            }
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            history[i] = make_float4(left[4 * i], left[4 * i + 1], left[4 * i + 2], left[4 * i + 3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTaps - 1; ++j) {
            window[j] = unpack4(*reinterpret_cast<const uint2*>(source - static_cast<size_t>(kTaps - 1 - j) * mixed_stride));
        }
    }
    __nv_bfloat16* target = qkv + row * channels + channel;
    const float unit = head < kDeltaKeyHeads ? 0.08838834764831845f : 1.0f;  // 128^-1/2 for q
#pragma unroll 1
    for (int begin = 0; begin < count; begin += kStepTokens) {
#pragma unroll
        for (int t = 0; t < kStepTokens; ++t) {
            window[kTaps - 1] = unpack4(raw[t]);
            if (kTileTokens > kStepTokens) {
                raw[t] = fetch(begin + kStepTokens + t);
            }
            Channels x = multiply(taps[0], window[0]);
#pragma unroll
            for (int j = 1; j < kTaps; ++j) {
                x = multiply_add(taps[j], window[j], x);
                window[j - 1] = window[j];
            }
            x = multiply(x, {sigmoid_pair(x.lo), sigmoid_pair(x.hi)});
            if (head < 2 * kDeltaKeyHeads) {
                const float total = warp_sum(x.lo.x * x.lo.x + x.lo.y * x.lo.y + x.hi.x * x.hi.x + x.hi.y * x.hi.y);
                const float inverse = rsqrtf(total + 1e-6f) * unit;
                const float2 both = make_float2(inverse, inverse);
                x = multiply(x, {both, both});
            }
            const __nv_bfloat162 lo = __floats2bfloat162_rn(x.lo.x, x.lo.y), hi = __floats2bfloat162_rn(x.hi.x, x.hi.y);
            if (begin + t < count) {  // (uniform over the CTA)
                *reinterpret_cast<uint2*>(target) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
            target += channels;
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
        !aligned(conv_weight) || !aligned(conv_state) || !aligned(qkv)) {
        return cudaErrorInvalidValue;
    }
    int* status = status_ptr();
    if (status == nullptr) {
        return cudaErrorInvalidValue;
    }
    const auto launch = [&](auto kernel, int tile_tokens) {
        const dim3 grid((2 * kDeltaKeyHeads + v_heads) / kPrepareWarps + 1, most_chunk_tiles(tokens, sequences, tile_tokens));
        return launch_chained(
            kernel, grid, dim3(kPrepareWarps * 32), 0, stream, static_cast<const __nv_bfloat16*>(mixed_qkv),
            static_cast<const __nv_bfloat16*>(a_projection), static_cast<const __nv_bfloat16*>(b_projection),
            static_cast<const __nv_bfloat16*>(conv_weight), static_cast<const __nv_bfloat16*>(a_log),
            static_cast<const __nv_bfloat16*>(dt_bias), static_cast<float*>(conv_state),
            static_cast<const uint32_t*>(state_slots), static_cast<const uint32_t*>(continues),
            static_cast<const uint32_t*>(chunk_begins), static_cast<__nv_bfloat16*>(qkv), static_cast<float*>(alpha),
            static_cast<float*>(beta), tokens, sequences, mixed_stride, gate_stride, v_heads, state_capacity, status);
    };
    // The shortest tile with no more than 1500 CTAs (three to four rounds of what is resident at once; a chunk's last tile
    // counts as one, however short it is), or the longest.
    // Measured (us, tiles of 8 / 16 / 32): 17 tokens, 32 heads 4.5 / 6.5 / 8.2; with 48 heads 512 tokens 9.6 / 9.8 / 13.7, 1088
    // tokens 15.2 / 15.3 / 15.9, 2100 tokens 27.1 / 24.6 / 25.4, 8192 tokens 96 / 82 / 79 (4.3 TB/s); 1088 tokens in 64 chunks
    // 27.3 / 23.3 / 22.4, in 128 chunks 40.5 / 32.4 / 31.1.
    const int ctas_per_tile = (2 * kDeltaKeyHeads + v_heads) / kPrepareWarps + 1;
    if (most_chunk_tiles(tokens, sequences, 8) * ctas_per_tile <= 1500) {
        return launch(delta_prepare_chunk_kernel<8>, 8);
    }
    if (most_chunk_tiles(tokens, sequences, 16) * ctas_per_tile <= 1500) {
        return launch(delta_prepare_chunk_kernel<16>, 16);
    }
    return launch(delta_prepare_chunk_kernel<32>, 32);
}
