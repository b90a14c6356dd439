// Attention of a ragged batch of chunks of new tokens over the paged e4m3 cache: token i of a chunk of n tokens stands at
// position context - n + i of its sequence (context_lengths count the chunk) and sees the positions up to its own.
//   o = sum_j softmax_j(scale q . k_j) v_j, times sigmoid(gate)
// Heads, cache and gate as in the decode attention (cuda/paged_attention.cu:1299-1713); the chunk's own keys and values
// are in the cache already.  A row that sees nothing is zero.
//
// A CTA has one token and one KV head, its warps take the positions w, w + 8, ... with the six query heads of the group in
// registers, and their sums meet in shared memory.

#include "chunk.cuh"

namespace qwc {
namespace {

constexpr int kWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void e4m3x8_to_float(const uint2& codes, float (&out)[8]) {
    const uint32_t words[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t lo, hi;
        cvt_e4m3x4_to_f16x2(words[i], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        out[4 * i] = a.x;
        out[4 * i + 1] = a.y;
        out[4 * i + 2] = b.x;
        out[4 * i + 3] = b.y;
    }
}

__global__ void __launch_bounds__(kWarps * 32) chunk_attention_kernel(
    const __nv_bfloat16* __restrict__ query, const __nv_bfloat16* __restrict__ gate, const uint8_t* __restrict__ keys,
    const uint8_t* __restrict__ values, const uint32_t* __restrict__ block_tables,
    const uint32_t* __restrict__ context_lengths, const uint32_t* __restrict__ begins,
    const float* __restrict__ key_scales, const float* __restrict__ value_scales, __nv_bfloat16* __restrict__ output,
    int tokens, int sequences, int max_blocks, int page_size, int num_blocks, int gate_stride, float softmax_scale) {
    pdl_launch_dependents();
    __shared__ float maxima[kWarps][kGqaGroup], sums[kWarps][kGqaGroup];
    __shared__ float partial[kWarps][kHeadDim];
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int kv_head = blockIdx.y;
    pdl_wait();
    const ChunkTile tile = find_chunk_tile(begins, sequences, tokens, 1, blockIdx.x);
    if (tile.sequence < 0) {
        return;
    }
    const size_t row = static_cast<size_t>(tile.span.begin) + tile.index;
    const uint32_t context =
        min(__ldcg(context_lengths + tile.sequence), static_cast<uint32_t>(max_blocks) * static_cast<uint32_t>(page_size));
    const int hidden_behind = tile.span.length - 1 - tile.index;  // later tokens of the chunk
    const int visible = static_cast<int>(context) - hidden_behind;
    const uint32_t* table = block_tables + static_cast<size_t>(tile.sequence) * max_blocks;
    const float scale = softmax_scale * kLog2e * (key_scales ? key_scales[kv_head] : 1.0f);
    float q[kGqaGroup][8], acc[kGqaGroup][8], running_max[kGqaGroup], running_sum[kGqaGroup];
#pragma unroll
    for (int h = 0; h < kGqaGroup; ++h) {
        const uint4 raw = *reinterpret_cast<const uint4*>(query + (row * kQueryHeads + kv_head * kGqaGroup + h) * kHeadDim + 8 * lane);
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[h][2 * i] = __uint_as_float(words[i] << 16) * scale;
            q[h][2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u) * scale;
            acc[h][2 * i] = acc[h][2 * i + 1] = 0.0f;
        }
        running_max[h] = -INFINITY;
        running_sum[h] = 0.0f;
    }
    for (int position = warp; position < visible; position += kWarps) {
        const uint32_t page = __ldg(table + position / page_size);
        const bool exists = page < static_cast<uint32_t>(num_blocks);
        const size_t at = ((static_cast<size_t>(page) * kKvHeads + kv_head) * page_size + position % page_size) * kHeadDim + 8 * lane;
        float k[8], v[8];
        e4m3x8_to_float(exists ? *reinterpret_cast<const uint2*>(keys + at) : make_uint2(0, 0), k);
        e4m3x8_to_float(exists ? *reinterpret_cast<const uint2*>(values + at) : make_uint2(0, 0), v);
#pragma unroll
        for (int h = 0; h < kGqaGroup; ++h) {
            float score = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                score = fmaf(q[h][i], k[i], score);
            }
            score = warp_sum(score);
            const float new_max = fmaxf(running_max[h], score);
            const float factor = exp2f(running_max[h] - new_max);
            const float weight = exp2f(score - new_max);
            running_sum[h] = fmaf(running_sum[h], factor, weight);
            running_max[h] = new_max;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[h][i] = fmaf(acc[h][i], factor, weight * v[i]);
            }
        }
    }
    if (lane == 0) {
#pragma unroll
        for (int h = 0; h < kGqaGroup; ++h) {
            maxima[warp][h] = running_max[h];
            sums[warp][h] = running_sum[h];
        }
    }
    __syncthreads();
    const float v_scale = value_scales ? value_scales[kv_head] : 1.0f;
    const int dim = threadIdx.x;
#pragma unroll
    for (int h = 0; h < kGqaGroup; ++h) {
        float highest = -INFINITY;
        for (int w = 0; w < kWarps; ++w) {
            highest = fmaxf(highest, maxima[w][h]);
        }
        const float factor = running_sum[h] > 0.0f ? exp2f(running_max[h] - highest) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            partial[warp][8 * lane + i] = acc[h][i] * factor;
        }
        __syncthreads();
        float total = 0.0f, denominator = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            total += partial[w][dim];
            denominator += sums[w][h] > 0.0f ? sums[w][h] * exp2f(maxima[w][h] - highest) : 0.0f;
        }
        float value = denominator > 0.0f ? total * v_scale / denominator : 0.0f;
        const int head = kv_head * kGqaGroup + h;
        if (gate != nullptr) {
            value *= 1.0f / (1.0f + __expf(-__bfloat162float(gate[row * gate_stride + head * (2 * kHeadDim) + kHeadDim + dim])));
        }
        output[(row * kQueryHeads + head) * kHeadDim + dim] = __float2bfloat16(value);
        __syncthreads();
    }
}

}  // namespace
}  // namespace qwc

extern "C" size_t qwc_paged_attention_chunk_workspace_bytes(void) { return 0; }

extern "C" int qwc_paged_attention_chunk_fp8(const void* query, const void* query_gate_projection, const void* key_cache,
                                             const void* value_cache, const void* block_tables,
                                             const void* context_lengths, const void* chunk_begins,
                                             const float* key_scales, const float* value_scales, void* output,
                                             void* workspace, size_t workspace_bytes, int tokens, int sequences,
                                             int max_blocks, int page_size, int num_blocks, int gate_stride,
                                             float softmax_scale, cudaStream_t stream) {
    using namespace qwc;
    const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (gate_stride == 0) {
        gate_stride = kQueryHeads * 2 * kHeadDim;
    }
    if (query == nullptr || key_cache == nullptr || value_cache == nullptr || block_tables == nullptr ||
        context_lengths == nullptr || chunk_begins == nullptr || output == nullptr || tokens <= 0 ||
        tokens > kMaxChunkTokens || sequences <= 0 || sequences > kMaxChunkSequences || max_blocks <= 0 ||
        (page_size != 16 && page_size != 64) || static_cast<long long>(max_blocks) * page_size > 0x7fffffffll ||
        num_blocks <= 0 || static_cast<long long>(num_blocks) * kKvHeads * page_size > 0x7fffffffll ||
        gate_stride < kQueryHeads * 2 * kHeadDim || gate_stride % 8 != 0 || !isfinite(softmax_scale) ||
        softmax_scale <= 0.0f || !aligned(query) || !aligned(query_gate_projection) || !aligned(key_cache) ||
        !aligned(value_cache) || !aligned(output) || !aligned(workspace) ||
        workspace_bytes < qwc_paged_attention_chunk_workspace_bytes()) {
        return cudaErrorInvalidValue;
    }
    return launch_chained(chunk_attention_kernel, dim3(tokens, kKvHeads), dim3(kWarps * 32), 0, stream,
                          static_cast<const __nv_bfloat16*>(query), static_cast<const __nv_bfloat16*>(query_gate_projection),
                          static_cast<const uint8_t*>(key_cache), static_cast<const uint8_t*>(value_cache),
                          static_cast<const uint32_t*>(block_tables), static_cast<const uint32_t*>(context_lengths),
                          static_cast<const uint32_t*>(chunk_begins), key_scales, value_scales,
                          static_cast<__nv_bfloat16*>(output), tokens, sequences, max_blocks, page_size, num_blocks,
                          gate_stride, softmax_scale);
}
