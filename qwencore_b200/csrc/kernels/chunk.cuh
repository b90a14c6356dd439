// What the operators on chunks of new tokens share: a ragged batch of `sequences` chunks lies in rows
// begins[s] .. begins[s + 1] of [tokens] rows (begins u32[sequences + 1], ascending).  Rows before the first and
// behind the last chunk belong to nobody and are left as they are; begins beyond `tokens` are cut there.
#pragma once

#include "common.cuh"

namespace qwc {

constexpr int kMaxChunkTokens = 65536;
constexpr int kMaxChunkSequences = 128;

struct ChunkSpan {
    int begin;   // first row
    int length;  // rows
};

__device__ __forceinline__ ChunkSpan chunk_span(const uint32_t* begins, int sequence, int tokens) {
    const uint32_t first = min(__ldcg(begins + sequence), static_cast<uint32_t>(tokens));
    const uint32_t end = min(__ldcg(begins + sequence + 1), static_cast<uint32_t>(tokens));
    return {static_cast<int>(first), end > first ? static_cast<int>(end - first) : 0};
}

// The status word as the operators on chunks take it.  A wait that gave up, anywhere, leaves results that nobody should build
// on: the kernels that wait do nothing then, and leave outputs and states as they were.  An id out of range (a slot, a unit of
// a copy) has left out its own chunk or pair and nothing else, so it does not stop them.
__device__ __forceinline__ bool is_range_code(int code) { return code == kStatusStateSlotRange || code == kStatusCopyRange; }

__device__ __forceinline__ int status_code(const int* status) { return *reinterpret_cast<const volatile int*>(status); }

__device__ __forceinline__ bool stops_chunks(int code) { return code != kStatusOk && !is_range_code(code); }

// A wait gave up: its code takes the place of an id out of range, which would not stop the kernels behind this one.
__device__ __forceinline__ void record_wait(int* status, int code) {
    const int before = atomicCAS(status, kStatusOk, code);
    if (is_range_code(before)) {
        atomicCAS(status, before, code);
    }
}

// 2^x and 1 / x of the unit for special functions, to 2^-22 of themselves, without the instructions that would save results
// below 2^-126.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float sigmoid_fast(float x) { return reciprocal_fast(1.0f + exp2_fast(x * -1.4426950408889634f)); }

// (The multiplications and additions of two take one instruction.)
__device__ __forceinline__ float2 sigmoid_pair(float2 x) {
    const float2 y = __fmul2_rn(x, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    const float2 z = __fadd2_rn(make_float2(exp2_fast(y.x), exp2_fast(y.y)), make_float2(1.0f, 1.0f));
    return make_float2(reciprocal_fast(z.x), reciprocal_fast(z.y));
}

// Every chunk is cut into tiles of `tile_tokens` from its own first row; tile numbers run through the chunks in order.
// For a converged warp: which chunk tile `tile` lies in (-1: there is no such tile), and its number inside it.
struct ChunkTile {
    int sequence;
    int index;
    ChunkSpan span;
};

__device__ __forceinline__ ChunkTile find_chunk_tile(const uint32_t* begins, int sequences, int tokens, int tile_tokens,
                                                     int tile) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
    for (int base = 0; base < sequences; base += 32) {
        ChunkSpan span = {0, 0};
        if (base + lane < sequences) {
            span = chunk_span(begins, base + lane, tokens);
        }
        const int mine = (span.length + tile_tokens - 1) / tile_tokens;
        int inclusive = mine;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, inclusive, offset);
            if (lane >= offset) {
                inclusive += other;
            }
        }
        const uint32_t past = __ballot_sync(0xffffffffu, tile < carry + inclusive);
        if (past != 0) {
            const int at = __ffs(past) - 1;
            ChunkTile found;
            found.sequence = base + at;
            found.index = tile - carry - __shfl_sync(0xffffffffu, inclusive - mine, at);
            found.span.begin = __shfl_sync(0xffffffffu, span.begin, at);
            found.span.length = __shfl_sync(0xffffffffu, span.length, at);
            return found;
        }
        carry += __shfl_sync(0xffffffffu, inclusive, 31);
    }
    return {-1, 0, {0, 0}};
}

// No more tiles than this, whatever the chunks are.
inline int most_chunk_tiles(int tokens, int sequences, int tile_tokens) {
    return (tokens + tile_tokens - 1) / tile_tokens + sequences;
}

}  // namespace qwc
