// Attention of a ragged batch of chunks of new tokens over the paged e4m3 cache: token i of a chunk of n tokens stands at
// position context - n + i of its sequence (context_lengths count the chunk) and sees the positions up to its own.
//   o = sum_j softmax_j(scale q . k_j) v_j, times sigmoid(gate)
// Heads, cache and gate as in the decode attention (cuda/paged_attention.cu:1299-1713); the chunk's own keys and values
// are in the cache already.  A row that sees nothing is zero.
//
// Bound by the tensor cores once a chunk has more than a few dozen tokens: 4 * 256 flops for each (row, position).
// Two SMs of a pair work on one item (chunk_plan.h), 42 tokens x 6 heads of a KV head: 126 rows each, of 128.  For every
// unit of 128 positions tcgen05.mma.cta_group::2 computes S = Q K^T and O += P V for all 256 rows; an SM fetches half of
// the operands, 64 of the keys and 128 of the value's dims, which is why it is a pair: alone, an SM would widen twice as
// many values, and read twice as much shared memory for the tensor cores.
//
//   * keys enter as they are stored (kind::f8f6f4).  A row's query is brought to [128, 256) by a power of two and becomes the
//     sum of an e4m3 and an e5m2, one multiplication each: four bits, and then what they leave in three, which holds a
//     bf16's eight bits for 14 binades below the row's largest element.  What is lost below, times the largest key there can
//     be, bounds the error of a score; where that is more than 2^-13 for any row of an item, the item's keys are
//     widened to f16 like the values, and its queries are f16, which hold eight bits for 29 binades;
//   * values are widened: an e4m3 is moved bit by bit into an f16 that is 2^-8 of it, exactly (a shift and two masks for two
//     of them; the factor goes into the scales).  A code that is no number becomes a finite one, so that it does no harm
//     where a probability is zero.  The masks take bytes 0 and 2, 1 and 3 of a word together, so the columns of O lie in
//     that order, and are put right when it is stored;
//   * two threads share a row of S, 64 columns each.  Probabilities go back as f16 into the tensor memory of their scores, as
//     the A operand of P V (their fp32 values are summed).  What they refer to follows the running maximum only when that has
//     grown by 2^4, so that O, which stays in tensor memory for the whole item, is hardly ever rescaled.  The largest is put
//     at 2^11 .. 2^15, near the upper end of what f16 holds: weights down to 2^-25 of the row's largest have eleven bits,
//     smaller ones are off by up to 2^-36 of the largest (a first token that draws the weight and has no value, with thousands
//     of others behind it, is their mean);
//   * tensor memory: two buffers of scores (2 x 128 columns) and O (256 columns).  S of unit n + 1 is issued before P V of unit n.
//
//   warps 0-7   softmax, and the item's result
//   warps 8-11  the query's digits, widening
//   warp 12     fetches K and V, rings of three and two stages
//   warp 13     issues the MMAs (in the pair's first CTA)

#include <algorithm>

#include "chunk.cuh"
#include "chunk_plan.h"
#include "tcgen05.cuh"

namespace qwc {
namespace {

constexpr int kSoftmaxWarps = 8;
constexpr int kFirstWidenWarp = kSoftmaxWarps;
constexpr int kWidenWarps = 4;
constexpr int kFetchWarp = kFirstWidenWarp + kWidenWarps;
constexpr int kMmaWarp = kFetchWarp + 1;
constexpr int kThreads = (kMmaWarp + 1) * 32;
constexpr int kRowTokens = kItemTokens / 2;              // of a CTA's rows
constexpr int kRows = 128;                               // ... 126 of them used
constexpr int kUnit = kPlanUnitTokens;
constexpr int kKeyTokens = kUnit / 2;                    // of a unit that a CTA widens
constexpr int kBoxTokens = 16;
constexpr int kBoxBytes = kBoxTokens * 128;
constexpr int kRawBytes = kKeyTokens * kHeadDim;         // K of a unit, or V: 16 KiB
constexpr int kKeyStages = 3;                           // (values leave theirs when they are widened, keys when they have been used)
constexpr int kValueStages = 2;
constexpr int kKeyBlock = kKeyTokens * 128;              // 64 dims of the widened keys
constexpr int kValueBlock = kUnit * 128;
constexpr int kQueryBlock = kRows * 128;
constexpr int kDigitBytes = 2 * kQueryBlock;             // a digit of the queries: [half of the dims][row][128 bytes]
constexpr int kTmemColumns = 512;
constexpr int kOutputColumn = 2 * kUnit;
constexpr int kMaxPairs = 96;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargest = 11.0f;                        // log2 of a row's largest probability, when its reference is set ...
constexpr float kRescaleAbove = 15.0f;                   // ... and where the reference has to be set again
constexpr float kPartialScale = 128.0f;                  // of partial results: a value code is at most 480
constexpr float kScoreError = 1.0f / 8192.0f;            // of a score, by digits that leave something
static_assert(kPlanHeads == kKvHeads && kRowTokens * kGqaGroup <= kRows, "the plan's items");

struct Smem {
    uint8_t q[4 * kQueryBlock];               // two digits, or f16 [64 dims][row][128 bytes]; 128-byte swizzle
    uint8_t wide[2][2 * kValueBlock];         // V of a unit: [64 dims][token][128 bytes]; or V and K ([64 dims][token][128 bytes])
    uint8_t raw_k[kKeyStages][kRawBytes];     // [half of the dims][token][128 bytes], e4m3, 128-byte swizzle
    uint8_t raw_v[kValueStages][kRawBytes];     // [token][128 bytes]
    uint64_t raw_k_full[kKeyStages], raw_k_empty[kKeyStages];
    uint64_t raw_v_full[kValueStages], raw_v_empty[kValueStages];
    // (those that the MMAs wait for, k_peer, k_wide, v_full, q_full, q_wide, p_full, o_free: the first CTA's count)
    uint64_t k_peer[kKeyStages];              // the other CTA's keys are there
    uint64_t k_wide, k_empty, v_full[2], v_empty[2];
    uint64_t q_full, q_wide, q_free, scales_ready;
    uint64_t flags_ready, mode_ready;         // of the words inexact and mode
    uint64_t s_full[2], p_full[2];
    uint64_t max_ready[2][4], sum_ready[4];   // of the two warps that share 32 rows
    uint64_t o_done[2], o_free;
    float row_max[2][2][kRows];
    float row_sum[2][kRows];
    float row_scale[kRows];                   // what the row's query times key has been divided by
    uint32_t inexact[2 * kWidenWarps];        // rows whose digits leave too much, by warp of the pair (first CTA)
    uint32_t mode;                            // what follows from that: queries and keys are widened
    ChunkSequence sequence[kMaxChunkSequences];
    long long sequence_line[kMaxChunkSequences];  // a head's length of line
    ChunkWalk start;
    long long total;
    uint32_t tmem_base;
    int stop;    // nothing is done: a wait of an earlier kernel has given up
    int failed;  // a wait gave up
};
static_assert(sizeof(Smem) + 1024 <= 232448, "shared memory of a CTA");

// What a pair leaves of an item that is cut: statistics and normalised rows of both CTAs, two slots for each pair.  The
// rows are f16, in units of the value scale / 128: eleven bits, and nothing below 2^-32 of the scale.
struct PartialStats {
    float maximum;  // log2
    float sum;
};
struct MergeItem {
    int sequence;  // -1: nothing to merge
    int head;
    int tile;
    int last_pair;
    int first_row;
    int rows;      // tokens
};
constexpr size_t kSlotRows = 2 * kRows;
constexpr size_t kOutBytes = static_cast<size_t>(kMaxPairs) * 2 * kSlotRows * kHeadDim * sizeof(__half);
constexpr size_t kStatsBytes = static_cast<size_t>(kMaxPairs) * 2 * kSlotRows * sizeof(PartialStats);
constexpr size_t kWorkspaceBytes = kOutBytes + kStatsBytes + kMaxPairs * sizeof(MergeItem);

struct Params {
    const __nv_bfloat16* query;
    const __nv_bfloat16* gate;
    const uint32_t* block_tables;
    const uint32_t* context_lengths;
    const uint32_t* begins;
    const float* key_scales;
    const float* value_scales;
    __nv_bfloat16* output;
    __half* partial_out;
    PartialStats* partial_stats;
    MergeItem* merge;
    int tokens, sequences, max_blocks, page_size, num_blocks, gate_stride;
    int wide_rows;  // gate, output and partial rows begin on 32-byte boundaries
    float softmax_scale;
    int* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return rank;
}

__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// An arrival at the barrier of the pair's first CTA, for what has been written to this CTA's tensor memory, or to its shared
// memory and handed to the tensor cores by a proxy fence.  (No release at the scope of the pair: that waits for every
// store of the warp, 2763 us instead of 2092 for 4096 tokens over 28672.)
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
    asm volatile(
        "{\n"
        ".reg .b32 remote;\n"
        "mapa.shared::cluster.u32 remote, %0, 0;\n"
        "mbarrier.arrive.shared::cluster.b64 _, [remote];\n"
        "}\n" ::"r"(smem_u32(bar))
        : "memory");
}

// A word for the same place of a CTA's shared memory; its four bytes count at the barrier beside it.
__device__ __forceinline__ void tell(uint32_t* word, uint32_t value, uint64_t* bar, uint32_t rank) {
    asm volatile(
        "{\n"
        ".reg .b32 remote, barrier;\n"
        "mapa.shared::cluster.u32 remote, %0, %3;\n"
        "mapa.shared::cluster.u32 barrier, %2, %3;\n"
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [remote], %1, [barrier];\n"
        "}\n" ::"r"(smem_u32(word)),
        "r"(value), "r"(smem_u32(bar)), "r"(rank)
        : "memory");
}

// Every role marches unit by unit with the others, so no wait is long: it gives up after 20 ms.
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, Smem& sm, int* status) {
    const long long start = clock64();
    for (;;) {
#pragma unroll 1
        for (int spin = 0; spin < 64; ++spin) {
            if (mbar_try_wait(bar, parity)) {
                return true;
            }
        }
        if (*reinterpret_cast<volatile int*>(&sm.failed) != 0) {
            return false;
        }
        if (clock64() - start > 40000000ll) {
            break;
        }
    }
    record_wait(status, kStatusChunkAttentionWait);
    *reinterpret_cast<volatile int*>(&sm.failed) = 1;
    return false;
}

// For a converged warp: the same answer in every lane.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Smem& sm, int* status) {
    const bool ok = mbar_try_wait(bar, parity) || wait_slow(bar, parity, sm, status);
    return __all_sync(0xffffffffu, ok);
}

// D[2 x 128][N] (+)= A[2 x 128][16] x B[N][16], f16, fp32 accumulate, both SMs of the pair: A from shared memory ...
__device__ __forceinline__ void pair_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// ... 32 eight-bit elements each ...
__device__ __forceinline__ void pair_mma_fp8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// ... or A from tensor memory.
__device__ __forceinline__ void pair_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One arrival at the barrier of both CTAs when every MMA issued so far has completed.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// Operand of 128-byte rows with the 128-byte swizzle, eight rows to an atom.  K-major: a row is one of M or N, its bytes 64
// of the contracted elements.  MN-major: a row is one of the contracted, its bytes 64 of M or N, the next 64 `block` bytes on.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t block) {
    const uint64_t lo = ((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16);
    const uint64_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return lo | (hi << 32);
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Largest of three; a NaN counts as nothing.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t out;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(hi), "f"(lo));
    return out;
}

// Two numbers below 256 as e4m3 and, of what that leaves, as e5m2, in f16 arithmetic; returns the magnitudes of what is left
// at last.  (A warp has its scheduler's attention for an instruction every three or four cycles here: what counts is how
// few there are.  Rounding to e5m2 with integer operations instead of conversions was slower, fp32 arithmetic too.)
__device__ __forceinline__ __half2 take_digits(float lo, float hi, uint32_t& d0, uint32_t& d1) {
    const uint32_t bits = pack_f16(lo, hi);
    uint16_t first, second;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(first) : "r"(bits));
    const uint32_t held = cvt_e4m3x2_to_f16x2(first);
    const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&bits), *reinterpret_cast<const __half2*>(&held));
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(second) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
    d0 = first;
    d1 = second;
    const uint32_t upper = __byte_perm(d1, 0u, 0x1404);  // an e5m2 is the upper byte of an f16
    return __habs2(__hsub2(rest, *reinterpret_cast<const __half2*>(&upper)));
}

// Four e4m3 -> two f16x2 of 2^-8 their value: bytes 0 and 2, bytes 1 and 3.
__device__ __forceinline__ void widen4(uint32_t word, uint32_t& even, uint32_t& odd) {
    even = ((word << 7) & 0x3f803f80u) | ((word << 8) & 0x80008000u);
    odd = ((word >> 1) & 0x3f803f80u) | (word & 0x80008000u);
}

// 64 bytes of eight raw rows of 128 bytes -> f16, by a warp: `half` of the row.  Sixteen bytes per lane; lanes 0-3 and 4-7 of
// a phase read rows that differ in bits 0 and 2, so that neither the loads nor the stores meet in a bank.
__device__ __forceinline__ void widen_rows(const uint8_t* raw, uint8_t* wide, int half, int lane) {
    const int group = lane >> 3;
    const int row = (lane & 4) != 0 ? group ^ 5 : group;
    const int piece = lane & 3;
    const uint4 codes = *reinterpret_cast<const uint4*>(raw + row * 128 + (((half * 4 + piece) ^ row) << 4));
    uint4 lo, hi;
    widen4(codes.x, lo.x, lo.y);
    widen4(codes.y, lo.z, lo.w);
    widen4(codes.z, hi.x, hi.y);
    widen4(codes.w, hi.z, hi.w);
    *reinterpret_cast<uint4*>(wide + row * 128 + (((2 * piece) ^ row) << 4)) = lo;
    *reinterpret_cast<uint4*>(wide + row * 128 + (((2 * piece + 1) ^ row) << 4)) = hi;
}

// 64 bytes of a row, half of it at a time where the rows begin on 32-byte boundaries (`wide`): whole sectors, of 32 rows
// in one instruction.
__device__ __forceinline__ void load64(const void* from, int wide, uint4 (&to)[4]) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(to[2 * i].x), "=r"(to[2 * i].y), "=r"(to[2 * i].z), "=r"(to[2 * i].w), "=r"(to[2 * i + 1].x),
                           "=r"(to[2 * i + 1].y), "=r"(to[2 * i + 1].z), "=r"(to[2 * i + 1].w)
                         : "l"(static_cast<const char*>(from) + 32 * i));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            to[i] = reinterpret_cast<const uint4*>(from)[i];
        }
    }
}

__device__ __forceinline__ void store64(void* to, int wide, const uint4 (&from)[4]) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(static_cast<char*>(to) + 32 * i),
                         "r"(from[2 * i].x), "r"(from[2 * i].y), "r"(from[2 * i].z), "r"(from[2 * i].w), "r"(from[2 * i + 1].x),
                         "r"(from[2 * i + 1].y), "r"(from[2 * i + 1].z), "r"(from[2 * i + 1].w)
                         : "memory");
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            reinterpret_cast<uint4*>(to)[i] = from[i];
        }
    }
}

// Cache pages as rows of 256 bytes, fetched in boxes of 16 tokens x 128 bytes.  A row beyond the cache arrives as zeros.
cudaError_t encode_pages(CUtensorMap* map, const void* cache, long long rows) {
    const EncodeTiled encode = tensor_map_encoder();
    if (encode == nullptr) {
        return cudaErrorNotSupported;
    }
    const cuuint64_t dims[2] = {kHeadDim, static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {kHeadDim};
    const cuuint32_t box[2] = {128, kBoxTokens};
    const cuuint32_t element_strides[2] = {1, 1};
    const CUresult result =
        encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(cache), dims, strides, box, element_strides,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return result == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

__device__ __forceinline__ ChunkSequence sequence_info(const Params& p, int sequence) {
    const ChunkSpan span = chunk_span(p.begins, sequence, p.tokens);
    const uint32_t capacity = static_cast<uint32_t>(p.max_blocks) * static_cast<uint32_t>(p.page_size);
    return {span.begin, span.length, static_cast<int>(min(__ldcg(p.context_lengths + sequence), capacity))};
}

// Where this pair's share of the line begins, by the whole CTA.
__device__ __forceinline__ void find_start(const Params& p, Smem& sm, int pair, int pairs) {
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    for (int s = warp; s < p.sequences; s += kThreads / 32) {
        const ChunkSequence info = sequence_info(p, s);
        const int tiles = item_tiles(info);
        long long sum = 0;
        for (int tile = lane; tile < tiles; tile += 32) {
            sum += item_units(info, tile) + kItemLead;
        }
#pragma unroll
        for (int offset = 16; offset > 0; offset >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, offset);
        }
        if (lane == 0) {
            sm.sequence[s] = info;
            sm.sequence_line[s] = sum;
        }
    }
    __syncthreads();
    if (warp != 0) {
        return;
    }
    long long total = 0;
    for (int s = lane; s < p.sequences; s += 32) {
        total += kPlanHeads * sm.sequence_line[s];
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, offset);
    }
    const int workers = plan_workers(total, pairs);
    const long long begin = share_begin(total, pair, workers);
    ChunkWalk walk = {};
    walk.left = pair < workers ? share_begin(total, pair + 1, workers) - begin : 0;
    // the sequence: a warp scan for 32 of them
    long long carry = 0;
    for (int base = 0; base < p.sequences && walk.left > 0; base += 32) {
        const long long mine = base + lane < p.sequences ? kPlanHeads * sm.sequence_line[base + lane] : 0;
        long long inclusive = mine;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, inclusive, offset);
            if (lane >= offset) {
                inclusive += other;
            }
        }
        const uint32_t past = __ballot_sync(0xffffffffu, begin < carry + inclusive);
        if (past != 0) {
            const int at = __ffs(past) - 1;
            walk.sequence = base + at;
            carry += __shfl_sync(0xffffffffu, inclusive - mine, at);
            break;
        }
        carry += __shfl_sync(0xffffffffu, inclusive, 31);
    }
    if (walk.left > 0) {
        walk.info = sm.sequence[walk.sequence];
        const long long head_line = sm.sequence_line[walk.sequence];
        for (; walk.head < kPlanHeads - 1 && begin >= carry + head_line; ++walk.head) {
            carry += head_line;
        }
        // ... and the tile
        const int tiles = item_tiles(walk.info);
        for (int base = 0; base < tiles; base += 32) {
            const long long mine = base + lane < tiles ? item_units(walk.info, base + lane) + kItemLead : 0;
            long long inclusive = mine;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const long long other = __shfl_up_sync(0xffffffffu, inclusive, offset);
                if (lane >= offset) {
                    inclusive += other;
                }
            }
            const uint32_t past = __ballot_sync(0xffffffffu, begin < carry + inclusive);
            if (past != 0) {
                const int at = __ffs(past) - 1;
                walk.tile = base + at;
                carry += __shfl_sync(0xffffffffu, inclusive - mine, at);
                break;
            }
            carry += __shfl_sync(0xffffffffu, inclusive, 31);
        }
        walk.skip = begin - carry;
        walk.at = carry;
    }
    if (lane == 0) {
        sm.start = walk;
        sm.total = total;
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    chunk_attention_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                           const __grid_constant__ Params p) {
    extern __shared__ unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int rank = static_cast<int>(cluster_rank());
    const int pair = blockIdx.x >> 1;
    const int pairs = gridDim.x >> 1;

    if (threadIdx.x == kFetchWarp * 32) {
        for (int i = 0; i < kKeyStages; ++i) {
            mbar_init(&sm.raw_k_full[i], 1);
            mbar_init(&sm.raw_k_empty[i], 1);
            mbar_init(&sm.k_peer[i], 1);
        }
        for (int i = 0; i < kValueStages; ++i) {
            mbar_init(&sm.raw_v_full[i], 1);
            mbar_init(&sm.raw_v_empty[i], kWidenWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.v_full[i], 2 * kWidenWarps);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 2 * kSoftmaxWarps);
            mbar_init(&sm.o_done[i], 1);
            for (int j = 0; j < 4; ++j) {
                mbar_init(&sm.max_ready[i][j], 2);
            }
        }
        for (int j = 0; j < 4; ++j) {
            mbar_init(&sm.sum_ready[j], 2);
        }
        mbar_init(&sm.k_wide, 2 * kWidenWarps);
        mbar_init(&sm.k_empty, 1);
        mbar_init(&sm.q_full, 2 * kWidenWarps);
        mbar_init(&sm.q_wide, 2 * kWidenWarps);
        mbar_init(&sm.q_free, 1 + kSoftmaxWarps);
        mbar_init(&sm.scales_ready, kWidenWarps);
        mbar_init(&sm.flags_ready, 1);
        mbar_init(&sm.mode_ready, 1);
        mbar_init(&sm.o_free, 2 * kSoftmaxWarps);
        sm.failed = 0;
        mbar_fence_init();
    }
    fence_proxy_async();
    __syncthreads();
    pair_sync();  // (the other CTA's shared memory is there)
    pdl_wait();
    // Tensor memory is asked for when the kernels before this one have given theirs back, and the next kernel may start
    // when this CTA has its own: CTAs of two kernels that each held some and asked for the rest would wait for each other.
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (rank == 0 && threadIdx.x < 2) {
        // both CTAs of a pair go by what the first one finds in the status word
        const uint32_t stop = stops_chunks(status_code(p.status)) ? 1u : 0u;
        asm volatile(
            "{\n"
            ".reg .b32 remote;\n"
            "mapa.shared::cluster.u32 remote, %0, %1;\n"
            "st.shared::cluster.u32 [remote], %2;\n"
            "}\n" ::"r"(smem_u32(&sm.stop)),
            "r"(threadIdx.x), "r"(stop)
            : "memory");
    }
    find_start(p, sm, pair, pairs);
    __syncthreads();
    pdl_launch_dependents();
    pair_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sm.tmem_base);
    const auto info = [&](int sequence) { return sm.sequence[sequence]; };
    ChunkWalk walk = sm.start;
    if (*reinterpret_cast<volatile int*>(&sm.stop) != 0) {
        walk.left = 0;
    }
    ChunkPiece piece;
    bool ok = true;
    int g = 0;     // units so far
    int item = 0;  // pieces so far

    if (warp == kFetchWarp) {
        // ---------------- lanes 0-7: K, 16 tokens x 128 bytes each; lanes 8-15: V ------------------
        const bool keys = lane < 8;
        const int token = keys ? rank * kKeyTokens + (lane >> 1) * kBoxTokens : (lane - 8) * kBoxTokens;  // of the unit
        const int x = keys ? (lane & 1) * 128 : rank * 128;
        const int page_shift = p.page_size == 16 ? 4 : 6;
        const int offset = keys ? (lane & 1) * kKeyTokens * 128 + (lane >> 1) * kBoxBytes : (lane - 8) * kBoxBytes;
        for (bool first = true; ok && next_piece(walk, first, p.sequences, info, piece); first = false) {
            const uint32_t* table = p.block_tables + static_cast<size_t>(walk.sequence) * p.max_blocks;
            for (int unit = piece.unit_begin; unit < piece.unit_end; ++unit, ++g) {
                const int k_slot = g % kKeyStages, v_slot = g % kValueStages;
                const long long position = static_cast<long long>(unit) * kUnit + token;
                int row = -kBoxTokens;  // in front of the cache: zeros
                if (lane < 16 && position < walk.info.context) {
                    const uint32_t page = __ldg(table + (position >> page_shift));
                    if (page < static_cast<uint32_t>(p.num_blocks)) {
                        row = (((static_cast<int>(page) * kKvHeads + walk.head) << page_shift) |
                              static_cast<int>(position & (p.page_size - 1)));
                    }
                }
                ok = wait(&sm.raw_k_empty[k_slot], ((g / kKeyStages) & 1) ^ 1, sm, p.status);
                if (!ok) {
                    break;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sm.raw_k_full[k_slot], kRawBytes);
                }
                __syncwarp();
                if (lane < 8) {
                    tma_box_g2s(sm.raw_k[k_slot] + offset, &key_map, x, row, &sm.raw_k_full[k_slot]);
                }
                __syncwarp();
                ok = wait(&sm.raw_v_empty[v_slot], ((g / kValueStages) & 1) ^ 1, sm, p.status);
                if (lane == 0) {
                    // (asked for or not: what is left out on giving up is not waited for)
                    if (ok) {
                        mbar_arrive_expect_tx(&sm.raw_v_full[v_slot], kRawBytes);
                    }
                }
                __syncwarp();
                if (ok && lane >= 8 && lane < 16) {
                    tma_box_g2s(sm.raw_v[v_slot] + offset, &value_map, x, row, &sm.raw_v_full[v_slot]);
                }
                __syncwarp();
                if (!ok) {
                    ++g;  // its keys are on their way
                    break;
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- tensor-core issue, for both CTAs ------------------------------------------
        if (rank == 0) {
            const uint32_t idesc_scores = (1u << 4) | (static_cast<uint32_t>(kUnit >> 3) << 17) | (16u << 24);
            const uint32_t idesc_rest = idesc_scores | (1u << 7);  // A is e5m2
            const uint32_t idesc_output = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(kHeadDim >> 3) << 17) | (16u << 24);
            const uint32_t q_base = smem_u32(sm.q);
            bool widened = false;
            int wide_items = 0, wide_units = 0;
            // P V of unit number `number`
            const auto issue_output = [&](int number, bool first_unit) {
                const int buffer = number & 1;
                if (!wait(&sm.p_full[buffer], (number >> 1) & 1, sm, p.status) ||
                    !wait(&sm.v_full[buffer], (number >> 1) & 1, sm, p.status)) {
                    return false;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint32_t v_base = smem_u32(sm.wide[widened ? 0 : buffer]);
#pragma unroll
                    for (int ks = 0; ks < kUnit / 16; ++ks) {
                        pair_mma_ts(tmem_base + kOutputColumn, tmem_base + buffer * kUnit + ks * 8,
                                    operand(v_base + ks * 2048, kValueBlock), idesc_output, first_unit && ks == 0 ? 0u : 1u);
                    }
                    pair_commit(&sm.v_empty[buffer]);
                    pair_commit(&sm.o_done[buffer]);
                }
                __syncwarp();
                return true;
            };
            for (bool first = true; ok && next_piece(walk, first, p.sequences, info, piece); first = false) {
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sm.flags_ready, 2 * kWidenWarps * 4);
                }
                __syncwarp();
                ok = wait(&sm.q_full, item & 1, sm, p.status) && wait(&sm.flags_ready, item & 1, sm, p.status);
                widened = __any_sync(0xffffffffu, lane < 2 * kWidenWarps && sm.inexact[lane & (2 * kWidenWarps - 1)] != 0);
                if (ok && lane < 2) {
                    tell(&sm.mode, widened ? 1u : 0u, &sm.mode_ready, lane);
                }
                __syncwarp();
                if (ok && widened) {
                    ok = wait(&sm.q_wide, wide_items & 1, sm, p.status);
                    ++wide_items;
                }
                for (int unit = piece.unit_begin; ok && unit < piece.unit_end; ++unit, ++g) {
                    const int buffer = g & 1;
                    if (!widened) {
                        ok = wait(&sm.raw_k_full[g % kKeyStages], (g / kKeyStages) & 1, sm, p.status) &&
                             wait(&sm.k_peer[g % kKeyStages], (g / kKeyStages) & 1, sm, p.status);
                    } else {
                        ok = wait(&sm.k_wide, wide_units & 1, sm, p.status);
                        ++wide_units;
                    }
                    if (!ok) {
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
                        const uint32_t d = tmem_base + buffer * kUnit;
                        if (!widened) {
                            const uint32_t k_base = smem_u32(sm.raw_k[g % kKeyStages]);
#pragma unroll
                            for (int ks = 0; ks < kHeadDim / 32; ++ks) {
                                const uint64_t keys = operand(k_base + (ks >> 2) * (kKeyTokens * 128) + (ks & 3) * 32, 16);
                                const uint32_t a = q_base + (ks >> 2) * kQueryBlock + (ks & 3) * 32;
                                pair_mma_fp8(d, operand(a, 16), keys, idesc_scores, ks > 0 ? 1u : 0u);
                                pair_mma_fp8(d, operand(a + kDigitBytes, 16), keys, idesc_rest, 1u);
                            }
                        } else {
                            const uint32_t k_base = smem_u32(sm.wide[1]);
#pragma unroll
                            for (int ks = 0; ks < kHeadDim / 16; ++ks) {
                                pair_mma_ss(d, operand(q_base + (ks >> 2) * kQueryBlock + (ks & 3) * 32, 16),
                                            operand(k_base + (ks >> 2) * kKeyBlock + (ks & 3) * 32, 16), idesc_scores, ks > 0 ? 1u : 0u);
                            }
                        }
                        pair_commit(&sm.s_full[buffer]);
                        pair_commit(&sm.raw_k_empty[g % kKeyStages]);
                        pair_commit(&sm.k_empty);
                        if (unit == piece.unit_end - 1) {
                            pair_commit(&sm.q_free);
                        }
                    }
                    __syncwarp();
                    if (unit == piece.unit_begin) {
                        // O of the item before has been read
                        ok = wait(&sm.o_free, (item & 1) ^ 1, sm, p.status);
                    } else {
                        ok = issue_output(g - 1, unit == piece.unit_begin + 1);
                    }
                }
                if (ok) {
                    ok = issue_output(g - 1, piece.unit_end - piece.unit_begin == 1);
                }
                ++item;
            }
        } else {
            // the second CTA's keys, told to the first
            for (bool first = true; ok && next_piece(walk, first, p.sequences, info, piece); first = false) {
                for (int unit = piece.unit_begin; ok && unit < piece.unit_end; ++unit, ++g) {
                    ok = wait(&sm.raw_k_full[g % kKeyStages], (g / kKeyStages) & 1, sm, p.status);
                    if (ok && lane == 0) {
                        arrive_first(&sm.k_peer[g % kKeyStages]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= kFirstWidenWarp) {
        // ---------------- the query's digits; V (and K) to f16 ------------------------------------------
        const int me = warp - kFirstWidenWarp;
        constexpr int kWarpRows = kRows / kWidenWarps;
        constexpr int kAhead = 8;  // rows in flight, eight dims per lane
        bool widened = false, was_widened = false;
        const auto widen_keys = [&](int number) {
            const int slot = number % kKeyStages;
            if (!wait(&sm.raw_k_full[slot], (number / kKeyStages) & 1, sm, p.status) ||
                !wait(&sm.k_empty, (number & 1) ^ 1, sm, p.status)) {
                return false;
            }
#pragma unroll 4
            for (int i = me; i < 32; i += kWidenWarps) {  // half of the dims, eight tokens, half of a raw row
                const int block = i >> 3, rows = (i & 7) * 8;
                widen_rows(sm.raw_k[slot] + (block >> 1) * (kKeyTokens * 128) + rows * 128,
                           sm.wide[1] + block * kKeyBlock + rows * 128, block & 1, lane);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                arrive_first(&sm.k_wide);
            }
            return true;
        };
        const auto widen_values = [&](int number) {
            const int slot = number % kValueStages;
            const int buffer = number & 1;
            if (!wait(&sm.raw_v_full[slot], (number / kValueStages) & 1, sm, p.status) ||
                !wait(&sm.v_empty[buffer], ((number >> 1) & 1) ^ 1, sm, p.status) ||
                // (all units in one buffer: the unit before, too)
                (widened && number > 0 && !wait(&sm.v_empty[buffer ^ 1], ((number - 1) >> 1) & 1, sm, p.status))) {
                return false;
            }
            uint8_t* to = sm.wide[widened ? 0 : buffer];
#pragma unroll 4
            for (int i = me; i < 32; i += kWidenWarps) {
                const int block = i & 1, rows = (i >> 1) * 8;
                widen_rows(sm.raw_v[slot] + rows * 128, to + block * kValueBlock + rows * 128, block, lane);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.raw_v_empty[slot]);
                arrive_first(&sm.v_full[buffer]);
            }
            return true;
        };
        for (bool first = true; ok && next_piece(walk, first, p.sequences, info, piece); first = false) {
            const int first_token = walk.tile * kItemTokens + rank * kRowTokens;
            // row r of the CTA: token r / 6, head r % 6 of the group; the warps take rows in turn
            const uint4* queries = reinterpret_cast<const uint4*>(
                                       p.query + ((static_cast<size_t>(walk.info.begin) + first_token) * kQueryHeads +
                                                  walk.head * kGqaGroup) * kHeadDim) + lane;
            const int live_rows = min(kRowTokens, walk.info.length - first_token) * kGqaGroup;
            const auto fetch_row = [&](int index) {
                const uint32_t r = index * kWidenWarps + me;
                constexpr uint32_t kRow = kHeadDim / 8, kToken = (kQueryHeads - kGqaGroup) * kRow;  // in uint4
                return static_cast<int>(r) < live_rows ? __ldg(queries + (r * kRow + r / kGqaGroup * kToken))
                                                                            : make_uint4(0, 0, 0, 0);
            };
            // The row's numbers with its largest in [2^top, 2^(top + 1)), and what they are multiplied with to be what they
            // were; infinities and NaN stay what they are, and rows that are (nearly) zero are not blown up without end.
            const auto scale_row = [&](const uint4& raw, int top, float (&x)[8]) {
                const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
                const uint32_t both = __vmaxu2(__vmaxu2(words[0] & 0x7fff7fffu, words[1] & 0x7fff7fffu),
                                               __vmaxu2(words[2] & 0x7fff7fffu, words[3] & 0x7fff7fffu));
                const uint32_t highest = __reduce_max_sync(0xffffffffu, max(both & 0xffffu, both >> 16));
                const uint32_t exponent = max(highest >> 7, 64u);
                const float up = exponent == 255u ? 1.0f : __uint_as_float((254u + top - exponent) << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 scaled = __fmul2_rn(make_float2(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u)),
                                                     make_float2(up, up));
                    x[2 * i] = scaled.x;
                    x[2 * i + 1] = scaled.y;
                }
                return exponent == 255u ? 1.0f : __uint_as_float((exponent - top) << 23);
            };
            uint4 raw[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                raw[j] = fetch_row(j);
            }
            ok = wait(&sm.q_free, (item & 1) ^ 1, sm, p.status);
            if (!ok) {
                break;
            }
            const float largest_key = 448.0f * p.softmax_scale * (p.key_scales ? fabsf(p.key_scales[walk.head]) : 1.0f);
            // (Four rows at a time, some 12000 cycles an item.  With all of them unrolled the warps waited for instructions:
            // 30000 to 45000.)
            float lost = 0.0f;  // by this lane's elements, over all rows
            float largest_scale = 0.0f;
#pragma unroll 1
            for (int base = 0; base < kWarpRows; base += 4) {
                if (base * kWidenWarps + me >= live_rows) {
                    // none of these rows, nor of those behind: zeros
                    for (int r = base * kWidenWarps + me; r < kRows; r += kWidenWarps) {
                        uint8_t* to = sm.q + (lane >> 4) * kQueryBlock + r * 128 + (lane & 15) * 8;
                        *reinterpret_cast<uint2*>(to) = make_uint2(0u, 0u);
                        *reinterpret_cast<uint2*>(to + kDigitBytes) = make_uint2(0u, 0u);
                        if (lane == 0) {
                            sm.row_scale[r] = 1.0f;
                        }
                    }
                    break;
                }
                const uint4 now[4] = {raw[0], raw[1], raw[2], raw[3]};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    raw[j] = raw[j + 4];
                    raw[j + 4] = fetch_row(base + kAhead + j);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = (base + j) * kWidenWarps + me;
                    float x[8];
                    const float scale = scale_row(now[j], 7, x);
                    uint32_t d0[4], d1[4];
                    __half2 left = __float2half2_rn(0.0f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        left = __hadd2(left, take_digits(x[2 * i], x[2 * i + 1], d0[i], d1[i]));
                    }
                    lost = fmaf(__low2float(left) + __high2float(left), scale, lost);
                    largest_scale = fmaxf(largest_scale, scale);
                    uint8_t* to = sm.q + (lane >> 4) * kQueryBlock + r * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
                    *reinterpret_cast<uint2*>(to) = make_uint2(d0[0] | d0[1] << 16, d0[2] | d0[3] << 16);
                    *reinterpret_cast<uint2*>(to + kDigitBytes) = make_uint2(d1[0] | d1[1] << 16, d1[2] | d1[3] << 16);
                    if (lane == 0) {
                        sm.row_scale[r] = scale;
                    }
                }
            }
            // A score of any row is off by no more than all rows' losses, and what f16 leaves of 256 elements (2^-25 of
            // each at most), times the largest key.  (A NaN or an infinity among the queries: too much.)  The pair's first
            // CTA decides.
            const bool exact = __all_sync(0xffffffffu, lost < INFINITY) &&
                               fmaf(largest_scale, 7.62939453125e-6f, warp_sum(lost)) * largest_key <= kScoreError;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                arrive_first(&sm.q_full);
                tell(&sm.inexact[rank * kWidenWarps + me], exact ? 0u : 1u, &sm.flags_ready, 0);
                if (me == 0) {
                    mbar_arrive_expect_tx(&sm.mode_ready, 4);
                }
            }
            __syncwarp();
            ok = wait(&sm.mode_ready, item & 1, sm, p.status);
            if (!ok) {
                break;
            }
            was_widened = widened;
            widened = *reinterpret_cast<volatile uint32_t*>(&sm.mode) != 0;
            if ((widened || was_widened) && g > 0) {
                // the buffers change their use: what has been issued has read them
                ok = wait(&sm.v_empty[(g - 1) & 1], ((g - 1) >> 1) & 1, sm, p.status);
                if (!ok) {
                    break;
                }
            }
            if (widened) {
#pragma unroll 2
                for (int j = 0; j < kWarpRows; ++j) {
                    const int r = j * kWidenWarps + me;
                    float x[8];
                    const float scale = scale_row(fetch_row(j), 14, x);
                    // (the dims in the order in which widened keys have them)
                    *reinterpret_cast<uint4*>(sm.q + (lane >> 3) * kQueryBlock + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) =
                        make_uint4(pack_f16(x[0], x[2]), pack_f16(x[1], x[3]), pack_f16(x[4], x[6]), pack_f16(x[5], x[7]));
                    if (lane == 0) {
                        sm.row_scale[r] = scale * 256.0f;
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    arrive_first(&sm.q_wide);
                }
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.scales_ready);
            }
            ok = !widened || widen_keys(g);
            for (int unit = piece.unit_begin; ok && unit < piece.unit_end; ++unit, ++g) {
                if (widened && unit + 1 < piece.unit_end) {
                    ok = widen_keys(g + 1);
                }
                ok = ok && widen_values(g);
                if (unit > piece.unit_begin) {
                    continue;
                }
                // Into L2: the gates that this item ends with, 512 bytes of a row ...
                if (p.gate != nullptr) {
                    const int r = me * kWarpRows + lane;
                    const int token = first_token + r / kGqaGroup;
                    if (r < live_rows) {
                        bulk_prefetch_l2(p.gate + (static_cast<size_t>(walk.info.begin) + token) * p.gate_stride +
                                             (walk.head * kGqaGroup + r % kGqaGroup) * (2 * kHeadDim) + kHeadDim,
                                         kHeadDim * 2);
                    }
                    __syncwarp();
                }
                {
                    // ... and the next item's queries, 6 heads of a token together
                    ChunkWalk ahead = walk;
                    ChunkPiece next;
                    if (me == 0 && next_piece(ahead, false, p.sequences, info, next)) {
                        const int token = ahead.tile * kItemTokens + rank * kRowTokens + lane;
                        if (lane < kRowTokens && token < ahead.info.length) {
                            bulk_prefetch_l2(p.query + ((static_cast<size_t>(ahead.info.begin) + token) * kQueryHeads +
                                                        ahead.head * kGqaGroup) * kHeadDim, kGqaGroup * kHeadDim * 2);
                        }
                        __syncwarp();
                    }
                }
            }
            ++item;
        }
        // the last commits have arrived in this CTA's shared memory before it ends
        if (ok && g > 0) {
            ok = (g < 2 || wait(&sm.v_empty[g & 1], ((g - 2) >> 1) & 1, sm, p.status)) &&
                 wait(&sm.v_empty[(g - 1) & 1], ((g - 1) >> 1) & 1, sm, p.status) &&
                 wait(&sm.q_free, (item - 1) & 1, sm, p.status);
            for (int i = g > kKeyStages ? g - kKeyStages : 0; i < g && ok; ++i) {
                ok = wait(&sm.raw_k_empty[i % kKeyStages], (i / kKeyStages) & 1, sm, p.status);
            }
            ok = ok && wait(&sm.k_empty, (g - 1) & 1, sm, p.status);
        }
    } else {
        // ---------------- softmax: two threads for a row ----------------------------------------------
        constexpr int kColumns = kUnit / 2;  // of a thread
        const int half = warp >> 2;
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const int row_token = r / kGqaGroup;
        if (threadIdx.x == 0 && rank == 0) {
            p.merge[pair].sequence = -1;  // nothing to merge, until an item turns out to be cut
        }
        for (bool first = true; ok && next_piece(walk, first, p.sequences, info, piece); first = false) {
            ok = wait(&sm.scales_ready, item & 1, sm, p.status);
            if (!ok) {
                break;
            }
            const int token = walk.tile * kItemTokens + rank * kRowTokens + row_token;  // of the chunk
            const bool live = r < kRowTokens * kGqaGroup && token < walk.info.length;
            // positions that the row sees, and that every live row of the CTA sees
            const int visible = live ? walk.info.context - walk.info.length + token + 1 : 0;
            const int visible_to_all = walk.info.context - walk.info.length + walk.tile * kItemTokens + rank * kRowTokens + 1;
            // scores in log2
            const float scale =
                fmaxf(p.softmax_scale * kLog2e * (p.key_scales ? p.key_scales[walk.head] : 1.0f) * sm.row_scale[r], 1e-37f);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.q_free);
            }
            float reference = -INFINITY;  // log2
            float sum = 0.0f;
            for (int unit = piece.unit_begin; unit < piece.unit_end; ++unit, ++g) {
                const int buffer = g & 1;
                ok = wait(&sm.s_full[buffer], (g >> 1) & 1, sm, p.status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t loaded[2][32];
                tmem_load32_issue(t_lane + buffer * kUnit + half * kColumns, loaded[0]);
                tmem_load32_issue(t_lane + buffer * kUnit + half * kColumns + 32, loaded[1]);
                tmem_load_wait();
                float s[kColumns];
#pragma unroll
                for (int i = 0; i < kColumns; ++i) {
                    asm volatile("" : "+r"(loaded[i / 32][i % 32]));  // (not to be taken before the wait)
                    s[i] = __uint_as_float(loaded[i / 32][i % 32]);
                }
                if ((unit + 1) * static_cast<long long>(kUnit) > visible_to_all) {
                    const long long limit = static_cast<long long>(visible) - static_cast<long long>(unit) * kUnit - half * kColumns;
                    const int seen = limit > kColumns ? kColumns : limit < 0 ? 0 : static_cast<int>(limit);
#pragma unroll
                    for (int i = 0; i < kColumns; ++i) {
                        s[i] = i < seen ? s[i] : -INFINITY;
                    }
                }
                float highest[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < kColumns; i += 8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        highest[j] = i + 4 + j < kColumns ? max3(highest[j], s[i + j], s[i + 4 + j]) : fmaxf(highest[j], s[i + j]);
                    }
                }
                const float mine = fmaxf(fmaxf(highest[0], highest[1]), fmaxf(highest[2], highest[3]));
                sm.row_max[buffer][half][r] = mine;
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.max_ready[buffer][quarter]);
                }
                ok = wait(&sm.max_ready[buffer][quarter], (g >> 1) & 1, sm, p.status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float top = fmaxf(mine, sm.row_max[buffer][half ^ 1][r]) * scale;
                // (a row without any score keeps its reference, and none at all counts as 0)
                const bool grown = top - reference > kRescaleAbove;
                if (__any_sync(0xffffffffu, grown)) {
                    const float lowered = top - kLargest;  // (beyond 2^27 a float may take more than that away)
                    const float moved = top - lowered > kRescaleAbove ? top : lowered;
                    const float factor = grown ? exp2_fast(reference - moved) : 1.0f;
                    if (unit > piece.unit_begin) {
                        // the first unit's O is not added to anything; after it, wait for the one before this
                        ok = wait(&sm.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1, sm, p.status);
                        if (!ok) {
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int c = half * 4; c < half * 4 + 4; ++c) {
                            uint32_t part[32];
                            tmem_load32_issue(t_lane + kOutputColumn + c * 32, part);
                            tmem_load_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                asm volatile("" : "+r"(part[i]));
                                part[i] = __float_as_uint(__uint_as_float(part[i]) * factor);
                            }
                            tmem_store32(t_lane + kOutputColumn + c * 32, part);
                        }
                        tmem_store_wait();
                    }
                    sum *= factor;
                    reference = grown ? moved : reference;
                }
                const float minus = reference == -INFINITY ? 0.0f : -reference;
                float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t packed[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float lo = exp2_fast(fmaf(s[2 * i], scale, minus));
                    const float hi = exp2_fast(fmaf(s[2 * i + 1], scale, minus));
                    sums[i & 3] += lo + hi;
                    packed[i] = pack_f16(lo, hi);
                }
                // (over scores of either half: both warps have read theirs when they met)
                tmem_store32(t_lane + buffer * kUnit + half * 32, packed);
                sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                tmem_store_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    arrive_first(&sm.p_full[buffer]);
                }
            }
            if (!ok) {
                break;
            }
            // ---- the piece's result
            const bool whole = piece.unit_begin == 0 && piece.unit_end == piece.units;
            const int slot = 2 * pair + (piece.unit_begin == 0 ? 1 : 0);
            const size_t partial_row = static_cast<size_t>(slot) * kSlotRows + rank * kRows + r;
            if (!whole && piece.unit_begin == 0 && threadIdx.x == 0 && rank == 0) {
                MergeItem merge;
                merge.sequence = walk.sequence;
                merge.head = walk.head;
                merge.tile = walk.tile;
                merge.last_pair = worker_of(sm.total, walk.item_end - 1, plan_workers(sm.total, pairs));
                merge.first_row = walk.info.begin + walk.tile * kItemTokens;
                merge.rows = min(kItemTokens, walk.info.length - walk.tile * kItemTokens);
                p.merge[pair] = merge;
            }
            sm.row_sum[half][r] = sum;
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.sum_ready[quarter]);
            }
            const size_t row = static_cast<size_t>(walk.info.begin) + token;
            const int head = walk.head * kGqaGroup + r % kGqaGroup;
            const int first_dim = half * (kHeadDim / 2);
            const bool gated = whole && p.gate != nullptr && live;
            const __nv_bfloat16* gate_row = p.gate + row * p.gate_stride + head * (2 * kHeadDim) + kHeadDim + first_dim;
            void* const target = whole ? static_cast<void*>(p.output + (row * kQueryHeads + head) * kHeadDim + first_dim)
                                       : static_cast<void*>(p.partial_out + partial_row * kHeadDim + first_dim);
            uint4 gates[4] = {};
            if (gated) {
                load64(gate_row, p.wide_rows, gates);
            }
            ok = wait(&sm.sum_ready[quarter], item & 1, sm, p.status);
            if (!ok) {
                break;
            }
            sum += sm.row_sum[half ^ 1][r];
            const float inverse = sum > 0.0f || isnan(sum) ? 256.0f / sum : 0.0f;  // (values are 2^-8 of themselves)
            const float v_scale = inverse * (p.value_scales ? p.value_scales[walk.head] : 1.0f);
            const float partial_scale = inverse * kPartialScale;
            // (a barrier for every second unit: P V of the unit before may still run, and on one barrier the parity of
            // this one would be that of the one before it)
            ok = wait(&sm.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1, sm, p.status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < kHeadDim / 64; ++c) {
                uint32_t part[32];
                const uint4 here[4] = {gates[0], gates[1], gates[2], gates[3]};
                if (gated && c + 1 < kHeadDim / 64) {
                    load64(gate_row + (c + 1) * 32, p.wide_rows, gates);
                }
                __syncwarp();
                tmem_load32_issue(t_lane + kOutputColumn + first_dim + c * 32, part);
                tmem_load_wait();
                float value[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    asm volatile("" : "+r"(part[i]));
                    // columns 4 i .. + 3 are dims 4 i + 0, 2, 1, 3
                    value[(i & ~3) | ((i & 1) << 1) | ((i >> 1) & 1)] = __uint_as_float(part[i]);
                }
                if (live && !whole) {
                    uint4 out[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        out[i] = make_uint4(pack_f16(value[8 * i] * partial_scale, value[8 * i + 1] * partial_scale),
                                           pack_f16(value[8 * i + 2] * partial_scale, value[8 * i + 3] * partial_scale),
                                           pack_f16(value[8 * i + 4] * partial_scale, value[8 * i + 5] * partial_scale),
                                           pack_f16(value[8 * i + 6] * partial_scale, value[8 * i + 7] * partial_scale));
                    }
                    store64(static_cast<__half*>(target) + c * 32, p.wide_rows, out);
                } else if (live) {
                    uint4 out[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t words[4];
                        const uint32_t gate_words[4] = {here[i].x, here[i].y, here[i].z, here[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float lo = value[8 * i + 2 * j] * v_scale, hi = value[8 * i + 2 * j + 1] * v_scale;
                            if (gated) {
                                lo *= sigmoid_fast(__uint_as_float(gate_words[j] << 16));
                                hi *= sigmoid_fast(__uint_as_float(gate_words[j] & 0xffff0000u));
                            }
                            const __nv_bfloat162 both = __floats2bfloat162_rn(lo, hi);
                            words[j] = *reinterpret_cast<const uint32_t*>(&both);
                        }
                        out[i] = make_uint4(words[0], words[1], words[2], words[3]);
                    }
                    store64(static_cast<__nv_bfloat16*>(target) + c * 32, p.wide_rows, out);
                }
                __syncwarp();
            }
            if (!whole && live && half == 0) {
                p.partial_stats[partial_row] = {reference, sum};
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                arrive_first(&sm.o_free);
            }
            ++item;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(&sm.failed) != 0) {
        // A wait gave up somewhere.  What was asked for and arrives by itself is waited for, 0.2 ms at most for each.
        const auto arrived = [](uint64_t* bar, uint32_t parity) {
            const long long start = clock64();
            while (!mbar_try_wait(bar, parity) && clock64() - start < 400000ll) {
            }
        };
        if (warp == kFetchWarp) {
            for (int i = g > kKeyStages ? g - kKeyStages : 0; i < g; ++i) {
                arrived(&sm.raw_k_full[i % kKeyStages], (i / kKeyStages) & 1);
            }
            for (int i = g > kValueStages ? g - kValueStages : 0; i < g; ++i) {
                arrived(&sm.raw_v_full[i % kValueStages], (i / kValueStages) & 1);
            }
        } else if (warp == kMmaWarp && rank == 0 && g > 0) {
            arrived(&sm.s_full[(g - 1) & 1], ((g - 1) >> 1) & 1);
            arrived(&sm.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
            if (g > 1) {
                arrived(&sm.o_done[g & 1], ((g - 2) >> 1) & 1);
            }
        }
    }
    __syncthreads();
    pair_sync();  // nobody leaves while the other may still arrive at its barriers, or while MMAs read its memory
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns) : "memory");
    }
}

// Items that were cut: a pair's last item began there and went on with the pairs after it.  A warp per row, eight dims
// per lane, the pieces in order.
constexpr int kMergeWarps = 8;
constexpr int kMergeDepth = 4;  // pieces in flight

__global__ void __launch_bounds__(kMergeWarps * 32) chunk_merge_kernel(const __grid_constant__ Params p) {
    pdl_launch_dependents();
    pdl_wait();
    const int pair = blockIdx.x;
    const MergeItem item = p.merge[pair];
    if (item.sequence < 0) {
        return;
    }
    const int lane = threadIdx.x & 31;
    const int index = blockIdx.y * kMergeWarps + (threadIdx.x >> 5);  // token and head of the group
    const int token = index / kGqaGroup;
    if (token >= item.rows) {
        return;
    }
    const int r = (token / kRowTokens) * kRows + (token % kRowTokens) * kGqaGroup + index % kGqaGroup;
    const auto slot = [&](int piece) {
        return (2 * static_cast<size_t>(pair + piece) + (piece == 0 ? 1 : 0)) * kSlotRows + r;
    };
    const int pieces = item.last_pair - pair + 1;
    const size_t row = static_cast<size_t>(item.first_row) + token;
    const int head = item.head * kGqaGroup + index % kGqaGroup;
    // everything that does not wait for something else is asked for at once: gates, the first pieces, the statistics
    uint4 gates = make_uint4(0, 0, 0, 0);
    if (p.gate != nullptr) {
        gates = __ldg(reinterpret_cast<const uint4*>(p.gate + row * p.gate_stride + head * (2 * kHeadDim) + kHeadDim) + lane);
    }
    uint4 raw[kMergeDepth];
    const auto fetch = [&](int first) {
#pragma unroll
        for (int j = 0; j < kMergeDepth; ++j) {
            raw[j] = make_uint4(0, 0, 0, 0);
            if (first + j < pieces) {
                raw[j] = reinterpret_cast<const uint4*>(p.partial_out + slot(first + j) * kHeadDim)[lane];
            }
        }
    };
    fetch(0);
    // a piece per lane: its weight (at most 96 pieces)
    float maximum = -INFINITY;
    PartialStats stats[(kMaxPairs + 31) / 32];
#pragma unroll
    for (int i = 0; i < (kMaxPairs + 31) / 32; ++i) {
        stats[i] = {-INFINITY, 0.0f};
        if (32 * i + lane < pieces) {
            stats[i] = p.partial_stats[slot(32 * i + lane)];
        }
        if (!(stats[i].sum <= 0.0f)) {
            maximum = fmaxf(maximum, stats[i].maximum);
        }
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        maximum = fmaxf(maximum, __shfl_xor_sync(0xffffffffu, maximum, offset));
    }
    float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    float denominator = 0.0f;
#pragma unroll
    for (int i = 0; i < (kMaxPairs + 31) / 32; ++i) {
        const float mine = !(stats[i].sum <= 0.0f) ? stats[i].sum * exp2f(stats[i].maximum - maximum) : 0.0f;
#pragma unroll 1
        for (int first = 32 * i; first < min(32 * i + 32, pieces); first += kMergeDepth) {
#pragma unroll
            for (int j = 0; j < kMergeDepth; ++j) {
                const float weight = __shfl_sync(0xffffffffu, mine, (first + j) & 31);
                if (first + j < pieces) {
                    denominator += weight;
                    const uint32_t words[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&words[d]));
                        acc[2 * d] = fmaf(weight, f.x, acc[2 * d]);
                        acc[2 * d + 1] = fmaf(weight, f.y, acc[2 * d + 1]);
                    }
                }
            }
            if (first + kMergeDepth < pieces) {
                fetch(first + kMergeDepth);
            }
        }
    }
    const float v_scale = (p.value_scales ? p.value_scales[item.head] : 1.0f) / kPartialScale;
    const float inverse = denominator > 0.0f || isnan(denominator) ? v_scale / denominator : 0.0f;
    const uint32_t gate_words[4] = {gates.x, gates.y, gates.z, gates.w};
    uint32_t words[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float lo = acc[2 * j] * inverse, hi = acc[2 * j + 1] * inverse;
        if (p.gate != nullptr) {
            lo *= sigmoid_fast(__uint_as_float(gate_words[j] << 16));
            hi *= sigmoid_fast(__uint_as_float(gate_words[j] & 0xffff0000u));
        }
        const __nv_bfloat162 both = __floats2bfloat162_rn(lo, hi);
        words[j] = *reinterpret_cast<const uint32_t*>(&both);
    }
    reinterpret_cast<uint4*>(p.output + (row * kQueryHeads + head) * kHeadDim)[lane] = make_uint4(words[0], words[1], words[2], words[3]);
}

}  // namespace
}  // namespace qwc

extern "C" size_t qwc_paged_attention_chunk_workspace_bytes(void) { return qwc::kWorkspaceBytes; }

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
        context_lengths == nullptr || chunk_begins == nullptr || output == nullptr || workspace == nullptr || tokens <= 0 ||
        tokens > kMaxChunkTokens || sequences <= 0 || sequences > kMaxChunkSequences || max_blocks <= 0 ||
        (page_size != 16 && page_size != 64) || static_cast<long long>(max_blocks) * page_size > 0x7fffffffll ||
        num_blocks <= 0 || static_cast<long long>(num_blocks) * kKvHeads * page_size > 0x7fffffffll ||
        gate_stride < kQueryHeads * 2 * kHeadDim || gate_stride % 8 != 0 || !isfinite(softmax_scale) ||
        softmax_scale <= 0.0f || !aligned(query) || !aligned(query_gate_projection) || !aligned(key_cache) ||
        !aligned(value_cache) || !aligned(output) || !aligned(workspace) || workspace_bytes < kWorkspaceBytes) {
        return cudaErrorInvalidValue;
    }
    int* status = status_ptr();
    if (status == nullptr) {
        return cudaErrorInvalidValue;
    }
    const int shared = static_cast<int>(sizeof(Smem)) + 1024;
    struct Setup {
        cudaError_t error;
        int pairs;
    };
    static PerDevice<Setup> per_device;
    const Setup* setup = per_device.get([shared]() {
        Setup found = {cudaSuccess, 0};
        int device = 0, sms = 0;
        found.error = cudaFuncSetAttribute(chunk_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (found.error == cudaSuccess) {
            found.error = cudaGetDevice(&device);
        }
        if (found.error == cudaSuccess) {
            found.error = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        }
        found.pairs = sms / 2 < 1 ? 1 : sms / 2 > kMaxPairs ? kMaxPairs : sms / 2;
        return found;
    });
    if (setup == nullptr) {
        return cudaErrorInvalidDevice;
    }
    if (setup->error != cudaSuccess) {
        return setup->error;
    }
    CUtensorMap key_map, value_map;
    const long long rows = static_cast<long long>(num_blocks) * kKvHeads * page_size;
    cudaError_t error = encode_pages(&key_map, key_cache, rows);
    if (error == cudaSuccess) {
        error = encode_pages(&value_map, value_cache, rows);
    }
    if (error != cudaSuccess) {
        return error;
    }
    Params p;
    p.query = static_cast<const __nv_bfloat16*>(query);
    p.gate = static_cast<const __nv_bfloat16*>(query_gate_projection);
    p.block_tables = static_cast<const uint32_t*>(block_tables);
    p.context_lengths = static_cast<const uint32_t*>(context_lengths);
    p.begins = static_cast<const uint32_t*>(chunk_begins);
    p.key_scales = key_scales;
    p.value_scales = value_scales;
    p.output = static_cast<__nv_bfloat16*>(output);
    p.partial_out = static_cast<__half*>(workspace);
    p.partial_stats = reinterpret_cast<PartialStats*>(static_cast<char*>(workspace) + kOutBytes);
    p.merge = reinterpret_cast<MergeItem*>(static_cast<char*>(workspace) + kOutBytes + kStatsBytes);
    p.tokens = tokens;
    p.sequences = sequences;
    p.max_blocks = max_blocks;
    p.page_size = page_size;
    p.num_blocks = num_blocks;
    p.gate_stride = gate_stride;
    p.softmax_scale = softmax_scale;
    p.wide_rows = ((reinterpret_cast<uintptr_t>(query_gate_projection) | reinterpret_cast<uintptr_t>(output) |
                    reinterpret_cast<uintptr_t>(workspace)) & 31) == 0 && gate_stride % 16 == 0;
    p.status = status;
    error = launch_chained(chunk_attention_kernel, dim3(2 * setup->pairs), dim3(kThreads), shared, stream, key_map, value_map, p);
    if (error != cudaSuccess) {
        return error;
    }
    const int item_rows = std::min(kItemTokens, tokens) * kGqaGroup;  // at most
    return launch_chained(chunk_merge_kernel, dim3(setup->pairs, (item_rows + kMergeWarps - 1) / kMergeWarps), dim3(kMergeWarps * 32),
                          0, stream, p);
}
