// The gated delta rule over the tokens of a ragged batch of chunks, on the slots' int8 state.
//
// Per token and value head, S [128 x 128] (rows: value dims, columns: key dims):
//   S <- alpha S;  u = beta (v - S k);  S <- S + u k^T;  o = S q
// (the recurrence of cuda/delta_net.cu:99-119 without the requantisation after every token: the state is read from its
// eight bits once per call, carried in fp32, and written back once, with the rounding of cuda/delta_net.cu:137-175).
//
// 64 tokens at a time (a block), with g_t the decay from the block's start, S0 the state there:
//   u_t = beta_t (v_t - g_t S0 k_t - sum_{j<t} (g_t / g_j) (k_t.k_j) u_j)
// is a triangular system, (1 + A) U = diag(beta) R with R_t = v_t - g_t S0 k_t and A_tj = beta_t (g_t / g_j) (k_t.k_j), and
//   o_t = g_t S0 q_t + sum_{j<=t} (g_t / g_j) (q_t.k_j) u_j,     S1 = g_end S0 + sum_j (g_end / g_j) u_j k_j^T.
// With T = (1 + A)^-1 diag(beta) and P the matrix of the second sum, W = [P T ; diag(g_end / g) T] (128 x 64) does not
// depend on the state: the first kernel makes it for all blocks and heads at once.  The second kernel walks through the
// blocks of a head, with everything the other way round, a value dim in a row:
//   X = S0 K^T,  Y = S0 Q^T;     [O | U'] = V^T W^T - (X diag(g)) W^T;     S1 = g_end S0 + U' K;     outputs O + Y diag(g).
//
// Bound by the chain S0 -> X -> U' -> S1, block after block.  All products run on the fifth-generation tensor cores, M = 128 value
// dims.  S (fp32, accumulated in place), X and U' never leave tensor memory: a thread has a row, turns 32 columns of an
// accumulator into the next product's A operand and puts it where the accumulator was.  The B operands, K, Q, V and W, come
// as they lie in memory.  What the chain does not wait for, V^T W^T, Y and the outputs, is issued where the tensor cores
// would wait for such a step.  K, Q and V are bf16 as they come; S, X, U' and W are the sum of two bf16, which hold 16 bits,
// and their products leave out only the lower part times the lower part.

#include <algorithm>
#include <cstddef>

#include "chunk.cuh"
#include "tcgen05.cuh"

namespace qwc {
namespace {

constexpr int kDim = kDeltaHeadDim;
constexpr int kBlock = 64;                               // tokens
constexpr int kTileBytes = 128 * 128;                    // 128 rows of 64 bf16, 128-byte swizzle
constexpr int kQkBytes = 2 * kTileBytes;                 // [half of the dims][q of the block's tokens, k][128 bytes]
constexpr int kWBytes = 2 * kTileBytes;                  // [upper, lower bf16][row][128 bytes]
constexpr int kVBytes = kTileBytes;                      // [half of the value dims][token][128 bytes]
constexpr int kProductBytes = kTileBytes;                // T of a block: [upper, lower][row][128 bytes]

// Workspace: images of the operands as shared memory has them.
struct Images {
    uint8_t* qk;    // [block][key head][kQkBytes]
    uint8_t* w;     // [block][value head][kWBytes]
    float* decay;   // [block][value head][kBlock]: from the block's start
    int4* order;    // the chunks, longest first: sequence, first row, length, first block
    int* taken;     // jobs that are not a CTA's first one
};

inline size_t images_bytes(int blocks, int v_heads) {
    return static_cast<size_t>(blocks) *
           (static_cast<size_t>(kDeltaKeyHeads) * kQkBytes + static_cast<size_t>(v_heads) * (kWBytes + kBlock * sizeof(float))) +
           kMaxChunkSequences * sizeof(int4) + sizeof(int);
}

inline Images images_at(void* workspace, int blocks, int v_heads) {
    Images at;
    at.qk = static_cast<uint8_t*>(workspace);
    at.w = at.qk + static_cast<size_t>(blocks) * kDeltaKeyHeads * kQkBytes;
    at.decay = reinterpret_cast<float*>(at.w + static_cast<size_t>(blocks) * v_heads * kWBytes);
    at.order = reinterpret_cast<int4*>(at.decay + static_cast<size_t>(blocks) * v_heads * kBlock);
    at.taken = reinterpret_cast<int*>(at.order + kMaxChunkSequences);
    return at;
}

// D[128][N] (+)= A[128][16] x B[N][16], bf16 from shared memory, fp32 accumulate.
__device__ __forceinline__ void mma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

constexpr uint32_t idesc_of(int columns) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(columns >> 3) << 17) | (8u << 24);
}
constexpr uint32_t kTransposeA = 1u << 15, kTransposeB = 1u << 16;

// Operand of 128-byte rows with the 128-byte swizzle, eight rows to an atom.  K-major: a row is one of M or N, its bytes 64
// of the contracted elements.  MN-major: a row is one of the contracted, its bytes 64 of M or N, the next 64 `block` bytes on.
// Made in two steps, the lower word of its beginning once and then the part of it that an MMA reads, one addition.
__device__ __forceinline__ uint32_t operand_base(uint32_t address, uint32_t block) {
    return ((address >> 4) & 0x3FFFu) | ((block >> 4) & 0x3FFFu) << 16;
}

__device__ __forceinline__ uint64_t operand_at(uint32_t base, uint32_t bytes) {
    constexpr uint32_t kUpper = (1024u >> 4) | (1u << 14) | (2u << 29);
    return static_cast<uint64_t>(kUpper) << 32 | (base + (bytes >> 4));
}

// Where 16 bytes of a row lie.
__device__ __forceinline__ int swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// Two numbers as two bf16 each.
__device__ __forceinline__ void split2(float x, float y, uint32_t& upper, uint32_t& lower) {
    const __nv_bfloat162 high = __floats2bfloat162_rn(x, y);
    upper = *reinterpret_cast<const uint32_t*>(&high);
    const __nv_bfloat162 low =
        __floats2bfloat162_rn(x - __uint_as_float(upper << 16), y - __uint_as_float(upper & 0xffff0000u));
    lower = *reinterpret_cast<const uint32_t*>(&low);
}

// 32 columns of a row of an operand in two parts, `parts` bytes apart.
__device__ __forceinline__ void store_split(uint8_t* at, int parts, int row, int first_piece, const float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint4 upper, lower;
        split2(x[8 * i], x[8 * i + 1], upper.x, lower.x);
        split2(x[8 * i + 2], x[8 * i + 3], upper.y, lower.y);
        split2(x[8 * i + 4], x[8 * i + 5], upper.z, lower.z);
        split2(x[8 * i + 6], x[8 * i + 7], upper.w, lower.w);
        *reinterpret_cast<uint4*>(at + swizzled(row, first_piece + i)) = upper;
        *reinterpret_cast<uint4*>(at + parts + swizzled(row, first_piece + i)) = lower;
    }
}

// Until the copies out of shared memory have been written.
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Bounded as in the other kernels: 20 ms, then the status word is set and the CTA's waits fail.
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, int* failed, int* status) {
    const long long start = clock64();
    for (;;) {
#pragma unroll 1
        for (int spin = 0; spin < 64; ++spin) {
            if (mbar_try_wait(bar, parity)) {
                return true;
            }
        }
        if (*reinterpret_cast<volatile int*>(failed) != 0) {
            return false;
        }
        if (clock64() - start > 40000000ll) {
            break;
        }
    }
    record_wait(status, kStatusChunkDeltaWait);
    *reinterpret_cast<volatile int*>(failed) = 1;
    return false;
}

// For a converged warp: the same answer in every lane.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* failed, int* status) {
    const bool ok = mbar_try_wait(bar, parity) || wait_slow(bar, parity, failed, status);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void load_columns(uint32_t taddr, float (&x)[32]) {
    uint32_t raw[32];
    tmem_load32_issue(taddr, raw);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        asm volatile("" : "+r"(raw[i]));  // (not to be taken before the wait)
        x[i] = __uint_as_float(raw[i]);
    }
}

// ---- W of every block and head ------------------------------------------------------------------------
//
// [Q ; K] K^T on the tensor cores gives P and A (a thread has a row), fp32 arithmetic the inverse: columns of the four 16 x 16
// blocks on the diagonal by substitution, then T_10 = -T_11 A_10 T_00 for blocks of 16 and of 32.  P T is a product on the tensor
// cores again.  Bound by the latencies of these steps: what counts is how many CTAs an SM holds.

constexpr int kFactorThreads = 128;
constexpr int kPitch = 68;  // floats of a row of the matrices in shared memory: rows begin in different banks

constexpr int kMaxRatio = 3;  // value heads of a key head
// Below this many blocks of a call a CTA takes one value head, from there on all of a key head, which share [Q ; K] K^T:
// 48 heads, 64 tokens 30.2 us with one head and 39.3 with three, 512 tokens 54 and 58, 1280 tokens 99 and 102, 1600
// tokens 119 and 116, 4 chunks of 8192 in all 338 and 319; 32 heads, 704 tokens 56.7 and 59.6, 1600 tokens 104.7 and 103.8.
constexpr int kFewBlocks = 24;

struct FactorSmem {
    union {
        uint8_t qk[kQkBytes];
        struct {
            uint8_t p[kProductBytes];             // [upper, lower][row][128 bytes]
            union {
                float t[kBlock * kPitch];         // A below the diagonal; it becomes (1 + A)^-1 where it is
                uint8_t product[kProductBytes];   // T diag(beta) in two parts
            };
        } m;
    };
    float2 log[kMaxRatio][kBlock];                // log2 of the decay from the start: a whole number and the rest
    float beta[kMaxRatio][kBlock];
    int length[kMaxChunkSequences];
    uint64_t done;
    uint32_t tmem_base;
    int stop;  // nothing is done: a wait of an earlier kernel has given up
    int failed;
};
static_assert(offsetof(FactorSmem, m.product) % 1024 == 0, "an operand's alignment");

// x += a * rows[0 .. 3][4 columns] for four steps of the sum, for kRows rows of a.
template <int kRows>
__device__ __forceinline__ void multiply4(float2 (&x)[kRows][2], const float4 (&a)[kRows], const float* rows) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float4 row = *reinterpret_cast<const float4*>(rows + k * kPitch);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float factor = k == 0 ? a[r].x : k == 1 ? a[r].y : k == 2 ? a[r].z : a[r].w;
            x[r][0] = __ffma2_rn({factor, factor}, {row.x, row.y}, x[r][0]);
            x[r][1] = __ffma2_rn({factor, factor}, {row.z, row.w}, x[r][1]);
        }
    }
}

// The chunks in the order of their length, for the second kernel: what takes longest begins first (20 chunks of 4000 tokens
// in all 164.5 us, 170 in the order of the batch, a CTA for each).  Of two alike the first is the longer.  By a CTA, a thread for a chunk.
__device__ __forceinline__ void find_order(int (&length)[kMaxChunkSequences], const uint32_t* begins, int tokens, int sequences,
                                           int4* order) {
    static_assert(kFactorThreads >= kMaxChunkSequences, "a thread for a chunk");
    const int mine = threadIdx.x;
    ChunkSpan span = {0, 0};
    if (mine < sequences) {
        span = chunk_span(begins, mine, tokens);
        length[mine] = span.length;
    }
    __syncthreads();
    if (mine < sequences) {
        int rank = 0, blocks_before = 0;
        for (int i = 0; i < sequences; ++i) {
            rank += length[i] > span.length || (length[i] == span.length && i < mine) ? 1 : 0;
            blocks_before += i < mine ? (length[i] + kBlock - 1) / kBlock : 0;
        }
        order[rank] = make_int4(mine, span.begin, span.length, blocks_before);
    }
}

// A CTA has a block with `per_cta` value heads of one key head: all of them, or one where CTAs are few (see the launch).
__global__ void __launch_bounds__(kFactorThreads, 4) delta_factor_kernel(
    const __nv_bfloat16* __restrict__ qkv, const float* __restrict__ alpha, const float* __restrict__ beta,
    const uint32_t* __restrict__ begins, const Images images, int tokens, int sequences, int v_heads, int per_cta,
    int* status) {
    extern __shared__ unsigned char smem_raw[];
    FactorSmem& sm = *reinterpret_cast<FactorSmem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    constexpr int kTmemFactor = 2 * kBlock;  // [Q ; K] K^T, P T
    const int tid = threadIdx.x;
    const int lane = tid & 31;
    const int warp = tid >> 5;
    const int ratio = v_heads / kDeltaKeyHeads;
    const int first_head = blockIdx.x * per_cta;
    const int key_head = first_head / ratio;
    const int block = blockIdx.y;
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDim;
    if (tid == 0) {
        mbar_init(&sm.done, 1);
        sm.failed = 0;
        mbar_fence_init();
    }
    pdl_wait();
    // Tensor memory is asked for when the kernels before this one have given theirs back, and the next kernel may start
    // when this CTA has its own: CTAs of two kernels that each held some and asked for the rest would wait for each other.
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                     "r"(kTmemFactor)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (blockIdx.x == 0 && block == 0) {
        find_order(sm.length, begins, tokens, sequences, images.order);
        if (tid == 0) {
            *images.taken = 0;
        }
    }
    const int code = status_code(status);
    const ChunkTile tile = find_chunk_tile(begins, sequences, tokens, kBlock, block);
    bool here = tile.sequence >= 0;
    const int first = tile.index * kBlock;
    const int count = here ? min(kBlock, tile.span.length - first) : 0;
    const size_t row0 = static_cast<size_t>(tile.span.begin) + first;
    if (here) {
        // q and k of the block, zeros behind it: 16 threads fetch the 256 bytes of a row
#pragma unroll
        for (int i = 0; i < 2 * kBlock * 16 / kFactorThreads; ++i) {
            const int row = (tid >> 4) + i * (kFactorThreads / 16), piece = tid & 15;
            const int token = row & (kBlock - 1);
            const __nv_bfloat16* from =
                qkv + (row0 + (token < count ? token : 0)) * channels + ((row < kBlock ? 0 : kDeltaKeyHeads) + key_head) * kDim + 8 * piece;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             smem_u32(sm.qk + (piece >> 3) * kTileBytes + swizzled(row, piece & 7))),
                         "l"(from), "r"(token < count ? 16 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (warp < per_cta) {
            // decay from the start, a warp for a head: a scan over the tokens, in whole numbers and rests below one
            const int head = first_head + warp;
            float whole[2], part[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = lane + 32 * i;
                // (beyond 2^-130 fp32 has nothing, and an alpha of 0 takes everything before it away; a NaN stays one)
                float log = token < count ? log2f(alpha[(row0 + token) * v_heads + head]) : 0.0f;
                log = log < -130.0f ? -130.0f : log;
                sm.beta[warp][token] = token < count ? beta[(row0 + token) * v_heads + head] : 0.0f;
                whole[i] = rintf(log);
                part[i] = log - whole[i];
            }
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float w = __shfl_up_sync(0xffffffffu, whole[i], offset);
                    const float p = __shfl_up_sync(0xffffffffu, part[i], offset);
                    whole[i] += lane >= offset ? w : 0.0f;
                    part[i] += lane >= offset ? p : 0.0f;
                }
            }
            whole[1] += __shfl_sync(0xffffffffu, whole[0], 31);
            part[1] += __shfl_sync(0xffffffffu, part[0], 31);
            float* decay = images.decay + (static_cast<size_t>(block) * v_heads + head) * kBlock;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sm.log[warp][lane + 32 * i] = make_float2(whole[i], part[i]);
                decay[lane + 32 * i] = exp2f(whole[i] + part[i]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    if (tid == 0) {
        sm.stop = stops_chunks(code) ? 1 : 0;
    }
    fence_proxy_async();
    __syncthreads();
    pdl_launch_dependents();
    here = here && *reinterpret_cast<volatile int*>(&sm.stop) == 0;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sm.tmem_base);
    const uint32_t tmem_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
    bool ok = here;
    if (here) {
        if (warp == 0) {
            if (elect_one()) {
                const uint32_t base = operand_base(smem_u32(sm.qk), 16);
#pragma unroll
                for (int ks = 0; ks < kDim / 16; ++ks) {
                    const uint32_t at = (ks >> 2) * kTileBytes + (ks & 3) * 32;
                    mma_bf16(tmem_base, operand_at(base, at), operand_at(base, at + kBlock * 128), idesc_of(kBlock), ks > 0 ? 1u : 0u);
                }
                umma_commit(&sm.done);
            }
            __syncwarp();
        }
        if (tid == 0 && first_head == key_head * ratio) {
            // the image of q and k, once for the key head
            bulk_s2g(images.qk + (static_cast<size_t>(block) * kDeltaKeyHeads + key_head) * kQkBytes, sm.qk, kQkBytes);
            bulk_commit();
        }
        ok = wait(&sm.done, 0, &sm.failed, status);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int t = tid & (kBlock - 1);
    const bool outputs = tid < kBlock;
#pragma unroll 1
    for (int h = 0; h < per_cta; ++h) {
        if (tid == 0) {
            bulk_wait_all_read();  // (what has been copied from shared memory)
        }
        __syncthreads();
        if (ok) {
            // thread t has row t of Q K^T, thread 64 + t of K K^T: P to its operand, A to shared memory
            const float2 mine = sm.log[h][t];
            const float strength = outputs ? 1.0f : sm.beta[h][t];
            const int limit = outputs ? t + 1 : t;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                float x[32];
                if (32 * c <= (t | 31)) {  // (the same for a warp)
                    load_columns(tmem_row + 32 * c, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const int j = 32 * c + i;
                        const float4 others = *reinterpret_cast<const float4*>(&sm.log[h][j]);
                        const float2 one = __fadd2_rn(mine, make_float2(-others.x, -others.y));
                        const float2 two = __fadd2_rn(mine, make_float2(-others.z, -others.w));
                        const float2 decay = make_float2(exp2_fast(one.x + one.y), exp2_fast(two.x + two.y));
                        const float2 both = __fmul2_rn(__fmul2_rn(decay, make_float2(strength, strength)), make_float2(x[i], x[i + 1]));
                        x[i] = j < limit ? both.x : 0.0f;
                        x[i + 1] = j + 1 < limit ? both.y : 0.0f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        x[i] = 0.0f;
                    }
                }
                if (outputs) {
                    store_split(sm.m.p, kProductBytes / 2, t, 4 * c, x);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        *reinterpret_cast<float4*>(&sm.m.t[t * kPitch + 32 * c + 4 * i]) =
                            make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        __syncthreads();
        if (ok && outputs) {
            // blocks of 16 on the diagonal: a column per thread
            const int b = tid >> 4, j = tid & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < i; k += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(&sm.m.t[(16 * b + i) * kPitch + 16 * b + k]);
                    sum = fmaf(a.x, x[k], sum);
                    sum = k + 1 < i ? fmaf(a.y, x[k + 1 < i ? k + 1 : 0], sum) : sum;
                    sum = k + 2 < i ? fmaf(a.z, x[k + 2 < i ? k + 2 : 0], sum) : sum;
                    sum = k + 3 < i ? fmaf(a.w, x[k + 3 < i ? k + 3 : 0], sum) : sum;
                }
                x[i] = i == j ? 1.0f : i < j ? 0.0f : -sum;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sm.m.t[(16 * b + i) * kPitch + 16 * b + j] = x[i];
            }
        }
        __syncthreads();
        // blocks of 32: T_10 = -T_11 (A_10 T_00) of 16, eight columns per warp, four columns of a row per lane
        {
            const int base = 32 * (warp >> 1), column = base + 8 * (warp & 1) + 4 * (lane >> 4);
            const int r = base + 16 + (lane & 15);
            float* at = &sm.m.t[r * kPitch + column];
            float2 x[1][2] = {};
            if (ok) {
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float4 left[1] = {*reinterpret_cast<const float4*>(&sm.m.t[r * kPitch + base + k])};
                    multiply4(x, left, &sm.m.t[(base + k) * kPitch + column]);
                }
            }
            __syncthreads();  // (A_10 has been read)
            if (ok) {
                *reinterpret_cast<float4*>(at) = make_float4(x[0][0].x, x[0][0].y, x[0][1].x, x[0][1].y);
                __syncwarp();
                float2 y[1][2] = {};
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float4 left[1] = {*reinterpret_cast<const float4*>(&sm.m.t[r * kPitch + base + 16 + k])};
                    multiply4(y, left, &sm.m.t[(base + 16 + k) * kPitch + column]);
                }
                __syncwarp();
                *reinterpret_cast<float4*>(at) = make_float4(-y[0][0].x, -y[0][0].y, -y[0][1].x, -y[0][1].y);
            }
        }
        __syncthreads();
        // the block of 32 below: eight columns per warp, four columns of two rows per lane (T_00 is zero above its
        // diagonal); in blocks of 32 tokens or fewer it is zero, as A is there
        if (count > 32) {
            const int column = 8 * warp + 4 * (lane >> 4);
            const int r = 32 + (lane & 15);
            float* at = &sm.m.t[r * kPitch + column];
            float2 x[2][2] = {};
            if (ok) {
                for (int k = 8 * warp; k < 32; k += 4) {
                    const float4 left[2] = {*reinterpret_cast<const float4*>(&sm.m.t[r * kPitch + k]),
                                            *reinterpret_cast<const float4*>(&sm.m.t[(r + 16) * kPitch + k])};
                    multiply4(x, left, &sm.m.t[k * kPitch + column]);
                }
            }
            __syncthreads();  // (A_10 has been read)
            if (ok) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    *reinterpret_cast<float4*>(at + 16 * i * kPitch) = make_float4(x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y);
                }
                __syncwarp();
                float2 y[2][2] = {};
#pragma unroll 2
                for (int k = 0; k < 32; k += 4) {
                    const float4 left[2] = {*reinterpret_cast<const float4*>(&sm.m.t[r * kPitch + 32 + k]),
                                            *reinterpret_cast<const float4*>(&sm.m.t[(r + 16) * kPitch + 32 + k])};
                    multiply4(y, left, &sm.m.t[(32 + k) * kPitch + column]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    *reinterpret_cast<float4*>(at + 16 * i * kPitch) = make_float4(-y[i][0].x, -y[i][0].y, -y[i][1].x, -y[i][1].y);
                }
            }
            __syncthreads();
        }
        // T diag(beta) as an operand: half a row per thread
        const int row = tid >> 1, half = tid & 1;
        float x[32];
        if (ok) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 value = *reinterpret_cast<const float4*>(&sm.m.t[row * kPitch + 32 * half + 4 * i]);
                const float4 strength = *reinterpret_cast<const float4*>(&sm.beta[h][32 * half + 4 * i]);
                const float2 lo = __fmul2_rn(make_float2(value.x, value.y), make_float2(strength.x, strength.y));
                const float2 hi = __fmul2_rn(make_float2(value.z, value.w), make_float2(strength.z, strength.w));
                x[4 * i] = lo.x;
                x[4 * i + 1] = lo.y;
                x[4 * i + 2] = hi.x;
                x[4 * i + 3] = hi.y;
            }
        }
        __syncthreads();  // (T has been read)
        if (ok) {
            store_split(sm.m.product, kProductBytes / 2, row, 4 * half, x);
            fence_proxy_async();
        }
        __syncthreads();
        if (ok) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (warp == 0) {
                if (elect_one()) {
                    // (rows 64 .. of this operand are whatever lies behind P: their results are not read)
                    const uint32_t a = operand_base(smem_u32(sm.m.p), 16), b = operand_base(smem_u32(sm.m.product), 16);
#pragma unroll
                    for (int ks = 0; ks < kBlock / 16; ++ks) {
                        const uint64_t upper = operand_at(a, ks * 32), lower = operand_at(a, kProductBytes / 2 + ks * 32);
                        const uint64_t t_upper = operand_at(b, ks * 2048), t_lower = operand_at(b, kProductBytes / 2 + ks * 2048);
                        mma_bf16(tmem_base + kBlock, upper, t_upper, idesc_of(kBlock) | kTransposeB, ks > 0 ? 1u : 0u);
                        mma_bf16(tmem_base + kBlock, upper, t_lower, idesc_of(kBlock) | kTransposeB, 1u);
                        mma_bf16(tmem_base + kBlock, lower, t_upper, idesc_of(kBlock) | kTransposeB, 1u);
                    }
                    umma_commit(&sm.done);
                }
                __syncwarp();
            }
            const float2 mine = sm.log[h][row], end = sm.log[h][kBlock - 1];
            const float to_end = exp2_fast((end.x - mine.x) + (end.y - mine.y));
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float2 both = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(to_end, to_end));
                x[i] = both.x;
                x[i + 1] = both.y;
            }
            ok = wait(&sm.done, (h + 1) & 1, &sm.failed, status);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (ok) {
            // W's halves where the operands were, and from there to memory in one piece each
            store_split(sm.m.product, kProductBytes / 2, row, 4 * half, x);
            if (outputs) {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    load_columns(tmem_row + kBlock + 32 * c, x);
                    store_split(sm.m.p, kProductBytes / 2, t, 4 * c, x);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
            fence_proxy_async();
        }
        __syncthreads();
        if (ok && tid == 0) {
            uint8_t* w = images.w + (static_cast<size_t>(block) * v_heads + first_head + h) * kWBytes;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                bulk_s2g(w + part * kTileBytes, sm.m.p + part * (kProductBytes / 2), kProductBytes / 2);
                bulk_s2g(w + part * kTileBytes + kTileBytes / 2, sm.m.product + part * (kProductBytes / 2), kProductBytes / 2);
            }
            bulk_commit();
        }
    }
    if (tid == 0) {
        bulk_wait_all();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemFactor) : "memory");
    }
}

// ---- the chain of blocks --------------------------------------------------------------------------------
//
//   warps 0-7    the chain: four quarters of the 128 rows, two groups of columns
//   warps 8-15   outputs: the same division, then rows of the batch, norm and gate
//   warp 16      issues the MMAs
//   warp 17      fetches K, Q, W and V of the next block, warp 18 the gates of the next outputs

constexpr int kChainWarps = 8;
constexpr int kOutputWarps = 8;
constexpr int kMmaWarp = kChainWarps + kOutputWarps;
constexpr int kLoadWarp = kMmaWarp + 1;
constexpr int kGateWarp = kLoadWarp + 1;
constexpr int kChainThreads = (kGateWarp + 1) * 32;
// tensor memory
constexpr int kStateColumn = 0;                          // fp32, 128 key dims
constexpr int kSplitColumn = 128;                        // upper (64 columns), lower
constexpr int kKeyColumn = 256;                          // X of 64 tokens; then -g X, 32 tokens upper and lower side by side
constexpr int kQueryColumn = 320;                        // Y
constexpr int kResultColumn = 384;                       // O, U'; then U' split as X
constexpr int kUpdateColumn = kResultColumn + kBlock;
constexpr int kTmemColumns = 512;                        // all of it: the address that the allocation returns is 0

struct ChunkOfJobs {
    int sequence, begin, length, first_block, slot;
};

struct ChainSmem {
    uint8_t qk[2][kQkBytes];
    uint8_t w[2][kWBytes];
    uint8_t v[kVBytes];
    float rows[kBlock * kDim];          // outputs of a block
    uint8_t gate[2][kBlock * kDim * 2]; // [token][256 bytes]
    float decay[2][kBlock];
    float peak[2][2][kDim];             // of every second job, by group
    ChunkOfJobs chunk[kMaxChunkSequences];  // longest first
    uint64_t qk_full[2], qk_empty[2], w_full[2], w_empty[2], v_full, v_empty;
    uint64_t s_ready, x_done, x_ready, u_done, u_ready, o_done, o_free, s_done;
    uint64_t rows_ready, rows_free, gate_full[2], gate_empty[2];
    uint64_t chain_met;                 // of the chain's warps
    uint64_t job_full[2], job_empty[2];
    int job[2];
    uint32_t tmem_base;
    int stop;  // as above; the first kernel of this call may have given up, too
    int failed;
};
static_assert(sizeof(ChainSmem) + 1024 <= 232448, "shared memory of a CTA");

// What follows the rule, where it is wanted: RMSNorm over a head's value dims, times weight, times silu(gate).
struct OutputNorm {
    const __nv_bfloat16* gate;    // null: not wanted
    const __nv_bfloat16* weight;
    int gate_stride;
    float epsilon;
};

__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_store_columns(uint32_t taddr, const float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t raw[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            raw[j] = __float_as_uint(x[16 * i + j]);
        }
        tmem_store16(taddr + 16 * i, raw);
    }
}

// 32 columns as an A operand in two parts of 16 columns.
__device__ __forceinline__ void tmem_store_split(uint32_t upper_at, uint32_t lower_at, const float (&x)[32]) {
    uint32_t upper[16], lower[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        split2(x[2 * i], x[2 * i + 1], upper[i], lower[i]);
    }
    tmem_store16(upper_at, upper);
    tmem_store16(lower_at, lower);
}

__global__ void __launch_bounds__(kChainThreads, 1) delta_chain_kernel(
    int8_t* __restrict__ state, float* __restrict__ state_scales, const uint32_t* __restrict__ state_slots,
    const uint32_t* __restrict__ continues, const __nv_bfloat16* __restrict__ qkv, const Images images, int images_blocks,
    __nv_bfloat16* __restrict__ out, int sequences, int v_heads, int state_capacity, const OutputNorm norm, int* status) {
    extern __shared__ unsigned char smem_raw[];
    ChainSmem& sm = *reinterpret_cast<ChainSmem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDim;
    pdl_wait();
    if (warp == kLoadWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    bool any = false;  // rows of the chunk that this thread looks at
    if (threadIdx.x < sequences) {
        const int4 chunk = __ldcg(images.order + threadIdx.x);
        any = chunk.z > 0;
        const uint32_t slot = __ldcg(state_slots + chunk.x);
        const bool there = slot < static_cast<uint32_t>(state_capacity);
        if (!there && chunk.z > 0) {
            // a slot beyond the pool: nothing of this chunk is read or written, the host learns of it through the status
            // word
            atomicCAS(status, 0, kStatusStateSlotRange);
        }
        sm.chunk[threadIdx.x] = {chunk.x, chunk.y, there ? chunk.z : 0, chunk.w, static_cast<int>(slot)};
    }
    if (threadIdx.x == kGateWarp * 32) {
        sm.stop = stops_chunks(status_code(status)) ? 1 : 0;
    }
    if (threadIdx.x == kMmaWarp * 32) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.qk_full[i], 1);
            mbar_init(&sm.qk_empty[i], 1);
            mbar_init(&sm.w_full[i], 1);
            mbar_init(&sm.w_empty[i], 1 + kOutputWarps);  // the MMAs, and who reads the decays
            mbar_init(&sm.gate_full[i], 1);
            mbar_init(&sm.job_full[i], 1);
            mbar_init(&sm.job_empty[i], kChainWarps + kOutputWarps + 2);
            mbar_init(&sm.gate_empty[i], kOutputWarps);
        }
        mbar_init(&sm.s_ready, kChainWarps);
        mbar_init(&sm.x_done, 1);
        mbar_init(&sm.x_ready, kChainWarps);
        mbar_init(&sm.u_done, 1);
        mbar_init(&sm.u_ready, kChainWarps);
        mbar_init(&sm.o_done, 1);
        mbar_init(&sm.o_free, kOutputWarps);
        mbar_init(&sm.s_done, 1);
        mbar_init(&sm.rows_ready, kOutputWarps);
        mbar_init(&sm.rows_free, kOutputWarps);
        mbar_init(&sm.v_full, 1);
        mbar_init(&sm.v_empty, 1);
        mbar_init(&sm.chain_met, kChainWarps);
        sm.failed = 0;
        mbar_fence_init();
    }
    fence_proxy_async();
    const int chunks = __syncthreads_count(any ? 1 : 0);  // the first ones
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    pdl_launch_dependents();  // (this CTA has its tensor memory)
    int* const failed = &sm.failed;
    bool ok = true;
    int n = 0;  // blocks so far
    // A job is a chunk with a value head, the longest first.  A CTA's first one is its own, then whoever is done takes the next;
    // the warp that loads takes it, and says which to the others.  -1: there is none.  (40 chunks of 1000 tokens in all: 192 us
    // with a CTA for each job, 173 so; 128 chunks of 4000: 592 and 529; one chunk of 4096: 225 and 226.)
    const int jobs = *reinterpret_cast<volatile int*>(&sm.stop) != 0 ? 0 : chunks * v_heads;
    int round = 0;
    const auto next_job = [&]() {
        const int slot = round & 1;
        int job = -1;
        if (wait(&sm.job_full[slot], (round >> 1) & 1, failed, status)) {
            job = sm.job[slot];
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.job_empty[slot]);
            }
        } else {
            ok = false;
        }
        ++round;
        return job;
    };

    if (warp == kLoadWarp) {
        // ---------------- operands of the blocks -------------------------------------------------------
        for (int job = blockIdx.x; ok; ++round) {
            const auto take = [&]() {
                const int taken = lane == 0 ? static_cast<int>(gridDim.x) + atomicAdd(images.taken, 1) : 0;
                return __shfl_sync(0xffffffffu, taken, 0);
            };
            while (job < jobs && sm.chunk[job / v_heads].length == 0) {
                job = take();  // (a chunk whose slot is beyond the pool)
            }
            const bool there = job < jobs;
            ok = wait(&sm.job_empty[round & 1], ((round >> 1) & 1) ^ 1, failed, status);
            if (ok && lane == 0) {
                sm.job[round & 1] = there ? job : -1;
                mbar_arrive(&sm.job_full[round & 1]);
            }
            __syncwarp();
            if (!ok || !there) {
                break;
            }
            const ChunkOfJobs& chunk = sm.chunk[job / v_heads];
            const int head = job % v_heads;
            if (lane == 0) {
                // (the chain asks for the state when it is done with the job before)
                bulk_prefetch_l2(state + (static_cast<size_t>(chunk.slot) * v_heads + head) * (kDim * kDim), kDim * kDim);
            }
            __syncwarp();
            const int length = chunk.length, first_block = chunk.first_block;
            const int key_head = head / (v_heads / kDeltaKeyHeads);
            const __nv_bfloat16* v_rows = qkv + static_cast<size_t>(chunk.begin) * channels + (2 * kDeltaKeyHeads + head) * kDim;
            const int blocks = (length + kBlock - 1) / kBlock;
            for (int at = 0; at < blocks && ok; ++at, ++n) {
                const int slot_of = n & 1;
                const uint32_t parity = ((n >> 1) & 1) ^ 1;
                // (chunks that overlap have more blocks than there is room for: what they get is nobody's, but it is there)
                const size_t block = static_cast<size_t>(min(first_block + at, images_blocks - 1));
                ok = wait(&sm.w_empty[slot_of], parity, failed, status);
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(&sm.w_full[slot_of], kWBytes + kBlock * 4);
                    bulk_g2s(sm.w[slot_of], images.w + (block * v_heads + head) * kWBytes, kWBytes, &sm.w_full[slot_of]);
                    bulk_g2s(sm.decay[slot_of], images.decay + (block * v_heads + head) * kBlock, kBlock * 4, &sm.w_full[slot_of]);
                }
                __syncwarp();
                ok = ok && wait(&sm.v_empty, (n & 1) ^ 1, failed, status);
                if (ok) {
                    // rows of v, zeros behind the chunk: sixteen lanes to a row
                    const int piece = lane & 15;
                    const int left = length - at * kBlock - (lane >> 4);
                    const __nv_bfloat16* from = v_rows + static_cast<size_t>(at * kBlock + (lane >> 4)) * channels + 8 * piece;
                    const uint32_t to = smem_u32(sm.v + (piece >> 3) * (kVBytes / 2));
#pragma unroll 8
                    for (int i = 0; i < kBlock / 2; ++i) {
                        const bool live = 2 * i < left;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         to + swizzled(2 * i + (lane >> 4), piece & 7)),
                                     "l"(live ? from + 2 * i * channels : v_rows), "r"(live ? 16 : 0)
                                     : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                ok = ok && wait(&sm.qk_empty[slot_of], parity, failed, status);
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(&sm.qk_full[slot_of], kQkBytes);
                    bulk_g2s(sm.qk[slot_of], images.qk + (block * kDeltaKeyHeads + key_head) * kQkBytes, kQkBytes, &sm.qk_full[slot_of]);
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                fence_proxy_async();
                __syncwarp();
                if (ok && lane == 0) {
                    mbar_arrive(&sm.v_full);
                }
                __syncwarp();
            }
            job = take();  // (not before: who has a long job would have the next one too)
        }
    } else if (warp == kGateWarp) {
        // ---------------- gates of the blocks' rows ---------------------------------------------------------
        const int piece = lane & 15;
        for (int job = next_job(); job >= 0; job = ok ? next_job() : -1) {
            if (norm.gate == nullptr) {
                continue;
            }
            const ChunkOfJobs& chunk = sm.chunk[job / v_heads];
            const int head = job % v_heads, length = chunk.length;
            const __nv_bfloat16* rows = norm.gate + static_cast<size_t>(chunk.begin) * norm.gate_stride + head * kDim + 8 * piece;
            const int blocks = (length + kBlock - 1) / kBlock;
            for (int at = 0; at < blocks && ok; ++at, ++n) {
                ok = wait(&sm.gate_empty[n & 1], ((n >> 1) & 1) ^ 1, failed, status);
                if (ok) {
                    const int left = length - at * kBlock - (lane >> 4);
                    const __nv_bfloat16* from = rows + static_cast<size_t>(at * kBlock + (lane >> 4)) * norm.gate_stride;
                    const uint32_t to = smem_u32(sm.gate[n & 1] + (lane >> 4) * (kDim * 2) + 16 * piece);
#pragma unroll 4
                    for (int i = 0; i < kBlock / 2; ++i) {
                        const bool live = 2 * i < left;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * (kDim * 4)), "l"(live ? from : rows),
                                     "r"(live ? 16 : 0)
                                     : "memory");
                        from += 2 * static_cast<size_t>(norm.gate_stride);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                __syncwarp();
                if (ok && lane == 0) {
                    mbar_arrive(&sm.gate_full[n & 1]);
                }
                __syncwarp();
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- tensor-core issue ------------------------------------------------------------
        constexpr uint32_t kWide = idesc_of(kDim), kNarrow = idesc_of(kBlock);
        const uint32_t qk_operand = operand_base(smem_u32(sm.qk[0]), 16), w_operand = operand_base(smem_u32(sm.w[0]), 16);
        const uint32_t k_across = operand_base(smem_u32(sm.qk[0]) + kBlock * 128, kTileBytes);  // k, dims across
        const uint32_t v_operand = operand_base(smem_u32(sm.v), kVBytes / 2);
        // [O | U'] begins as V^T W^T
        const auto issue_values = [&](int number) {
            const int slot_of = number & 1;
            if (!wait(&sm.w_full[slot_of], (number >> 1) & 1, failed, status) ||
                !wait(&sm.v_full, number & 1, failed, status) ||
                !wait(&sm.o_free, (number & 1) ^ 1, failed, status)) {
                return false;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                const uint32_t w_base = w_operand + slot_of * (kWBytes >> 4);
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    const uint64_t a = operand_at(v_operand, ks * 2048);
                    mma_bf16(kResultColumn, a, operand_at(w_base, ks * 32), kWide | kTransposeA, ks > 0 ? 1u : 0u);
                    mma_bf16(kResultColumn, a, operand_at(w_base, kTileBytes + ks * 32), kWide | kTransposeA, 1u);
                }
                umma_commit(&sm.v_empty);
            }
            __syncwarp();
            return true;
        };
        const auto next_blocks = [&]() {
            const int job = next_job();
            return job < 0 ? 0 : (sm.chunk[job / v_heads].length + kBlock - 1) / kBlock;
        };
        int end = next_blocks();  // of the blocks of the job at hand
        ok = ok && (end == 0 || issue_values(0));
        for (; n < end && ok; ++n) {
            const uint32_t parity = n & 1;
            const uint32_t qk_offset = (n & 1) * (kQkBytes >> 4);
            const uint32_t qk_base = qk_operand + qk_offset, w_base = w_operand + (n & 1) * (kWBytes >> 4);
            ok = wait(&sm.qk_full[n & 1], (n >> 1) & 1, failed, status) && wait(&sm.s_ready, parity, failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                // X, then Y
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const uint32_t rows = part == 0 ? kBlock * 128 : 0;
                    const uint32_t d = part == 0 ? kKeyColumn : kQueryColumn;
#pragma unroll
                    for (int ks = 0; ks < kDim / 16; ++ks) {
                        const uint64_t b = operand_at(qk_base, rows + (ks >> 2) * kTileBytes + (ks & 3) * 32);
                        umma_f16(d, kSplitColumn + ks * 8, b, kNarrow, ks > 0 ? 1u : 0u);
                        umma_f16(d, kSplitColumn + 64 + ks * 8, b, kNarrow, 1u);
                    }
                    if (part == 0) {
                        umma_commit(&sm.x_done);
                    }
                }
            }
            __syncwarp();
            ok = wait(&sm.x_ready, parity, failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                // U', then O
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const uint32_t rows = part == 0 ? kBlock * 128 : 0;
                    const uint32_t d = part == 0 ? kUpdateColumn : kResultColumn;
#pragma unroll
                    for (int ks = 0; ks < kBlock / 16; ++ks) {
                        const uint32_t x = kKeyColumn + (ks >> 1) * 32 + (ks & 1) * 8;
                        const uint64_t upper = operand_at(w_base, rows + ks * 32), lower = operand_at(w_base, rows + kTileBytes + ks * 32);
                        umma_f16(d, x, upper, kNarrow, 1u);
                        umma_f16(d, x + 16, upper, kNarrow, 1u);
                        umma_f16(d, x, lower, kNarrow, 1u);
                    }
                    umma_commit(part == 0 ? &sm.u_done : &sm.o_done);
                }
                umma_commit(&sm.w_empty[n & 1]);
            }
            __syncwarp();
            ok = wait(&sm.u_ready, parity, failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    const uint32_t u = kUpdateColumn + (ks >> 1) * 32 + (ks & 1) * 8;
                    const uint64_t b = operand_at(k_across + qk_offset, ks * 2048);
                    umma_f16(kStateColumn, u, b, kWide | kTransposeB, 1u);
                    umma_f16(kStateColumn, u + 16, b, kWide | kTransposeB, 1u);
                }
                umma_commit(&sm.s_done);
                umma_commit(&sm.qk_empty[n & 1]);
            }
            __syncwarp();
            if (n + 1 == end) {
                end += next_blocks();
            }
            if (ok && n + 1 < end) {
                ok = issue_values(n + 1);
            }
        }
        // the last commits that nobody else waits for have arrived in this CTA's shared memory before it ends
        if (ok && n > 0) {
            for (int i = n > 2 ? n - 2 : 0; i < n && ok; ++i) {
                ok = wait(&sm.qk_empty[i & 1], (i >> 1) & 1, failed, status) && wait(&sm.w_empty[i & 1], (i >> 1) & 1, failed, status);
            }
            ok = ok && wait(&sm.v_empty, (n - 1) & 1, failed, status);
        }
    } else if (warp < kChainWarps) {
        // ---------------- the chain --------------------------------------------------------------------
        const int quarter = warp & 3;
        const int group = warp >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t tmem = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t held = tmem + kStateColumn + group * 64;                // 64 key dims of the row
        const uint32_t upper = tmem + kSplitColumn + group * 32, lower = upper + 64;
        const uint32_t x_at = tmem + kKeyColumn + group * 32, u_at = tmem + kUpdateColumn + group * 32;
        int done = 0;  // jobs
        for (int job = next_job(); job >= 0; job = next_job()) {
            const ChunkOfJobs& chunk = sm.chunk[job / v_heads];
            const int blocks = (chunk.length + kBlock - 1) / kBlock;
            const size_t state_row = (static_cast<size_t>(chunk.slot) * v_heads + job % v_heads) * kDim + row;
            {
                const bool holds = continues == nullptr || __ldcg(continues + chunk.sequence) != 0;
                const float scale = holds ? state_scales[state_row] : 0.0f;
                const uint4* codes = reinterpret_cast<const uint4*>(state + state_row * kDim + group * 64);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float s[32];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 raw = codes[2 * c + i];
                        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            s[16 * i + j] = holds ? static_cast<float>(static_cast<int8_t>(words[j >> 2] >> (8 * (j & 3)))) * scale : 0.0f;
                        }
                    }
                    tmem_store_columns(held + 32 * c, s);
                    tmem_store_split(upper + 16 * c, lower + 16 * c, s);
                }
            }
            tmem_store_wait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.s_ready);
            }
            for (int at = 0; at < blocks; ++at, ++n) {
                const uint32_t parity = n & 1;
                const float* decay = sm.decay[n & 1];
                float x[32];
                ok = wait(&sm.w_full[n & 1], (n >> 1) & 1, failed, status) && wait(&sm.x_done, parity, failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_columns(x_at, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 g = *reinterpret_cast<const float4*>(decay + group * 32 + 4 * i);
                    x[4 * i] *= -g.x;
                    x[4 * i + 1] *= -g.y;
                    x[4 * i + 2] *= -g.z;
                    x[4 * i + 3] *= -g.w;
                }
                tmem_store_split(x_at, x_at + 16, x);
                const float end = decay[kBlock - 1];  // (before x_ready: behind it the place may get the block after next)
                tmem_store_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.x_ready);
                }
                // the state decays while U' is made
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    load_columns(held + 32 * c, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 both = __fmul2_rn({x[i], x[i + 1]}, {end, end});
                        x[i] = both.x;
                        x[i + 1] = both.y;
                    }
                    tmem_store_columns(held + 32 * c, x);
                }
                ok = wait(&sm.u_done, parity, failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_columns(u_at, x);
                tmem_store_split(u_at, u_at + 16, x);
                tmem_store_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.u_ready);
                }
                ok = wait(&sm.s_done, parity, failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (at + 1 < blocks) {
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        load_columns(held + 32 * c, x);
                        tmem_store_split(upper + 16 * c, lower + 16 * c, x);
                    }
                    tmem_store_wait();
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sm.s_ready);
                    }
                }
            }
            if (!ok) {
                break;
            }
            // the state's eight bits, 64 of a row
            float peak = 0.0f;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                float s[32];
                load_columns(held + 32 * c, s);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    peak = fmaxf(peak, fabsf(s[i]));
                }
            }
            sm.peak[done & 1][group][row] = peak;
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.chain_met);
            }
            // (bounded as everything: a warp that has given up does not come)
            ok = wait(&sm.chain_met, done & 1, failed, status);
            if (!ok) {
                break;
            }
            peak = fmaxf(peak, sm.peak[done & 1][group ^ 1][row]);
            ++done;
            const float inverse = peak == 0.0f ? 0.0f : __fdiv_rn(127.0f, peak);
            uint4* codes = reinterpret_cast<uint4*>(state + state_row * kDim + group * 64);
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                float s[32];
                load_columns(held + 32 * c, s);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t words[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        words[j >> 2] |= (static_cast<uint32_t>(__float2int_rn(s[16 * i + j] * inverse)) & 0xffu) << (8 * (j & 3));
                    }
                    codes[2 * c + i] = make_uint4(words[0], words[1], words[2], words[3]);
                }
            }
            if (group == 0) {
                state_scales[state_row] = __fmul_rn(peak, 1.0f / 127.0f);
            }
        }
    } else {
        // ---------------- outputs ----------------------------------------------------------------------
        const int quarter = warp & 3;
        const int group = (warp - kChainWarps) >> 2;
        const int row = quarter * 32 + lane;     // value dim
        const uint32_t tmem = (static_cast<uint32_t>(quarter * 32) << 16) + group * 32;
        const int piece = lane & 15;             // later: value dims 4 piece .. + 3 and 64 + 4 piece .. + 3 of a token
        float2 gain[4] = {};
        if (norm.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint2 raw = *reinterpret_cast<const uint2*>(norm.weight + 64 * i + 4 * piece);
                gain[2 * i] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u)};
                gain[2 * i + 1] = {__uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u)};
            }
        }
        const int stride = v_heads * kDim;
        const int first = (warp - kChainWarps) * 8 + (lane >> 4);  // of a block: this thread's first token
        for (int job = next_job(); job >= 0; job = ok ? next_job() : -1) {
            const ChunkOfJobs& chunk = sm.chunk[job / v_heads];
            __nv_bfloat16* target = out + (static_cast<size_t>(chunk.begin) + first) * stride + job % v_heads * kDim + 4 * piece;
            for (int left = chunk.length; left > 0; left -= kBlock, ++n) {
                const uint32_t parity = n & 1;
                ok = wait(&sm.w_full[n & 1], (n >> 1) & 1, failed, status) && wait(&sm.o_done, parity, failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float x[32];
                {
                    float y[32];
                    load_columns(tmem + kResultColumn, x);
                    load_columns(tmem + kQueryColumn, y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 g = *reinterpret_cast<const float4*>(&sm.decay[n & 1][group * 32 + 4 * i]);
                        const float2 lo = __ffma2_rn({g.x, g.y}, {y[4 * i], y[4 * i + 1]}, {x[4 * i], x[4 * i + 1]});
                        const float2 hi = __ffma2_rn({g.z, g.w}, {y[4 * i + 2], y[4 * i + 3]}, {x[4 * i + 2], x[4 * i + 3]});
                        x[4 * i] = lo.x;
                        x[4 * i + 1] = lo.y;
                        x[4 * i + 2] = hi.x;
                        x[4 * i + 3] = hi.y;
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.o_free);
                    mbar_arrive(&sm.w_empty[n & 1]);
                }
                ok = wait(&sm.rows_free, parity ^ 1, failed, status);
                if (!ok) {
                    break;
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    sm.rows[(group * 32 + i) * kDim + row] = x[i];
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.rows_ready);
                }
                ok = wait(&sm.rows_ready, parity, failed, status) &&
                     (norm.gate == nullptr || wait(&sm.gate_full[n & 1], (n >> 1) & 1, failed, status));
                if (!ok) {
                    break;
                }
                // rows of the batch: eight tokens of this warp, two at a time
                float2 o[4][4];
                float inverse[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 lo = *reinterpret_cast<const float4*>(&sm.rows[(first + 2 * i) * kDim + 4 * piece]);
                    const float4 hi = *reinterpret_cast<const float4*>(&sm.rows[(first + 2 * i) * kDim + 64 + 4 * piece]);
                    o[i][0] = {lo.x, lo.y};
                    o[i][1] = {lo.z, lo.w};
                    o[i][2] = {hi.x, hi.y};
                    o[i][3] = {hi.z, hi.w};
                }
                if (norm.gate != nullptr) {
                    // (the four sums go through the warp side by side)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float2 sums = __fmul2_rn(o[i][0], o[i][0]);
#pragma unroll
                        for (int j = 1; j < 4; ++j) {
                            sums = __ffma2_rn(o[i][j], o[i][j], sums);
                        }
                        inverse[i] = sums.x + sums.y;
                    }
#pragma unroll
                    for (int offset = 1; offset < 16; offset <<= 1) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            inverse[i] += __shfl_xor_sync(0xffffffffu, inverse[i], offset);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        inverse[i] = rsqrtf(inverse[i] / static_cast<float>(kDim) + norm.epsilon);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = first + 2 * i;
                    if (norm.gate != nullptr) {
                        const uint2 gate_lo = *reinterpret_cast<const uint2*>(sm.gate[n & 1] + t * (kDim * 2) + 8 * piece);
                        const uint2 gate_hi = *reinterpret_cast<const uint2*>(sm.gate[n & 1] + t * (kDim * 2) + kDim + 8 * piece);
                        const uint32_t words[4] = {gate_lo.x, gate_lo.y, gate_hi.x, gate_hi.y};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 z = {__uint_as_float(words[j] << 16), __uint_as_float(words[j] & 0xffff0000u)};
                            const float2 silu = __fmul2_rn(z, sigmoid_pair(z));
                            o[i][j] = __fmul2_rn(__fmul2_rn(o[i][j], {inverse[i], inverse[i]}), __fmul2_rn(gain[j], silu));
                        }
                    }
                    if (t < left) {
                        __nv_bfloat16* to = target + 2 * i * stride;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const __nv_bfloat162 lo = __floats2bfloat162_rn(o[i][2 * j].x, o[i][2 * j].y);
                            const __nv_bfloat162 hi = __floats2bfloat162_rn(o[i][2 * j + 1].x, o[i][2 * j + 1].y);
                            *reinterpret_cast<uint2*>(to + 64 * j) =
                                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.rows_free);
                    mbar_arrive(&sm.gate_empty[n & 1]);
                }
                target += kBlock * stride;
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(failed) != 0) {
        // A wait gave up somewhere.  What was asked for and arrives by itself is waited for, 0.2 ms at most for each.
        const auto arrived = [](uint64_t* bar, uint32_t parity) {
            const long long start = clock64();
            while (!mbar_try_wait(bar, parity) && clock64() - start < 400000ll) {
            }
        };
        if (warp == kLoadWarp) {
            for (int i = n > 2 ? n - 2 : 0; i <= n; ++i) {
                arrived(&sm.qk_full[i & 1], (i >> 1) & 1);
                arrived(&sm.w_full[i & 1], (i >> 1) & 1);
            }
        } else if (warp == kMmaWarp) {
            arrived(&sm.v_empty, n & 1);
            arrived(&sm.o_done, n & 1);
            arrived(&sm.s_done, n & 1);
            for (int i = n > 1 ? n - 1 : 0; i <= n; ++i) {
                arrived(&sm.qk_empty[i & 1], (i >> 1) & 1);
                arrived(&sm.w_empty[i & 1], (i >> 1) & 1);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kLoadWarp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(0), "r"(kTmemColumns) : "memory");
    }
}

}  // namespace
}  // namespace qwc

extern "C" size_t qwc_delta_chunk_workspace_bytes(int tokens, int sequences) {
    using namespace qwc;
    if (tokens <= 0 || tokens > kMaxChunkTokens || sequences <= 0 || sequences > kMaxChunkSequences) {
        return 0;
    }
    return images_bytes(most_chunk_tiles(tokens, sequences, kBlock), current_shape().delta_value_heads);
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
        !aligned(out) || workspace == nullptr || !aligned(workspace) ||
        workspace_bytes < qwc_delta_chunk_workspace_bytes(tokens, sequences)) {
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
    struct Setup {
        cudaError_t error;
        int sms;
    };
    static PerDevice<Setup> per_device;
    const Setup* setup = per_device.get([]() {
        Setup found = {cudaSuccess, 0};
        int device = 0;
        found.error = cudaFuncSetAttribute(delta_factor_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(sizeof(FactorSmem)) + 1024);
        if (found.error == cudaSuccess) {
            found.error = cudaFuncSetAttribute(delta_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(sizeof(ChainSmem)) + 1024);
        }
        if (found.error == cudaSuccess) {
            found.error = cudaGetDevice(&device);
        }
        if (found.error == cudaSuccess) {
            found.error = cudaDeviceGetAttribute(&found.sms, cudaDevAttrMultiProcessorCount, device);
        }
        return found;
    });
    if (setup == nullptr) {
        return cudaErrorInvalidDevice;
    }
    if (setup->error != cudaSuccess) {
        return setup->error;
    }
    const int blocks = most_chunk_tiles(tokens, sequences, kBlock);
    const Images images = images_at(workspace, blocks, v_heads);
    const int per_cta = blocks < kFewBlocks ? 1 : v_heads / kDeltaKeyHeads;
    const cudaError_t launched = launch_chained(
        delta_factor_kernel, dim3(v_heads / per_cta, blocks), dim3(kFactorThreads), sizeof(FactorSmem) + 1024, stream,
        static_cast<const __nv_bfloat16*>(qkv), static_cast<const float*>(alpha), static_cast<const float*>(beta),
        static_cast<const uint32_t*>(chunk_begins), images, tokens, sequences, v_heads, per_cta, status);
    if (launched != cudaSuccess) {
        return launched;
    }
    const OutputNorm norm = {static_cast<const __nv_bfloat16*>(gate), static_cast<const __nv_bfloat16*>(norm_weight),
                             gate_stride, epsilon};
    return launch_chained(delta_chain_kernel, dim3(std::min(v_heads * sequences, setup->sms)), dim3(kChainThreads), sizeof(ChainSmem) + 1024, stream,
                          static_cast<int8_t*>(state), state_scales, static_cast<const uint32_t*>(state_slots),
                          static_cast<const uint32_t*>(continues), static_cast<const __nv_bfloat16*>(qkv), images, blocks,
                          static_cast<__nv_bfloat16*>(out), sequences, v_heads, state_capacity, norm, status);
}
