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
// blocks of a head with three products,
//   [Q ; K] S0^T  ->  R  ->  W R = [outputs within the block ; updates U']  ->  S1^T = g_end S0^T + K^T U'.
//
// Bound by the chain of these products: each waits for the one before, block after block, 64 columns of the state (value
// dims) at a time.  They run on the fifth-generation tensor cores, M = 128 rows, accumulators in tensor memory.  q and k
// are bf16 as they come; S, R, U' and W are written as the sum of two bf16, which hold 16 bits, and their products leave
// out only the lower part times the lower part.  The state itself stays in fp32 registers: a thread is a key dim of 32
// value dims.

#include <cstddef>

#include "chunk.cuh"
#include "tcgen05.cuh"

namespace qwc {
namespace {

constexpr int kDim = kDeltaHeadDim;
constexpr int kBlock = 64;                               // tokens
constexpr int kColumns = 64;                             // value dims of a chain
constexpr int kTileBytes = 128 * 128;                    // 128 rows of 64 bf16, 128-byte swizzle
constexpr int kQkBytes = 2 * kTileBytes;                 // [half of the dims][q of the block's tokens, k][128 bytes]
constexpr int kWBytes = 2 * kTileBytes;                  // [upper, lower bf16][row][128 bytes]
constexpr int kSBytes = 2 * kTileBytes;                  // [upper, lower][key dim][128 bytes]
constexpr int kRBytes = kTileBytes;                      // [upper, lower][token][128 bytes]

// Workspace: images of the operands as shared memory has them.
struct Images {
    uint8_t* qk;    // [block][key head][kQkBytes]
    uint8_t* w;     // [block][value head][kWBytes]
    float* decay;   // [block][value head][kBlock]: from the block's start
};

inline size_t images_bytes(int blocks, int v_heads) {
    return static_cast<size_t>(blocks) *
           (static_cast<size_t>(kDeltaKeyHeads) * kQkBytes + static_cast<size_t>(v_heads) * (kWBytes + kBlock * sizeof(float)));
}

inline Images images_at(void* workspace, int blocks, int v_heads) {
    Images at;
    at.qk = static_cast<uint8_t*>(workspace);
    at.w = at.qk + static_cast<size_t>(blocks) * kDeltaKeyHeads * kQkBytes;
    at.decay = reinterpret_cast<float*>(at.w + static_cast<size_t>(blocks) * v_heads * kWBytes);
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

constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kColumns >> 3) << 17) | (8u << 24);
constexpr uint32_t kTransposeA = 1u << 15, kTransposeB = 1u << 16;

// Operand of 128-byte rows with the 128-byte swizzle, eight rows to an atom.  K-major: a row is one of M or N, its bytes 64
// of the contracted elements.  MN-major: a row is one of the contracted, its bytes 64 of M or N, the next 64 `block` bytes on.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t block) {
    const uint64_t lo = ((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16);
    const uint64_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return lo | (hi << 32);
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

__device__ __forceinline__ void unpack_bf16(const uint4& raw, float* out) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[2 * i] = __uint_as_float(words[i] << 16);
        out[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
    }
}

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
    atomicCAS(status, 0, kStatusChunkDeltaWait);
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
// blocks on the diagonal by substitution, then T_10 = -T_11 A_10 T_00 for blocks of 16 and of 32.  W is a product again,
// [P ; diag(g_end / g)] times T.

constexpr int kFactorThreads = 128;
constexpr int kPitch = 68;  // floats of a row of the matrices in shared memory: rows begin in different banks

struct FactorSmem {
    uint8_t operand[kQkBytes];            // q and k, then [P ; diag] in two parts
    float t[kBlock * kPitch];             // (1 + A)^-1
    union {
        float a[kBlock * kPitch];         // A, below the diagonal
        uint8_t product[kRBytes];         // T in two parts
    };
    float2 log[kBlock];                   // log2 of the decay from the start: a whole number and the rest
    float beta[kBlock];
    uint64_t done;
    uint32_t tmem_base;
    int failed;
};
static_assert(offsetof(FactorSmem, a) % 1024 == 0, "an operand's alignment");

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x += a * rows[0 .. 3][8 columns] for four steps of the sum.
__device__ __forceinline__ void multiply4(float (&x)[8], const float4& a, const float* rows) {
    const float factors[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float4 lo = *reinterpret_cast<const float4*>(rows + k * kPitch);
        const float4 hi = *reinterpret_cast<const float4*>(rows + k * kPitch + 4);
        const float row[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            x[c] = fmaf(factors[k], row[c], x[c]);
        }
    }
}

__global__ void __launch_bounds__(kFactorThreads) delta_factor_kernel(
    const __nv_bfloat16* __restrict__ qkv, const float* __restrict__ alpha, const float* __restrict__ beta,
    const uint32_t* __restrict__ begins, const Images images, int tokens, int sequences, int v_heads, int* status) {
    extern __shared__ unsigned char smem_raw[];
    FactorSmem& sm = *reinterpret_cast<FactorSmem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x;
    const int lane = tid & 31;
    const int warp = tid >> 5;
    const int head = blockIdx.x;
    const int block = blockIdx.y;
    const int ratio = v_heads / kDeltaKeyHeads;
    const int key_head = head / ratio;
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDim;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(64)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (tid == 0) {
        mbar_init(&sm.done, 1);
        sm.failed = 0;
        mbar_fence_init();
    }
    __syncthreads();
    // (Not before this CTA has its tensor memory: a CTA of the next kernel that took some of it first would wait for this
    // kernel's end, and this CTA for that one's.)
    pdl_launch_dependents();
    pdl_wait();
    const ChunkTile tile = find_chunk_tile(begins, sequences, tokens, kBlock, block);
    const bool here = tile.sequence >= 0;
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
                             smem_u32(sm.operand + (piece >> 3) * kTileBytes + swizzled(row, piece & 7))),
                         "l"(from), "r"(token < count ? 16 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (warp == 0) {
            // decay from the start: a scan over the tokens, in whole numbers and rests below one
            float whole[2], part[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = lane + 32 * i;
                // (beyond 2^-130 fp32 has nothing, and an alpha of 0 takes everything before it away)
                const float log = token < count ? fmaxf(log2f(alpha[(row0 + token) * v_heads + head]), -130.0f) : 0.0f;
                sm.beta[token] = token < count ? beta[(row0 + token) * v_heads + head] : 0.0f;
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
                sm.log[lane + 32 * i] = make_float2(whole[i], part[i]);
                decay[lane + 32 * i] = exp2f(whole[i] + part[i]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    fence_proxy_async();
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sm.tmem_base);
    const uint32_t tmem_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
    bool ok = here;
    if (here) {
        if (warp == 0) {
            if (elect_one()) {
                const uint32_t base = smem_u32(sm.operand);
#pragma unroll
                for (int ks = 0; ks < kDim / 16; ++ks) {
                    const uint32_t at = base + (ks >> 2) * kTileBytes + (ks & 3) * 32;
                    mma_bf16(tmem_base, operand(at, 16), operand(at + kBlock * 128, 16), kIdesc, ks > 0 ? 1u : 0u);
                }
                umma_commit(&sm.done);
            }
            __syncwarp();
        }
        if (head == key_head * ratio) {
            // the image of q and k, by the key head's first value head
            uint4* to = reinterpret_cast<uint4*>(images.qk + (static_cast<size_t>(block) * kDeltaKeyHeads + key_head) * kQkBytes);
#pragma unroll 4
            for (int i = tid; i < kQkBytes / 16; i += kFactorThreads) {
                to[i] = reinterpret_cast<const uint4*>(sm.operand)[i];
            }
        }
        ok = wait(&sm.done, 0, &sm.failed, status);
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    __syncthreads();  // (the image has been read)
    const int t = tid & (kBlock - 1);
    const bool outputs = tid < kBlock;
    if (ok) {
        // thread t has row t of Q K^T, thread 64 + t of K K^T: P to its operand, A to shared memory
        const float2 mine = sm.log[t];
        const float strength = outputs ? 1.0f : sm.beta[t];
        const int limit = outputs ? t + 1 : t;
        const float to_end = exp2_fast((sm.log[kBlock - 1].x - mine.x) + (sm.log[kBlock - 1].y - mine.y));
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
            float x[32];
            if (32 * c <= (t | 31)) {  // (the same for a warp)
                load_columns(tmem_row + 32 * c, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int j = 32 * c + i;
                    const float2 other = sm.log[j];
                    const float decay = exp2_fast((mine.x - other.x) + (mine.y - other.y));
                    x[i] = j < limit ? strength * decay * x[i] : 0.0f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = 0.0f;
                }
            }
            if (outputs) {
                store_split(sm.operand, kTileBytes, t, 4 * c, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    *reinterpret_cast<float4*>(&sm.a[t * kPitch + 32 * c + 4 * i]) =
                        make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = 32 * c + i == t ? to_end : 0.0f;
                }
                store_split(sm.operand, kTileBytes, kBlock + t, 4 * c, x);
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncthreads();
    if (ok) {
        if (outputs) {
            // blocks of 16 on the diagonal: a column per thread
            const int b = tid >> 4, j = tid & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < i; k += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(&sm.a[(16 * b + i) * kPitch + 16 * b + k]);
                    sum = fmaf(a.x, x[k], sum);
                    sum = k + 1 < i ? fmaf(a.y, x[k + 1 < i ? k + 1 : 0], sum) : sum;
                    sum = k + 2 < i ? fmaf(a.z, x[k + 2 < i ? k + 2 : 0], sum) : sum;
                    sum = k + 3 < i ? fmaf(a.w, x[k + 3 < i ? k + 3 : 0], sum) : sum;
                }
                x[i] = i == j ? 1.0f : i < j ? 0.0f : -sum;
                sm.t[(16 * b + i) * kPitch + 16 * b + j] = x[i];
            }
        } else {
            // zeros above the diagonal, in blocks of 16
            const int b = t >> 4;
            for (int j = 16 * (b + 1); j < kBlock; j += 4) {
                *reinterpret_cast<float4*>(&sm.t[t * kPitch + j]) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    }
    __syncthreads();
    if (ok) {
        // blocks of 32: T_10 = -T_11 (A_10 T_00) of 16, eight columns per thread of one row of 32
        const int pair = tid >> 5;  // two threads' columns of two blocks: pair & 1 the columns' half, pair >> 1 the block
        const int base = 32 * (pair >> 1), column = base + 8 * (pair & 1);
        const int r = lane & 15;    // (lanes 16-31 do the same again)
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            multiply4(x, *reinterpret_cast<const float4*>(&sm.a[(base + 16 + r) * kPitch + base + k]), &sm.t[(base + k) * kPitch + column]);
        }
        float* at = &sm.t[(base + 16 + r) * kPitch + column];
        if (lane < 16) {
            *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(at + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
        __syncwarp();
        float y[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            multiply4(y, *reinterpret_cast<const float4*>(&sm.t[(base + 16 + r) * kPitch + base + 16 + k]),
                      &sm.t[(base + 16 + k) * kPitch + column]);
        }
        __syncwarp();
        if (lane < 16) {
            *reinterpret_cast<float4*>(at) = make_float4(-y[0], -y[1], -y[2], -y[3]);
            *reinterpret_cast<float4*>(at + 4) = make_float4(-y[4], -y[5], -y[6], -y[7]);
        }
    }
    __syncthreads();
    if (ok) {
        // the block of 32 below: a row per lane, eight columns per warp (T_00 is zero above its diagonal)
        const int column = 8 * warp;
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = column; k < 32; k += 4) {
            multiply4(x, *reinterpret_cast<const float4*>(&sm.a[(32 + lane) * kPitch + k]), &sm.t[k * kPitch + column]);
        }
        float* at = &sm.t[(32 + lane) * kPitch + column];
        *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(at + 4) = make_float4(x[4], x[5], x[6], x[7]);
        __syncwarp();
        float y[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
        for (int k = 0; k < 32; k += 4) {
            multiply4(y, *reinterpret_cast<const float4*>(&sm.t[(32 + lane) * kPitch + 32 + k]), &sm.t[(32 + k) * kPitch + column]);
        }
        __syncwarp();
        *reinterpret_cast<float4*>(at) = make_float4(-y[0], -y[1], -y[2], -y[3]);
        *reinterpret_cast<float4*>(at + 4) = make_float4(-y[4], -y[5], -y[6], -y[7]);
    }
    __syncthreads();
    if (ok) {
        // T diag(beta) as an operand: half a row per thread
        const int row = tid >> 1, half = tid & 1;
        float x[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 value = *reinterpret_cast<const float4*>(&sm.t[row * kPitch + 32 * half + 4 * i]);
            const float4 strength = *reinterpret_cast<const float4*>(&sm.beta[32 * half + 4 * i]);
            x[4 * i] = value.x * strength.x;
            x[4 * i + 1] = value.y * strength.y;
            x[4 * i + 2] = value.z * strength.z;
            x[4 * i + 3] = value.w * strength.w;
        }
        store_split(sm.product, kRBytes / 2, row, 4 * half, x);
        fence_proxy_async();
    }
    __syncthreads();
    if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (warp == 0) {
            if (elect_one()) {
                const uint32_t a = smem_u32(sm.operand), b = smem_u32(sm.product);
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    const uint64_t upper = operand(a + ks * 32, 16), lower = operand(a + kTileBytes + ks * 32, 16);
                    const uint64_t t_upper = operand(b + ks * 2048, 16), t_lower = operand(b + kRBytes / 2 + ks * 2048, 16);
                    mma_bf16(tmem_base, upper, t_upper, kIdesc | kTransposeB, ks > 0 ? 1u : 0u);
                    mma_bf16(tmem_base, upper, t_lower, kIdesc | kTransposeB, 1u);
                    mma_bf16(tmem_base, lower, t_upper, kIdesc | kTransposeB, 1u);
                }
                umma_commit(&sm.done);
            }
            __syncwarp();
        }
        ok = wait(&sm.done, 1, &sm.failed, status);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (ok) {
        uint8_t* w = images.w + (static_cast<size_t>(block) * v_heads + head) * kWBytes;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
            float x[32];
            load_columns(tmem_row + 32 * c, x);
            store_split(w, kTileBytes, tid, 4 * c, x);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(64) : "memory");
    }
}

// ---- the chain of blocks --------------------------------------------------------------------------------

constexpr int kChainWarps = 8;  // of a chain: four quarters of the rows, two halves of its columns

// Two chains (both halves of a head's value dims) to a CTA, or one.
template <int kChains>
struct ChainSmem {
    uint8_t qk[2][kQkBytes];
    uint8_t w[kWBytes];
    uint8_t s[kChains][kSBytes];
    uint8_t r[kChains][kRBytes];  // R of a block, then U'
    uint64_t qk_full[2], qk_empty[2], w_full, w_empty;
    uint64_t s_ready[kChains], d1_done[kChains], r_ready[kChains], d2_done[kChains], u_ready[kChains], d3_done[kChains];
    float peak[kChains][4][kColumns];
    uint32_t tmem_base;
    int failed;
};

template <int kChains>
__global__ void __launch_bounds__((kChains * (kChainWarps + 1) + 1) * 32, 1) delta_chain_kernel(
    int8_t* __restrict__ state, float* __restrict__ state_scales, const uint32_t* __restrict__ state_slots,
    const uint32_t* __restrict__ continues, const uint32_t* __restrict__ begins, const __nv_bfloat16* __restrict__ qkv,
    const Images images, __nv_bfloat16* __restrict__ out, int tokens, int v_heads, int state_capacity, int* status) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = ChainSmem<kChains>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    constexpr int kFirstMmaWarp = kChains * kChainWarps;
    constexpr int kLoadWarp = kFirstMmaWarp + kChains;
    constexpr int kTmemColumns = kChains == 1 ? 256 : 512;
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int head = blockIdx.x / (2 / kChains);
    const int first_chain = kChains == 1 ? blockIdx.x & 1 : 0;  // of the head's two
    const int key_head = head / (v_heads / kDeltaKeyHeads);
    const int channels = (2 * kDeltaKeyHeads + v_heads) * kDim;
    const int sequence = blockIdx.y;
    pdl_wait();
    const ChunkSpan span = chunk_span(begins, sequence, tokens);
    const uint32_t slot = __ldcg(state_slots + sequence);
    if (span.length == 0) {
        return;
    }
    if (slot >= static_cast<uint32_t>(state_capacity)) {
        // a slot beyond the pool: nothing of this chunk is read or written, the host learns of it through the status
        // word (the whole CTA takes this branch)
        if (threadIdx.x == 0) {
            atomicCAS(status, 0, kStatusStateSlotRange);
        }
        return;
    }
    const int blocks = (span.length + kBlock - 1) / kBlock;
    if (warp == kLoadWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.qk_full[i], 1);
            mbar_init(&sm.qk_empty[i], kChains);
        }
        mbar_init(&sm.w_full, 1);
        mbar_init(&sm.w_empty, kChains);
        for (int i = 0; i < kChains; ++i) {
            mbar_init(&sm.s_ready[i], kChainWarps);
            mbar_init(&sm.d1_done[i], 1);
            mbar_init(&sm.r_ready[i], kChainWarps / 2);
            mbar_init(&sm.d2_done[i], 1);
            mbar_init(&sm.u_ready[i], kChainWarps / 2);
            mbar_init(&sm.d3_done[i], 1);
        }
        sm.failed = 0;
        mbar_fence_init();
    }
    fence_proxy_async();
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    pdl_launch_dependents();  // (this CTA has its tensor memory)
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sm.tmem_base);
    bool ok = true;
    int n = 0;  // blocks so far
    float s[32];

    if (warp == kLoadWarp) {
        // ---------------- operands of the blocks -------------------------------------------------------
        int first_block = 0;  // of this chunk, in the order of the first kernel
        for (int i = lane; i < sequence; i += 32) {
            first_block += (chunk_span(begins, i, tokens).length + kBlock - 1) / kBlock;
        }
        first_block = static_cast<int>(__reduce_add_sync(0xffffffffu, first_block));
        for (; n < blocks && ok; ++n) {
            const size_t block = static_cast<size_t>(first_block) + n;
            ok = wait(&sm.qk_empty[n & 1], ((n >> 1) & 1) ^ 1, &sm.failed, status);
            if (ok && lane == 0) {
                mbar_arrive_expect_tx(&sm.qk_full[n & 1], kQkBytes);
                bulk_g2s(sm.qk[n & 1], images.qk + (block * kDeltaKeyHeads + key_head) * kQkBytes, kQkBytes, &sm.qk_full[n & 1]);
            }
            __syncwarp();
            ok = ok && wait(&sm.w_empty, (n & 1) ^ 1, &sm.failed, status);
            if (ok && lane == 0) {
                mbar_arrive_expect_tx(&sm.w_full, kWBytes);
                bulk_g2s(sm.w, images.w + (block * v_heads + head) * kWBytes, kWBytes, &sm.w_full);
            }
            __syncwarp();
        }
    } else if (warp >= kFirstMmaWarp) {
        // ---------------- tensor-core issue of a chain ---------------------------------------------------
        const int chain = warp - kFirstMmaWarp;
        const uint32_t d1 = tmem_base + chain * 256, d2 = d1 + kColumns, d3 = d2 + kColumns;
        const uint32_t s_base = smem_u32(sm.s[chain]), r_base = smem_u32(sm.r[chain]), w_base = smem_u32(sm.w);
        for (; n < blocks; ++n) {
            const uint32_t parity = n & 1;
            const uint32_t qk_base = smem_u32(sm.qk[n & 1]);
            ok = wait(&sm.qk_full[n & 1], (n >> 1) & 1, &sm.failed, status) &&
                 wait(&sm.s_ready[chain], parity, &sm.failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < kDim / 16; ++ks) {
                    const uint64_t a = operand(qk_base + (ks >> 2) * kTileBytes + (ks & 3) * 32, 16);
                    mma_bf16(d1, a, operand(s_base + ks * 2048, 16), kIdesc | kTransposeB, ks > 0 ? 1u : 0u);
                    mma_bf16(d1, a, operand(s_base + kTileBytes + ks * 2048, 16), kIdesc | kTransposeB, 1u);
                }
                umma_commit(&sm.d1_done[chain]);
            }
            __syncwarp();
            ok = wait(&sm.w_full, parity, &sm.failed, status) && wait(&sm.r_ready[chain], parity, &sm.failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    const uint64_t upper = operand(w_base + ks * 32, 16), lower = operand(w_base + kTileBytes + ks * 32, 16);
                    const uint64_t r_upper = operand(r_base + ks * 2048, 16), r_lower = operand(r_base + kRBytes / 2 + ks * 2048, 16);
                    mma_bf16(d2, upper, r_upper, kIdesc | kTransposeB, ks > 0 ? 1u : 0u);
                    mma_bf16(d2, upper, r_lower, kIdesc | kTransposeB, 1u);
                    mma_bf16(d2, lower, r_upper, kIdesc | kTransposeB, 1u);
                }
                umma_commit(&sm.d2_done[chain]);
                umma_commit(&sm.w_empty);
            }
            __syncwarp();
            ok = wait(&sm.u_ready[chain], parity, &sm.failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    const uint64_t a = operand(qk_base + kBlock * 128 + ks * 2048, kTileBytes);  // k, dims across
                    mma_bf16(d3, a, operand(r_base + ks * 2048, 16), kIdesc | kTransposeA | kTransposeB, ks > 0 ? 1u : 0u);
                    mma_bf16(d3, a, operand(r_base + kRBytes / 2 + ks * 2048, 16), kIdesc | kTransposeA | kTransposeB, 1u);
                }
                umma_commit(&sm.d3_done[chain]);
                umma_commit(&sm.qk_empty[n & 1]);
            }
            __syncwarp();
        }
    } else {
        // ---------------- state, R, U' and the outputs -----------------------------------------------------
        const int chain = warp / kChainWarps;
        const int quarter = warp & 3;
        const int group = (warp >> 2) & 1;                       // of 32 columns
        const int row = quarter * 32 + lane;                     // key dim; or q (0 .. 63) and k (64 ..) of a token
        const int t = row & (kBlock - 1);
        const int column = (first_chain + chain) * kColumns + group * 32;  // first value dim
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t d1 = tmem_base + chain * 256 + lanes + group * 32, d2 = d1 + kColumns, d3 = d2 + kColumns;
        int first_block = 0;
        for (int i = lane; i < sequence; i += 32) {
            first_block += (chunk_span(begins, i, tokens).length + kBlock - 1) / kBlock;
        }
        first_block = static_cast<int>(__reduce_add_sync(0xffffffffu, first_block));
        const float* decays = images.decay + (static_cast<size_t>(first_block) * v_heads + head) * kBlock;
        const size_t state_row = (static_cast<size_t>(slot) * v_heads + head) * kDim + column;
        if (continues == nullptr || __ldcg(continues + sequence) != 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                s[i] = state[(state_row + i) * kDim + row] * state_scales[state_row + i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                s[i] = 0.0f;
            }
        }
        const __nv_bfloat16* v_rows = qkv + static_cast<size_t>(span.begin) * channels + (2 * kDeltaKeyHeads + head) * kDim + column;
        uint4 v_next[4] = {};
        if (quarter >= 2 && t < span.length) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v_next[i] = *(reinterpret_cast<const uint4*>(v_rows + static_cast<size_t>(t) * channels) + i);
            }
        }
        float decay_next = decays[t], end_next = decays[kBlock - 1];
        store_split(sm.s[chain], kTileBytes, row, 4 * group, s);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&sm.s_ready[chain]);
        }
        for (; n < blocks; ++n) {
            const uint32_t parity = n & 1;
            const int token = n * kBlock + t;
            const bool live = token < span.length;
            const float decay = decay_next, end = end_next;
            if (n + 1 < blocks) {
                decays += static_cast<size_t>(v_heads) * kBlock;
                decay_next = decays[t];
                end_next = decays[kBlock - 1];
            }
            if (quarter >= 2) {
                float v[32], x[32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unpack_bf16(v_next[i], v + 8 * i);
                }
                if (token + kBlock < span.length) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v_next[i] = *(reinterpret_cast<const uint4*>(v_rows + static_cast<size_t>(token + kBlock) * channels) + i);
                    }
                }
                ok = wait(&sm.d1_done[chain], parity, &sm.failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_columns(d1, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = live ? fmaf(-decay, x[i], v[i]) : 0.0f;
                }
                store_split(sm.r[chain], kRBytes / 2, t, 4 * group, x);
                fence_proxy_async();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.r_ready[chain]);
                }
                ok = wait(&sm.d2_done[chain], parity, &sm.failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                load_columns(d2, x);
                store_split(sm.r[chain], kRBytes / 2, t, 4 * group, x);
                fence_proxy_async();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.u_ready[chain]);
                }
            } else {
                ok = wait(&sm.d2_done[chain], parity, &sm.failed, status);
                if (!ok) {
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float x[32], y[32];
                load_columns(d1, x);
                load_columns(d2, y);
                if (live) {
                    uint4* to = reinterpret_cast<uint4*>(out + ((static_cast<size_t>(span.begin) + token) * v_heads + head) * kDim + column);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t words[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int e = 8 * i + 2 * j;
                            const __nv_bfloat162 pair = __floats2bfloat162_rn(fmaf(decay, x[e], y[e]), fmaf(decay, x[e + 1], y[e + 1]));
                            words[j] = *reinterpret_cast<const uint32_t*>(&pair);
                        }
                        to[i] = make_uint4(words[0], words[1], words[2], words[3]);
                    }
                }
                __syncwarp();
            }
            ok = wait(&sm.d3_done[chain], parity, &sm.failed, status);
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[32];
            load_columns(d3, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                s[i] = fmaf(end, s[i], x[i]);
            }
            if (n + 1 < blocks) {
                store_split(sm.s[chain], kTileBytes, row, 4 * group, s);
                fence_proxy_async();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.s_ready[chain]);
                }
            }
        }
        // the largest of a row of the state: over the warp's key dims, then over the quarters
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float highest;
            asm volatile("redux.sync.max.abs.f32 %0, %1, 0xffffffff;" : "=f"(highest) : "f"(s[i]));
            if (lane == i) {
                sm.peak[chain][quarter][group * 32 + i] = highest;
            }
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
        if (warp == kLoadWarp) {
            for (int i = n > 2 ? n - 2 : 0; i < n; ++i) {
                arrived(&sm.qk_full[i & 1], (i >> 1) & 1);
            }
            if (n > 0) {
                arrived(&sm.w_full, (n - 1) & 1);
            }
        } else if (warp >= kFirstMmaWarp) {
            const int chain = warp - kFirstMmaWarp;
            arrived(&sm.d1_done[chain], n & 1);
            arrived(&sm.d2_done[chain], n & 1);
            arrived(&sm.d3_done[chain], n & 1);
        }
        __syncthreads();
    } else if (warp < kFirstMmaWarp) {
        const int chain = warp / kChainWarps;
        const int quarter = warp & 3, group = (warp >> 2) & 1;
        const int row = quarter * 32 + lane;
        const size_t state_row = (static_cast<size_t>(slot) * v_heads + head) * kDim + (first_chain + chain) * kColumns + group * 32;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float* peaks = &sm.peak[chain][0][group * 32 + i];
            const float peak = fmaxf(fmaxf(peaks[0], peaks[kColumns]), fmaxf(peaks[2 * kColumns], peaks[3 * kColumns]));
            const float inverse = peak == 0.0f ? 0.0f : __fdiv_rn(127.0f, peak);
            state[(state_row + i) * kDim + row] = static_cast<int8_t>(__float2int_rn(s[i] * inverse));
            if (quarter == 0 && lane == i) {
                state_scales[state_row + i] = __fmul_rn(peak, 1.0f / 127.0f);
            }
        }
    }
    if (warp == kLoadWarp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns) : "memory");
    }
}

// RMSNorm over the 128 dims of a value head, times weight, times silu(gate): in place on the bf16 rows of the batch's
// chunks, one rounding.  Sixteen lanes to a token and head, eight dims each; a warp has eight rows in flight.
constexpr int kNormWarps = 8;
constexpr int kNormRows = 8;  // of a warp

__global__ void __launch_bounds__(kNormWarps * 32) delta_norm_rows_kernel(
    __nv_bfloat16* __restrict__ rows, const __nv_bfloat16* __restrict__ gate, const __nv_bfloat16* __restrict__ weight,
    const uint32_t* __restrict__ begins, int sequences, int tokens, int v_heads, int gate_stride, float epsilon) {
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int piece = lane & 15;
    const uint32_t first = (blockIdx.x * kNormWarps + (threadIdx.x >> 5)) * kNormRows + (lane >> 4);
    float gain[8];
    unpack_bf16(*(reinterpret_cast<const uint4*>(weight) + piece), gain);
    pdl_wait();
    const uint32_t low = __ldcg(begins), high = min(__ldcg(begins + sequences), static_cast<uint32_t>(tokens));
    uint4 raw[kNormRows / 2], gates[kNormRows / 2];
#pragma unroll
    for (int i = 0; i < kNormRows / 2; ++i) {
        const uint32_t row = first + 2 * i;
        const uint32_t token = row / v_heads, head = row % v_heads;
        raw[i] = gates[i] = make_uint4(0, 0, 0, 0);
        if (token >= low && token < high) {
            raw[i] = *(reinterpret_cast<const uint4*>(rows + static_cast<size_t>(row) * kDim) + piece);
            gates[i] = *(reinterpret_cast<const uint4*>(gate + static_cast<size_t>(token) * gate_stride + head * kDim) + piece);
        }
    }
#pragma unroll
    for (int i = 0; i < kNormRows / 2; ++i) {
        const uint32_t row = first + 2 * i;
        const uint32_t token = row / v_heads;
        float x[8], z[8];
        unpack_bf16(raw[i], x);
        unpack_bf16(gates[i], z);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = fmaf(x[j], x[j], sum);
        }
#pragma unroll
        for (int offset = 1; offset < 16; offset <<= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, offset);
        }
        const float inverse = rsqrtf(sum / static_cast<float>(kDim) + epsilon);
        uint32_t words[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] *= inverse * gain[j] * __fdividef(z[j], 1.0f + __expf(-z[j]));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            words[j] = *reinterpret_cast<const uint32_t*>(&pair);
        }
        if (token >= low && token < high) {
            *(reinterpret_cast<uint4*>(rows + static_cast<size_t>(row) * kDim) + piece) = make_uint4(words[0], words[1], words[2], words[3]);
        }
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
            found.error = cudaFuncSetAttribute(delta_chain_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(sizeof(ChainSmem<1>)) + 1024);
        }
        if (found.error == cudaSuccess) {
            found.error = cudaFuncSetAttribute(delta_chain_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(sizeof(ChainSmem<2>)) + 1024);
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
    cudaError_t launched = launch_chained(
        delta_factor_kernel, dim3(v_heads, blocks), dim3(kFactorThreads), sizeof(FactorSmem) + 1024, stream,
        static_cast<const __nv_bfloat16*>(qkv), static_cast<const float*>(alpha), static_cast<const float*>(beta),
        static_cast<const uint32_t*>(chunk_begins), images, tokens, sequences, v_heads, status);
    if (launched != cudaSuccess) {
        return launched;
    }
    // A head's two chains on an SM each as long as there are SMs for all of them.
    const bool apart = 2 * v_heads * sequences <= setup->sms;
    launched = launch_chained(
        apart ? delta_chain_kernel<1> : delta_chain_kernel<2>, dim3(apart ? 2 * v_heads : v_heads, sequences),
        dim3((apart ? kChainWarps + 2 : 2 * kChainWarps + 3) * 32),
        (apart ? sizeof(ChainSmem<1>) : sizeof(ChainSmem<2>)) + 1024, stream, static_cast<int8_t*>(state), state_scales,
        static_cast<const uint32_t*>(state_slots), static_cast<const uint32_t*>(continues),
        static_cast<const uint32_t*>(chunk_begins), static_cast<const __nv_bfloat16*>(qkv), images,
        static_cast<__nv_bfloat16*>(out), tokens, v_heads, state_capacity, status);
    if (launched != cudaSuccess || gate == nullptr) {
        return launched;
    }
    const int items = tokens * v_heads;  // at most 65536 * 48
    constexpr int kItems = kNormWarps * kNormRows;
    return launch_chained(delta_norm_rows_kernel, dim3((items + kItems - 1) / kItems), dim3(kNormWarps * 32), 0, stream,
                           static_cast<__nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(gate),
                          static_cast<const __nv_bfloat16*>(norm_weight), static_cast<const uint32_t*>(chunk_begins),
                          sequences, tokens, v_heads, gate_stride, epsilon);
}
