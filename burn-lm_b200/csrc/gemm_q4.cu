// Products with 4-bit weights: y[N, M] = x[N, K] W^T, W[m, k] = scale[m, k / group] * v, v a whole number of -8 .. 7.
//
// A scale has five significant bits, so scale * v is a bfloat16 number exactly: whichever kernel forms the product, the weights are
// the same numbers, and the only roundings are those of float32 sums (and of the result to its type).
//
// Weights are packed once, by tiles of 16 rows and 64 places of K, 512 bytes each: 16 bytes for every lane (g, t) of a warp, one word
// for each of four steps of 16 places (mma.sync.m16n8k16's K).  Lane (g, t)'s places of step s are 32 (s / 2) + 8 t + 4 (s % 2) + j,
// j = 0 .. 3, of rows g and g + 8; the nibbles of a word are, from the lowest, (g, 0) (g + 8, 0) (g, 2) (g + 8, 2) (g, 1) (g + 8, 1)
// (g, 3) (g + 8, 3): a shift and a mask by 0x000f000f leave two neighbours of one row in the two halves of a register.  A nibble
// holds v + 8.  Scales are bfloat16 [rows][one for every 32 places where groups have 32, else for every 64 (a group of 128 has its own
// twice)], filled up to whole stretches of 256 places.
#include "tcgen05.cuh"

BLM_API const char* blm_gemm_q4_last_error() { return g_blm_error; }

namespace q4 {

constexpr int kTileBytes = 512;      // of a tile of 16 rows x 64 places
constexpr int kBatch = 4;            // tiles that a warp loads together: 256 places, whole groups of any size
enum { END_STORE = 0, END_ADD = 1, END_GATED = 2 };

struct Args {
    const uint4* w;                  // [row tiles][k tiles][32]
    const __nv_bfloat16* scales;     // [row tiles * 16][groups]
    const __nv_bfloat16* x;          // [N, K], rows ldx apart
    long long ldx;
    void* y;                         // [N, M] (END_GATED: [N, M / 2]), rows ldy apart; END_ADD: float32, added to
    long long ldy;
    int y_f32, end;
    int N, M, K, k_tiles, row_scales, per_tile;      // scales of a row, and of a tile: 1 or 2
};

__device__ __forceinline__ void mma16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two whole numbers of a word: 0x43 in front of a nibble is the bfloat16 number 128 + nibble, and the nibble is v + 8.
__device__ __forceinline__ unsigned pair(unsigned word, int p) {
    const unsigned biased = ((word >> (4 * p)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), __float2bfloat162_rn(136.f));
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float bf16_of(unsigned two, int which) { return __uint_as_float(which ? two & 0xffff0000u : two << 16); }

// Few tokens: a block has R tiles of 16 rows and up to 8 NT tokens; its warps take stretches of 256 places of K in turn and meet in
// shared memory.  Bound by the weights' bytes: every lane loads R x 64 bytes of weights before it waits for anything.
constexpr int kWarps = 8;
template <int R, int NT>
__global__ void __launch_bounds__(kWarps * 32) skinny_kernel(const Args a) {
    __shared__ float sums[kWarps][R * 16][8 * NT + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int tile0 = blockIdx.x * R, n = a.N, tiles = (a.M + 15) / 16;
    pdl_launch_dependents();
    float total[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[r][i][e] = 0.f;
    bool waited = false;
    for (int kt = warp * kBatch; kt < a.k_tiles; kt += kWarps * kBatch) {
        uint4 w[R][kBatch];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                w[r][j] = tile0 + r < tiles && kt + j < a.k_tiles ? load_once(a.w + ((size_t)(tile0 + r) * a.k_tiles + kt + j) * 32 + lane)
                                                                  : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        // the stretch's scales of rows g and g + 8: of each tile's first and second 32 places
        unsigned sc[R][2][kBatch];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __nv_bfloat16* s = a.scales + (size_t)(min(tile0 + r, tiles - 1) * 16 + g + 8 * h) * a.row_scales + kt * a.per_tile;
                if (a.per_tile == 2) {
                    const uint4 v = *reinterpret_cast<const uint4*>(s);
                    sc[r][h][0] = v.x; sc[r][h][1] = v.y; sc[r][h][2] = v.z; sc[r][h][3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(s);
                    sc[r][h][0] = __byte_perm(v.x, 0, 0x1010); sc[r][h][1] = __byte_perm(v.x, 0, 0x3232);
                    sc[r][h][2] = __byte_perm(v.y, 0, 0x1010); sc[r][h][3] = __byte_perm(v.y, 0, 0x3232);
                }
            }
        if (!waited) { pdl_wait(); waited = true; }      // the tokens are the work of the kernel before
        uint4 x[kBatch][NT][2];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = (kt + j) * 64 + 32 * h + 8 * t, tok = 8 * i + g;
                    x[j][i][h] = tok < n && k < a.K ? *reinterpret_cast<const uint4*>(a.x + (size_t)tok * a.ldx + k) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float part[NT][4];
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) part[i][e] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const unsigned word = h ? (s ? w[r][j].w : w[r][j].z) : (s ? w[r][j].y : w[r][j].x);
                        const unsigned a0 = pair(word, 0), a1 = pair(word, 1), a2 = pair(word, 2), a3 = pair(word, 3);
#pragma unroll
                        for (int i = 0; i < NT; ++i) mma16(part[i], a0, a1, a2, a3, s ? x[j][i][h].z : x[j][i][h].x, s ? x[j][i][h].w : x[j][i][h].y);
                    }
                    const float s0 = bf16_of(sc[r][0][j], h), s1 = bf16_of(sc[r][1][j], h);
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        total[r][i][0] = fmaf(s0, part[i][0], total[r][i][0]);
                        total[r][i][1] = fmaf(s0, part[i][1], total[r][i][1]);
                        total[r][i][2] = fmaf(s1, part[i][2], total[r][i][2]);
                        total[r][i][3] = fmaf(s1, part[i][3], total[r][i][3]);
                    }
                }
    }
    if (!waited) pdl_wait();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[warp][r * 16 + g + 8 * (e >> 1)][8 * i + 2 * t + (e & 1)] = total[r][i][e];
    __syncthreads();
    const int rows = a.end == END_GATED ? R * 8 : R * 16, m_out = a.end == END_GATED ? a.M / 2 : a.M;
    for (int i = threadIdx.x; i < rows * n; i += kWarps * 32) {
        const int row = i % rows, tok = i / rows, out = tile0 * (a.end == END_GATED ? 8 : 16) + row;
        if (out >= m_out) continue;
        const int at = a.end == END_GATED ? (row >> 3) * 16 + (row & 7) : row;
        float y = 0.f, up = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) y += sums[k][at][tok];
        if (a.end == END_GATED) {
#pragma unroll
            for (int k = 0; k < kWarps; ++k) up += sums[k][at + 8][tok];
            y = y / (1.0f + __expf(-y)) * up;
        }
        const size_t to = (size_t)tok * a.ldy + out;
        if (a.end == END_ADD) reinterpret_cast<float*>(a.y)[to] += y;
        else if (a.y_f32) reinterpret_cast<float*>(a.y)[to] = y;
        else reinterpret_cast<__nv_bfloat16*>(a.y)[to] = __float2bfloat16_rn(y);
    }
}

template <int R, int NT>
static void launch_skinny(const Args& a, cudaStream_t stream) {
    const dim3 grid(((a.M + 15) / 16 + R - 1) / R);
    blm_launch_dependent(skinny_kernel<R, NT>, grid, dim3(kWarps * 32), 0, stream, a);
}

// ---- many tokens -----------------------------------------------------------------------------------------------------------
// The tcgen05 product with the weight's rows as the 128 rows of the accumulator and N tokens (32 to 256) as its columns.  A stage holds
// 128 places of K: one thread fetches the tokens (TMA, 128-byte swizzle, zeros beyond the last token and place), one issues the products,
// and sixteen warps turn a tile of 16 rows x 64 places each into bfloat16 in shared memory: a lane fetches its 16 bytes of packed weights
// with cp.async, kAhead stages ahead, and writes four pieces of eight places where the tensor core's swizzle wants them (a number is the
// whole number times its scale, exactly; three and a half instructions for two).  With 64 places a stage the threads' waits for one
// another, not the arithmetic, were what took the time (0.36 us a tile of 128 x 64 weights whatever the tokens).  Where a weight has too few rows to fill the SMs, K is cut
// over the blocks of a cluster.  The sums go from tensor memory to shared memory as they are, a row a lane; then each token's results
// are read, four rows a thread (from all the cluster's blocks, in their order), finished, and written as whole lines.  Waits are bounded.
enum { Q4_TIMEOUT_PRODUCT = 53 };
__host__ __device__ constexpr int rho_of(int g) { return (g & 1) << 2 | g >> 1; }         // and back: (r & 3) << 1 | r >> 2

struct WideArgs {
    Args a;
    int share;                   // k tiles of a block of the cluster, a multiple of 4 where there are several
    int vec;                     // rows of y and their beginnings allow four results at once
    int* status;
};

template <int N> struct Wide {
    static constexpr int kBlocks = N <= 64 ? 2 : 1;          // of an SM
    static constexpr int kStages = N == 128 ? 3 : 2, kAhead = N == 64 ? 1 : 3;
    static constexpr int kWidenWarps = 16, kThreads = (2 + kWidenWarps) * 32;
    static constexpr int kABytes = 128 * 128, kBBytes = N * 128;                           // of a tile of 64 places of K
    static constexpr int kStage = 2 * (kABytes + kBBytes);                                 // two: weights, weights, tokens, tokens
    static constexpr int kUnit = kTileBytes + 128;           // a warp's tile, and the scales of its pair: [16 rows][8 bytes]
    static constexpr int kSums = N * 128 * 4;
    static constexpr int kRing = kStages * kStage > kSums ? kStages * kStage : kSums;
    static constexpr int kSmem = kRing + kWidenWarps * kAhead * kUnit + 1024 + 256;
};

__device__ __forceinline__ void copy_async(unsigned dst, const void* src, int bytes) {
    if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
    else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float4 shared_of(unsigned mine, int rank) {                    // the same place in the shared memory of a block of the cluster
    unsigned at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(mine), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

template <int N>
__global__ void __launch_bounds__(Wide<N>::kThreads, Wide<N>::kBlocks) wide_kernel(const WideArgs wa, const __grid_constant__ CUtensorMap xmap) {
    using namespace tc5;
    using W = Wide<N>;
    constexpr int S = W::kStages, AHEAD = W::kAhead;
    const Args& a = wa.a;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);     // [S][weights 128 x 128 bytes, tokens N x 128 bytes]
    unsigned char* packed = ring + W::kRing;                                               // [warps][AHEAD][unit]
    unsigned long long* full = reinterpret_cast<unsigned long long*>(packed + W::kWidenWarps * AHEAD * W::kUnit);
    unsigned long long* empty = full + S;
    unsigned long long* done = empty + S;
    unsigned* slot = reinterpret_cast<unsigned*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x, ranks = gridDim.x, row0 = blockIdx.y * 128, tok0 = blockIdx.z * N;
    const int kt0 = rank * wa.share, n_k = max(0, min(a.k_tiles - kt0, wa.share));          // this block's tiles of K
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, 1 + W::kWidenWarps);     // the tokens and every warp's weights
            mbar_init(empty + s, 1);
        }
        mbar_init(done, 1);
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(slot, N);
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = *slot;
    const int pairs = (n_k + 1) / 2;

    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();                                  // the tokens are the work of the kernel before
            int i = 0;
            for (; i < pairs; ++i) {
                const int s = i % S;
                if (i >= S && !mbar_wait(empty + s, (i / S - 1) & 1)) { atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT); break; }
                const int n = min(2, n_k - 2 * i);       // (an odd last tile has no second)
                mbar_expect_tx(full + s, n * W::kBBytes);
                for (int x = 0; x < n; ++x)
                    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                                     smem_u32(ring + s * W::kStage + 2 * W::kABytes + x * W::kBBytes)),
                                 "l"(&xmap), "r"((kt0 + 2 * i + x) * 64), "r"(tok0), "r"(smem_u32(full + s))
                                 : "memory");
            }
            for (int k = max(0, i - S); k < i; ++k) mbar_wait(full + k % S, (k / S) & 1);   // nothing is on its way when the block ends
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr unsigned id = instruction(N);
            int s = 0;
            unsigned phase = 0;
            for (int i = 0; i < pairs; ++i) {
                if (!mbar_wait(full + s, phase)) { atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT); break; }
                fence_after();
                const unsigned long long ad = operand(ring + s * W::kStage, 2, 1024), bd = operand(ring + s * W::kStage + 2 * W::kABytes, 2, 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma(tmem, ad + 2 * k, bd + 2 * k, id, i > 0 || k > 0);
                if (2 * i + 1 < n_k)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma(tmem, ad + (W::kABytes >> 4) + 2 * k, bd + (W::kBBytes >> 4) + 2 * k, id, true);
                commit(empty + s);
                if (++s == S) { s = 0; phase ^= 1; }
            }
            commit(done);                                // when all products so far are over
        }
    } else {
        // ---- weights: this warp's tile of 16 rows, the first or the second of every pair of K tiles ----
        const int rows16 = (warp - 2) & 7, x = (warp - 2) >> 3;
        const int tiles = (a.M + 15) / 16, tile = min(row0 / 16 + rows16, tiles - 1), g = lane >> 2, t = lane & 3;
        const bool here = row0 / 16 + rows16 < tiles, two = a.per_tile == 2;      // (rows beyond the last tile are not written: any numbers do)
        unsigned char* mine = packed + (warp - 2) * AHEAD * W::kUnit;
        const unsigned at = smem_u32(mine);
        const uint4* w_at = a.w + ((size_t)tile * a.k_tiles + kt0 + x) * 32 + lane;
        const __nv_bfloat16* s_at = a.scales + (size_t)(tile * 16 + (lane & 15)) * a.row_scales + kt0 * a.per_tile;      // lanes 0 .. 15: a row each
        auto fetch = [&](int p, int slot_of) {
            if (here && 2 * p + x < n_k) {
                const unsigned to = at + slot_of * W::kUnit;
                copy_async(to + lane * 16, w_at + (size_t)p * 64, 16);
                if (lane < 16) copy_async(to + kTileBytes + lane * 8, s_at + p * 2 * a.per_tile, 4 * a.per_tile);
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) fetch(j, j);
        auto times = [](unsigned v, unsigned m) {
            const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&m));
            return *reinterpret_cast<const unsigned*>(&r);
        };
        // Row g of the tile becomes row rho(g) of the accumulator, so that the eight lanes of a phase (two g) meet in no bank: the swizzle
        // puts piece t of rows 0 .. 3 (mod 8) into one half of a row's 128 bytes and of rows 4 .. 7 into the other.
        const unsigned rho = rho_of(g), first_at = x * W::kABytes + ((t ^ rho) << 4) + (rows16 * 16 + rho) * 128;
        // the scale of the tile's first (second) 32 places, twice, from the pair's 4 or 8 bytes
        const unsigned sel_first = x == 1 && !two ? 0x3232u : 0x1010u, sel_second = x == 1 || two ? 0x3232u : 0x1010u;
        int s = 0, held = 0;                             // the next stage; the slot of the next tile
        unsigned parity = 1;                             // of the phase before the first: a new barrier counts as past it
        for (int p = 0; p < pairs; ++p) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(AHEAD - 1) : "memory");
            __syncwarp();                                // the scales are other lanes' copies
            const unsigned char* unit = mine + held * W::kUnit;
            const uint4 now = *reinterpret_cast<const uint4*>(unit + lane * 16);
            const unsigned s0 = *reinterpret_cast<const unsigned*>(unit + kTileBytes + g * 8 + (two ? 4 * x : 0));
            const unsigned s8 = *reinterpret_cast<const unsigned*>(unit + kTileBytes + (g + 8) * 8 + (two ? 4 * x : 0));
            __syncwarp();
            fetch(p + AHEAD, held);
            held = held + 1 == AHEAD ? 0 : held + 1;
            if (!mbar_wait(empty + s, parity)) {
                if (lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
                break;
            }
            if (2 * p + x < n_k) {
                unsigned char* stage = ring + s * W::kStage;
                auto half = [&](unsigned lo, unsigned hi, unsigned sel, unsigned at) {
                    const unsigned m0 = __byte_perm(s0, 0, sel), m8 = __byte_perm(s8, 0, sel);
                    *reinterpret_cast<uint4*>(stage + at) = make_uint4(times(pair(lo, 0), m0), times(pair(lo, 2), m0), times(pair(hi, 0), m0), times(pair(hi, 2), m0));
                    *reinterpret_cast<uint4*>(stage + at + 8 * 128) =
                        make_uint4(times(pair(lo, 1), m8), times(pair(lo, 3), m8), times(pair(hi, 1), m8), times(pair(hi, 3), m8));
                };
                half(now.x, now.y, sel_first, first_at);
                half(now.z, now.w, sel_second, first_at ^ 64u);
                fence_async_smem();
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(full + s);
            if (++s == S) { s = 0; parity ^= 1; }
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    }
    __syncwarp();

    // ---- the sums to shared memory, [N][128], when the products have read the ring: a lane a row ----
    float* sums = reinterpret_cast<float*>(ring);
    bool over = true;
    if (warp >= 2) {
        over = mbar_wait(done, 0);
        if (!over && lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
        fence_after();
        // (warps 2 .. 17: quarters 2 3 0 1 2 3 0 1 .., four warps to each)
        const int quarter = warp & 3, row = quarter * 32 + lane;
        float* to = sums + (row & ~7) + ((row & 3) << 1 | (row & 7) >> 2);       // the weight's row behind this row of the accumulator
        for (int c = (warp - 2) / 4 * 16; c < N; c += 64) {
            float v[16];
            if (n_k > 0) {
                tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c, v);
                wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) to[(c + e) * 128] = n_k > 0 ? v[e] : 0.f;
        }
    }
    fence_before();
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    else __syncthreads();

    // ---- and out: four rows of a token a thread; the tokens shared by the cluster's blocks ----
    if (warp >= 2 && over) {
        pdl_wait();                                      // (what is added to, or what the kernel before still reads)
        const bool gated = a.end == END_GATED;
        const int each = N / ranks, n_here = min(each, a.N - tok0 - rank * each), per = gated ? 16 : 32;
        const int m_out = gated ? a.M / 2 : a.M, m0 = gated ? row0 / 2 : row0;
        const unsigned base = smem_u32(sums + rank * each * 128);
        for (int i = threadIdx.x - 64; i < n_here * per; i += W::kWidenWarps * 32) {
            const int c = i / per, q = i % per, out = m0 + q * 4;
            if (out >= m_out) continue;
            const int row = gated ? q / 2 * 16 + q % 2 * 4 : q * 4;
            const unsigned place = base + (unsigned)(c * 128 + row) * 4;
            float y[4] = {0.f, 0.f, 0.f, 0.f}, up[4] = {0.f, 0.f, 0.f, 0.f};
            for (int r = 0; r < ranks; ++r) {
                const float4 v = shared_of(place, r);
                y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
                if (gated) {
                    const float4 u = shared_of(place + 32, r);
                    up[0] += u.x; up[1] += u.y; up[2] += u.z; up[3] += u.w;
                }
            }
            if (gated)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __fdividef(y[e], 1.0f + __expf(-y[e])) * up[e];
            const size_t to = (size_t)(tok0 + rank * each + c) * a.ldy + out;
            float* yf = reinterpret_cast<float*>(a.y) + to;
            __nv_bfloat16* yb = reinterpret_cast<__nv_bfloat16*>(a.y) + to;
            if (wa.vec && out + 4 <= m_out) {
                if (a.end == END_ADD) {
                    float4 v = *reinterpret_cast<float4*>(yf);
                    v.x += y[0]; v.y += y[1]; v.z += y[2]; v.w += y[3];
                    *reinterpret_cast<float4*>(yf) = v;
                } else if (a.y_f32) {
                    *reinterpret_cast<float4*>(yf) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
                    const __nv_bfloat162 l = __floats2bfloat162_rn(y[0], y[1]), h = __floats2bfloat162_rn(y[2], y[3]);
                    *reinterpret_cast<uint2*>(yb) = make_uint2(*reinterpret_cast<const unsigned*>(&l), *reinterpret_cast<const unsigned*>(&h));
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (out + e >= m_out) break;
                if (a.end == END_ADD) yf[e] += y[e];
                else if (a.y_f32) yf[e] = y[e];
                else yb[e] = __float2bfloat16_rn(y[e]);
            }
        }
    }
    __syncwarp();
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (warp == 1) {
        fence_after();
        tmem_free(tmem, N);
    }
}

template <int N>
static int launch_wide(const Args& a, int* status, cudaStream_t stream) {
    using W = Wide<N>;
    CUtensorMap map;
    const long long dims[2] = {a.K, a.N}, strides[1] = {a.ldx * 2};
    const int box[2] = {64, N};
    if (!tc5::make_map<2>(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
        return blm_fail(BLM_CUDA_ERROR, "gemm_q4: no tensor map for %d tokens of %d places, rows %lld apart", a.N, a.K, a.ldx);
    // blocks of a cluster: as many as it takes to have blocks for four of five SMs, each with a stretch of 256 places at least
    const int row_blocks = (a.M + 127) / 128, tok_blocks = (a.N + N - 1) / N;
    int ranks = 1;
    while (ranks < 8 && (long long)row_blocks * tok_blocks * ranks * 5 < (long long)blm_sm_count() * W::kBlocks * 4 && a.k_tiles >= ranks * 2 * kBatch) ranks *= 2;
    const int share = (a.k_tiles + ranks - 1) / ranks, unit = a.end == END_ADD || a.y_f32 ? 16 : 8;
    const WideArgs wa{a, ranks == 1 ? share : (share + 3) / 4 * 4, a.ldy % 4 == 0 && (size_t)a.y % unit == 0, status};
    static bool opted_in[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !opted_in[dev]) {
        if (cudaFuncSetAttribute(wide_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::kSmem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "gemm_q4: %s", cudaGetErrorString(cudaGetLastError()));
        if (dev >= 0 && dev < 64) opted_in[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, row_blocks, tok_blocks);
    cfg.blockDim = dim3(W::kThreads);
    cfg.dynamicSmemBytes = W::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, wide_kernel<N>, wa, map);
    return blm_check_launch("gemm_q4");
}
}  // namespace q4

BLM_API int blm_gemm_q4(const void* w, const void* scales, int row_scales, int group, const void* x, long long ldx, void* y, long long ldy, int y_f32,
                        int end, int n, int m, int k, int* status, cudaStream_t stream) {
    using namespace q4;
    if (n == 0 || m == 0) return BLM_OK;
    BLM_REQUIRE(group == 32 || group == 64 || group == 128, "gemm_q4: groups of %d places (32, 64 or 128)", group);
    BLM_REQUIRE(k > 0 && k % 8 == 0 && ldx % 8 == 0 && ((size_t)x & 15) == 0, "gemm_q4: rows of tokens in pieces of 16 bytes");
    BLM_REQUIRE(end != END_GATED || m % 16 == 0, "gemm_q4: gated rows come in tiles of 16, got %d", m);
    const int k_tiles = (k + 63) / 64;
    const int per_tile = group == 32 ? 2 : 1;
    BLM_REQUIRE(row_scales == (k_tiles + kBatch - 1) / kBatch * kBatch * per_tile, "gemm_q4: %d scales a row for %d places", row_scales, k);
    const Args a{(const uint4*)w, (const __nv_bfloat16*)scales, (const __nv_bfloat16*)x, ldx, y, ldy, y_f32, end, n, m, k, k_tiles, row_scales, per_tile};
    if (n > 16) {
        BLM_REQUIRE((m + 127) / 128 <= 65535 && (n + 255) / 256 <= 65535, "gemm_q4: %d tokens, %d rows", n, m);
        return n <= 32 ? launch_wide<32>(a, status, stream) : n <= 64 ? launch_wide<64>(a, status, stream)
               : n <= 128 ? launch_wide<128>(a, status, stream) : launch_wide<256>(a, status, stream);
    }
    if (n <= 8) launch_skinny<2, 1>(a, stream); else launch_skinny<2, 2>(a, stream);
    return blm_check_launch("gemm_q4");
}
