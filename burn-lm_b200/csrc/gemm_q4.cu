// Products with 4-bit weights: y[N, M] = x[N, K] W^T, W[m, k] = scale[m, k / group] * v, v a whole number of -8 .. 7.
//
// A scale has five significant bits, so scale * v is a bfloat16 number exactly: whichever kernel forms the product, the weights are
// the same numbers, and the only roundings are those of float32 sums (and of the result to its type).
//
// Weights are packed once, by tiles of 16 rows and 64 places of K, 512 bytes each: 16 bytes for every lane (g, t) of a warp, one word
// for each of four steps of 16 places (mma.sync.m16n8k16's K).  Lane (g, t)'s places of step s are 32 (s / 2) + 8 t + 4 (s % 2) + j,
// j = 0 .. 3, of rows g and g + 8; the nibbles of a word are, from the lowest, (g, 0) (g + 8, 0) (g, 2) (g + 8, 2) (g, 1) (g + 8, 1)
// (g, 3) (g + 8, 3): a shift and a mask by 0x000f000f leave two neighbours of one row in the two halves of a register.  A nibble
// holds v + 8.  Scales are bfloat16 [rows][groups], the groups filled up to whole stretches of 256 places.
#include "tcgen05.cuh"

BLM_API const char* blm_gemm_q4_last_error() { return g_blm_error; }

namespace q4 {

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
    int N, M, K, k_tiles, groups, group;
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
        // the stretch's scales of rows g and g + 8: one for every `group` places
        const int per = kBatch * 64 / a.group;           // 2, 4 or 8 of them
        unsigned sc[R][2][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = min((tile0 + r) * 16 + g + 8 * h, tiles * 16 - 1);
                const __nv_bfloat16* s = a.scales + (size_t)row * a.groups + kt / kBatch * per;
                if (per == 8) {
                    const uint4 v = *reinterpret_cast<const uint4*>(s);
                    sc[r][h][0] = v.x; sc[r][h][1] = v.y; sc[r][h][2] = v.z; sc[r][h][3] = v.w;
                } else if (per == 4) {                   // a scale a tile: both halves of a tile's word
                    const uint2 v = *reinterpret_cast<const uint2*>(s);
                    sc[r][h][0] = __byte_perm(v.x, 0, 0x1010); sc[r][h][1] = __byte_perm(v.x, 0, 0x3232);
                    sc[r][h][2] = __byte_perm(v.y, 0, 0x1010); sc[r][h][3] = __byte_perm(v.y, 0, 0x3232);
                } else {
                    const unsigned v = *reinterpret_cast<const unsigned*>(s);
                    sc[r][h][0] = sc[r][h][1] = __byte_perm(v, 0, 0x1010);
                    sc[r][h][2] = sc[r][h][3] = __byte_perm(v, 0, 0x3232);
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
// The tcgen05 product with the weight's rows as the 128 rows of the accumulator and N tokens (32 to 256) as its columns.  Ten warps:
// one thread fetches the tokens of 64 places of K at a time (TMA, 128-byte swizzle, zeros beyond the last token and place), one issues
// the products, and eight warps turn the weights into bfloat16 in shared memory: a lane has 16 bytes of packed weights a tile, six or
// eight tiles ahead in registers, and writes four pieces of eight places where the tensor core's swizzle wants them (a number is the
// whole number times its scale, exactly; three and a half instructions for two).  A block of 128 x 256 x 64 takes the tensor core some
// 500 cycles, and its 8,192 weights about 200 issue slots of each of the four schedulers, so that prompts are bound by the tensor cores;
// few tokens by the weights' bytes.  Where a weight has too few rows to fill the SMs, K is cut over the blocks of a cluster, whose sums
// meet in distributed shared memory, in the order of the blocks.  The eight warps read the accumulator, a lane a row: a token's results
// are written 32 rows at a time, gate and up of an output lie eight lanes apart.  Waits are bounded.
enum { Q4_TIMEOUT_PRODUCT = 53 };
constexpr int kDequantWarps = 8, kWideThreads = (2 + kDequantWarps) * 32;

struct WideArgs {
    Args a;
    int share;                   // k tiles of a block of the cluster
    int* status;
};

template <int N> struct Wide {
    static constexpr int kStages = N == 256 || N == 64 ? 4 : 5, kAhead = N <= 64 ? 6 : 8;       // (up to 64 tokens: two blocks an SM)
    static constexpr int kABytes = 128 * 128, kBBytes = N * 128, kStage = kABytes + kBBytes;
    static constexpr int kSmem = kStages * kStage + 1024 + 256;
};

template <int N>
__global__ void __launch_bounds__(kWideThreads, N <= 64 ? 2 : 1) wide_kernel(const WideArgs wa, const __grid_constant__ CUtensorMap xmap) {
    using namespace tc5;
    using W = Wide<N>;
    constexpr int S = W::kStages, kAhead = W::kAhead;
    const Args& a = wa.a;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);     // [S][weights 128 x 128 bytes, tokens N x 128 bytes]
    unsigned long long* full_x = reinterpret_cast<unsigned long long*>(ring + S * W::kStage);
    unsigned long long* full_w = full_x + S;
    unsigned long long* empty = full_w + S;
    unsigned long long* done = empty + S;
    unsigned* slot = reinterpret_cast<unsigned*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x, ranks = gridDim.x, row0 = blockIdx.y * 128, tok0 = blockIdx.z * N;
    const int kt0 = rank * wa.share, n_k = max(0, min(a.k_tiles - kt0, wa.share));          // this block's tiles of K
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_x + s, 1);
            mbar_init(full_w + s, kDequantWarps);
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

    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();                                  // the tokens are the work of the kernel before
            int i = 0;
            for (; i < n_k; ++i) {
                const int s = i % S;
                if (i >= S && !mbar_wait(empty + s, (i / S - 1) & 1)) { atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT); break; }
                mbar_expect_tx(full_x + s, W::kBBytes);
                asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                                 smem_u32(ring + s * W::kStage + W::kABytes)),
                             "l"(&xmap), "r"((kt0 + i) * 64), "r"(tok0), "r"(smem_u32(full_x + s))
                             : "memory");
            }
            for (int k = max(0, i - S); k < i; ++k) mbar_wait(full_x + k % S, (k / S) & 1);   // nothing is on its way when the block ends
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr unsigned id = instruction(N);
            bool ok = true;
            for (int i = 0; i < n_k && ok; ++i) {
                const int s = i % S;
                ok = mbar_wait(full_x + s, (i / S) & 1) && mbar_wait(full_w + s, (i / S) & 1);
                if (!ok) { atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT); break; }
                fence_after();
                const unsigned long long ad = operand(ring + s * W::kStage, 2, 1024), bd = operand(ring + s * W::kStage + W::kABytes, 2, 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma(tmem, ad + 2 * k, bd + 2 * k, id, i > 0 || k > 0);
                commit(empty + s);
            }
            commit(done);                                // when all products so far are over
        }
    } else {
        // ---- weights: this warp's tile of 16 rows ----
        const int tile = row0 / 16 + warp - 2, tiles = (a.M + 15) / 16, g = lane >> 2, t = lane & 3;
        const bool here = tile < tiles;
        const uint4* w_at = a.w + ((size_t)min(tile, tiles - 1) * a.k_tiles + kt0) * 32 + lane;
        const __nv_bfloat16* s_at = a.scales + (size_t)(min(tile, tiles - 1) * 16 + g) * a.groups;
        auto fetch = [&](int i) { return here && i < n_k ? load_once(w_at + (size_t)i * 32) : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u); };
        // the scales of a tile: of its first and its second 32 places, for row g and row g + 8 (halves of a word)
        auto scale_of = [&](int i, int h) -> unsigned {
            const int k = min(kt0 + i, a.k_tiles - 1) * 64;
            const __nv_bfloat16* s = s_at + (size_t)8 * h * a.groups;
            if (a.group == 32) return *reinterpret_cast<const unsigned*>(s + k / 32);
            const unsigned v = *reinterpret_cast<const unsigned short*>(s + k / a.group);
            return v | v << 16;
        };
        uint4 w[kAhead];
        unsigned sc[kAhead][2];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            w[j] = fetch(j);
            sc[j][0] = scale_of(j, 0);
            sc[j][1] = scale_of(j, 1);
        }
        const bool odd = g & 1;
        bool ok = true;
        for (int i0 = 0; i0 < n_k && ok; i0 += kAhead) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = i0 + j, s = i % S;
                if (i >= n_k || !ok) break;
                const uint4 now = w[j];
                const unsigned s0 = sc[j][0], s8 = sc[j][1];
                w[j] = fetch(i + kAhead);
                sc[j][0] = scale_of(i + kAhead, 0);
                sc[j][1] = scale_of(i + kAhead, 1);
                if (i >= S && !mbar_wait(empty + s, (i / S - 1) & 1)) {
                    if (lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
                    ok = false;
                    break;
                }
                unsigned char* rows = ring + s * W::kStage + ((warp - 2) * 16 + g) * 128;
                // (odd rows write their second half first: no two lanes of a phase meet in a bank)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const bool second = (x == 1) != odd;
                    const unsigned lo = second ? now.z : now.x, hi = second ? now.w : now.y;
                    const unsigned sel = second ? 0x3232u : 0x1010u;
                    const unsigned m0 = __byte_perm(s0, 0, sel), m8 = __byte_perm(s8, 0, sel);
                    auto times = [](unsigned v, unsigned m) {
                        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&m));
                        return *reinterpret_cast<const unsigned*>(&r);
                    };
                    const int chunk = ((second ? 4 + t : t) ^ g) << 4;
                    *reinterpret_cast<uint4*>(rows + chunk) = make_uint4(times(pair(lo, 0), m0), times(pair(lo, 2), m0), times(pair(hi, 0), m0), times(pair(hi, 2), m0));
                    *reinterpret_cast<uint4*>(rows + 8 * 128 + chunk) =
                        make_uint4(times(pair(lo, 1), m8), times(pair(lo, 3), m8), times(pair(hi, 1), m8), times(pair(hi, 3), m8));
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full_w + s);
            }
        }
    }

    __syncwarp();
    // ---- the sums: a lane a row, the columns of its quarter shared by two warps ----
    bool over = true;
    if (warp >= 2) {
        over = mbar_wait(done, 0);
        if (!over && lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
        fence_after();
    }
    const int quarter = warp & 3, half = (warp - 2) / 4, row = quarter * 32 + lane;        // (warps 2 .. 9: quarters 2 3 0 1 2 3 0 1)
    float* partial = reinterpret_cast<float*>(ring);     // [N][128], when the products have read the ring
    const int n_here = min(N, a.N - tok0);
    // a row's result for one token, all lanes of the warp together
    auto end = [&](float y, int tok) {
        const int m = row0 + row;
        float up = 0.f;
        if (a.end == END_GATED) up = __shfl_down_sync(0xffffffffu, y, 8);
        if (m >= a.M || tok >= n_here) return;
        int out = m;
        if (a.end == END_GATED) {
            if (lane & 8) return;
            out = m / 16 * 8 + (m & 7);
            y = y / (1.0f + __expf(-y)) * up;
        }
        const size_t to = (size_t)(tok0 + tok) * a.ldy + out;
        if (a.end == END_ADD) reinterpret_cast<float*>(a.y)[to] += y;
        else if (a.y_f32) reinterpret_cast<float*>(a.y)[to] = y;
        else reinterpret_cast<__nv_bfloat16*>(a.y)[to] = __float2bfloat16_rn(y);
    };
    if (warp >= 2) {
        pdl_wait();                                      // (what is added to, or what the kernel before still reads)
        for (int c = half * (N / 2); c < (half + 1) * (N / 2); c += 16) {
            float v[16];
            if (n_k > 0) {
                tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c, v);
                wait_ld();
            }
            if (ranks == 1) {
                if (over)
#pragma unroll
                    for (int e = 0; e < 16; ++e) end(v[e], c + e);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) partial[(c + e) * 128 + row] = n_k > 0 ? v[e] : 0.f;
            }
        }
    }
    if (ranks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (warp >= 2 && over) {
            // this block's columns of the cluster's sums
            const int each = N / ranks, c0 = rank * each;
            const unsigned mine = smem_u32(partial);
            for (int c = c0 + half; c < c0 + each; c += 2) {
                float y = 0.f;
                for (int r = 0; r < ranks; ++r) {
                    unsigned at;
                    float v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(mine + (unsigned)(c * 128 + row) * 4), "r"(r));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
                    y += v;
                }
                end(y, c);
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    if (warp == 1) tmem_free(tmem, N);
}

template <int N>
static int launch_wide(const Args& a, int* status, cudaStream_t stream) {
    using W = Wide<N>;
    CUtensorMap map;
    const long long dims[2] = {a.K, a.N}, strides[1] = {a.ldx * 2};
    const int box[2] = {64, N};
    if (!tc5::make_map<2>(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
        return blm_fail(BLM_CUDA_ERROR, "gemm_q4: no tensor map for %d tokens of %d places, rows %lld apart", a.N, a.K, a.ldx);
    // blocks of a cluster: as many as it takes to have a block for four of five SMs, each with a stretch of 256 places at least
    const int row_blocks = (a.M + 127) / 128, tok_blocks = (a.N + N - 1) / N;
    int ranks = 1;
    while (ranks < 8 && (long long)row_blocks * tok_blocks * ranks * 5 < (long long)blm_sm_count() * 4 && a.k_tiles >= ranks * 2 * kBatch) ranks *= 2;
    const WideArgs wa{a, (a.k_tiles + ranks - 1) / ranks, status};
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
    cfg.blockDim = dim3(kWideThreads);
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

BLM_API int blm_gemm_q4(const void* w, const void* scales, int groups, int group, const void* x, long long ldx, void* y, long long ldy, int y_f32,
                        int end, int n, int m, int k, int* status, cudaStream_t stream) {
    using namespace q4;
    if (n == 0 || m == 0) return BLM_OK;
    BLM_REQUIRE(group == 32 || group == 64 || group == 128, "gemm_q4: groups of %d places (32, 64 or 128)", group);
    BLM_REQUIRE(k > 0 && k % 8 == 0 && ldx % 8 == 0 && ((size_t)x & 15) == 0, "gemm_q4: rows of tokens in pieces of 16 bytes");
    BLM_REQUIRE(end != END_GATED || m % 16 == 0, "gemm_q4: gated rows come in tiles of 16, got %d", m);
    const int k_tiles = (k + 63) / 64;
    BLM_REQUIRE(groups == (k_tiles + kBatch - 1) / kBatch * (kBatch * 64 / group), "gemm_q4: %d groups a row for %d places", groups, k);
    const Args a{(const uint4*)w, (const __nv_bfloat16*)scales, (const __nv_bfloat16*)x, ldx, y, ldy, y_f32, end, n, m, k, k_tiles, groups, group};
    if (n > 16) {
        BLM_REQUIRE((m + 127) / 128 <= 65535 && (n + 255) / 256 <= 65535, "gemm_q4: %d tokens, %d rows", n, m);
        return n <= 32 ? launch_wide<32>(a, status, stream) : n <= 64 ? launch_wide<64>(a, status, stream)
               : n <= 128 ? launch_wide<128>(a, status, stream) : launch_wide<256>(a, status, stream);
    }
    if (n <= 8) launch_skinny<2, 1>(a, stream); else launch_skinny<2, 2>(a, stream);
    return blm_check_launch("gemm_q4");
}
