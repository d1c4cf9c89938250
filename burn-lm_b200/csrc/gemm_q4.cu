// Products with 4-bit weights: y[N, M] = x[N, K] W^T, W[m, k] = scale[m, k / group] * v, v a whole number of -8 .. 7.
//
// A scale has five significant bits, so scale * v is a bfloat16 number exactly: whichever kernel forms the product, the weights are
// the same numbers, and the only roundings are those of float32 sums (and of the result to its type).
//
// Weights are packed once, by tiles of 16 rows and stretches of 256 places of K (four tiles of 64), 512 bytes a tile: 16 bytes for every
// lane (g, t) of a warp, one word for each of four steps of 16 places (mma.sync.m16n8k16's K).  Lane (g, t)'s places of step s are
// 32 (s / 2) + 8 t + 4 (s % 2) + j, j = 0 .. 3, of rows g and g + 8; the nibbles of a word are, from the lowest, (g, 0) (g + 8, 0) (g, 2)
// (g + 8, 2) (g, 1) (g + 8, 1) (g, 3) (g + 8, 3): a shift and a mask by 0x000f000f leave two neighbours of one row in the two halves of
// a register.  A nibble holds v + 8.  Behind a stretch's four tiles stand its scales, bfloat16 [16 rows][4], one for every 64 places (a
// group of 128 has its own twice), or [16 rows][8] where groups have 32: one copy of 2,176 or 2,304 bytes brings all that a warp needs.
#include "cluster.cuh"
#include "tcgen05.cuh"

BLM_API const char* blm_gemm_q4_last_error() { return g_blm_error; }

namespace q4 {

constexpr int kTileBytes = 512;      // of a tile of 16 rows x 64 places
constexpr int kBatch = 4;            // tiles that a warp loads together: 256 places, whole groups of any size
enum { END_STORE = 0, END_ADD = 1, END_GATED = 2 };

struct Args {
    const unsigned char* w;          // [row tiles][stretches][unit]
    const __nv_bfloat16* x;          // [N, K], rows ldx apart
    long long ldx;
    void* y;                         // [N, M] (END_GATED: [N, M / 2]), rows ldy apart; END_ADD: float32, added to
    long long ldy;
    int y_f32, end;
    int N, M, K, k_tiles, stretches, unit, per_tile; // bytes of a stretch of a tile of rows; scales of a tile of 64 places: 1 or 2
};

__device__ __forceinline__ void mma16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16_onto(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// Two whole numbers of a word times their scale, exactly, where a rotation to the right by `by` brings the nibbles to bits 3 .. 6 of the
// halves: behind the bits of 16 they are the bfloat16 numbers 16 + v + 8, and 24 times the scale, which is taken off their product,
// has seven bits.  (At bits 0 .. 3 it would be 136 times, ten bits, and take a subtraction and a product.)
__device__ __forceinline__ unsigned scaled_two(unsigned word, int by, __nv_bfloat162 scale, __nv_bfloat162 less) {
    const unsigned biased = (__funnelshift_r(word, word, by) & 0x00780078u) | 0x41804180u;
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&biased), scale, less);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float bf16_of(unsigned two, int which) { return __uint_as_float(which ? two & 0xffff0000u : two << 16); }

// ---- few tokens ------------------------------------------------------------------------------------------------------------
// Up to 8 tokens.  A cluster's blocks cut K into chunks of 2,048 places, a block's eight warps a
// chunk into stretches of 256, so that a warp meets the same tokens for every row: their fragments stay in its registers, and it does
// nothing but stream its places of one tile of 16 rows after the other, AHEAD tiles ahead.  What bounds it beside the weights' bytes is
// the instructions that make operands of them, so they are used as they are: sixteen bits that hold a whole number n below 256 are the
// bfloat16 number n 2^-133 (below 2^-126, and still with that step in the next binade), so a mask by 0x000f000f or 0x00f000f0 and one
// shift of a word by eight bits give all of its weights, of rows g as n = v + 8, of rows g + 8 as 16 (v + 8).  The tokens are multiplied by
// a power of two that brings the largest of a warp's stretch to 2^120 (exactly: bfloat16 has the exponents for it), so that products and
// sums are of ordinary size.  The 8 is not taken off the weights: a part's sum starts at -8 (-128) times the sum of its tokens' places,
// formed by the tensor cores, once.  A part's scale multiplies its sum.  The warps' sums meet in shared memory, the cluster's blocks in
// distributed shared memory, in a fixed order.
constexpr int kWarps = 8, kChunk = kWarps * kBatch;      // k tiles of a block
enum { Q4_TIMEOUT_WEIGHTS = 54 };
struct Few {
    static constexpr int kAhead = 3, kBlocks = 2;                                  // tiles of rows on their way a warp; blocks of an SM
    static constexpr int kUnit = kBatch * kTileBytes + 256;                        // room for a stretch of a tile of rows
    static constexpr int kSlots = 12;                                              // tiles of rows between two meetings
    static constexpr int kSums = 16 * 8;                                           // of a tile: [16 rows][8 tokens]
    static constexpr int kSmem = kWarps * kAhead * kUnit + kSlots * (kWarps + 1) * kSums * 4 + kWarps * kAhead * 8;
};

struct FewArgs {
    Args a;
    int chunks, clusters;        // blocks of a cluster, clusters
    int* status;
};

// An infinity or a NaN among a token's numbers makes all its sums none in the kernel (n = v + 8 times it, and -8 times it).  What they are is the sum
// of weight times such a number, none where the weight is zero: for a row of a tile and the row 8 behind it, from memory, and seldom.
template <bool TWO>
__device__ __noinline__ float2 odd_sums(const unsigned char* w, const __nv_bfloat16* x, int K, int stretches, int unit_bytes, int tile, int row, float y, float behind) {
    bool any = false;
    float sum[2] = {0.f, 0.f};
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
        const float v = __bfloat162float(x[k]);
        if (fabsf(v) < INFINITY) continue;
        any = true;
        const unsigned char* unit = w + ((size_t)tile * stretches + k / 256) * unit_bytes;
        const int j = k / 64 % 4, h = k / 32 % 2, at = TWO ? 2 * j + h : j;
        const unsigned word = *reinterpret_cast<const unsigned*>(unit + j * kTileBytes + ((row & 7) * 4 + k / 8 % 4) * 16 + (2 * h + k / 4 % 2) * 4);
        const unsigned two = word >> (16 * (k & 1) + 8 * (k >> 1 & 1));
        const __nv_bfloat16* scales = reinterpret_cast<const __nv_bfloat16*>(unit + kBatch * kTileBytes) + (row & 7) * (TWO ? 8 : 4) + at;
        sum[0] += (float)((int)(two & 15) - 8) * __bfloat162float(scales[0]) * v;
        sum[1] += (float)((int)(two >> 4 & 15) - 8) * __bfloat162float(scales[8 * (TWO ? 8 : 4)]) * v;
    }
    if (any) {
        y = row < 8 ? sum[0] : sum[1];
        behind = sum[1];
    }
    return make_float2(y, behind);
}

template <bool TWO>
__global__ void __launch_bounds__(kWarps * 32, Few::kBlocks) few_kernel(const FewArgs fa) {
    using F = Few;
    constexpr int AHEAD = F::kAhead, PARTS = TWO ? 2 : 1;                          // parts of a tile with a scale of their own
    const Args& a = fa.a;
    extern __shared__ __align__(128) unsigned char smem_few[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem_few + warp * AHEAD * F::kUnit;                      // this warp's units
    float* partial = reinterpret_cast<float*>(smem_few + kWarps * AHEAD * F::kUnit);       // [slots][warps][16][8], then [slots][16][8]
    float* sums = partial + F::kSlots * kWarps * F::kSums;
    unsigned long long* full = reinterpret_cast<unsigned long long*>(sums + F::kSlots * F::kSums) + warp * AHEAD;
    const int rank = blockIdx.x % fa.chunks, cluster = blockIdx.x / fa.chunks, n = a.N;
    const int stretch = rank * kWarps + warp, kt = stretch * kBatch, tiles = (a.M + 15) / 16;
    const int t_lo = (int)((long long)tiles * cluster / fa.clusters), t_hi = (int)((long long)tiles * (cluster + 1) / fa.clusters);
    const bool here = stretch < a.stretches;
    const int total_units = here ? t_hi - t_lo : 0;
    pdl_launch_dependents();
    // the weights, AHEAD units ahead: one lane copies
    const unsigned char* w_at = a.w + ((size_t)t_lo * a.stretches + (here ? stretch : 0)) * a.unit;
    const size_t w_step = (size_t)a.stretches * a.unit;
    auto fetch = [&](int slot) {
        tc5::mbar_expect_tx(full + slot, a.unit);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(ring + slot * F::kUnit)),
                     "l"(w_at), "r"(a.unit), "r"(smem_u32(full + slot))
                     : "memory");
        w_at += w_step;
    };
    if (lane == 0) {
        for (int j = 0; j < AHEAD; ++j) tc5::mbar_init(full + j, 1);
        tc5::mbar_init_fence();
        for (int j = 0; j < AHEAD && j < total_units; ++j) fetch(j);
    }
    __syncwarp();
    pdl_wait();                                          // the tokens are the work of the kernel before
    uint4 x[kBatch][2];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
        for (int h = 0; h < 2; ++h) {
            const int k = (kt + j) * 64 + 32 * h + 8 * t;
            x[j][h] = g < n && k < a.K ? *reinterpret_cast<const uint4*>(a.x + (size_t)g * a.ldx + k) : make_uint4(0u, 0u, 0u, 0u);
        }
    // times a power of two: the largest of this stretch to 2^120 (zeros as they are; infinities and NaN too, whose sums odd_sums puts right)
    float back[2];                                   // of tokens 2 t and 2 t + 1: what takes that and the weights' 2^-133 off again, over 2^40
    {
        unsigned top = 0;                                // of two magnitudes' bits at once
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 v = x[j][h];
                top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu));
            }
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(max(top & 0xffffu, top >> 16) >> 7);                  // the largest exponent, 127 too large
        const int by = e == 0 || e == 255 ? 0 : min(127, 247 - e);                // (-7 at least)
        const unsigned factor = (unsigned)(127 + by) << 7, both = factor << 16 | factor;
        auto times = [&](unsigned v) {
            const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&both));
            return *reinterpret_cast<const unsigned*>(&r);
        };
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4& v = x[j][h];
                v = make_uint4(times(v.x), times(v.y), times(v.z), times(v.w));
            }
        // 2^(133 - 40 - by), of token g: sums with scales of up to 2^80 stay floats times the 2^40, those of 2^-110 times the rest of it
        const float mine = __uint_as_float((unsigned)(127 + 93 - by) << 23);
        back[0] = __shfl_sync(0xffffffffu, mine, 8 * t);
        back[1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
    }
    // where a part's sum starts: -8 times the sum of its places for row g, -128 times for row g + 8
    float start[kBatch][PARTS][4];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float (&d)[4] = start[j][TWO ? h : 0];
            if (TWO || h == 0) d[0] = d[1] = d[2] = d[3] = 0.f;
            constexpr unsigned k8 = 0x80088008u, k128 = 0x80808080u;
            mma16(d, k8, k128, k8, k128, x[j][h].x, x[j][h].y);
            mma16(d, k8, k128, k8, k128, x[j][h].z, x[j][h].w);
        }

    const int m_out = a.end == END_GATED ? a.M / 2 : a.M, rows = a.end == END_GATED ? 8 : 16;
    int unit = 0, slot = 0;                              // the next of this warp's, and where it lies
    unsigned phase = 0;
    bool ok = true;
    for (int b0 = t_lo; b0 < t_hi; b0 += F::kSlots) {
        const int count = min(F::kSlots, t_hi - b0);
        float* to = partial + warp * F::kSums + g * 8 + 2 * t;
#pragma unroll 1
        for (int r = 0; r < count; ++r, to += kWarps * F::kSums) {
            float total[4] = {0.f, 0.f, 0.f, 0.f};
            if (here && ok) {
                if (!tc5::mbar_wait(full + slot, phase)) {
                    if (lane == 0) atomicCAS(fa.status, 0, Q4_TIMEOUT_WEIGHTS);
                    ok = false;
                }
                const unsigned char* at_unit = ring + slot * F::kUnit;
                uint4 w[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) w[j] = *reinterpret_cast<const uint4*>(at_unit + j * kTileBytes + lane * 16);
                unsigned sc[2][2 * PARTS];               // rows g and g + 8: the stretch's 4 or 8 scales
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned char* s = at_unit + kBatch * kTileBytes + (g + 8 * h) * (TWO ? 16 : 8);
                    if (TWO) {
                        const uint4 v = *reinterpret_cast<const uint4*>(s);
                        sc[h][0] = v.x; sc[h][1] = v.y; sc[h][2 * PARTS - 2] = v.z; sc[h][2 * PARTS - 1] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(s);
                        sc[h][0] = v.x; sc[h][1] = v.y;
                    }
                }
                __syncwarp();                            // the unit is in registers
                ++unit;
                if (lane == 0 && unit + AHEAD <= total_units && ok) fetch(slot);
                if (++slot == AHEAD) { slot = 0; phase ^= 1; }
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        float part[4];
#pragma unroll
                        for (int q = 0; q < 4 / PARTS; ++q) {
                            const int s = p * 2 + q;
                            const unsigned lo = s == 0 ? w[j].x : s == 1 ? w[j].y : s == 2 ? w[j].z : w[j].w, hi = lo >> 8;
                            const unsigned a0 = lo & 0x000f000fu, a1 = lo & 0x00f000f0u, a2 = hi & 0x000f000fu, a3 = hi & 0x00f000f0u;
                            const uint4& v = x[j][s >> 1];
                            mma16_onto(part, a0, a1, a2, a3, s & 1 ? v.z : v.x, s & 1 ? v.w : v.y, q == 0 ? start[j][p] : part);
                        }
                        const int at = j * PARTS + p;    // of the stretch's scales
                        const float m0 = bf16_of(sc[0][at >> 1], at & 1), m8 = bf16_of(sc[1][at >> 1], at & 1);
                        total[0] = fmaf(m0, part[0], total[0]);
                        total[1] = fmaf(m0, part[1], total[1]);
                        total[2] = fmaf(m8, part[2], total[2]);
                        total[3] = fmaf(m8, part[3], total[3]);
                    }
            }
            *reinterpret_cast<float2*>(to) = make_float2(total[0] * 0x1p40f * back[0], total[1] * 0x1p40f * back[1]);
            *reinterpret_cast<float2*>(to + 8 * 8) = make_float2(total[2] * 0x1p36f * back[0], total[3] * 0x1p36f * back[1]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count * F::kSums; i += kWarps * 32) {
            const float* from = partial + i / F::kSums * kWarps * F::kSums + i % F::kSums;
            float y = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) y += from[k * F::kSums];
            sums[i] = y;
        }
        if (fa.chunks > 1) cluster_sync();
        else __syncthreads();
        // out: the cluster's blocks take tiles in turn
        const unsigned base = smem_u32(sums);
        const int mine = (count - rank + fa.chunks - 1) / fa.chunks;
        for (int i = threadIdx.x; i < mine * rows * n; i += kWarps * 32) {
            const int row = i % rows, tok = i / rows % n, slot = i / (rows * n) * fa.chunks + rank, out = (b0 + slot) * rows + row;
            if (out >= m_out) continue;
            const unsigned at = base + (unsigned)((slot * 16 + row) * 8 + tok) * 4;
            float y = 0.f, up = 0.f;
            for (int r = 0; r < fa.chunks; ++r) {
                y += cluster_float(at, r);
                if (a.end == END_GATED) up += cluster_float(at + 8 * 8 * 4, r);
            }
            if (__builtin_expect(!(fabsf(y) < INFINITY && fabsf(up) < INFINITY), 0)) {
                const float2 both = odd_sums<TWO>(a.w, a.x + (size_t)tok * a.ldx, a.K, a.stretches, a.unit, b0 + slot, row, y, up);
                y = both.x;
                up = both.y;
            }
            if (a.end == END_GATED) y = y / (1.0f + __expf(-y)) * up;
            const size_t to = (size_t)tok * a.ldy + out;
            if (a.end == END_ADD) reinterpret_cast<float*>(a.y)[to] += y;
            else if (a.y_f32) reinterpret_cast<float*>(a.y)[to] = y;
            else reinterpret_cast<__nv_bfloat16*>(a.y)[to] = __float2bfloat16_rn(y);
        }
        // nobody writes sums again while another block reads them, nor leaves
        if (fa.chunks > 1) cluster_sync();
        else if (b0 + F::kSlots < t_hi) __syncthreads();
    }
    // (a wait that ran out: what is still on its way lands before the block ends)
    if (!ok && lane == 0)
        for (int j = 0; j < AHEAD && unit + j < total_units; ++j) tc5::mbar_wait(full + (slot + j) % AHEAD, slot + j < AHEAD ? phase : phase ^ 1);
}

// Which kernel: up to 8 tokens the one for few, as far as a cluster of eight blocks reaches (16,384 places).  Measured, 1 and 8 tokens
// against the other kernel: 2,048 x 2,048 3.1 and 3.3 us against 4.0 and 4.2; 6,144 x 4,096 6.7 and 7.6 against 8.2 and 8.5; 28,672 x 4,096
// 16.5 and 18.5 against 28 and 27; 4,096 x 14,336 11.5 and 12.8 against 14.7 and 15.0.  (With two products a piece of weights for 16
// tokens: 3.9, 10.6, 30 and 23 against 4.4, 8.7, 27 and 15.3.)
static bool few_take(int n, int k_tiles) { return n <= 8 && k_tiles <= 8 * kChunk; }

template <bool TWO>
static int launch_few(const Args& a, int* status, cudaStream_t stream) {
    using F = Few;
    FewArgs fa{a, (a.stretches + kWarps - 1) / kWarps, 0, status};
    const int tiles = (a.M + 15) / 16;
    static bool opted_in[64] = {};
    static int resident[64][9] = {};                     // clusters of so many blocks that the device holds at once
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return blm_fail(BLM_CUDA_ERROR, "gemm_q4: device %d", dev);
    if (!opted_in[dev]) {
        if (cudaFuncSetAttribute(few_kernel<TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "gemm_q4: %s", cudaGetErrorString(cudaGetLastError()));
        opted_in[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = fa.chunks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = fa.chunks > 1 ? 2 : 1;
    if (resident[dev][fa.chunks] == 0) {
        // (a cluster lies in one group of SMs, which a number of blocks need not divide)
        int fit = blm_sm_count() * F::kBlocks;
        cfg.gridDim = dim3(fa.chunks);
        if (fa.chunks > 1 && (cudaOccupancyMaxActiveClusters(&fit, few_kernel<TWO>, &cfg) != cudaSuccess || fit < 1)) {
            cudaGetLastError();
            fit = blm_sm_count() * F::kBlocks / (2 * fa.chunks);
        }
        resident[dev][fa.chunks] = fit < 1 ? 1 : fit;
    }
    fa.clusters = resident[dev][fa.chunks];
    if (fa.clusters > tiles) fa.clusters = tiles;
    if (fa.clusters < 1) fa.clusters = 1;
    cfg.gridDim = dim3(fa.chunks * fa.clusters);
    cudaLaunchKernelEx(&cfg, few_kernel<TWO>, fa);
    return blm_check_launch("gemm_q4");
}

// ---- many tokens -----------------------------------------------------------------------------------------------------------
// The tcgen05 product with the weight's rows as the 128 rows of the accumulator and N tokens (32 to 256) as its columns.  A stage holds
// 64 places of K: one thread fetches the tokens (TMA, 128-byte swizzle, zeros beyond the last token and place), one warp issues the
// products, and the other warps turn weights into bfloat16 in tensor memory, a row a lane, each group of four warps every kGroups-th tile
// of K: a lane copies 16 bytes of each of the warp's two tiles of rows, kAhead tiles ahead (cp.async), reads its row's four pieces (which
// hold row g + 8 too), and makes two numbers in three instructions, each the whole number times its scale, exactly.  (Weights in shared
// memory instead, written and then read by the products beside 256 tokens, took 100 KB of its traffic a tile, 780 cycles for 512 of the
// tensor core's.)  Where a weight has too few rows to fill the SMs, K is cut over the blocks of a cluster.  The sums go from tensor memory
// to shared memory as they are, a row a lane; then each token's results are read, four rows a thread (from all the cluster's blocks, in
// their order), finished, and written as whole lines.  Waits are bounded.
// Measured, with groups of 64: 512 tokens by 28,672 x 4,096 93 to 96 us (1,250 to 1,296 TFLOP/s), 2,048 by 16,384 x 2,048 117 us (1,180), 64 by
// 28,672 x 4,096 30 us (2.2 TB/s of weights).  A tile of K with 256 tokens takes 0.34 us for 0.28 of products, a block's beginning and end
// 7 us, which nothing hides; with few tokens it is the widening, 0.2 us a tile of 128 x 64 weights.
enum { Q4_TIMEOUT_PRODUCT = 53 };

// A grid that fills the SMs some times and leaves a few blocks is two launches: WAVES, whole times, then the REST with K cut over clusters.
// The rest may run beside the last of the others: what both read is ready once WAVES has waited for the kernel before it, so that is when it
// lets the rest begin, and the rest waits for WAVES at its end only (so that what follows waits for both).
enum { ALONE = 0, WAVES = 1, REST = 2 };
struct WideArgs {
    Args a;
    int share;                   // k tiles of a block of the cluster, whole stretches
    int vec;                     // rows of y and their beginnings allow four results at once
    int ranks;                   // blocks of a cluster
    int first, tok_blocks, part; // this launch's first block of rows and tokens (tokens first), blocks of tokens; ALONE, WAVES or REST
    int* status;
};

template <int N> struct Wide {
    static constexpr int kBlocks = N <= 128 ? 2 : 1;         // of an SM (128 tokens by 28,672 x 4,096: 36 us with two, 52 with one of 18 warps)
    static constexpr int kStages = N == 256 ? 5 : N == 128 ? 4 : N == 64 ? 6 : 7;
    static constexpr int kGroups = N <= 128 ? 2 : 4, kThreads = (2 + 4 * kGroups) * 32;
    static constexpr int kCols = N <= 128 ? 256 : 512;       // of tensor memory: N of sums, 32 a stage of weights
    static constexpr int kStage = N * 128;                   // bytes of the tokens of a tile of 64 places
    static constexpr int kSums = N * 128 * 4;
    static constexpr int kRing = kStages * kStage > kSums ? kStages * kStage : kSums;
    static constexpr int kAhead = N == 256 ? 3 : N == 128 ? 4 : 6;               // packed tiles of a warp on their way
    static constexpr int kUnit = 2 * kTileBytes + 128;       // two tiles of 16 rows, a scale (two, where groups have 32) a row
    static constexpr int kSmem = kRing + 4 * kGroups * kAhead * kUnit + 1024 + 256;
    static_assert(N + 32 * kStages <= kCols && kBlocks * kCols <= 512, "tensor memory");
};

__device__ __forceinline__ void copy_async16(unsigned to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy_async4(unsigned to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(from) : "memory"); }

template <int N>
__global__ void __launch_bounds__(Wide<N>::kThreads, Wide<N>::kBlocks) wide_kernel(const WideArgs wa, const __grid_constant__ CUtensorMap xmap) {
    using namespace tc5;
    using tc5::smem_u32;
    using W = Wide<N>;
    constexpr int S = W::kStages, KG = W::kGroups;
    const Args& a = wa.a;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);     // [S][N tokens x 128 bytes]
    unsigned char* packed = ring + W::kRing;                                               // [warps][kAhead][unit]
    unsigned long long* full = reinterpret_cast<unsigned long long*>(packed + 4 * KG * W::kAhead * W::kUnit);
    unsigned long long* empty = full + S;
    unsigned long long* done = empty + S;
    unsigned* slot = reinterpret_cast<unsigned*>(done + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int ranks = wa.ranks, rank = blockIdx.x % ranks, block = wa.first + blockIdx.x / ranks, row0 = block / wa.tok_blocks * 128, tok0 = block % wa.tok_blocks * N;
    const int kt0 = rank * wa.share, n_k = max(0, min(a.k_tiles - kt0, wa.share));          // this block's tiles of K
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, 1 + 4);                  // the tokens and four warps' weights
            mbar_init(empty + s, 1);
        }
        mbar_init(done, 1);
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(slot, W::kCols);
    fence_before();
    __syncthreads();
    fence_after();
    if (wa.part != WAVES) pdl_launch_dependents();        // (not before this block has its tensor memory: the next kernel may take some too)
    const unsigned tmem = __shfl_sync(0xffffffffu, *slot, 0);

    if (warp == 0) {
        if (lane == 0) {
            if (wa.part != REST) pdl_wait();             // the tokens are the work of the kernel before
            if (wa.part == WAVES) pdl_launch_dependents();
            int i = 0;
            for (; i < n_k; ++i) {
                const int s = i % S;
                if (i >= S && !mbar_wait(empty + s, (i / S - 1) & 1)) { atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT); break; }
                mbar_expect_tx(full + s, W::kStage);
                asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
                                 smem_u32(ring + s * W::kStage)),
                             "l"(&xmap), "r"((kt0 + i) * 64), "r"(tok0), "r"(smem_u32(full + s))
                             : "memory");
            }
            for (int k = max(0, i - S); k < i; ++k) mbar_wait(full + k % S, (k / S) & 1);   // nothing is on its way when the block ends
        }
    } else if (warp == 1) {
        // (the whole warp, so that what a product is issued with is known to be one number for all its lanes: behind `lane == 0` the
        // issue of a product took 65 cycles and a wait 400)
        constexpr unsigned id = instruction(N);
        int s = 0;
        unsigned phase = 0;
        for (int i = 0; i < n_k; ++i) {
            if (!mbar_wait(full + s, phase)) {
                if (lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
                break;
            }
            fence_after();
            if (elect()) {
                const unsigned long long bd = operand(ring + s * W::kStage, 2, 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_ts(tmem, tmem + N + s * 32 + 8 * k, bd + 2 * k, id, i > 0 || k > 0);
                commit(empty + s);
            }
            __syncwarp();
            if (++s == S) { s = 0; phase ^= 1; }
        }
        if (elect()) commit(done);                       // when all products so far are over
    } else {
        // ---- weights: the quarter of the rows that the warp's lanes of tensor memory are, a row a lane ----
        const int quarter = warp & 3, first = (warp - 2) / 4, row = row0 + quarter * 32 + lane, tiles = (a.M + 15) / 16;
        const int g = lane & 7;                          // (rows beyond the last tile are not written: any numbers do)
        const int by0 = lane & 8 ? 1 : 29, by2 = lane & 8 ? 9 : 5;                          // (of a byte's two nibbles the second is row g + 8's)
        const int tile_lo = min((row - lane) >> 4, tiles - 1), tile_hi = min(((row - lane) >> 4) + 1, tiles - 1);      // the warp's two
        const size_t lo = ((size_t)tile_lo * a.stretches + kt0 / kBatch) * a.unit, hi = ((size_t)tile_hi * a.stretches + kt0 / kBatch) * a.unit;
        const unsigned char* mine = packed + (warp - 2) * W::kAhead * W::kUnit;
        // a lane brings piece (g, t) of both tiles and its row's scale; pieces stand at t ^ (g / 2), so that eight rows' meet in no bank
        const unsigned put = smem_u32(mine) + ((lane & ~3) + ((lane & 3) ^ (lane >> 3))) * 16;
        auto fetch = [&](int kt, int at) {
            if (kt < n_k) {
                const unsigned char* from = a.w + (size_t)(kt / kBatch) * a.unit + kt % kBatch * kTileBytes + lane * 16;
                copy_async16(put + at * W::kUnit, from + lo);
                copy_async16(put + at * W::kUnit + kTileBytes, from + hi);
                copy_async4(smem_u32(mine) + at * W::kUnit + 2 * kTileBytes + lane * 4,
                            a.w + (lane < 16 ? lo : hi) + (size_t)(kt / kBatch) * a.unit + kBatch * kTileBytes +
                                ((lane & 15) * 2 * a.per_tile + (a.per_tile == 2 ? kt % kBatch : kt % kBatch / 2)) * 4);
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
        for (int i = 0; i < W::kAhead; ++i) fetch(first + i * KG, i);
        for (int kt = first, held = 0; kt < n_k; kt += KG) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(W::kAhead - 1) : "memory");
            __syncwarp();                                // the pieces are other lanes' copies
            const unsigned char* unit = mine + held * W::kUnit;
            uint4 now[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) now[t] = *reinterpret_cast<const uint4*>(unit + (lane >> 4) * kTileBytes + (4 * g + (t ^ (g >> 1))) * 16);
            unsigned scales = *reinterpret_cast<const unsigned*>(unit + 2 * kTileBytes + lane * 4);
            if (a.per_tile == 1) scales = __byte_perm(scales, 0, kt & 1 ? 0x3232 : 0x1010);
            __syncwarp();
            fetch(kt + W::kAhead * KG, held);
            held = held + 1 == W::kAhead ? 0 : held + 1;
            unsigned w[2][16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned both = __byte_perm(scales, 0, h == 0 ? 0x1010 : 0x3232);
                const __nv_bfloat162 scale = *reinterpret_cast<const __nv_bfloat162*>(&both), less = __hmul2(scale, __float2bfloat162_rn(-24.f));
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned word = h == 0 ? (e == 0 ? now[t].x : now[t].y) : (e == 0 ? now[t].z : now[t].w);
                        w[h][4 * t + 2 * e] = scaled_two(word, by0, scale, less);
                        w[h][4 * t + 2 * e + 1] = scaled_two(word, by2, scale, less);
                    }
            }
            const int s = kt % S;
            if (kt >= S && !mbar_wait(empty + s, (kt / S - 1) & 1)) {
                if (lane == 0) atomicCAS(wa.status, 0, Q4_TIMEOUT_PRODUCT);
                break;
            }
            fence_after();
            const unsigned to = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(N + s * 32);
            tmem_st16(to, w[0]);
            tmem_st16(to + 16, w[1]);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + s);
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
        // (warps 2 and up: quarters 2 3 0 1 2 3 0 1 .., kGroups warps to each)
        const int quarter = warp & 3;
        float* to = sums + quarter * 32 + lane;
        for (int c = (warp - 2) / 4 * 16; c < N; c += KG * 16) {
            float v[16];
            if (n_k > 0) {
                tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c, v);
                wait_ld(v);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) to[(c + e) * 128] = n_k > 0 ? v[e] : 0.f;
        }
    }
    fence_before();
    if (ranks > 1) cluster_sync();
    else __syncthreads();

    // ---- and out: four rows of a token a thread; the tokens shared by the cluster's blocks ----
    if (warp >= 2 && over) {
        if (wa.part != REST) pdl_wait();                 // (what is added to, or what the kernel before still reads)
        const bool gated = a.end == END_GATED;
        const int each = N / ranks, n_here = min(each, a.N - tok0 - rank * each), at_once = gated ? 4 : 5;        // (log2 of a token's threads)
        const int m_out = gated ? a.M / 2 : a.M, m0 = gated ? row0 / 2 : row0;
        // a thread has the same rows of every token it finishes, so that a token costs few instructions beside its reads and its write:
        // places worked out anew for each took 6.5 us of a block of 256 tokens
        const int i = threadIdx.x - 64, q = i & ((1 << at_once) - 1), out = m0 + q * 4, step = KG * 128 >> at_once;
        const int rows = min(4, m_out - out);
        const float* from = sums + rank * each * 128 + (gated ? q / 2 * 16 + q % 2 * 4 : q * 4);
        auto sum_of = [&](const float* mine) {
            if (ranks == 1) return *reinterpret_cast<const float4*>(mine);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < ranks; ++r) {
                const float4 x = cluster_float4(smem_u32(mine), r);
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
            return v;
        };
        if (rows > 0)
#pragma unroll 4
            for (int c = i >> at_once; c < n_here; c += step) {
                const size_t to = (size_t)(tok0 + rank * each + c) * a.ldy + out;
                float* yf = reinterpret_cast<float*>(a.y) + to;
                __nv_bfloat16* yb = reinterpret_cast<__nv_bfloat16*>(a.y) + to;
                float4 y = sum_of(from + c * 128);
                if (gated) {
                    const float4 up = sum_of(from + c * 128 + 8);
                    y.x = __fdividef(y.x, 1.0f + __expf(-y.x)) * up.x;
                    y.y = __fdividef(y.y, 1.0f + __expf(-y.y)) * up.y;
                    y.z = __fdividef(y.z, 1.0f + __expf(-y.z)) * up.z;
                    y.w = __fdividef(y.w, 1.0f + __expf(-y.w)) * up.w;
                }
                if (wa.vec && rows == 4) {
                    if (a.end == END_ADD) {
                        const float4 v = *reinterpret_cast<const float4*>(yf);
                        y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
                    }
                    if (a.y_f32) *reinterpret_cast<float4*>(yf) = y;
                    else {
                        const __nv_bfloat162 l = __floats2bfloat162_rn(y.x, y.y), h = __floats2bfloat162_rn(y.z, y.w);
                        *reinterpret_cast<uint2*>(yb) = make_uint2(*reinterpret_cast<const unsigned*>(&l), *reinterpret_cast<const unsigned*>(&h));
                    }
                    continue;
                }
                const float one[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e >= rows) break;
                    if (a.end == END_ADD) yf[e] += one[e];
                    else if (a.y_f32) yf[e] = one[e];
                    else yb[e] = __float2bfloat16_rn(one[e]);
                }
            }
    }
    __syncwarp();
    if (wa.part == REST) pdl_wait();
    if (ranks > 1) cluster_sync();
    if (warp == 1) {
        fence_after();
        tmem_free(tmem, W::kCols);
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
    static bool opted_in[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !opted_in[dev]) {
        if (cudaFuncSetAttribute(wide_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::kSmem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "gemm_q4: %s", cudaGetErrorString(cudaGetLastError()));
        if (dev >= 0 && dev < 64) opted_in[dev] = true;
    }
    const int row_blocks = (a.M + 127) / 128, tok_blocks = (a.N + N - 1) / N, at_once = blm_sm_count() * W::kBlocks;
    const int unit = a.end == END_ADD || a.y_f32 ? 16 : 8, vec = a.ldy % 4 == 0 && (size_t)a.y % unit == 0;
    auto launch = [&](int first, int blocks, int part) {
        // blocks of a cluster: the number with the shortest time, that of so many turns of a share of K each and, about as long as 16
        // tiles of K, a block's beginning and end; no share below a stretch of 256 places
        int ranks = 1;
        auto tiles = [&](int r) { return ((long long)blocks * r + at_once - 1) / at_once * ((a.k_tiles + r - 1) / r + 16); };
        for (int r = 2; r <= 8 && a.k_tiles >= r * kBatch; r *= 2)
            if (tiles(r) < tiles(ranks)) ranks = r;
        const int share = (a.k_tiles + ranks - 1) / ranks;
        const WideArgs wa{a, ranks == 1 ? share : (share + 3) / 4 * 4, vec, ranks, first, tok_blocks, part, status};
        blm_launch_cluster(wide_kernel<N>, ranks, dim3(ranks * blocks), dim3(W::kThreads), W::kSmem, stream, wa, map);
    };
    // (512 tokens by 28,672 x 4,096 are 448 blocks for 148 SMs: 104 us in four times, the last of 4 blocks)
    const int blocks = row_blocks * tok_blocks, rest = blocks % at_once;
    if (blocks > at_once && rest > 0 && 2 * rest <= at_once && a.k_tiles >= 2 * kBatch) {
        launch(0, blocks - rest, WAVES);
        launch(blocks - rest, rest, REST);
    } else launch(0, blocks, ALONE);
    return blm_check_launch("gemm_q4");
}
}  // namespace q4

BLM_API int blm_gemm_q4(const void* w, int stretches, int group, const void* x, long long ldx, void* y, long long ldy, int y_f32, int end, int n, int m,
                        int k, int* status, cudaStream_t stream) {
    using namespace q4;
    if (n == 0 || m == 0) return BLM_OK;
    BLM_REQUIRE(group == 32 || group == 64 || group == 128, "gemm_q4: groups of %d places (32, 64 or 128)", group);
    BLM_REQUIRE(k > 0 && k % 8 == 0 && ldx % 8 == 0 && ((size_t)x & 15) == 0, "gemm_q4: rows of tokens in pieces of 16 bytes");
    BLM_REQUIRE(((size_t)w & 15) == 0, "gemm_q4: weights begin at a multiple of 16 bytes");
    BLM_REQUIRE(end != END_GATED || m % 16 == 0, "gemm_q4: gated rows come in tiles of 16, got %d", m);
    const int k_tiles = (k + 63) / 64, per_tile = group == 32 ? 2 : 1;
    BLM_REQUIRE(stretches == (k_tiles + kBatch - 1) / kBatch, "gemm_q4: %d stretches a row for %d places", stretches, k);
    const Args a{(const unsigned char*)w, (const __nv_bfloat16*)x, ldx, y, ldy, y_f32, end, n, m, k, k_tiles, stretches, kBatch * kTileBytes + 128 * per_tile, per_tile};
    if (!few_take(n, k_tiles)) {
        BLM_REQUIRE((long long)((m + 127) / 128) * ((n + 255) / 256) < 1 << 28, "gemm_q4: %d tokens, %d rows", n, m);
        return n <= 32 ? launch_wide<32>(a, status, stream) : n <= 64 ? launch_wide<64>(a, status, stream)
               : n <= 128 ? launch_wide<128>(a, status, stream) : launch_wide<256>(a, status, stream);
    }
    return per_tile == 2 ? launch_few<true>(a, status, stream) : launch_few<false>(a, status, stream);
}
