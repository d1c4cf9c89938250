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
#include "common.cuh"

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

__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
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
    const int tile0 = blockIdx.x * R, tok0 = blockIdx.y * 8 * NT, n = min(8 * NT, a.N - tok0), tiles = (a.M + 15) / 16;
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
                    x[j][i][h] = tok < n && k < a.K ? *reinterpret_cast<const uint4*>(a.x + (size_t)(tok0 + tok) * a.ldx + k) : make_uint4(0u, 0u, 0u, 0u);
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
                        for (int i = 0; i < NT; ++i) mma(part[i], a0, a1, a2, a3, s ? x[j][i][h].z : x[j][i][h].x, s ? x[j][i][h].w : x[j][i][h].y);
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
        const size_t to = (size_t)(tok0 + tok) * a.ldy + out;
        if (a.end == END_ADD) reinterpret_cast<float*>(a.y)[to] += y;
        else if (a.y_f32) reinterpret_cast<float*>(a.y)[to] = y;
        else reinterpret_cast<__nv_bfloat16*>(a.y)[to] = __float2bfloat16_rn(y);
    }
}

template <int R, int NT>
static void launch_skinny(const Args& a, cudaStream_t stream) {
    const dim3 grid(((a.M + 15) / 16 + R - 1) / R, (a.N + 8 * NT - 1) / (8 * NT));
    blm_launch_dependent(skinny_kernel<R, NT>, grid, dim3(kWarps * 32), 0, stream, a);
}
}  // namespace q4

BLM_API int blm_gemm_q4(const void* w, const void* scales, int groups, int group, const void* x, long long ldx, void* y, long long ldy, int y_f32,
                        int end, int n, int m, int k, cudaStream_t stream) {
    using namespace q4;
    if (n == 0 || m == 0) return BLM_OK;
    BLM_REQUIRE(group == 32 || group == 64 || group == 128, "gemm_q4: groups of %d places (32, 64 or 128)", group);
    BLM_REQUIRE(k > 0 && k % 8 == 0 && ldx % 8 == 0 && ((size_t)x & 15) == 0, "gemm_q4: rows of tokens in pieces of 16 bytes");
    BLM_REQUIRE(end != END_GATED || m % 16 == 0, "gemm_q4: gated rows come in tiles of 16, got %d", m);
    const int k_tiles = (k + 63) / 64;
    BLM_REQUIRE(groups == (k_tiles + kBatch - 1) / kBatch * (kBatch * 64 / group), "gemm_q4: %d groups a row for %d places", groups, k);
    BLM_REQUIRE((n + 7) / 8 <= 65535, "gemm_q4: %d tokens", n);
    const Args a{(const uint4*)w, (const __nv_bfloat16*)scales, (const __nv_bfloat16*)x, ldx, y, ldy, y_f32, end, n, m, k, k_tiles, groups, group};
    if (n <= 8) launch_skinny<2, 1>(a, stream); else launch_skinny<2, 2>(a, stream);
    return blm_check_launch("gemm_q4");
}
