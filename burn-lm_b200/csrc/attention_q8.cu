// A cache line in 8 bits: appending to it with the rotation of queries and keys, and attention over it.
//
// A cache page holds a block of 64 positions.  The keys (values) of one kv head in a COMPLETE block are 8-bit whole numbers with
// one float32 scale: s = max|x| / 127 over the block's 64 x D numbers, q = round(x / s), and q s is what attention reads.  A block
// is stored when its last position arrives, from rows that were kept unrounded: the rows of a sequence's unfinished block lie in
// its `tail` in the compute type.  A query reads the blocks before its own in 8 bits and the keys of its own block unrounded.  So
// what a position's attention gives depends on the tokens alone, not on how a prompt was cut into steps (a scale that grew while
// its block fills would make the block's first numbers depend on when they were read, and a token run ahead and forgotten would
// leave its mark).
//
// A step of several tokens a sequence may fill the block it found unfinished and begin others: the rows it found in the tail are
// copied to `old` (one entry a sequence of the step) before the tail takes the last block's, and attention reads the step's own
// rows from the rotated projection and the rows before them from `old`.  Steps of one token a sequence read the tail itself.
//
// Layout of a kv head's part of a page: keys [64][D] bytes, then values so that the decode kernel's tensor-core fragments are
// 16-byte pieces: for keys 16 w + 4 t + e and lanes d = g (D / 8) + n the byte at
//     w (16 Dp) + (n / 4) 512 + (4 g + t) 16 + (n % 4) 4 + e,     Dp = D rounded up to a multiple of 32:
// thread (g, t) of a warp finds four lanes of four keys in 16 bytes.
#include <math.h>

#include "common.cuh"

BLM_API const char* blm_attention_q8_last_error() { return g_blm_error; }

namespace q8 {
constexpr int kPage = 64;
enum { PAIRS_HALVES = 0, PAIRS_INTERLEAVED = 1, PAIRS_TILED = 2 };

__host__ __device__ constexpr int padded(int hd) { return (hd + 31) / 32 * 32; }
__host__ __device__ constexpr int line_bytes(int hd) { return kPage * (hd + padded(hd)); }       // of one kv head in a page

// where the word of the values of keys k .. k + 3 (k a multiple of 4) and lane d lies, from the start of the values
__device__ __forceinline__ int value_word(int k, int d, int hd) {
    const int per = hd / 8, g = d / per, n = d - g * per;
    return (k >> 4) * (16 * padded(hd)) + (n >> 2) * 512 + (4 * g + ((k >> 2) & 3)) * 16 + (n & 3) * 4;
}

// The page of a slot's block b; -1 where the table holds none that the pool has.
__device__ __forceinline__ int page_of(const int* block_table, int table_stride, int slot, int b, int n_pages) {
    const int page = b < table_stride ? block_table[(size_t)slot * table_stride + b] : -1;
    return page < n_pages ? page : -1;
}

// sixteen bytes of T, as floats
template <typename T> struct Vec { static constexpr int n = 16 / sizeof(T); };
__device__ __forceinline__ void load_vec(const float* p, float* o) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float* o) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(b[i]);
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
    }
}
template <int N> __device__ __forceinline__ void load_n(const float* p, float* o) {
#pragma unroll
    for (int i = 0; i < N; i += 4) load_vec(p + i, o + i);
}
template <int N> __device__ __forceinline__ void load_n(const __nv_bfloat16* p, float* o) {
#pragma unroll
    for (int i = 0; i < N; i += 8) load_vec(p + i, o + i);
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
    __nv_bfloat162 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(b);
}

// ---- the append ------------------------------------------------------------------------------------------------------------
struct AppendArgs {
    const void* qkv;             // [N, n_heads + 2 n_kv, hd]
    void* out;                   // the same shape: q and k rotated, v; may be qkv itself
    const int* cu_seqlens;
    const int* slot_of_seq;
    const int* start_pos;
    const int* block_table;
    int table_stride;
    const double* inv_freq;
    const float2* table;         // (cos, sin) of the positions below table_len, already times turn_scale
    int table_len;
    float turn_scale;
    int rot, pairing;
    signed char* pool;           // [pages][n_kv][line_bytes]
    float* scales;               // [pages][n_kv][2]
    void* tail;                  // [slots][2][n_kv][64][hd]
    void* old;                   // [n_seqs][2][n_kv][64][hd], or null when every sequence brings one token
    int n_heads, n_kv, hd, n_pages;
};

__device__ __forceinline__ float2 turn_of(const AppendArgs& a, int pos, int pair) {
    if (pos < a.table_len) return a.table[(size_t)pos * (a.rot / 2) + pair];
    double s, c;
    sincos((double)pos * a.inv_freq[pair], &s, &c);
    return make_float2(a.turn_scale * (float)c, a.turn_scale * (float)s);
}
// (a, b) turned: products and sums rounded one by one, so that the numbers do not depend on how they are contracted
__device__ __forceinline__ void turn(float& x, float& y, float2 cs) {
    const float nx = __fsub_rn(__fmul_rn(x, cs.x), __fmul_rn(y, cs.y));
    y = __fadd_rn(__fmul_rn(y, cs.x), __fmul_rn(x, cs.y));
    x = nx;
}

// Unit u of a row (16 lanes, one thread): rotates it when it belongs to a query or key and lies among the rotated lanes, writes it
// to `dst` and, where given, to `dst2` and `dst3`.  VEC: the rotated lanes are a multiple of 16, so that a unit is eight pairs in
// two pieces of eight lanes; otherwise lane by lane.
template <typename T, bool VEC>
__device__ __forceinline__ void unit(const AppendArgs& a, const T* src, T* dst, T* dst2, T* dst3, int u, int pos, bool rotates) {
    const int rot = rotates ? a.rot : 0;
    if (VEC || rot == 0) {
        const bool turns = u < rot / 16;
        const bool halves = turns && a.pairing == PAIRS_HALVES;
        const int la = halves ? 8 * u : 16 * u, lb = halves ? rot / 2 + 8 * u : 16 * u + 8;
        float x[8], y[8];
        load_n<8>(src + la, x);
        load_n<8>(src + lb, y);
        if (turns) {
            if (a.pairing == PAIRS_INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    turn(x[2 * i], x[2 * i + 1], turn_of(a, pos, 8 * u + i));
                    turn(y[2 * i], y[2 * i + 1], turn_of(a, pos, 8 * u + 4 + i));
                }
            } else {
                float2 cs[8];
                if (pos < a.table_len) {
                    const float4* t = reinterpret_cast<const float4*>(a.table + (size_t)pos * (rot / 2) + 8 * u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 f = t[i];
                        cs[2 * i] = make_float2(f.x, f.y);
                        cs[2 * i + 1] = make_float2(f.z, f.w);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) cs[i] = turn_of(a, pos, 8 * u + i);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) turn(x[i], y[i], cs[i]);
            }
        }
        store8(dst + la, x);
        store8(dst + lb, y);
        if (dst2) { store8(dst2 + la, x); store8(dst2 + lb, y); }
        if (dst3) { store8(dst3 + la, x); store8(dst3 + lb, y); }
        return;
    }
    // any even number of rotated lanes: pairs 8 u .. 8 u + 7 and, of the lanes that stand still, eight at a time and their next eight
    auto put = [&](int d, float v) {
        const T t = from_f32<T>(v);
        dst[d] = t;
        if (dst2) dst2[d] = t;
        if (dst3) dst3[d] = t;
    };
    for (int i = 8 * u; i < 8 * u + 8; ++i) {
        if (i < rot / 2) {
            const int la = a.pairing == PAIRS_INTERLEAVED ? 2 * i : i, lb = a.pairing == PAIRS_INTERLEAVED ? 2 * i + 1 : i + rot / 2;
            float x = to_f32(src[la]), y = to_f32(src[lb]);
            turn(x, y, turn_of(a, pos, i));
            put(la, x);
            put(lb, y);
        } else {                                         // pairs beyond the rotated ones: two lanes that stand still
            put(2 * i, to_f32(src[2 * i]));
            put(2 * i + 1, to_f32(src[2 * i + 1]));
        }
    }
}

// Stores a complete block of one kv head's keys (VALUES: values): rows(key) gives a row's address.  All 128 threads.
template <typename T, bool VALUES, typename Rows>
__device__ void store_block(const AppendArgs& a, Rows rows, int page, int kvh, float* red) {
    if (page < 0) return;                                // (uniform)
    const int hd = a.hd, pieces = hd / 8, tid = threadIdx.x;
    unsigned top = 0;                                    // of the magnitudes' bits: infinities and NaN stand above every number
    for (int i = tid; i < kPage * pieces; i += 128) {
        float x[8];
        load_n<8>(rows(i / pieces) + (i % pieces) * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();                                     // (red is free, whatever used it before)
    if ((tid & 31) == 0) red[tid >> 5] = __uint_as_float(top);
    __syncthreads();
    top = max(max(__float_as_uint(red[0]), __float_as_uint(red[1])), max(__float_as_uint(red[2]), __float_as_uint(red[3])));
    const float scale = __fdiv_rn(__uint_as_float(top), 127.0f);
    auto eight = [&](float x) -> unsigned {
        const int q = scale == 0.f ? 0 : __float2int_rn(__fdiv_rn(x, scale));
        return (unsigned)max(-127, min(127, q)) & 0xffu;
    };
    signed char* line = a.pool + ((size_t)page * a.n_kv + kvh) * line_bytes(hd);
    if (tid == 0) a.scales[((size_t)page * a.n_kv + kvh) * 2 + (VALUES ? 1 : 0)] = scale;
    if (!VALUES) {
        for (int i = tid; i < kPage * pieces; i += 128) {
            const int key = i / pieces, c = i % pieces;
            float x[8];
            load_n<8>(rows(key) + c * 8, x);
            uint2 w;
            w.x = eight(x[0]) | eight(x[1]) << 8 | eight(x[2]) << 16 | eight(x[3]) << 24;
            w.y = eight(x[4]) | eight(x[5]) << 8 | eight(x[6]) << 16 | eight(x[7]) << 24;
            *reinterpret_cast<uint2*>(line + key * hd + c * 8) = w;
        }
    } else {
        signed char* values = line + kPage * hd;
        for (int i = tid; i < 16 * pieces; i += 128) {
            const int key = (i / pieces) * 4, c = i % pieces;
            unsigned w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[8];
                load_n<8>(rows(key + j) + c * 8, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] |= eight(x[e]) << (8 * j);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<unsigned*>(values + value_word(key, c * 8 + e, hd)) = w[e];
        }
    }
}

// Steps of one token a sequence: a block is (kv head, sequence) and has that head's queries, its key and its value.  Bound by its
// launch; the rare block that completes a page reads the tail's 63 rows and stores them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) append_token_kernel(const AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T* own = reinterpret_cast<T*>(smem_raw);             // [2][hd]: the new key and value
    float* red = reinterpret_cast<float*>(own + 2 * a.hd);
    pdl_wait();
    const int kvh = blockIdx.x, seq = blockIdx.y, tok = a.cu_seqlens[seq];
    if (a.cu_seqlens[seq + 1] == tok) return;
    const int pos = a.start_pos[seq], slot = a.slot_of_seq[seq], at = pos % kPage;
    const bool completes = at == kPage - 1;
    const int group = a.n_heads / a.n_kv, units = a.hd / 16, width = a.n_heads + 2 * a.n_kv;
    const T* src = reinterpret_cast<const T*>(a.qkv) + (size_t)tok * width * a.hd;
    T* dst = reinterpret_cast<T*>(a.out) + (size_t)tok * width * a.hd;
    T* tail = reinterpret_cast<T*>(a.tail) + ((size_t)slot * 2 * a.n_kv + kvh) * kPage * a.hd;     // the keys' rows of this head
    const size_t to_values = (size_t)a.n_kv * kPage * a.hd;
    for (int i = threadIdx.x; i < (group + 2) * units; i += 128) {
        const int r = i / units, u = i % units;          // the group's queries, the key, the value
        const int head = r < group ? kvh * group + r : (r == group ? a.n_heads + kvh : a.n_heads + a.n_kv + kvh);
        T* keep = nullptr;
        if (r >= group) keep = completes ? own + (r - group) * a.hd : tail + (r == group ? 0 : to_values) + (size_t)at * a.hd;
        unit<T, VEC>(a, src + (size_t)head * a.hd, dst + (size_t)head * a.hd, keep, nullptr, u, pos, r <= group);
    }
    if (!completes) return;
    __syncthreads();
    const int page = page_of(a.block_table, a.table_stride, slot, pos / kPage, a.n_pages);
    const T* kt = tail;
    const T* vt = tail + to_values;
    const T* mine = own;
    const int hd = a.hd;
    store_block<T, false>(a, [=](int key) { return key == kPage - 1 ? mine : kt + (size_t)key * hd; }, page, kvh, red);
    store_block<T, true>(a, [=](int key) { return key == kPage - 1 ? mine + hd : vt + (size_t)key * hd; }, page, kvh, red);
}

// Steps of several tokens: a block is (64-position block x of the sequence's new tokens, head of q, k or v, sequence).  Bound by the
// memory: every row is read once and written once (keys and values pass through shared memory on their way into 8 bits).  The rows
// that the step found in the tail and the rows of its last, unfinished block belong to one thread block (x = 0), which reads the
// tail before it writes it.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) append_prompt_kernel(const AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T* rows = reinterpret_cast<T*>(smem_raw);            // [64][hd + 16 bytes]
    const int hd = a.hd, ld = hd + 16 / (int)sizeof(T), units = hd / 16, width = a.n_heads + 2 * a.n_kv;
    float* red = reinterpret_cast<float*>(rows + kPage * ld);
    pdl_wait();
    const int seq = blockIdx.z, head = blockIdx.y, tok0 = a.cu_seqlens[seq], n = a.cu_seqlens[seq + 1] - tok0;
    if (n <= 0) return;
    const int start = a.start_pos[seq], end = start + n, first = start / kPage, last = (end - 1) / kPage;
    int b = first + (int)blockIdx.x;
    if (b > last) return;
    const bool query = head < a.n_heads, value = head >= a.n_heads + a.n_kv;
    const bool last_open = end % kPage != 0;
    if (!query && b > first && b == last && last_open) return;         // the block x = 0 has it
    const int slot = a.slot_of_seq[seq], kvh = value ? head - a.n_heads - a.n_kv : head - a.n_heads;
    const T* qkv = reinterpret_cast<const T*>(a.qkv);
    T* out = reinterpret_cast<T*>(a.out);
    const size_t line = (((size_t)slot * 2 + (value ? 1 : 0)) * a.n_kv + kvh) * kPage * hd;
    T* tail = reinterpret_cast<T*>(a.tail) + (query ? 0 : line);
    for (;;) {
        const int p0 = b * kPage, lo = max(start, p0), hi = min(end, p0 + kPage);
        const bool complete = hi == p0 + kPage;
        for (int i = threadIdx.x; i < (hi - lo) * units; i += 128) {
            const int pos = lo + i / units;
            const size_t at = ((size_t)(tok0 + pos - start) * width + head) * hd;
            T* keep = nullptr;
            if (!query) keep = complete ? rows + (pos - p0) * ld : tail + (size_t)(pos - p0) * hd;
            unit<T, VEC>(a, qkv + at, out + at, keep, nullptr, i % units, pos, !value);
        }
        if (query) return;
        if (b == first && start > p0) {
            // the rows found in the tail: to `old`, and to the block that is being completed
            T* old = reinterpret_cast<T*>(a.old) + (((size_t)seq * 2 + (value ? 1 : 0)) * a.n_kv + kvh) * kPage * hd;
            constexpr int V = Vec<T>::n;
            for (int i = threadIdx.x; i < (start - p0) * (hd / V); i += 128) {
                const int r = i / (hd / V), c = (i % (hd / V)) * V;
                const uint4 v = *reinterpret_cast<const uint4*>(tail + (size_t)r * hd + c);
                *reinterpret_cast<uint4*>(old + (size_t)r * hd + c) = v;
                if (complete) *reinterpret_cast<uint4*>(rows + r * ld + c) = v;
            }
        }
        if (complete) {
            __syncthreads();
            const int page = page_of(a.block_table, a.table_stride, slot, b, a.n_pages);
            const T* r = rows;
            if (value) store_block<T, true>(a, [=](int key) { return r + key * ld; }, page, kvh, red);
            else store_block<T, false>(a, [=](int key) { return r + key * ld; }, page, kvh, red);
        }
        if (b != first || last == first || !last_open) return;
        __syncthreads();                                  // the tail's rows have been read
        b = last;
    }
}

// ---- pages as the numbers they stand for ----------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(128) values_kernel(const signed char* __restrict__ pool, const float* __restrict__ scales, const int* __restrict__ pages,
                                                     T* __restrict__ out, int n_kv, int hd, int n_pages) {
    const int i = blockIdx.x, kvh = blockIdx.y, page = pages[i];
    if (page < 0 || page >= n_pages) return;
    const signed char* line = pool + ((size_t)page * n_kv + kvh) * line_bytes(hd);
    const float ks = scales[((size_t)page * n_kv + kvh) * 2], vs = scales[((size_t)page * n_kv + kvh) * 2 + 1];
    T* ko = out + ((size_t)i * 2 * n_kv + kvh) * kPage * hd;
    T* vo = ko + (size_t)n_kv * kPage * hd;
    for (int j = threadIdx.x; j < kPage * hd; j += 128) {
        const int key = j / hd, d = j % hd;
        ko[j] = from_f32<T>(line[j] * ks);
        vo[j] = from_f32<T>(line[kPage * hd + value_word(key & ~3, d, hd) + (key & 3)] * vs);
    }
}

// ---- attention -------------------------------------------------------------------------------------------------------------
struct AttendArgs {
    const void* rotated;         // [N, n_heads + 2 n_kv, hd]: the append's output
    const signed char* pool;
    const float* scales;
    const void* found;           // rows of the unfinished blocks: the tail (by slot), or `old` (by sequence)
    int found_by_slot;
    const int* block_table;
    int table_stride;
    const int* cu_seqlens;
    const int* slot_of_seq;
    const int* start_pos;
    void* out;                   // [N, n_heads hd]
    int n_seqs, n_heads, n_kv, hd, n_pages, window;
    float scale_log2e;
};

// The general kernel: any type, head size and number of heads.  A block is (token, head); its warps take pages in turn, a lane a key
// for the scores and D / 32 lanes for the sums, each warp with its own running maximum and sum; they meet in shared memory.
constexpr int kGeneralWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kGeneralWarps * 32) attend_general_kernel(const AttendArgs a) {
    __shared__ __align__(16) float q[256];
    __shared__ float sm_acc[kGeneralWarps][256], sm_m[kGeneralWarps], sm_l[kGeneralWarps];
    pdl_wait();
    const int head = blockIdx.x % a.n_heads, tok = blockIdx.x / a.n_heads, hd = a.hd, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the sequence of this row: the last one that begins at or before it
    int lo_s = 0, hi_s = a.n_seqs;
    if (tok >= a.cu_seqlens[hi_s]) return;               // a row of no sequence
    while (hi_s - lo_s > 1) {
        const int mid = (lo_s + hi_s) / 2;
        if (a.cu_seqlens[mid] <= tok) lo_s = mid; else hi_s = mid;
    }
    const int seq = lo_s, tok0 = a.cu_seqlens[seq], start = a.start_pos[seq], pos = start + tok - tok0, slot = a.slot_of_seq[seq];
    const int kvh = head / (a.n_heads / a.n_kv), width = a.n_heads + 2 * a.n_kv;
    const int key_lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0, mine = pos / kPage;
    const T* rows = reinterpret_cast<const T*>(a.rotated);
    for (int d = tid; d < hd; d += blockDim.x) q[d] = to_f32(rows[((size_t)tok * width + head) * hd + d]) * a.scale_log2e;
    __syncthreads();
    float m_run = -INFINITY, l_run = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    const T* found = reinterpret_cast<const T*>(a.found) + ((size_t)(a.found_by_slot ? slot : seq) * 2 * a.n_kv + kvh) * kPage * hd;
    for (int c = key_lo / 32 + warp; c <= pos / 32; c += kGeneralWarps) {        // 32 keys a step
        const int b = c / 2, key = c * 32 + lane;
        const bool own = b == mine, seen = key <= pos && key >= key_lo;
        // where a row of the own block lies
        auto own_row = [&](int k, int which) -> const T* {
            if (k >= start) return rows + ((size_t)(tok0 + k - start) * width + a.n_heads + which * a.n_kv + kvh) * hd;
            return found + ((size_t)which * a.n_kv * kPage + k % kPage) * hd;
        };
        const signed char* line = nullptr;
        float ks = 0.f, vs = 0.f;
        if (!own) {
            const int page = page_of(a.block_table, a.table_stride, slot, b, a.n_pages);
            if (page < 0) continue;
            line = a.pool + ((size_t)page * a.n_kv + kvh) * line_bytes(hd);
            ks = a.scales[((size_t)page * a.n_kv + kvh) * 2];
            vs = a.scales[((size_t)page * a.n_kv + kvh) * 2 + 1];
        }
        float s = -INFINITY;
        if (seen) {
            float sum = 0.f;
            if (own) {
                const T* kr = own_row(key, 0);
                for (int d = 0; d < hd; d += 8) {
                    float x[8];
                    load_n<8>(kr + d, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fmaf(q[d + e], x[e], sum);
                }
            } else {
                const signed char* kr = line + (key % kPage) * hd;
                for (int d = 0; d < hd; d += 16) {
                    const int4 w = *reinterpret_cast<const int4*>(kr + d);
                    const signed char* x = reinterpret_cast<const signed char*>(&w);
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum = fmaf(q[d + e], (float)x[e], sum);
                }
                sum *= ks;
            }
            s = sum;
        }
        const float m_new = fmaxf(m_run, warp_max(s));
        if (m_new == -INFINITY) continue;
        const float alpha = m_run == -INFINITY ? 0.f : exp2f(m_run - m_new), p = seen ? exp2f(s - m_new) : 0.f;
        m_run = m_new;
        l_run = l_run * alpha + warp_sum(p);
        const float pv = own ? p : p * vs;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= alpha;
        // keys that are not seen are not read: what lies there may be anything
        const int k_first = max(c * 32, key_lo), k_last = min(c * 32 + 31, pos);
        if (own) {
            for (int k = k_first; k <= k_last; ++k) {
                const float w = __shfl_sync(0xffffffffu, pv, k & 31);
                const T* vr = own_row(k, 1);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (lane + 32 * i < hd) acc[i] = fmaf(w, to_f32(vr[lane + 32 * i]), acc[i]);
            }
        } else {
            for (int k = (c * 32) % kPage; k < (c * 32) % kPage + 32; k += 4) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __shfl_sync(0xffffffffu, pv, (k & 31) + e);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (lane + 32 * i < hd) {
                        const char4 v = *reinterpret_cast<const char4*>(line + kPage * hd + value_word(k, lane + 32 * i, hd));
                        acc[i] = fmaf(w[0], (float)v.x, fmaf(w[1], (float)v.y, fmaf(w[2], (float)v.z, fmaf(w[3], (float)v.w, acc[i]))));
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < hd) sm_acc[warp][lane + 32 * i] = acc[i];
    if (lane == 0) { sm_m[warp] = m_run; sm_l[warp] = l_run; }
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < kGeneralWarps; ++w) m = fmaxf(m, sm_m[w]);
    for (int w = 0; w < kGeneralWarps; ++w) l += sm_m[w] == -INFINITY ? 0.f : sm_l[w] * exp2f(sm_m[w] - m);
    for (int d = tid; d < hd; d += blockDim.x) {
        float o = 0.f;
        for (int w = 0; w < kGeneralWarps; ++w) o += sm_m[w] == -INFINITY ? 0.f : sm_acc[w][d] * exp2f(sm_m[w] - m);
        reinterpret_cast<T*>(a.out)[((size_t)tok * a.n_heads + head) * hd + d] = from_f32<T>(o / l);
    }
}

template <typename T, bool VEC>
static int launch_append(const AppendArgs& a, int n_seqs, int max_q_len, cudaStream_t stream) {
    if (max_q_len == 1) {
        const size_t smem = 2 * a.hd * sizeof(T) + 4 * sizeof(float);
        blm_launch_dependent(append_token_kernel<T, VEC>, dim3(a.n_kv, n_seqs), dim3(128), smem, stream, a);
    } else {
        const size_t smem = (size_t)kPage * (a.hd + 16 / sizeof(T)) * sizeof(T) + 4 * sizeof(float);
        if (smem > 48 * 1024 &&
            cudaFuncSetAttribute(append_prompt_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "rope_append_q8: no room for a block's rows");
        // a run of max_q_len tokens touches this many blocks at most, wherever it begins
        const dim3 grid((max_q_len + kPage - 2) / kPage + 1, a.n_heads + 2 * a.n_kv, n_seqs);
        blm_launch_dependent(append_prompt_kernel<T, VEC>, grid, dim3(128), smem, stream, a);
    }
    return blm_check_launch("rope_append_q8");
}
}  // namespace q8

BLM_API int blm_rope_append_q8(const void* qkv, void* out, int dtype, const int* cu_seqlens, const int* slot_of_seq, const int* start_pos,
                               const int* block_table, int table_stride, const double* inv_freq, int rot, int pairing, const float* table,
                               int table_len, float turn_scale, void* pool, float* scales, void* tail, void* old, int n_seqs, int max_q_len,
                               int n_heads, int n_kv, int hd, int n_pages, cudaStream_t stream) {
    using namespace q8;
    if (n_seqs == 0 || max_q_len == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0, "rope_append_q8: heads of %d lanes (multiples of 16 from 16 to 256)", hd);
    BLM_REQUIRE(n_kv > 0 && n_heads % n_kv == 0, "rope_append_q8: %d heads do not divide into %d kv heads", n_heads, n_kv);
    BLM_REQUIRE(rot >= 0 && rot <= hd && rot % 2 == 0, "rope_append_q8: %d rotated lanes of a head of %d", rot, hd);
    BLM_REQUIRE(rot == 0 || inv_freq != nullptr, "rope_append_q8: no frequencies");
    BLM_REQUIRE(pairing >= 0 && pairing <= 2 && (pairing != PAIRS_TILED || rot % 16 == 0), "rope_append_q8: pairing %d of %d lanes", pairing, rot);
    BLM_REQUIRE(n_seqs <= 65535 && n_heads + 2 * n_kv <= 65535, "rope_append_q8: %d sequences, %d heads (at most 65535 of either)", n_seqs, n_heads + 2 * n_kv);
    BLM_REQUIRE(dtype == BLM_F32 || dtype == BLM_BF16, "rope_append_q8: dtype %d", dtype);
    const AppendArgs a{qkv, out, cu_seqlens, slot_of_seq, start_pos, block_table, table_stride, inv_freq, (const float2*)table, table ? table_len : 0,
                       turn_scale, rot, pairing, (signed char*)pool, scales, tail, old, n_heads, n_kv, hd, n_pages};
    const bool vec = rot % 16 == 0;
    if (dtype == BLM_F32) return vec ? launch_append<float, true>(a, n_seqs, max_q_len, stream) : launch_append<float, false>(a, n_seqs, max_q_len, stream);
    return vec ? launch_append<__nv_bfloat16, true>(a, n_seqs, max_q_len, stream) : launch_append<__nv_bfloat16, false>(a, n_seqs, max_q_len, stream);
}

BLM_API int blm_q8_values(const void* pool, const float* scales, const int* pages, void* out, int dtype, int n, int n_kv, int hd, int n_pages,
                          cudaStream_t stream) {
    using namespace q8;
    if (n == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0 && n_kv <= 65535, "q8_values: %d heads of %d lanes", n_kv, hd);
    const dim3 grid(n, n_kv);
    if (dtype == BLM_F32) values_kernel<<<grid, 128, 0, stream>>>((const signed char*)pool, scales, pages, (float*)out, n_kv, hd, n_pages);
    else if (dtype == BLM_BF16) values_kernel<<<grid, 128, 0, stream>>>((const signed char*)pool, scales, pages, (__nv_bfloat16*)out, n_kv, hd, n_pages);
    else return blm_fail(BLM_BAD_ARGUMENT, "q8_values: dtype %d", dtype);
    return blm_check_launch("q8_values");
}

BLM_API int blm_attention_q8(const void* rotated, const void* pool, const float* scales, const void* found, int found_by_slot, int dtype,
                             const int* block_table, int table_stride, const int* cu_seqlens, const int* slot_of_seq, const int* start_pos,
                             void* out, int n_tokens, int n_seqs, int n_heads, int n_kv, int hd, int n_pages, int window, float scale,
                             cudaStream_t stream) {
    using namespace q8;
    if (n_tokens == 0 || n_seqs == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0, "attention_q8: heads of %d lanes (multiples of 16 from 16 to 256)", hd);
    BLM_REQUIRE(n_kv > 0 && n_heads % n_kv == 0, "attention_q8: %d heads do not divide into %d kv heads", n_heads, n_kv);
    BLM_REQUIRE((long long)n_tokens * n_heads < (1ll << 31), "attention_q8: %d tokens of %d heads in one step", n_tokens, n_heads);
    const AttendArgs a{rotated, (const signed char*)pool, scales, found, found_by_slot, block_table, table_stride, cu_seqlens, slot_of_seq, start_pos,
                       out, n_seqs, n_heads, n_kv, hd, n_pages, window, scale * 1.4426950408889634f};
    const dim3 grid(n_heads * n_tokens);
    if (dtype == BLM_F32) blm_launch_dependent(attend_general_kernel<float>, grid, dim3(kGeneralWarps * 32), 0, stream, a);
    else if (dtype == BLM_BF16) blm_launch_dependent(attend_general_kernel<__nv_bfloat16>, grid, dim3(kGeneralWarps * 32), 0, stream, a);
    else return blm_fail(BLM_BAD_ARGUMENT, "attention_q8: dtype %d", dtype);
    return blm_check_launch("attention_q8");
}
