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
// Layout of a kv head's part of a page: keys [64][D] bytes, where D is a multiple of 32 with the 16-byte pieces of odd rows exchanged
// pairwise (so that the decode kernel's reads of neighbouring rows meet in no bank of shared memory); then the values, so that the decode
// kernel's tensor-core fragments are 16-byte pieces: for keys 16 w + 4 t + e and lanes d = g (D / 8) + n the byte at
//     w (16 Dp) + (n / 4) 512 + (4 g + t) 16 + (n % 4) 4 + e,     Dp = D rounded up to a multiple of 32:
// thread (g, t) of a warp finds four lanes of four keys in 16 bytes; then 16 bytes whose first eight are the two scales, so that one
// copy brings all that a block needs.  A byte holds q + 128: behind the byte 0x64 it is the half-precision number 1024 + 128 + q, so that
// one byte permutation makes two numbers.
#include <cuda_fp16.h>
#include <math.h>

#include "cluster.cuh"
#include "tcgen05.cuh"

BLM_API const char* blm_attention_q8_last_error() { return g_blm_error; }

namespace q8 {
constexpr int kPage = 64;
enum { PAIRS_HALVES = 0, PAIRS_INTERLEAVED = 1, PAIRS_TILED = 2 };

__host__ __device__ constexpr int padded(int hd) { return (hd + 31) / 32 * 32; }
__host__ __device__ constexpr int number_bytes(int hd) { return kPage * (hd + padded(hd)); }     // of one kv head in a page
__host__ __device__ constexpr int line_bytes(int hd) { return number_bytes(hd) + 16; }             // ... and its scales
__device__ __forceinline__ const float2* scales_of(const void* line, int hd) { return reinterpret_cast<const float2*>((const signed char*)line + number_bytes(hd)); }

// where lanes d .. d + 15 (d a multiple of 16) of key k lie, from the start of the keys
__device__ __forceinline__ int key_piece(int k, int d, int hd) { return k * hd + (hd % 32 == 0 ? d ^ ((k & 1) << 4) : d); }
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

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}

// Steps of several tokens have a block of threads for every block of `unit` positions that a sequence touches.  The one with number `at`,
// the sequences in turn, each one's from its last (which walk furthest): its sequence, -1 where there are fewer, and its number from the
// sequence's last.  A warp asks together.  (With a grid of the longest sequence's blocks for every sequence, a prompt of 2,000 tokens
// beside 63 single ones was 287 us of attention, most of it blocks that had nothing to do.)
__device__ __forceinline__ int find_block(const int* cu_seqlens, const int* start_pos, int n_seqs, int unit, int at, int& from_last) {
    const int lane = threadIdx.x & 31;
    if (n_seqs == 1) {                                   // (a quarter of a microsecond sooner)
        const int n = cu_seqlens[1] - cu_seqlens[0], start = start_pos[0];
        from_last = at;
        return n > 0 && at <= (start + n - 1) / unit - start / unit ? 0 : -1;
    }
    for (int base = 0; base < n_seqs; base += 32) {
        const int s = base + lane;
        int count = 0;
        if (s < n_seqs) {
            const int n = cu_seqlens[s + 1] - cu_seqlens[s], start = start_pos[s];
            if (n > 0) count = (start + n - 1) / unit - start / unit + 1;
        }
        int sum = count;
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, sum, w);
            if (lane >= w) sum += below;
        }
        const int total = __shfl_sync(0xffffffffu, sum, 31);
        if (at < total) {
            const int of = __ffs(__ballot_sync(0xffffffffu, at < sum)) - 1;
            from_last = at - __shfl_sync(0xffffffffu, sum - count, of);
            return base + of;
        }
        at -= total;
    }
    from_last = 0;
    return -1;
}
// the most that sequences with n_tokens together touch
static inline long long most_blocks(long long n_tokens, long long n_seqs, int unit) { return (n_tokens + n_seqs * (unit - 2)) / unit + n_seqs; }

// the halves of two bfloat16 numbers that are infinities or NaN, as masks
__device__ __forceinline__ unsigned odd_two(unsigned v) {
    return ((v & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((v & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
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
    void* tail;                  // [slots][2][n_kv][64][hd]
    void* old;                   // [n_seqs][2][n_kv][64][hd], or null when every sequence brings one token
    int n_heads, n_kv, hd, n_pages, n_seqs;
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
// to `dst` and, where given, to `dst2`.  VEC: the rotated lanes are a multiple of 16, so that a unit is eight pairs in
// two pieces of eight lanes; otherwise lane by lane.
template <typename T, bool VEC>
__device__ __forceinline__ void unit(const AppendArgs& a, const T* src, T* dst, T* dst2, int u, int pos, bool rotates) {
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
        return;
    }
    // any even number of rotated lanes: pairs 8 u .. 8 u + 7 and, of the lanes that stand still, eight at a time and their next eight
    auto put = [&](int d, float v) {
        const T t = from_f32<T>(v);
        dst[d] = t;
        if (dst2) dst2[d] = t;
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

constexpr int kAppendThreads = 256;
// Stores a complete block of one kv head's keys or values from its rows in shared memory, `ld` apart.  All 256 threads.
template <typename T>
__device__ void store_block(const AppendArgs& a, const T* rows, int ld, bool value, int page, int kvh, float* red) {
    if (page < 0) return;                                // (uniform)
    const int hd = a.hd, pieces = hd / 8, tid = threadIdx.x;
    unsigned top = 0;                                    // of the magnitudes' bits: infinities and NaN stand above every number
    for (int i = tid; i < kPage * pieces; i += kAppendThreads) {
        float x[8];
        load_n<8>(rows + i / pieces * ld + i % pieces * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();                                     // (red is free, whatever used it before)
    if ((tid & 31) == 0) red[tid >> 5] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, __float_as_uint(red[w]));
    const float scale = __fdiv_rn(__uint_as_float(top), 127.0f);
    auto eight = [&](float v) -> unsigned {
        const int q = scale == 0.f ? 0 : __float2int_rn(__fdiv_rn(v, scale));
        return (unsigned)(max(-127, min(127, q)) + 128);
    };
    signed char* line = a.pool + ((size_t)page * a.n_kv + kvh) * line_bytes(hd);
    if (tid == 0) reinterpret_cast<float*>(line + number_bytes(hd))[value ? 1 : 0] = scale;
    // four lanes of four keys a thread: a word of each key, or of each lane
    for (int i = tid; i < 4 * hd; i += kAppendThreads) {
        const int key = i / (hd / 4) * 4, d = i % (hd / 4) * 4;
        unsigned q[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const T* x = rows + (key + r) * ld + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[r][e] = eight(to_f32(x[e]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (value) *reinterpret_cast<unsigned*>(line + kPage * hd + value_word(key, d + e, hd)) = q[0][e] | q[1][e] << 8 | q[2][e] << 16 | q[3][e] << 24;
            else *reinterpret_cast<unsigned*>(line + key_piece(key + e, d & ~15, hd) + (d & 15)) = q[e][0] | q[e][1] << 8 | q[e][2] << 16 | q[e][3] << 24;
        }
    }
}
// Rows of hd numbers, 16 bytes a thread.
template <typename T>
__device__ __forceinline__ void copy_rows(const T* src, T* dst, int ld, T* dst2, int n, int hd) {
    constexpr int V = Vec<T>::n;
    for (int i = threadIdx.x; i < n * (hd / V); i += kAppendThreads) {
        const int r = i / (hd / V), c = i % (hd / V) * V;
        const uint4 v = *reinterpret_cast<const uint4*>(src + (size_t)r * hd + c);
        if (dst) *reinterpret_cast<uint4*>(dst + r * ld + c) = v;
        if (dst2) *reinterpret_cast<uint4*>(dst2 + (size_t)r * hd + c) = v;
    }
}

// Steps of one token a sequence: a block is (kv head, sequence, 0: that head's queries and its key, 1: its value).  Bound by its launch
// and the few loads that wait for one another; the block that completes a page reads the tail's 63 rows and stores them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_token_kernel(const AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T* rows = reinterpret_cast<T*>(smem_raw);            // [64][hd + 16 bytes], of a block that is completed
    const int ld = a.hd + 16 / (int)sizeof(T);
    float* red = reinterpret_cast<float*>(rows + kPage * ld);
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.x, seq = blockIdx.y, tok = a.cu_seqlens[seq], next = a.cu_seqlens[seq + 1];
    const int pos = a.start_pos[seq], slot = a.slot_of_seq[seq], at = pos % kPage;
    if (next == tok) return;
    const bool completes = at == kPage - 1, value = blockIdx.z == 1;
    const int page = completes ? page_of(a.block_table, a.table_stride, slot, pos / kPage, a.n_pages) : -1;
    const int group = a.n_heads / a.n_kv, units = a.hd / 16, width = a.n_heads + 2 * a.n_kv, hd = a.hd;
    const T* src = reinterpret_cast<const T*>(a.qkv) + (size_t)tok * width * hd;
    T* dst = reinterpret_cast<T*>(a.out) + (size_t)tok * width * hd;
    T* tail = reinterpret_cast<T*>(a.tail) + (((size_t)slot * 2 + (value ? 1 : 0)) * a.n_kv + kvh) * kPage * hd;
    if (completes) copy_rows<T>(tail, rows, ld, nullptr, kPage - 1, hd);
    const int first = value ? group + 1 : 0, count = value ? 1 : group + 1;
    for (int i = threadIdx.x; i < count * units; i += kAppendThreads) {
        const int r = first + i / units, u = i % units;  // the group's queries, the key, the value
        const int head = r < group ? kvh * group + r : (r == group ? a.n_heads + kvh : a.n_heads + a.n_kv + kvh);
        T* keep = nullptr;
        if (r >= group) keep = completes ? rows + at * ld : tail + (size_t)at * hd;
        unit<T, VEC>(a, src + (size_t)head * hd, dst + (size_t)head * hd, keep, u, pos, r <= group);
    }
    if (!completes) return;
    __syncthreads();
    store_block<T>(a, rows, ld, value, page, kvh, red);
}

// Steps of several tokens: a block is (64-position block that a sequence touches, head of q, k or v).  Every row is read once and written
// once (keys and values pass through shared memory on their way into 8 bits, which is read twice: for the largest magnitude, then for the
// numbers).  The rows that the step found in the tail and the rows of the sequence's last, unfinished block belong to the thread block of
// the sequence's first, which reads the tail before it writes it.  2,048 tokens of 32 heads of 64 to 8: 18.8 us (float32 21.2), 4.3 of
// them the memory's.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_prompt_kernel(const AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T* rows = reinterpret_cast<T*>(smem_raw);            // [64][hd + 16 bytes]
    const int hd = a.hd, ld = hd + 16 / (int)sizeof(T), units = hd / 16, width = a.n_heads + 2 * a.n_kv;
    float* red = reinterpret_cast<float*>(rows + kPage * ld);
    pdl_launch_dependents();
    pdl_wait();
    int from_last;
    const int seq = find_block(a.cu_seqlens, a.start_pos, a.n_seqs, kPage, (int)blockIdx.x, from_last), head = blockIdx.y;
    if (seq < 0) return;
    const int tok0 = a.cu_seqlens[seq], n = a.cu_seqlens[seq + 1] - tok0;
    const int start = a.start_pos[seq], end = start + n, first = start / kPage, last = (end - 1) / kPage;
    int b = last - from_last;
    const bool query = head < a.n_heads, value = head >= a.n_heads + a.n_kv;
    const bool last_open = end % kPage != 0;
    if (!query && b > first && b == last && last_open) return;         // the block of the sequence's first has it
    const int slot = a.slot_of_seq[seq], kvh = value ? head - a.n_heads - a.n_kv : head - a.n_heads;
    const T* qkv = reinterpret_cast<const T*>(a.qkv);
    T* out = reinterpret_cast<T*>(a.out);
    const size_t line = (((size_t)slot * 2 + (value ? 1 : 0)) * a.n_kv + kvh) * kPage * hd;
    T* tail = reinterpret_cast<T*>(a.tail) + (query ? 0 : line);
    for (;;) {
        const int p0 = b * kPage, lo = max(start, p0), hi = min(end, p0 + kPage);
        const bool complete = hi == p0 + kPage;
        for (int i = threadIdx.x; i < (hi - lo) * units; i += kAppendThreads) {
            const int pos = lo + i / units;
            const size_t at = ((size_t)(tok0 + pos - start) * width + head) * hd;
            T* keep = nullptr;
            if (!query) keep = complete ? rows + (pos - p0) * ld : tail + (size_t)(pos - p0) * hd;
            unit<T, VEC>(a, qkv + at, out + at, keep, i % units, pos, !value);
        }
        if (query) return;
        if (b == first && start > p0) {
            // the rows found in the tail: to `old`, and to the block that is being completed
            T* old = reinterpret_cast<T*>(a.old) + (((size_t)seq * 2 + (value ? 1 : 0)) * a.n_kv + kvh) * kPage * hd;
            copy_rows<T>(tail, complete ? rows : nullptr, ld, old, start - p0, hd);
        }
        if (complete) {
            __syncthreads();
            const int page = page_of(a.block_table, a.table_stride, slot, b, a.n_pages);
            store_block<T>(a, rows, ld, value, page, kvh, red);
        }
        if (b != first || last == first || !last_open) return;
        __syncthreads();                                  // the tail's rows have been read
        b = last;
    }
}

// ---- pages as the numbers they stand for ----------------------------------------------------------------------------------
// A thread has four lanes of four keys: four words of keys, four of values.
template <typename T>
__global__ void __launch_bounds__(256) values_kernel(const signed char* __restrict__ pool, const int* __restrict__ pages, T* __restrict__ out, int n_kv, int hd,
                                                     int n_pages) {
    const int kvh = blockIdx.y, page = pages[blockIdx.x], i = blockIdx.z * 256 + threadIdx.x;
    if (i >= 4 * hd) return;
    const int key = i / (hd / 4) * 4, d = i % (hd / 4) * 4;
    const signed char* line = pool + ((size_t)max(page, 0) * n_kv + kvh) * line_bytes(hd);
    const bool is = page >= 0 && page < n_pages;
    const float2 scale = is ? *scales_of(line, hd) : make_float2(0.f, 0.f);
    unsigned k[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u}, v[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
    if (is) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k[e] = *reinterpret_cast<const unsigned*>(line + key_piece(key + e, d & ~15, hd) + (d & 15));
            v[e] = *reinterpret_cast<const unsigned*>(line + kPage * hd + value_word(key, d + e, hd));
        }
    }
    T* ko = out + (((size_t)blockIdx.x * 2 * n_kv + kvh) * kPage + key) * hd + d;
    T* vo = ko + (size_t)n_kv * kPage * hd;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            ko[e * hd + f] = from_f32<T>((float)((int)(k[e] >> (8 * f) & 0xffu) - 128) * scale.x);
            vo[e * hd + f] = from_f32<T>((float)((int)(v[f] >> (8 * e) & 0xffu) - 128) * scale.y);
        }
}

// ---- attention -------------------------------------------------------------------------------------------------------------
struct AttendArgs {
    const void* rotated;         // [N, n_heads + 2 n_kv, hd]: the append's output
    const signed char* pool;
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

// The general kernel: any type, head size and number of tokens, on mma.sync.  A block owns 32 rows, HB query heads of a kv head by 32 / HB
// positions inside one 64-position block of a sequence, and walks the sequence's pages, whose numbers are widened once into shared memory
// for all of them; a cluster's blocks take the pages in turn.  Four warps have 16 rows by 32 keys of a page each, with a maximum, sums and
// a result of their own, which meet at the end.  The whole numbers of a page are exact in bfloat16; a float32 operand is the sum of three
// bfloat16 numbers (8 bits each of its 24), so three products with a page's numbers are exact, and six of the nine with the own block's
// float32 rows leave out 2^-25 of a product.  The tensor cores cut their 32-bit sums off, so a page's result is formed from zero and added
// to the others as a float.  (On the 32-bit units, 4 by 4 results a thread: 63 us against 32 for 137 tokens behind 700 in float32;
// what bounded it was reads of shared memory.)  The next page's bytes are on their way into registers meanwhile.
constexpr int kTileThreads = 128, kTileRows = 32;
template <typename T> struct Tile {
    static constexpr int kPieces = sizeof(T) == 4 ? 3 : 1, kSlots = kPieces < 2 ? 2 : kPieces;       // of a query; room for the pieces of keys or values
    static constexpr size_t smem(int hd) { return (size_t)(kPieces * kTileRows + kSlots * kPage) * (hd + 8) * 2; }
};
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix4_turned(unsigned (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x and y as bfloat16 numbers side by side, and what is left of them
__device__ __forceinline__ unsigned take_two(float& x, float& y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    x -= __low2float(v);
    y -= __high2float(v);
    return *reinterpret_cast<const unsigned*>(&v);
}

template <typename T, int NL>
__global__ void __launch_bounds__(kTileThreads, NL == 1 ? 3 : 1) attend_tile_kernel(const AttendArgs a, int hb, int ranks, int single) {
    constexpr int PIECES = Tile<T>::kPieces;
    extern __shared__ __align__(16) unsigned char tile_shared[];
    // bits: keys of the own block whose values hold an infinity or a NaN; that hold one themselves (where a number is several pieces, which an
    // infinity has not)
    __shared__ __align__(16) unsigned odd_keys[4];
    unsigned* odd_scores = odd_keys + 2;
    __shared__ float met_m[2][kTileRows], met_l[2][kTileRows], weights[2 * kTileRows];
    const int hd = a.hd, row_of = hd + 8;                // numbers between rows: eight rows' 16-byte pieces meet in no bank
    __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(tile_shared);            // [PIECES][32 rows][hd + 8]
    __nv_bfloat16* page = q + (size_t)PIECES * kTileRows * row_of;               // [slots][64 keys][hd + 8]
    float* met = reinterpret_cast<float*>(tile_shared);                          // [2 halves][32 rows][hd + 4], at the end
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.n_heads / a.n_kv, per_kv = group / hb, tb = kTileRows / hb;
    const int n_groups = a.n_kv * per_kv, rank = blockIdx.x % ranks, heads = blockIdx.x / ranks % n_groups, at = blockIdx.x / ranks / n_groups;
    const int kvh = heads / per_kv, head0 = kvh * group + heads % per_kv * hb;
    pdl_wait();
    pdl_launch_dependents();
    int from_last = 0;
    const int seq = single ? at : find_block(a.cu_seqlens, a.start_pos, a.n_seqs, tb, at, from_last);
    if (seq < 0) return;                                 // (the whole cluster)
    const int tok0 = a.cu_seqlens[seq], n = a.cu_seqlens[seq + 1] - tok0, start = a.start_pos[seq], slot = a.slot_of_seq[seq], end = start + n;
    if (n <= 0) return;
    const int tile = (end - 1) / tb - from_last;
    const int t0 = tile * tb, mine = t0 / kPage, p0 = mine * kPage, width = a.n_heads + 2 * a.n_kv;
    auto first_key = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; };
    const int pg_lo = first_key(max(start, t0)) / kPage;
    const T* rows = reinterpret_cast<const T*>(a.rotated);
    const T* found = reinterpret_cast<const T*>(a.found) + ((size_t)(a.found_by_slot ? slot : seq) * 2 * a.n_kv + kvh) * kPage * hd;
    auto own_row = [&](int pos, int which) -> const T* { // of a position of the own block before the sequence's end
        return pos >= start ? rows + ((size_t)(tok0 + pos - start) * width + a.n_heads + which * a.n_kv + kvh) * hd
                            : found + ((size_t)which * a.n_kv * kPage + pos % kPage) * hd;
    };
    // eight numbers as pieces, `apart` numbers between the pieces
    auto put = [&](__nv_bfloat16* to, size_t apart, float (&x)[8]) {
        if (PIECES > 1) {                                // what would round to an infinity is cut off first: its last bits are nothing beside it
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned bits = __float_as_uint(x[e]), size = bits & 0x7fffffffu;
                if (size >= 0x7f7f8000u && size < 0x7f800000u) x[e] = __uint_as_float(bits & 0xffff0000u);
            }
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            *reinterpret_cast<uint4*>(to + i * apart) = make_uint4(take_two(x[0], x[1]), take_two(x[2], x[3]), take_two(x[4], x[5]), take_two(x[6], x[7]));
    };
    if (tid < 4) odd_keys[tid] = 0u;
    for (int i = tid; i < kTileRows * (hd / 8); i += kTileThreads) {
        const int r = i % kTileRows, d = i / kTileRows * 8, pos = t0 + r / hb;
        float x[8] = {};
        if (pos >= start && pos < end) load_n<8>(rows + ((size_t)(tok0 + pos - start) * width + head0 + r % hb) * hd + d, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= PIECES > 1 ? a.scale_log2e : 1.f;    // (a bfloat16 query stays as it is: its scores are multiplied)
        put(q + (size_t)r * row_of + d, (size_t)kTileRows * row_of, x);
    }
    // this warp's 16 rows and 32 keys of a page; a thread has rows g and g + 8 and columns 2 t, 2 t + 1 of every eight
    const int m0 = (warp & 1) * 16, half = warp >> 1, g = lane >> 2, t = lane & 3;
    const bool idle = t0 + m0 / hb >= end || t0 + (m0 + 15) / hb < start;        // (single tokens have 16 rows of the 32 at most)
    const int pos_of[2] = {t0 + (m0 + g) / hb, t0 + (m0 + g + 8) / hb}, lo_of[2] = {first_key(pos_of[0]), first_key(pos_of[1])};
    // where a lane's row of the 8 x 8 matrices begins: of 16 rows by 16 numbers of q; of 16 keys by 16 numbers; turned, of 16 keys by 16 lanes
    const unsigned q_at = tc5::smem_u32(q + (size_t)(m0 + (lane & 15)) * row_of + (lane >> 4) * 8);
    const unsigned k_at = tc5::smem_u32(page + (size_t)(half * 32 + (lane & 7) + (lane >> 4) * 8) * row_of + (lane >> 3 & 1) * 8);
    const unsigned v_at = tc5::smem_u32(page + (size_t)(half * 32 + (lane & 15)) * row_of + (lane >> 4) * 8);
    const unsigned q_piece = kTileRows * row_of * 2, page_piece = kPage * row_of * 2;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[8 * NL][4];
#pragma unroll
    for (int i = 0; i < 8 * NL; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const int pieces = 4 * hd, chunks = 4 * padded(hd), per = hd / 8;            // of sixteen bytes: of a page's keys, of its values
    // where a thread's pieces lie in a page, and go (worked out once: it takes longer than their widening)
    int k_from[2 * NL], k_to[2 * NL], v_to[2 * NL], v_lanes[2 * NL];
#pragma unroll
    for (int i = 0; i < 2 * NL; ++i) {
        const int c = tid + i * kTileThreads, rem = c % padded(hd), piece = rem & 31, lanes0 = rem / 32 * 4;
        k_from[i] = key_piece(c % kPage, c / kPage * 16, hd);
        k_to[i] = c % kPage * row_of + c / kPage * 16;
        v_to[i] = (kPage + c / padded(hd) * 16 + (piece & 3) * 4) * row_of + (piece >> 2) * per + lanes0;
        v_lanes[i] = min(4, per - lanes0);               // (the last piece of a row may have fewer)
    }
    uint4 next_k[2 * NL], next_v[2 * NL];
    float2 next_scale = make_float2(0.f, 0.f);
    bool next_there = false;
    auto fetch = [&](int b) {
        const int number = page_of(a.block_table, a.table_stride, slot, b, a.n_pages);
        next_there = number >= 0;
        if (!next_there) return;
        const signed char* line = a.pool + ((size_t)number * a.n_kv + kvh) * line_bytes(hd);
        next_scale = *scales_of(line, hd);
#pragma unroll
        for (int i = 0; i < 2 * NL; ++i) {
            const int c = tid + i * kTileThreads;
            if (c < pieces) next_k[i] = *reinterpret_cast<const uint4*>(line + k_from[i]);
            if (c < chunks) next_v[i] = *reinterpret_cast<const uint4*>(line + kPage * hd + c * 16);
        }
    };
    // a byte behind 0x4b0000 is 2^23 + 128 + a whole number
    auto wide = [](unsigned word, int e) { return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 | e)) - 8388736.f; };
    if (pg_lo + rank < mine) fetch(pg_lo + rank);
    for (int b = pg_lo + rank; b <= mine; b += ranks) {
        const bool own = b == mine;
        float2 scale = own ? make_float2(1.f, 1.f) : next_scale;
        if (PIECES == 1) scale.x *= a.scale_log2e;
        __syncthreads();                                 // (the page before has been read)
        if (!own) {
            if (!next_there) {                           // (the same for the whole block)
                if (b + ranks < mine) fetch(b + ranks);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 2 * NL; ++i) {
                const int c = tid + i * kTileThreads;
                if (c < pieces) {
                    uint4* to = reinterpret_cast<uint4*>(page + k_to[i]);
                    auto four = [&](unsigned w) { return make_uint2(pack_bf16(wide(w, 0), wide(w, 1)), pack_bf16(wide(w, 2), wide(w, 3))); };
                    const uint2 x = four(next_k[i].x), y = four(next_k[i].y), z = four(next_k[i].z), w = four(next_k[i].w);
                    to[0] = make_uint4(x.x, x.y, y.x, y.y);
                    to[1] = make_uint4(z.x, z.y, w.x, w.y);
                }
                if (c < chunks) {                        // four lanes of four keys
                    __nv_bfloat16* to = page + v_to[i];
                    const unsigned w[4] = {next_v[i].x, next_v[i].y, next_v[i].z, next_v[i].w};
                    if (per % 4 == 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<uint2*>(to + e * row_of) = make_uint2(pack_bf16(wide(w[0], e), wide(w[1], e)), pack_bf16(wide(w[2], e), wide(w[3], e)));
                    } else {                             // (rows of an odd number of pairs of lanes)
#pragma unroll
                        for (int x = 0; x < 4; x += 2)
                            if (x < v_lanes[i])
#pragma unroll
                                for (int e = 0; e < 4; ++e) *reinterpret_cast<unsigned*>(to + e * row_of + x) = pack_bf16(wide(w[x], e), wide(w[x + 1], e));
                    }
                }
            }
            if (b + ranks < mine) fetch(b + ranks);
        } else {
            for (int c = tid; c < kPage * per; c += kTileThreads) {
                const int key = c % kPage, d = c / kPage * 8;
                float x[8] = {};
                if (p0 + key < end) load_n<8>(own_row(p0 + key, 0) + d, x);
                if (PIECES > 1) {
                    unsigned top = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                    if (top >= 0x7f800000u) {
                        atomicOr(odd_scores + (key >> 5), 1u << (key & 31));
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = 0.f;
                    }
                }
                put(page + (size_t)key * row_of + d, (size_t)kPage * row_of, x);
            }
        }
        __syncthreads();
        // 16 rows by four times eight keys; the products of lower pieces by themselves, so that fewer sums of full size are cut off
        float s[4][4] = {}, low[PIECES > 1 ? 4 : 1][4] = {};
#pragma unroll 4
        for (int k = 0; k < (idle ? 0 : hd / 16); ++k) {
            unsigned x[PIECES][4];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) ldmatrix4(x[i], q_at + i * q_piece + k * 32);
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {           // (a page's keys have one piece)
                if (j > 0 && !own) break;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    unsigned y[4];
                    ldmatrix4(y, k_at + j * page_piece + c * 16 * row_of * 2 + k * 32);
#pragma unroll
                    for (int i = 0; i < PIECES - j; ++i) {
                        mma_bf16(i + j == 0 ? s[2 * c] : low[PIECES > 1 ? 2 * c : 0], x[i], y[0], y[1]);
                        mma_bf16(i + j == 0 ? s[2 * c + 1] : low[PIECES > 1 ? 2 * c + 1 : 0], x[i], y[2], y[3]);
                    }
                }
            }
        }
        if (PIECES > 1)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i / 4][i % 4] += low[PIECES > 1 ? i / 4 : 0][i % 4];
        if (PIECES > 1 && own) {                         // (left out here: at the end the rows that see such a key ask what its score is)
            const unsigned hidden = odd_scores[half] >> (2 * t);
            if (hidden != 0)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (hidden >> (i / 4 * 8 + (i & 1)) & 1) s[i / 4][i % 4] = -INFINITY;
        }
        float alpha[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = b * kPage + half * 32 + i / 2 * 8 + 2 * t + (i & 1);
                float& x = s[i / 2][2 * r + (i & 1)];
                x = key <= pos_of[r] && key >= lo_of[r] ? x * scale.x : -INFINITY;
                top = fmaxf(top, x);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[r], top), ref = now == -INFINITY ? 0.f : now;
            alpha[r] = exp2f(m[r] - ref);
            m[r] = now;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = b * kPage + half * 32 + i / 2 * 8 + 2 * t + (i & 1);
                float& x = s[i / 2][2 * r + (i & 1)];
                const float e = exp2f(x - ref);
                const bool seen = key <= pos_of[r] && key >= lo_of[r];
                x = seen ? e * scale.y : 0.f;            // (of what is not seen, whatever the scale)
                sum += seen ? e : 0.f;
            }
            l[r] = l[r] * alpha[r] + sum;                // of the thread's keys; the four threads of a row meet at the end
        }
        unsigned p[2][PIECES][4];                        // 16 rows by twice sixteen keys
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[c][i][e] = take_two(s[2 * c + e / 2][2 * (e & 1)], s[2 * c + e / 2][2 * (e & 1) + 1]);
        if (own) {                                       // the values take the keys' place
            __syncthreads();
            for (int c = tid; c < kPage * per; c += kTileThreads) {
                const int key = c % kPage, d = c / kPage * 8;
                float x[8] = {};
                if (p0 + key < end) load_n<8>(own_row(p0 + key, 1) + d, x);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    // (a probability of zero does not silence an infinity or a NaN: those are put in at the end, by the rows that see them)
                    if (!(fabsf(x[e]) < INFINITY)) {
                        x[e] = 0.f;
                        atomicOr(odd_keys + (key >> 5), 1u << (key & 31));
                    }
                put(page + (size_t)key * row_of + d, (size_t)kPage * row_of, x);
            }
            __syncthreads();
        }
        const unsigned values_at = v_at + (own ? 0u : page_piece);
#pragma unroll
        for (int d = 0; d < 4 * NL; ++d) {               // sixteen lanes at a time
            if (d * 16 >= hd || idle) break;
            float part[2][4] = {}, less[2][4] = {};
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                if (j > 0 && !own) break;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    unsigned y[4];
                    ldmatrix4_turned(y, values_at + j * page_piece + c * 16 * row_of * 2 + d * 32);
#pragma unroll
                    for (int i = 0; i < PIECES - j; ++i) {
                        mma_bf16(i + j == 0 ? part[0] : less[0], p[c][i], y[0], y[1]);
                        mma_bf16(i + j == 0 ? part[1] : less[1], p[c][i], y[2], y[3]);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[2 * d + x][e] = fmaf(acc[2 * d + x][e], alpha[e >> 1], PIECES > 1 ? part[x][e] + less[x][e] : part[x][e]);
        }
    }
    __syncthreads();
    // ---- the warps' halves and the cluster's blocks meet, a share of the rows each ----
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t == 0) {
            met_m[half][m0 + g + 8 * r] = m[r];
            met_l[half][m0 + g + 8 * r] = l[r];
        }
    }
    auto met_at = [&](int h, int row, int d) { return met + ((size_t)h * kTileRows + row) * (hd + 4) + d; };
#pragma unroll
    for (int i = 0; i < 8 * NL; ++i)
        if (i * 8 < hd)
#pragma unroll
            for (int r = 0; r < 2; ++r) *reinterpret_cast<float2*>(met_at(half, m0 + g + 8 * r, i * 8 + 2 * t)) = make_float2(acc[i][2 * r], acc[i][2 * r + 1]);
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    const int parts = 2 * ranks, share = kTileRows / ranks, last = (mine - pg_lo) % ranks;       // (whose step was the own block)
    const float4 odd_bits = ranks > 1 ? cluster_float4(tc5::smem_u32(odd_keys), last) : *reinterpret_cast<const float4*>(odd_keys);
    const unsigned long long odd = (unsigned long long)__float_as_uint(odd_bits.y) << 32 | __float_as_uint(odd_bits.x);
    const unsigned long long odd_k = PIECES > 1 ? (unsigned long long)__float_as_uint(odd_bits.w) << 32 | __float_as_uint(odd_bits.z) : 0;
    if (tid < share * parts) {                           // the parts' weights, a thread each: a row's are neighbours
        const int row = rank * share + tid / parts, k = tid % parts;
        const float mk = cluster_float(tc5::smem_u32(&met_m[k & 1][row]), k >> 1), lk = cluster_float(tc5::smem_u32(&met_l[k & 1][row]), k >> 1);
        float top = mk;
        for (int w = 1; w < parts; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        // (a part that the row saw nothing of has nothing; one whose scores were no numbers has none, which its sum tells)
        const float by = mk == top ? 1.f : exp2f(mk - (top == -INFINITY ? 0.f : top));
        float total = lk * by;
        for (int w = 1; w < parts; w *= 2) total += __shfl_xor_sync(0xffffffffu, total, w);
        weights[tid] = by / total;
    }
    __syncthreads();
    for (int i = tid; i < share * (hd / 4); i += kTileThreads) {
        const int here = i / (hd / 4), row = rank * share + here, d = i % (hd / 4) * 4, pos = t0 + row / hb;
        if (pos < start || pos >= end) continue;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
            const float* at = met_at(k & 1, row, d);
            const float4 v = ranks == 1 ? *reinterpret_cast<const float4*>(at) : cluster_float4(tc5::smem_u32(at), k >> 1);
            const float by = weights[here * parts + k];
            o[0] = fmaf(v.x, by, o[0]); o[1] = fmaf(v.y, by, o[1]); o[2] = fmaf(v.z, by, o[2]); o[3] = fmaf(v.w, by, o[3]);
        }
        T* out = reinterpret_cast<T*>(a.out) + ((size_t)(tok0 + pos - start) * a.n_heads + head0 + row % hb) * hd + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = from_f32<T>(o[e]);
    }
    // infinities and NaN of the own block, by the rows that see them: of a value they join the result; a key's leave it only where its score is
    // minus infinity (the thread that wrote a place looks at it again)
    if ((odd | odd_k) != 0)
        for (int i = tid; i < share * (hd / 4); i += kTileThreads) {
            const int row = rank * share + i / (hd / 4), d = i % (hd / 4) * 4, pos = t0 + row / hb, head = head0 + row % hb;
            if (pos < start || pos >= end) continue;
            T* out = reinterpret_cast<T*>(a.out) + ((size_t)(tok0 + pos - start) * a.n_heads + head) * hd + d;
            const T* q_row = rows + ((size_t)(tok0 + pos - start) * width + head) * hd;
            for (int k = max(p0, first_key(pos)); k <= pos; ++k) {
                float score = -INFINITY;
                if (odd_k >> (k - p0) & 1) {
                    score = 0.f;
                    for (int x = 0; x < hd; ++x) score = fmaf(to_f32(q_row[x]) * a.scale_log2e, to_f32(own_row(k, 0)[x]), score);
                }
                for (int e = 0; e < 4; ++e) {
                    const float v = to_f32(own_row(k, 1)[d + e]);
                    if (!(score == -INFINITY)) out[e] = from_f32<T>(NAN);
                    else if (odd >> (k - p0) & 1 && !(fabsf(v) < INFINITY)) out[e] = from_f32<T>(to_f32(out[e]) + v);
                }
            }
        }
    if (ranks > 1) cluster_sync();                       // what others read stays until they have
}

template <typename T, int NL>
static int launch_tile(const AttendArgs& a, int n_tokens, int max_q_len, int max_kv_len, cudaStream_t stream) {
    const int group = a.n_heads / a.n_kv, hb = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1, tb = kTileRows / hb;
    // a walk of several pages is shared by the blocks of a cluster, as far as they are resident together: three an SM with heads of up to 64
    // lanes, two of up to 128 (60 tokens behind 1,000 in float32, heads of 64: 26 us so, 35 with four; 8 single tokens behind 2,000 with
    // heads of 80: 27 us with two blocks of all the registers they want, 35 with three)
    const size_t smem = Tile<T>::smem(a.hd);
    const int at_once = blm_sm_count() * (NL == 1 ? 3 : NL == 2 ? 2 : 1);
    const int tiles = a.n_kv * (group / hb) * ((n_tokens + tb - 1) / tb + a.n_seqs - 1);
    int pages = (max_kv_len + kPage - 1) / kPage, ranks = 1;
    if (a.window > 0 && pages > a.window / kPage + 2) pages = a.window / kPage + 2;
    while (ranks < 8 && (long long)tiles * ranks * 2 <= at_once && pages >= 2 * ranks) ranks *= 2;
    const long long blocks = (long long)a.n_kv * (group / hb) * ranks * (max_q_len <= 1 ? a.n_seqs : most_blocks(n_tokens, a.n_seqs, tb));
    BLM_REQUIRE(blocks < 1ll << 31, "attention_q8: %d tokens of %d heads in one step", n_tokens, a.n_heads);
    if (cudaFuncSetAttribute(attend_tile_kernel<T, NL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return blm_fail(BLM_CUDA_ERROR, "attention_q8: %s", cudaGetErrorString(cudaGetLastError()));
    blm_launch_cluster(attend_tile_kernel<T, NL>, ranks, dim3((unsigned)blocks), dim3(kTileThreads), smem, stream, a, hb, ranks, max_q_len <= 1);
    return blm_check_launch("attention_q8");
}
template <typename T>
static int launch_tile(const AttendArgs& a, int n_tokens, int max_q_len, int max_kv_len, cudaStream_t stream) {
    return a.hd <= 64 ? launch_tile<T, 1>(a, n_tokens, max_q_len, max_kv_len, stream) : a.hd <= 128 ? launch_tile<T, 2>(a, n_tokens, max_q_len, max_kv_len, stream)
                                                                                      : launch_tile<T, 4>(a, n_tokens, max_q_len, max_kv_len, stream);
}

// ---- single tokens -----------------------------------------------------------------------------------------------------------
// One new token a sequence, bfloat16, heads of 64 or 128 lanes: a block owns (share of the sequence's pages, up to eight query heads
// of a kv head, sequence).  Its producer warp streams the pages into a ring in shared memory, one bulk copy of 8 or 16 KB each (keys,
// values and scales of the kv head), completion on mbarriers; four consumer warps, WPP of them to a page, form scores and sums with
// 16 keys (lanes) by the query heads a tensor-core tile.  What bounds it, beside the memory, is the instructions that turn bytes into
// operands, so:
//   * keys and lanes are the 16 rows of a product and the heads its 8 columns (with the heads as rows half of a product would be empty:
//     20 to 30 % slower); probabilities change their place from one product's result to the other's operand by movmatrix;
//   * a thread reads its bytes as 16-byte pieces that hold its fragments, and everything is in half precision: a byte behind 0x64 is
//     1024 + 128 + q exactly, one permutation for two numbers;
//   * of the keys the 1152 is not taken off: a score's sum starts at -1152 times the sum of its query, which is exact in what it takes
//     off and costs 2^-23 of 1152 |q| a step in 32-bit sums (1e-6 of the largest score the block's keys could have);
//   * the queries are multiplied by a power of two that brings their largest lane to 16 .. 32 (bfloat16 numbers above 2^-18 of it stay
//     exact), the scores divided by it again;
//   * the values' scale rides in the exponent: p' = 2^(score + log2 vs - m), with the maximum m taken of that sum, is at most 1, its
//     product with the whole numbers needs no scale, and the sum of the probabilities gets p' / vs.  p' is rounded to half precision
//     times 2^12 (11 bits from the largest down to 2^-26 of it).
// Warps keep their own running maximum, sum and output and merge at the end; up to eight shares of a sequence meet in their cluster, more
// in a second kernel.  The own block's keys, unrounded, are read straight from the tail and the step's rows by the four warps of the last
// share, while the first pages are on their way; their probabilities are bfloat16 numbers 2^(score - m), as large as 2^112 where a key's
// values are small.  Waits are bounded; one that runs out leaves a code in the status word.
struct TokenArgs {
    AttendArgs a;
    float* part_acc;             // [N, n_heads, n_splits, hd]
    float* part_ml;              // [N, n_heads, n_splits, 2]: maximum (base 2) and sum
    int n_splits, head_tiles, heads_a_tile, pages_per_split;
    int clustered;               // the shares of a sequence are the blocks of a cluster, and meet in it
    int* status;
};
enum { Q8_TIMEOUT_PAGE = 51, Q8_TIMEOUT_FREE = 52 };
using tc5::mbar_arrive;
using tc5::mbar_expect_tx;
using tc5::mbar_init;
using tc5::mbar_wait;
using tc5::smem_u32;

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
template <bool HALF>
__device__ __forceinline__ void mma_sync(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    if (HALF)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit numbers, a row's two a lane, transposed
__device__ __forceinline__ unsigned transposed(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}
// Bytes LO and LO + 1 of a word as two half-precision numbers, 1152 too large, and without that.
template <int LO>
__device__ __forceinline__ unsigned biased_two(unsigned word) { return __byte_perm(word, 0x64u, LO == 0 ? 0x4140 : 0x4342); }
template <int LO>
__device__ __forceinline__ unsigned two_of(unsigned word) {
    const unsigned p = biased_two<LO>(word);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&p), __float2half2_rn(1152.f));
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float ex2(float x) {          // 2^x (x = -inf gives 0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// three numbers' largest, and two sums or products with a sum at once
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ void fma_two(float& x, float& y, float by, float plus) {
    asm("{\n.reg .b64 v, b, p;\nmov.b64 v, {%0, %1};\nmov.b64 b, {%2, %2};\nmov.b64 p, {%3, %3};\nfma.rn.f32x2 v, v, b, p;\nmov.b64 {%0, %1}, v;\n}\n" : "+f"(x), "+f"(y) : "f"(by), "f"(plus));
}
__device__ __forceinline__ void add_two(float& x, float& y, float a, float b) {
    asm("{\n.reg .b64 v, w;\nmov.b64 v, {%0, %1};\nmov.b64 w, {%2, %3};\nadd.rn.f32x2 v, v, w;\nmov.b64 {%0, %1}, v;\n}\n" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}

// How many of the n_splits shares of a sequence work: one per `pages_per_split` pages of 8-bit blocks.
__host__ __device__ inline int active_splits(int n_pages, int n_splits, int pages_per_split) {
    const int want = (n_pages + pages_per_split - 1) / pages_per_split;
    return want < 1 ? 1 : (want > n_splits ? n_splits : want);
}

constexpr float kPShift = 12.f;          // probabilities are kept times 2^12

// What a warp knows of its eight heads: thread (g, t) has heads 2 t and 2 t + 1, of the sums lanes g HD / 8 + n, n = 0 .. HD / 8 - 1:
// o[n / 2][n % 2 * 2 + head].
template <int HD>
struct TokenState {
    float o[HD / 16][4], m[2], l[2];
    // the thread's largest new scores of its two heads: moves the references and gives what is to be added to a score in the exponent
    __device__ __forceinline__ void refer(float top0, float top1, float& shift0, float& shift1) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        const float now0 = fmaxf(m[0], top0), now1 = fmaxf(m[1], top1);
        const float ref0 = now0 == -INFINITY ? 0.f : now0, ref1 = now1 == -INFINITY ? 0.f : now1;
        if (__any_sync(0xffffffffu, now0 != m[0] || now1 != m[1])) {
            const float a0 = ex2(m[0] - ref0), a1 = ex2(m[1] - ref1);
            l[0] *= a0;
            l[1] *= a1;
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                o[n][0] *= a0; o[n][1] *= a1; o[n][2] *= a0; o[n][3] *= a1;
            }
        }
        m[0] = now0;
        m[1] = now1;
        shift0 = kPShift - ref0;
        shift1 = kPShift - ref1;
    }
};

constexpr int kTokenWarps = 4;           // consumers of a block
template <int HD, int WPP>
__global__ void __launch_bounds__((kTokenWarps + 1) * 32) attend_token_kernel(const TokenArgs ta) {
    constexpr int WARPS = kTokenWarps, NG = WARPS / WPP, CH = 4 / WPP;   // groups of warps, 16-key chunks of a page that a warp has
    constexpr int S = NG;                                                // pages of the ring; a stage always serves the same group
    constexpr int KS = HD / 16, PIECES = HD / 64;                        // PIECES: 16-byte pieces of a key row in a thread
    constexpr unsigned STAGE = line_bytes(HD);
    const AttendArgs& a = ta.a;
    __shared__ float2 met[8];                                            // maximum and sum of this share's heads, for the cluster
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* ring = smem_raw;                                      // [S][keys, values, scales]
    float* sm_acc = reinterpret_cast<float*>(ring);                      // [WARPS][8][HD], when the ring has been read
    float* sm_m = reinterpret_cast<float*>(ring + (size_t)S * STAGE);
    float* sm_l = sm_m + WARPS * 8;
    unsigned long long* full = reinterpret_cast<unsigned long long*>(sm_l + WARPS * 8);
    unsigned long long* empty = full + S;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, kvh = blockIdx.y / ta.head_tiles, tile = blockIdx.y % ta.head_tiles, seq = blockIdx.z;
    const int group = a.n_heads / a.n_kv, head0 = kvh * group + tile * ta.heads_a_tile, G = min(ta.heads_a_tile, group - tile * ta.heads_a_tile);
    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, WPP);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    pdl_wait();
    const int tok = a.cu_seqlens[seq], next = a.cu_seqlens[seq + 1], pos = a.start_pos[seq], slot = a.slot_of_seq[seq];
    const int key_lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0, mine = pos / kPage;
    const int pg_first = key_lo / kPage, n_pg = max(0, mine - pg_first);          // blocks in 8 bits
    const int active = active_splits(n_pg, ta.n_splits, ta.pages_per_split);
    if (next <= tok) return;                             // (the whole cluster)
    if (split >= active) {                               // (the whole block; the kernel that merges computes the same number)
        if (ta.clustered && active > 1) {
            cluster_sync();
            cluster_sync();
        }
        return;
    }
    const int per = (n_pg + active - 1) / active;
    const int pg_lo = pg_first + split * per, pg_hi = min(pg_first + n_pg, pg_lo + per);
    __syncthreads();

    if (warp == WARPS) {
        // ---- producer: page numbers 32 at a time, copies by lane 0 ----
        int s = -1, i = 0;
        unsigned phase = 0;
        bool failed = false;
        for (int base = pg_lo; base < pg_hi; base += 32) {
            const int n = min(32, pg_hi - base);
            const int my_page = lane < n ? page_of(a.block_table, a.table_stride, slot, base + lane, a.n_pages) : -1;
            for (int j = 0; j < n; ++j) {
                const int page = __shfl_sync(0xffffffffu, my_page, j);
                if (lane != 0 || failed) continue;
                if (++s == S) { s = 0; phase ^= 1; }
                if (i >= S && !mbar_wait(empty + s, phase ^ 1)) {
                    atomicCAS(ta.status, 0, Q8_TIMEOUT_FREE);
                    failed = true;
                    continue;
                }
                ++i;
                unsigned char* stage = ring + (size_t)s * STAGE;
                if (page < 0) {                          // none of the pool's: the consumers know it by a scale below zero
                    *const_cast<float2*>(scales_of(stage, HD)) = make_float2(0.f, -1.f);
                    tc5::fence_async_smem();             // (a copy may write the same place next)
                    mbar_arrive(full + s);
                    continue;
                }
                mbar_expect_tx(full + s, STAGE);
                bulk_copy(stage, a.pool + ((size_t)page * a.n_kv + kvh) * STAGE, STAGE, full + s);
            }
        }
        // every copy has landed before the ring is used otherwise or the block ends, whatever became of the consumers
        if (lane == 0)
            for (int k = max(0, i - S); k < i; ++k) mbar_wait(full + k % S, (k / S) & 1);
    } else {
        // Q as the A operand: thread t's lanes of a row are t HD / 4 .. + HD / 4, four of them a step of K
        const int width = a.n_heads + 2 * a.n_kv;
        const __nv_bfloat16* rows = reinterpret_cast<const __nv_bfloat16*>(a.rotated) + (size_t)tok * width * HD;
        unsigned qf[KS][2];
        {
            const uint4* q = reinterpret_cast<const uint4*>(rows + (size_t)(head0 + min(g, G - 1)) * HD + t * (HD / 4));
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
                const uint4 v = g < G ? q[i] : make_uint4(0u, 0u, 0u, 0u);
                qf[2 * i][0] = v.x; qf[2 * i][1] = v.y; qf[2 * i + 1][0] = v.z; qf[2 * i + 1][1] = v.w;
            }
        }
        TokenState<HD> st;
        st.m[0] = st.m[1] = -INFINITY;
        st.l[0] = st.l[1] = 0.f;
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[n][e] = 0.f;

        for (int quarter = warp; split == active - 1 && quarter < 4 && quarter * 16 <= pos % kPage; quarter += WARPS) {
            // ---- the own block: 16 of its rows, unrounded ----
            const __nv_bfloat16* found = reinterpret_cast<const __nv_bfloat16*>(a.found) + ((size_t)slot * 2 * a.n_kv + kvh) * kPage * HD;
            auto row = [&](int k, int which) -> const __nv_bfloat16* {            // k of the own block, at most pos
                if (mine * kPage + k == pos) return rows + (size_t)(a.n_heads + which * a.n_kv + kvh) * HD;
                return found + ((size_t)which * a.n_kv * kPage + k) * HD;
            };
            const int own_lo = max(0, key_lo - mine * kPage), own_hi = pos % kPage;      // the keys seen
            const int k0 = quarter * 16 + 4 * (g >> 1) + (g & 1);                        // the thread's rows: k0 and k0 + 2
            const bool seen0 = k0 <= own_hi && k0 >= own_lo, seen2 = k0 + 2 <= own_hi && k0 + 2 >= own_lo;
            const uint4* r0 = reinterpret_cast<const uint4*>(row(min(k0, own_hi), 0) + t * (HD / 4));
            const uint4* r2 = reinterpret_cast<const uint4*>(row(min(k0 + 2, own_hi), 0) + t * (HD / 4));
            // all loads before the first use: one latency
            uint4 k_of[2][KS / 2], v[HD / 64][4];        // (v: lanes g HD / 8 .. + HD / 8 of keys 4 t .. 4 t + 3)
#pragma unroll
            for (int j = 0; j < KS / 2; ++j) {
                k_of[0][j] = r0[j];
                k_of[1][j] = r2[j];
            }
            bool sees[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = quarter * 16 + 4 * t + e;
                sees[e] = key <= own_hi && key >= own_lo;
                const uint4* from = reinterpret_cast<const uint4*>(row(min(key, own_hi), 1) + g * (HD / 8));
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) v[j][e] = from[j];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < HD / 64; ++j)
                    if (!sees[e]) v[j][e] = make_uint4(0u, 0u, 0u, 0u);
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS / 2; ++j) {
                const uint4 x = seen0 ? k_of[0][j] : make_uint4(0u, 0u, 0u, 0u), y = seen2 ? k_of[1][j] : make_uint4(0u, 0u, 0u, 0u);
                mma_sync<false>(c, x.x, y.x, x.y, y.y, qf[2 * j][0], qf[2 * j][1]);
                mma_sync<false>(c, x.z, y.z, x.w, y.w, qf[2 * j + 1][0], qf[2 * j + 1][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = (e < 2 ? seen0 : seen2) ? c[e] * a.scale_log2e : -INFINITY;
            // what a key's values weigh, as log2 of 2^-7 of the largest magnitude among them: the reference is one of score times value here
            // too, so that neither these rows nor the pages leave the range of the pages' half precision (with the scores alone, values of 1e-8
            // behind pages were off by a tenth).  Two keys a word, their magnitudes' bits.
            unsigned size[2];
            auto look = [&](bool all) {                  // (a value that is no number says nothing about the others)
                size[0] = size[1] = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned top = 0;                    // of two magnitudes' bits at once
#pragma unroll
                    for (int j = 0; j < HD / 64; ++j) {
                        uint4 x = v[j][e];
                        if (!all) x = make_uint4(x.x & ~odd_two(x.x), x.y & ~odd_two(x.y), x.z & ~odd_two(x.z), x.w & ~odd_two(x.w));
                        top = __vmaxu2(__vmaxu2(top, x.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(x.y & 0x7fff7fffu, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu));
                    }
                    size[e >> 1] |= max(top & 0xffffu, top >> 16) << (16 * (e & 1));
                }
            };
            look(true);
            if (__any_sync(0xffffffffu, odd_two(size[0]) != 0 || odd_two(size[1]) != 0)) look(false);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) size[w] = __vmaxu2(size[w], __shfl_xor_sync(0xffffffffu, size[w], x));
                size[w] = __shfl_sync(0xffffffffu, size[w], g >> 1) >> (16 * (g & 1)) & 0xffffu;      // of keys k0 and k0 + 2
            }
            const float lv0 = (float)max((int)(size[0] >> 7) - 134, -100), lv2 = (float)max((int)(size[1] >> 7) - 134, -100);
            float shift0, shift1;
            st.refer(fmaxf(c[0] + lv0, c[2] + lv2), fmaxf(c[1] + lv0, c[3] + lv2), shift0, shift1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = ex2(c[e] + (e & 1 ? shift1 : shift0));
                st.l[e & 1] += c[e];
            }
            const unsigned b0 = transposed(pack_bf16(c[0], c[1])), b1 = transposed(pack_bf16(c[2], c[3]));
#pragma unroll
            for (int j = 0; j < HD / 64; ++j)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    auto word = [&](const uint4& u) { return n == 0 ? u.x : n == 1 ? u.y : n == 2 ? u.z : u.w; };
                    const unsigned w0 = word(v[j][0]), w1 = word(v[j][1]), w2 = word(v[j][2]), w3 = word(v[j][3]);
                    mma_sync<false>(st.o[4 * j + n], __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410), __byte_perm(w2, w3, 0x7632), b0, b1);
                }
        }

        // the queries in half precision: times a power of two that brings the row's largest lane to 16 .. 32
        float start0, start1, to_log2_0, to_log2_1;         // of the thread's two heads
        {
            float q[KS][4], top = 0.f, sum = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    q[k][2 * h] = __uint_as_float(qf[k][h] << 16);
                    q[k][2 * h + 1] = __uint_as_float(qf[k][h] & 0xffff0000u);
                    top = fmaxf(top, fmaxf(fabsf(q[k][2 * h]), fabsf(q[k][2 * h + 1])));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int exponent = (int)(__float_as_uint(top) >> 23);               // 0: zero or next to it; 255: an infinity
            const int by = exponent == 0 || exponent == 255 ? 127 : min(254, max(1, 258 - exponent));
            const float factor = __uint_as_float((unsigned)by << 23);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const __half2 v = __floats2half2_rn(q[k][2 * h] * factor, q[k][2 * h + 1] * factor);
                    qf[k][h] = *reinterpret_cast<const unsigned*>(&v);
                    const float2 f = __half22float2(v);
                    sum += f.x + f.y;
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            // (until here the lanes of a quad have head g)
            start0 = -1152.f * __shfl_sync(0xffffffffu, sum, 8 * t);
            start1 = -1152.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            to_log2_0 = a.scale_log2e / __shfl_sync(0xffffffffu, factor, 8 * t);
            to_log2_1 = a.scale_log2e / __shfl_sync(0xffffffffu, factor, 8 * t + 4);
        }

        // ---- the pages: this warp's group takes every NG-th, the warp CH chunks of 16 keys of each ----
        const int grp = warp / WPP, part = warp % WPP;
        const int s = grp;
        unsigned phase = 1;
        for (int pg = pg_lo + grp; pg < pg_hi; pg += NG) {
            phase ^= 1;
            if (!mbar_wait(full + s, phase)) {
                if (lane == 0) atomicCAS(ta.status, 0, Q8_TIMEOUT_PAGE);
                break;
            }
            const unsigned char* keys = ring + (size_t)s * STAGE;
            const unsigned char* values = keys + kPage * HD;
            const float2 scale = *scales_of(keys, HD);
            // (a block whose values are all next to zero: any scale will do; a NaN stays one)
            const float vs = scale.y < 0x1p-100f ? 0x1p-100f : scale.y, lv = __log2f(vs);
            // (a block of keys with an infinity: its numbers are zeros, whose score's sum need not come out as exactly 0 here; times an infinity it
            // must be none all the same, not minus infinity)
            const float ks = fmaf(scale.x, 0.f, scale.x), f0 = to_log2_0 * ks, f1 = to_log2_1 * ks;
            float sc[CH][4], top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                // the thread's rows of the chunk: keys k0 and k0 + 2
                float (&c)[4] = sc[ch];
                c[0] = c[2] = start0;
                c[1] = c[3] = start1;
                const int k0 = (part * CH + ch) * 16 + 4 * (g >> 1) + (g & 1);
                const uint4* kr = reinterpret_cast<const uint4*>(keys + k0 * HD);
#pragma unroll
                for (int j = 0; j < PIECES; ++j) {
                    const uint4 x = kr[(t * PIECES + j) ^ (g & 1)], y = kr[2 * HD / 16 + ((t * PIECES + j) ^ (g & 1))];
                    const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_sync<true>(c, biased_two<0>(xw[i]), biased_two<0>(yw[i]), biased_two<2>(xw[i]), biased_two<2>(yw[i]), qf[4 * j + i][0], qf[4 * j + i][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = fmaf(c[e], e & 1 ? f1 : f0, lv);
                top0 = fmaxf(top0, fmaxf(c[0], c[2]));
                top1 = fmaxf(top1, fmaxf(c[1], c[3]));
            }
            if (pg * kPage < key_lo) {                   // the window's edge
                top0 = top1 = -INFINITY;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (pg * kPage + (part * CH + ch) * 16 + 4 * (g >> 1) + (g & 1) + (e & 2) < key_lo) sc[ch][e] = -INFINITY;
                        if (e & 1) top1 = fmaxf(top1, sc[ch][e]); else top0 = fmaxf(top0, sc[ch][e]);
                    }
            }
            if (!(scale.y < 0.f)) {
                float shift0, shift1, sum0 = 0.f, sum1 = 0.f;
                st.refer(top0, top1, shift0, shift1);
                const float to_sum = 1.f / vs;
                const uint4* vr = reinterpret_cast<const uint4*>(values + part * CH * (16 * HD)) + lane;
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) {
                    const float p0 = ex2(sc[ch][0] + shift0), p1 = ex2(sc[ch][1] + shift1), p2 = ex2(sc[ch][2] + shift0), p3 = ex2(sc[ch][3] + shift1);
                    sum0 += p0 + p2;
                    sum1 += p1 + p3;
                    const unsigned b0 = transposed(pack_half(p0, p1)), b1 = transposed(pack_half(p2, p3));
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) {
                        const uint4 v = vr[(ch * (HD / 32) + j) * 32];
                        mma_sync<true>(st.o[2 * j], two_of<0>(v.x), two_of<0>(v.y), two_of<2>(v.x), two_of<2>(v.y), b0, b1);
                        mma_sync<true>(st.o[2 * j + 1], two_of<0>(v.z), two_of<0>(v.w), two_of<2>(v.z), two_of<2>(v.w), b0, b1);
                    }
                }
                st.l[0] = fmaf(sum0, to_sum, st.l[0]);   // this thread's share
                st.l[1] = fmaf(sum1, to_sum, st.l[1]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + s);
        }
#pragma unroll
        for (int x = 4; x < 32; x *= 2) {
            st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], x);
            st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], x);
        }
        if (g == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) { sm_m[warp * 8 + 2 * t + h] = st.m[h]; sm_l[warp * 8 + 2 * t + h] = st.l[h]; }
        }
        // the ring is free when all consumers and the producer are here (named barrier: all threads of the block)
        asm volatile("bar.sync 1, %0;\n" ::"r"((WARPS + 1) * 32) : "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < HD / 16; n += 2)
                *reinterpret_cast<float4*>(sm_acc + (warp * 8 + 2 * t + h) * HD + g * (HD / 8) + 2 * n) =
                    make_float4(st.o[n][h], st.o[n][2 + h], st.o[n + 1][h], st.o[n + 1][2 + h]);
    }
    if (warp == WARPS) asm volatile("bar.sync 1, %0;\n" ::"r"((WARPS + 1) * 32) : "memory");
    __syncthreads();
    const bool meet = ta.clustered && active > 1;
    for (int i = tid; i < G * HD; i += blockDim.x) {
        const int h = i / HD, d = i % HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sm_m[w * 8 + h]);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = ex2(sm_m[w * 8 + h] - ref);
            l += sm_l[w * 8 + h] * f;
            o += sm_acc[(w * 8 + h) * HD + d] * f;
        }
        const size_t row = (size_t)tok * a.n_heads + head0 + h;
        if (active == 1) {
            reinterpret_cast<__nv_bfloat16*>(a.out)[row * HD + d] = __float2bfloat16_rn(o / l);
        } else if (meet) {
            sm_acc[h * HD + d] = o;                      // (no other thread reads or writes lane d of head h)
            if (d == 0) met[h] = make_float2(m, l);
        } else {
            const size_t part = row * ta.n_splits + split;
            ta.part_acc[part * HD + d] = o;
            if (d == 0) { ta.part_ml[part * 2] = m; ta.part_ml[part * 2 + 1] = l; }
        }
    }
    if (!meet) return;
    // the cluster's shares: some of the heads each, four lanes a thread, all reads before the first use
    cluster_sync();
    const int heads = (G - split + active - 1) / active;
    for (int i = tid; i < heads * (HD / 4); i += blockDim.x) {
        const int h = split + i / (HD / 4) * active, d = i % (HD / 4) * 4;
        float m[8], l[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < active) {
                m[k] = cluster_float(smem_u32(&met[h].x), k);
                l[k] = cluster_float(smem_u32(&met[h].y), k);
                v[k] = cluster_float4(smem_u32(sm_acc + h * HD + d), k);
            }
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < active) top = fmaxf(top, m[k]);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < active) {
                const float w = ex2(m[k] - ref);
                total = fmaf(l[k], w, total);
                o.x = fmaf(v[k].x, w, o.x); o.y = fmaf(v[k].y, w, o.y); o.z = fmaf(v[k].z, w, o.z); o.w = fmaf(v[k].w, w, o.w);
            }
        const float by = 1.f / total;
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)tok * a.n_heads + head0 + h) * HD + d) =
            make_uint2(pack_bf16(o.x * by, o.y * by), pack_bf16(o.z * by, o.w * by));
    }
    cluster_sync();                                      // what others read stays until they have
}

// Merges the shares: a block per (sequence, head); 512 / HD groups of threads take shares in turn, four lanes a thread.
template <int HD>
__global__ void __launch_bounds__(128) merge_kernel(const TokenArgs ta) {
    constexpr int LANES = HD / 4, GROUPS = 128 / LANES;
    const AttendArgs& a = ta.a;
    __shared__ float weight[64];
    __shared__ float2 red[2];
    __shared__ float4 sums[128];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, head = blockIdx.x, seq = blockIdx.y, tok = a.cu_seqlens[seq], next = a.cu_seqlens[seq + 1], pos = a.start_pos[seq];
    const int key_lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const int active = active_splits(max(0, pos / kPage - key_lo / kPage), ta.n_splits, ta.pages_per_split);
    if (next <= tok || active == 1) return;              // written by the block itself
    const size_t row = (size_t)tok * a.n_heads + head;
    const float4* acc = reinterpret_cast<const float4*>(ta.part_acc + row * ta.n_splits * HD) + tid % LANES;
    if (tid < 64) {                                      // two warps: maximum and sum of up to 64 shares
        const float2 x = tid < active ? reinterpret_cast<const float2*>(ta.part_ml)[row * ta.n_splits + tid] : make_float2(-INFINITY, 0.f);
        const float m = warp_max(x.x), ref = m == -INFINITY ? 0.f : m;
        const float w = ex2(x.x - ref), l = warp_sum(x.y * w);
        weight[tid] = w;
        if (tid % 32 == 0) red[tid / 32] = make_float2(m, l);
    }
    __syncthreads();
    const float m = fmaxf(red[0].x, red[1].x), ref = m == -INFINITY ? 0.f : m;
    const float f0 = ex2(red[0].x - ref), f1 = ex2(red[1].x - ref), l = red[0].y * f0 + red[1].y * f1;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = tid / LANES; z < active; z += GROUPS) {
        const float w = weight[z] * (z < 32 ? f0 : f1);
        const float4 v = acc[(size_t)z * LANES];
        o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
    }
    sums[tid] = o;
    __syncthreads();
    if (tid >= LANES) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
        const float4 v = sums[i * LANES + tid];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    const float by = 1.f / l;
    uint2 w;
    w.x = pack_bf16(o.x * by, o.y * by);
    w.y = pack_bf16(o.z * by, o.w * by);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + row * HD + tid * 4) = w;
}

// The plan of a step of single tokens, the same for the caller that provides the scratch and for the launch.
struct TokenPlan { int splits, pages_per_split, wpp, head_tiles, heads_a_tile; };
constexpr int kClusterShares = 8;        // so many shares, the blocks of a cluster, meet in it; more in a second kernel
static TokenPlan plan_tokens(int n_seqs, int n_heads, int n_kv, int hd, int max_kv_len, int window) {
    TokenPlan p;
    const int group = n_heads / n_kv, sms = blm_sm_count();
    p.head_tiles = (group + 7) / 8;
    p.heads_a_tile = (group + p.head_tiles - 1) / p.head_tiles;
    int pages = (max_kv_len + kPage - 1) / kPage;
    if (window > 0 && pages > window / kPage + 2) pages = window / kPage + 2;
    if (pages < 1) pages = 1;
    const int rows = n_seqs * n_kv * p.head_tiles;       // blocks of an unsplit step
    // Walks are cut, as far as the shares' blocks are resident together (three of heads of 128 an SM, four of 64: one block more than that
    // is a second turn): into up to eight of two pages or more, which meet in a cluster, and long ones into shares of eight pages, which
    // meet in a second kernel.  Measured, heads of 128, 32 to 8: one sequence of 500, 2,000, 4,000 tokens 6.0, 7.0, 9.4 us (with shares of
    // eight pages and the second kernel 6.9, 10.3, 11.4); 8 of 2,000 14.0 in five or six shares, 19.8 in seven, which are 448 blocks;
    // 32 of 1,000 20.0 in one, 27 in two; one of 32,000 20.1 in 55 and 20.5 in 37.
    const int eights = (pages + 7) / 8, twos = (pages + 1) / 2, to_fill = (hd == 128 ? 3 : 4) * sms / rows;
    const int by_length = eights > kClusterShares ? eights : twos < kClusterShares ? twos : kClusterShares;
    p.splits = by_length < to_fill ? by_length : to_fill;
    if (p.splits > 64) p.splits = 64;
    if (p.splits < 1) p.splits = 1;
    const int blocks = rows * p.splits, each = (pages + p.splits - 1) / p.splits;
    p.pages_per_split = blocks > 2 * sms ? each : 1;
    // Four warps with a page each and a ring of four, three (heads of 128 lanes) or four blocks an SM; where three an SM are too few for
    // all the blocks of heads of 128, two warps to a page and a ring of two pages, four an SM.  Measured, 64 sequences of 1,000 tokens
    // with heads of 128: 30.4 us against 37.0; 8 of 8,000: 30.6 against 36.9.  Eight warps a block: 39.3 and 32.6 us.
    p.wpp = hd == 128 && blocks > 3 * sms ? 2 : 1;
    return p;
}

template <int HD, int WPP>
static int launch_tokens_as(const TokenArgs& ta, cudaStream_t stream) {
    const dim3 grid(ta.n_splits, ta.a.n_kv * ta.head_tiles, ta.a.n_seqs);
    constexpr size_t smem = (size_t)kTokenWarps / WPP * (line_bytes(HD) + 16) + (size_t)kTokenWarps * 8 * 2 * 4;
    static bool opted_in[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !opted_in[dev]) {
        if (cudaFuncSetAttribute(attend_token_kernel<HD, WPP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "attention_q8: %s", cudaGetErrorString(cudaGetLastError()));
        if (dev >= 0 && dev < 64) opted_in[dev] = true;
    }
    blm_launch_cluster(attend_token_kernel<HD, WPP>, ta.clustered ? ta.n_splits : 1, grid, dim3((kTokenWarps + 1) * 32), smem, stream, ta);
    if (ta.n_splits > 1 && !ta.clustered) blm_launch_dependent(merge_kernel<HD>, dim3(ta.a.n_heads, ta.a.n_seqs), dim3(128), 0, stream, ta);
    return blm_check_launch("attention_q8");
}
// bfloat16 steps of single tokens with heads of 64 or 128 lanes
static bool tokens_take(int dtype, int hd, int max_q_len, int n_seqs, int n_kv, int n_heads) {
    return dtype == BLM_BF16 && (hd == 64 || hd == 128) && max_q_len == 1 && n_seqs <= 65535 && (n_heads / n_kv + 7) / 8 * n_kv <= 65535;
}

// ---- several tokens ------------------------------------------------------------------------------------------------------
// bfloat16 portions with heads of 64 or 128 lanes, on tcgen05.  A block owns the queries of one 64-position block of a sequence for up to
// four heads of a kv head, in one or two tiles of 128 rows (two heads by 64 positions), and walks the sequence's blocks: those before its
// own in 8 bits, unmasked but for a window's edge, then its own, unrounded and causal.  So every border of a page is a border of the mask.
//   warp 13 copies pages (one bulk copy each: keys, values, scales) into a ring of three;
//   warps 8 .. 11 turn a page into operands, once for both tiles: keys [64][D] and values transposed, [D][64], bfloat16 with the 128-byte
//     swizzle, into rings of three each; a byte q + 128 in sixteen bits is the bfloat16 number (q + 128) 2^-133, and one subtraction makes
//     it q 2^-133: two instructions for two numbers.  The values' rows stand in an order that keeps their eight-byte writes to two a bank;
//   warp 12 issues S = Q K^T and O += P V of both tiles.  Q lies in tensor memory (as a second operand in shared memory its
//     reads, 32 KB a page and tile, would cost more than the products);
//   warps 0 .. 7 are the softmax, a row a thread: Q times a power of two that brings the row's largest lane to 2^60 (the keys' 2^-133 has to
//     meet ordinary numbers), scores times the keys' scale, a reference maximum m of score + log2 vs (vs: the values' scale; 2^-21 of the own
//     block) that moves when one exceeds it by 2^8, probabilities 2^(score + log2 vs - m + 112), of the own block 2^(score - 21 - m), rounded
//     to bfloat16, over the scores' columns.  So they stay below 2^121 whatever the values' size, and their products with values of about
//     1e-20 to 1e28 above 2^-126 down to probabilities of 2^-20.
// A tile's scores of the next page are issued behind its product of this one, by the same warp, so one set of columns does.  Measured, a
// page takes 2,200 cycles: a tile's softmax 1,400 (max, exponent and sum in pairs) and its product and next scores 730, one after the
// other, the two tiles half a page apart; products alone would take 1,024, exponentials as much.  (Two sets of columns for the scores, with
// the queries in shared memory to make room, took as long: 2,100; sixteen softmax warps of half a row each 2,300.)  The products are issued
// by a whole warp: behind `lane == 0`, where what an instruction needs is not known to be one number for the warp, each took 65 cycles to
// issue and each wait 400, and a page 2,900.  2,048 tokens, 32 heads of 128 to 8: 49 us (705 TFLOP/s).
constexpr int kPromptThreads = 14 * 32, kPromptStages = 3;
enum { Q8_TIMEOUT_PROMPT = 55 };
struct PromptArgs {
    AttendArgs a;
    int head_groups, heads_a_group;      // of a kv head's queries: at most four heads each
    int ranks;                           // blocks of a cluster, which share a walk
    int* status;
};
template <int HD> struct Prompt {
    static constexpr int kTile = 64 * HD * 2;                                // bytes of a page's keys (or values) as operands
    static constexpr int kRaw = (line_bytes(HD) + 127) / 128 * 128;
    static constexpr int kRows = 256 * HD * 2;                               // queries on their way in, sums on their way out
    static constexpr int kSmem = kPromptStages * (2 * kTile + kRaw) + kRows + 4 * 16 + 24 * 8 + 16 + 1024;
};
// two bytes of a word as two bfloat16 numbers, (byte - 128) 2^-133
template <int LO>
__device__ __forceinline__ unsigned tiny_two(unsigned word) {
    const unsigned p = __byte_perm(word, 0u, LO == 0 ? 0x4140 : 0x4342), less = 0x00800080u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&p), *reinterpret_cast<const __nv_bfloat162*>(&less));
    return *reinterpret_cast<const unsigned*>(&v);
}

template <int HD>
__global__ void __launch_bounds__(kPromptThreads, 1) attend_prompt_kernel(const PromptArgs pa) {
    using P = Prompt<HD>;
    constexpr int KS = kPromptStages;
    const AttendArgs& a = pa.a;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* keys = smem;                                              // [KS][HD / 64][64 keys][128 bytes]
    unsigned char* values = keys + KS * P::kTile;                            // [KS][HD lanes][128 bytes: 64 keys]
    unsigned char* raw = values + KS * P::kTile;                             // [KS][page]
    unsigned char* staged = raw + KS * P::kRaw;                              // [8 warps][32 rows][HD], the 16-byte pieces of row r at c ^ (r & 7)
    float4* scales = reinterpret_cast<float4*>(staged + P::kRows);           // [4] of the pages in the works: what the softmax makes of their scales
    unsigned long long* raw_full = reinterpret_cast<unsigned long long*>(scales + 4);
    unsigned long long* raw_free = raw_full + KS;
    unsigned long long* k_full = raw_free + KS;
    unsigned long long* k_free = k_full + KS;
    unsigned long long* v_full = k_free + KS;
    unsigned long long* v_free = v_full + KS;
    unsigned long long* s_full = v_free + KS;                                // [2] a tile's scores are formed
    unsigned long long* p_full = s_full + 2;                                 // [2] its probabilities are written
    unsigned long long* q_full = p_full + 2;
    unsigned long long* o_done = q_full + 1;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(o_done + 1);
    unsigned* odd_values = tmem_slot + 1;                                    // [2] bits: keys of the own block whose values hold an infinity or a NaN
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int ranks = pa.ranks, rank = blockIdx.x % ranks, n_groups = a.n_kv * pa.head_groups, kv_group = blockIdx.x / ranks % n_groups;
    const int kvh = kv_group / pa.head_groups, hg = kv_group % pa.head_groups;
    const int group = a.n_heads / a.n_kv, head0 = kvh * group + hg * pa.heads_a_group;
    const int G = min(pa.heads_a_group, group - hg * pa.heads_a_group), tiles = (G + 1) / 2;
    if (threadIdx.x == 0) {
        for (int s = 0; s < KS; ++s) {
            mbar_init(raw_full + s, 1);
            mbar_init(raw_free + s, 4);
            mbar_init(k_full + s, 4);
            mbar_init(k_free + s, 1);
            mbar_init(v_full + s, 4);
            mbar_init(v_free + s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
        }
        mbar_init(q_full, 4 * tiles);
        mbar_init(o_done, 1);
        odd_values[0] = odd_values[1] = 0u;
        tc5::mbar_init_fence();
    }
    if (warp == 12) tc5::tmem_alloc(tmem_slot, 512);      // (while the kernel before ends)
    pdl_wait();
    int from_last;
    const int found = find_block(a.cu_seqlens, a.start_pos, a.n_seqs, kPage, blockIdx.x / ranks / n_groups, from_last);
    const bool none_here = found < 0;                    // (the whole cluster)
    auto one = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };               // (one number for a warp: it need not have a register in each thread)
    const int seq = one(max(found, 0)), tok0 = one(a.cu_seqlens[seq]), start = one(a.start_pos[seq]), slot = one(a.slot_of_seq[seq]);
    const int end = start + one(a.cu_seqlens[seq + 1]) - tok0, mine = (end - 1) / kPage - one(from_last);
    const int p0 = mine * kPage;
    auto first_key = [&](int pos) { return a.window > 0 ? max(0, pos + 1 - a.window) : 0; };
    // this block's share of the walk (some may have none); the last step of the last is the own block
    const int pg_first = first_key(max(start, p0)) / kPage, share = max(1, (mine - pg_first + ranks) / ranks);
    const int pg_lo = pg_first + rank * share, steps = max(0, min(share, mine + 1 - pg_lo)), own_rank = (mine - pg_first) / share;
    const int own_step = rank == own_rank ? steps - 1 : steps;
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    pdl_launch_dependents();                              // (not before this block has its tensor memory: the next kernel may take some too)
    if (none_here) {
        if (warp == 12) tc5::tmem_free(*tmem_slot, 512);
        return;
    }
    // a tile's columns: 64 of scores (and probabilities), HD of sums, HD / 2 of queries
    const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);                 // (one number for a warp: what the products are issued with)
    constexpr unsigned kTileCols = 256, kOCol = 64, kQCol = 64 + HD;
    const int width = a.n_heads + 2 * a.n_kv;
    const __nv_bfloat16* rows = reinterpret_cast<const __nv_bfloat16*>(a.rotated);
    // where the cluster's blocks leave their sums, over the rings: [256 rows][HD] with row r's 16-byte pieces at c ^ (r & 7), then maxima and sums
    static_assert(256 * (HD + 2) * 4 <= KS * (2 * P::kTile + P::kRaw), "room for the sums");
    auto met_at = [&](int row, int c) { return reinterpret_cast<float4*>(smem + row * (HD * 4) + ((c ^ (row & 7)) << 4)); };
    float* met_m = reinterpret_cast<float*>(smem + 256 * HD * 4);
    float* met_l = met_m + 256;
    auto gave_up = [&] { atomicCAS(pa.status, 0, Q8_TIMEOUT_PROMPT); };

    if (warp == 13) {
        // ---- pages ----
        int i = 0;
        bool failed = false;
        for (int base = pg_lo; base < pg_lo + own_step; base += 32) {
            const int count = min(32, pg_lo + own_step - base);
            const int my_page = lane < count ? page_of(a.block_table, a.table_stride, slot, base + lane, a.n_pages) : -1;
            for (int j = 0; j < count; ++j) {
                const int page = __shfl_sync(0xffffffffu, my_page, j);
                if (lane != 0 || failed) continue;
                const int s = i % KS;
                if (i >= KS && !mbar_wait(raw_free + s, (i / KS - 1) & 1)) { gave_up(); failed = true; continue; }
                ++i;
                unsigned char* stage = raw + s * P::kRaw;
                if (page < 0) {                          // none of the pool's: known by a scale below zero
                    *const_cast<float2*>(scales_of(stage, HD)) = make_float2(0.f, -1.f);
                    tc5::fence_async_smem();             // (a copy may write the same place next)
                    mbar_arrive(raw_full + s);
                    continue;
                }
                mbar_expect_tx(raw_full + s, line_bytes(HD));
                bulk_copy(stage, a.pool + ((size_t)page * a.n_kv + kvh) * line_bytes(HD), line_bytes(HD), raw_full + s);
            }
        }
        if (lane == 0)
            for (int k = max(0, i - KS); k < i; ++k) mbar_wait(raw_full + k % KS, (k / KS) & 1);     // nothing is on its way when the block ends
    } else if (warp == 12) {
        // ---- products ----
        {
            constexpr unsigned kScores = tc5::instruction(64), kSums = tc5::instruction(HD);
            const unsigned long long k_desc = tc5::operand(keys, 2, 1024), v_desc = tc5::operand(values, 2, 1024);
            auto scores = [&](int i, int j) {
                if (tc5::elect()) {
                const unsigned long long kd = k_desc + (unsigned)((j % KS) * (P::kTile >> 4));
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    tc5::mma_ts(tmem + i * kTileCols, tmem + i * kTileCols + kQCol + 8 * k, kd + (unsigned)((k >> 2) * (8192 >> 4) + 2 * (k & 3)), kScores, k > 0);
                tc5::commit(s_full + i);
                if (i == tiles - 1) tc5::commit(k_free + j % KS);
                }
            };
            bool ok = mbar_wait(q_full, 0) && (steps == 0 || mbar_wait(k_full, 0));
            if (ok && steps > 0) {
                tc5::fence_after();
                for (int i = 0; i < tiles; ++i) scores(i, 0);
            }
            for (int j = 0; j < steps && ok; ++j) {
                const int s = j % KS;
                for (int i = 0; i < tiles && ok; ++i) {
                    ok = mbar_wait(p_full + i, j & 1) && (i > 0 || mbar_wait(v_full + s, (j / KS) & 1));
                    if (!ok) break;
                    tc5::fence_after();
                    if (tc5::elect()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc5::mma_ts(tmem + i * kTileCols + kOCol, tmem + i * kTileCols + 8 * k, v_desc + (unsigned)(s * (P::kTile >> 4) + 2 * k), kSums, j > 0 || k > 0);
                    if (i == tiles - 1) tc5::commit(v_free + s);
                    }
                    __syncwarp();
                    if (j + 1 == steps) continue;
                    ok = i > 0 || mbar_wait(k_full + (j + 1) % KS, ((j + 1) / KS) & 1);
                    if (!ok) break;
                    tc5::fence_after();
                    scores(i, j + 1);
                }
            }
            if (!ok && lane == 0) gave_up();
            if (tc5::elect()) tc5::commit(o_done);                         // when all products so far are over
        }
    } else if (warp >= 8) {
        // ---- operands ----
        const int me = threadIdx.x - 256, cw = warp - 8;
        bool ok = true;
        for (int j = 0; j < steps && ok; ++j) {
            const int s = j % KS, parity = (j / KS - 1) & 1;
            const bool own = j == own_step;
            unsigned char* kt = keys + s * P::kTile;
            unsigned char* vt = values + s * P::kTile;
            const unsigned char* page = raw + s * P::kRaw;
            // row r of the own block: from the step, from what the step found, or none
            auto own_row = [&](int r, int which) -> const __nv_bfloat16* {
                const int pos = p0 + r;
                if (pos >= end) return nullptr;
                if (pos >= start) return rows + ((size_t)(tok0 + pos - start) * width + a.n_heads + which * a.n_kv + kvh) * HD;
                return reinterpret_cast<const __nv_bfloat16*>(a.found) + ((((size_t)seq * 2 + which) * a.n_kv + kvh) * kPage + r) * HD;
            };
            if (!own && !mbar_wait(raw_full + s, (j / KS) & 1)) { ok = false; break; }
            const float2 scale = own ? make_float2(1.f, 1.f) : *scales_of(page, HD);
            const bool none = scale.y < 0.f;
            // a thread's pieces: of the keys sixteen lanes, four pieces of a 64-lane half by eight keys a warp; of the values four lanes of four keys
            constexpr int kPieces = HD / 32;
            auto key_at = [&](int i, int& half, int& r) {
                const int at = i * 4 + cw;
                half = HD == 128 ? at & 1 : 0;
                r = (HD == 128 ? at >> 1 : at) * 8 + (lane >> 2);
            };
            if (j >= KS && !mbar_wait(k_free + s, parity)) { ok = false; break; }
            if (own || none) {
                constexpr int kEach = HD / 16;           // (all loads before the first use: one latency, not eight)
                uint4 v[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int r = (me + i * 128) / (HD / 8), c = me % (HD / 8);
                    const __nv_bfloat16* from = own ? own_row(r, 0) : nullptr;
                    v[i] = from ? reinterpret_cast<const uint4*>(from)[c] : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int r = (me + i * 128) / (HD / 8), c = me % (HD / 8);
                    *reinterpret_cast<uint4*>(kt + (c >> 3) * 8192 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    int half, r;
                    key_at(i, half, r);
                    const uint4 v = *reinterpret_cast<const uint4*>(page + key_piece(r, (half * 4 + (lane & 3)) * 16, HD));
                    unsigned char* to = kt + half * 8192 + r * 128;
                    const int c = (lane & 3) * 2;
                    *reinterpret_cast<uint4*>(to + ((c ^ (r & 7)) << 4)) = make_uint4(tiny_two<0>(v.x), tiny_two<2>(v.x), tiny_two<0>(v.y), tiny_two<2>(v.y));
                    *reinterpret_cast<uint4*>(to + (((c + 1) ^ (r & 7)) << 4)) = make_uint4(tiny_two<0>(v.z), tiny_two<2>(v.z), tiny_two<0>(v.w), tiny_two<2>(v.w));
                }
            }
            if (me == 0) {
                // Scores are multiplied by the first number (times the row's own).  The third is the log2 of the values' scale, which the reference
                // is taken with; of the own block, whose values have none and whose probabilities leave 2^133 smaller, -21, so that they stay
                // below 2^8 and that the block seldom moves the reference (0 for it: 2,048 tokens 49.5 us instead of 48.9).  Their sum, the
                // pages' times 2^-112, counts the fourth times, in units of 2^10.  (A block whose values are all next to zero: any scale will
                // do.)  The second is below zero for a page that is none.
                const float vs = scale.y < 0x1p-100f ? 0x1p-100f : scale.y;
                scales[j & 3] = own ? make_float4(0x1p-67f, 1.f, -21.f, 0x1p11f) : make_float4(0x1p66f * scale.x, scale.y, __log2f(vs), 0x1p-10f / vs);
            }
            tc5::fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full + s);
            if (j >= KS && !mbar_wait(v_free + s, parity)) { ok = false; break; }
            // the value of lane d stands in row d % (HD / 8) * 8 + d / (HD / 8)
            if (own || none) {
                constexpr int kEach = HD / 64;
                uint4 v[kEach][4];
#pragma unroll
                for (int i = 0; i < kEach; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __nv_bfloat16* from = own ? own_row((me + i * 128) / (HD / 8) * 4 + e, 1) : nullptr;
                        v[i][e] = from ? reinterpret_cast<const uint4*>(from)[me % (HD / 8)] : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int k = (me + i * 128) / (HD / 8) * 4, d = me % (HD / 8) * 8;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // (a probability of zero does not silence an infinity or a NaN: those are put in at the end, by the rows that see them)
                        uint4& u = v[i][e];
                        const uint4 odd = make_uint4(odd_two(u.x), odd_two(u.y), odd_two(u.z), odd_two(u.w));
                        if (odd.x | odd.y | odd.z | odd.w) {
                            u = make_uint4(u.x & ~odd.x, u.y & ~odd.y, u.z & ~odd.z, u.w & ~odd.w);
                            atomicOr(odd_values + ((k + e) >> 5), 1u << ((k + e) & 31));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        auto word = [&](const uint4& u) { return x < 2 ? u.x : x < 4 ? u.y : x < 6 ? u.z : u.w; };
                        const int row = (d + x) % (HD / 8) * 8 + (d + x) / (HD / 8);
                        *reinterpret_cast<uint2*>(vt + row * 128 + (((k >> 3) ^ (row & 7)) << 4) + (k & 4) * 2) =
                            make_uint2(__byte_perm(word(v[i][0]), word(v[i][1]), x & 1 ? 0x7632 : 0x5410), __byte_perm(word(v[i][2]), word(v[i][3]), x & 1 ? 0x7632 : 0x5410));
                    }
                }
            } else {
                const int g = lane >> 2, t = lane & 3;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const uint4 v = *reinterpret_cast<const uint4*>(page + kPage * HD + cw * (16 * HD) + i * 512 + lane * 16);      // keys 16 cw .. 16 cw + 15
                    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int row = (4 * i + x) * 8 + g, c = 2 * cw + (t >> 1);
                        *reinterpret_cast<uint2*>(vt + row * 128 + ((c ^ g) << 4) + (t & 1) * 8) = make_uint2(tiny_two<0>(w[x]), tiny_two<2>(w[x]));
                    }
                }
            }
            tc5::fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(v_full + s);
                if (!own) mbar_arrive(raw_free + s);
            }
        }
        if (!ok && lane == 0) gave_up();
    } else if (warp < 4 * tiles) {
        // ---- softmax: a row a thread ----
        const int tile = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, pos = p0 + (r & 63), h = 2 * tile + (r >> 6);
        const bool live = h < G && pos >= start && pos < end;
        const unsigned at = tmem + tile * kTileCols + ((unsigned)(quarter * 32) << 16);
        uint4* my_rows = reinterpret_cast<uint4*>(staged) + warp * (32 * HD / 8);
        constexpr int kRowsAtOnce = 256 / HD;            // of the warp's 32, whole ones, between the threads and memory
        const int my_row = lane / (HD / 8), my_piece = lane % (HD / 8);
        float to_log2;                                   // of a score of unrounded keys; of the others 2^133 times that
        {
            unsigned q[HD / 2];
            // (a row a thread from memory itself would be 32 places a load: 3 us before the first product, and 4.5 for the sums' way out)
            uint4 v[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const int row = i * kRowsAtOnce + my_row, p = p0 + (quarter & 1) * 32 + row;
                const bool there = h < G && p >= start && p < end;
                v[i] = there ? reinterpret_cast<const uint4*>(rows + ((size_t)(tok0 + p - start) * width + head0 + h) * HD)[my_piece] : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const int row = i * kRowsAtOnce + my_row;
                my_rows[row * (HD / 8) + (my_piece ^ (row & 7))] = v[i];
            }
            __syncwarp();
            unsigned top = 0;                            // of two magnitudes' bits at once
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint4 v = my_rows[lane * (HD / 8) + (i ^ (lane & 7))];
                q[4 * i] = v.x; q[4 * i + 1] = v.y; q[4 * i + 2] = v.z; q[4 * i + 3] = v.w;
                top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu));
            }
            const int e = (int)(max(top & 0xffffu, top >> 16) >> 7), by = e == 0 || e == 255 ? 60 : max(-59, min(127, 187 - e));
            const unsigned factor = (unsigned)(127 + by) << 7, both = factor << 16 | factor;
#pragma unroll
            for (int i = 0; i < HD / 2; ++i) {
                const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&q[i]), *reinterpret_cast<const __nv_bfloat162*>(&both));
                q[i] = *reinterpret_cast<const unsigned*>(&v);
            }
#pragma unroll
            for (int c = 0; c < HD / 2; c += 16) {
                unsigned part[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) part[i] = q[c + i];
                tc5::tmem_st16(at + kQCol + c, part);
            }
            tc5::wait_st();
            to_log2 = a.scale_log2e * __uint_as_float((unsigned)(127 + 67 - by) << 23);    // times 2^66, or 2^-67
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const int lo = first_key(pos), warp_lo = first_key(p0 + (quarter & 1) * 32 + 31);          // the latest first key of the warp's rows
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < steps; ++j) {
            if (!mbar_wait(s_full + tile, j & 1)) { ok = false; break; }
            tc5::fence_after();
            const bool own = j == own_step;
            const int key0 = (pg_lo + j) * kPage;
            const float4 scale = scales[j & 3];
            float f = to_log2 * scale.x, lv = scale.z, to_sum = scale.w;
            float x[64];
#pragma unroll
            for (int c = 0; c < 64; c += 16) tc5::tmem_ld16(at + c, x + c);
            tc5::wait_ld(x);
            const bool masked = own || key0 < warp_lo || scale.y < 0.f;
            if (masked) {
                const int from = scale.y < 0.f ? 64 : lo - key0, to = own ? pos - key0 : 63;
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i < from || i > to) x[i] = -INFINITY;
                if (f == 0.f) f = 0x1p-126f;             // (keys of zeros: a hidden one's score stays minus infinity)
                if (from > 63) {                         // of a page that the row sees nothing of, whatever its scales
                    f = 0x1p-126f;
                    lv = to_sum = 0.f;
                }
            }
            float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int i = 4; i < 60; i += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) top[k] = max3(top[k], x[i + k], x[i + k + 4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], x[60 + k]);
            const float mx = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), f, lv);
            // (nothing seen: the product is minus infinity, or none where f is zero or none: neither moves the reference)
            const bool move = mx > m + 8.f;
            if (__any_sync(0xffffffffu, move)) {
                const float alpha = move ? ex2(m - mx) : 1.f;
                if (move) {
                    m = mx;
                    l *= alpha;
                }
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tc5::tmem_ld16(at + kOCol + c, o);
                        tc5::wait_ld(o);
                        unsigned w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[i] * alpha);
                        tc5::tmem_st16(at + kOCol + c, w);
                    }
                }
            }
            const float less = lv + (own ? 0.f : 112.f) - (m == -INFINITY ? 0.f : m);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
                fma_two(x[i], x[i + 1], f, less);
                x[i] = ex2(x[i]);
                x[i + 1] = ex2(x[i + 1]);
                add_two(sum[i & 2], sum[(i & 2) + 1], x[i], x[i + 1]);
            }
#pragma unroll
            for (int c = 0; c < 32; c += 16) {
                unsigned w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = pack_bf16(x[2 * (c + i)], x[2 * (c + i) + 1]);
                tc5::tmem_st16(at + c, w);
            }
            l = fmaf(((sum[0] + sum[1]) + (sum[2] + sum[3])) * (own ? 1.f : 0x1p-112f), to_sum, l);
            tc5::wait_st();
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + tile);
        }
        if (ok) ok = mbar_wait(o_done, 0);
        if (!ok && lane == 0) gave_up();
        tc5::fence_after();
        if (ok && ranks > 1) {                           // the sums as they are, for the cluster
            met_m[r + tile * 128] = m;
            met_l[r + tile * 128] = l;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {          // columns n 8 + g: lanes g HD / 8 + n
                float o[64];
#pragma unroll
                for (int i = 0; i < 64; i += 16) {
                    if (steps > 0) tc5::tmem_ld16(at + kOCol + c * 64 + i, o + i);
                    else
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[i + k] = 0.f;
                }
                tc5::wait_ld(o);
#pragma unroll
                for (int g = 0; g < 8; ++g)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        *met_at(tile * 128 + r, g * (HD / 32) + c * 2 + x) = make_float4(o[32 * x + g], o[32 * x + 8 + g], o[32 * x + 16 + g], o[32 * x + 24 + g]);
            }
        } else if (ok) {
            const float by = 1.f / l;
            // the odd values among the keys that the row sees in its block
            unsigned long long seen_odd = (unsigned long long)odd_values[1] << 32 | odd_values[0];
            if (seen_odd != 0) {
                seen_odd &= ~0ull >> (63 - (r & 63));
                if (lo > p0) seen_odd &= ~0ull << (lo - p0);
            }
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {          // columns n 8 + g: lanes g HD / 8 + n
                float o[64];
#pragma unroll
                for (int i = 0; i < 64; i += 16) tc5::tmem_ld16(at + kOCol + c * 64 + i, o + i);
                tc5::wait_ld(o);
                const float times = 0x1p11f * by;                                // (units of 2^-133 2^112 over those of 2^-10)
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    my_rows[lane * (HD / 8) + ((g * (HD / 64) + c) ^ (lane & 7))] =
                        make_uint4(pack_bf16(o[g] * times, o[8 + g] * times), pack_bf16(o[16 + g] * times, o[24 + g] * times),
                                   pack_bf16(o[32 + g] * times, o[40 + g] * times), pack_bf16(o[48 + g] * times, o[56 + g] * times));
            }
            if (live && seen_odd != 0)
                for (int k = 0; k < 64; ++k)
                    if (seen_odd >> k & 1) {
                        const int p = p0 + k;
                        const __nv_bfloat16* from = p >= start ? rows + ((size_t)(tok0 + p - start) * width + a.n_heads + a.n_kv + kvh) * HD
                                                               : reinterpret_cast<const __nv_bfloat16*>(a.found) + ((((size_t)seq * 2 + 1) * a.n_kv + kvh) * kPage + k) * HD;
                        for (int d = 0; d < HD; ++d) {
                            const float v = __bfloat162float(from[d]);
                            __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(my_rows + lane * (HD / 8) + ((d >> 3) ^ (lane & 7))) + (d & 7);
                            if (!(fabsf(v) < INFINITY)) *o = __float2bfloat16(__bfloat162float(*o) + v);
                        }
                    }
            __syncwarp();
#pragma unroll 4
            for (int i = 0; i < HD / 8; ++i) {
                const int row = i * kRowsAtOnce + my_row, p = p0 + (quarter & 1) * 32 + row;
                if (h < G && p >= start && p < end)
                    reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)(tok0 + p - start) * a.n_heads + head0 + h) * HD)[my_piece] =
                        my_rows[row * (HD / 8) + (my_piece ^ (row & 7))];
            }
        }
    }
    __syncwarp();
    tc5::fence_before();
    if (ranks > 1) {
        // ---- the cluster's shares meet: some of the rows each, four lanes a thread ----
        cluster_sync();
        const int some = tiles * 128 / ranks;
        unsigned long long odd = 0;
        for (int w = 0; w < 2; ++w) odd |= (unsigned long long)__float_as_uint(cluster_float(smem_u32(odd_values + w), own_rank)) << (32 * w);
        // the shares' weights, a thread each: a row's are neighbours
        float* weights = reinterpret_cast<float*>(staged);                       // [rows][ranks]
        if (threadIdx.x < some * ranks) {
            const int row = rank * some + threadIdx.x / ranks, k = threadIdx.x % ranks;
            const float mk = cluster_float(smem_u32(met_m + row), k), lk = cluster_float(smem_u32(met_l + row), k);
            float top = mk;
            for (int w = 1; w < ranks; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float by = mk == top ? 1.f : ex2(mk - top);
            float l = lk * by;
            for (int w = 1; w < ranks; w *= 2) l += __shfl_xor_sync(0xffffffffu, l, w);
            weights[threadIdx.x] = by * (0x1p11f / l);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < some * (HD / 4); i += kPromptThreads) {
            const int mine = i / (HD / 4), row = rank * some + mine, c = i % (HD / 4), pos = p0 + (row & 63), h = row >> 6;
            if (h >= G || pos < start || pos >= end) continue;
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            float4 v[8];                                 // (all reads before the first use)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < ranks) v[k] = cluster_float4(smem_u32(met_at(row, c)), k);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < ranks) {
                    const float by = weights[mine * ranks + k];
                    o[0] = fmaf(v[k].x, by, o[0]); o[1] = fmaf(v[k].y, by, o[1]); o[2] = fmaf(v[k].z, by, o[2]); o[3] = fmaf(v[k].w, by, o[3]);
                }
            const int lo = first_key(pos);
            __nv_bfloat16 y[4];
            for (int e = 0; e < 4; ++e) {
                float x = o[e];
                if (odd != 0)
                    for (int k = max(lo, p0); k <= pos; ++k)
                        if (odd >> (k - p0) & 1) {
                            const __nv_bfloat16* from = k >= start ? rows + ((size_t)(tok0 + k - start) * width + a.n_heads + a.n_kv + kvh) * HD
                                                                   : reinterpret_cast<const __nv_bfloat16*>(a.found) + ((((size_t)seq * 2 + 1) * a.n_kv + kvh) * kPage + k - p0) * HD;
                            const float v = __bfloat162float(from[c * 4 + e]);
                            if (!(fabsf(v) < INFINITY)) x += v;
                        }
                y[e] = __float2bfloat16(x);
            }
            *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)(tok0 + pos - start) * a.n_heads + head0 + h) * HD + c * 4) = *reinterpret_cast<const uint2*>(y);
        }
        cluster_sync();                                  // what others read stays until they have
    } else {
        __syncthreads();
    }
    if (warp == 12) {
        tc5::fence_after();
        tc5::tmem_free(tmem, 512);
    }
}

// `touched` 64-position blocks of all sequences, the longest walk of so many `pages`.
template <int HD>
static int launch_prompt(PromptArgs pa, int n_tokens, long long touched, int pages, cudaStream_t stream) {
    static int resident[64][4] = {};                     // clusters of 1, 2, 4 and 8 blocks that the device holds at once
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return blm_fail(BLM_CUDA_ERROR, "attention_q8: device %d", dev);
    if (resident[dev][0] == 0) {
        if (cudaFuncSetAttribute(attend_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<HD>::kSmem) != cudaSuccess)
            return blm_fail(BLM_CUDA_ERROR, "attention_q8: %s", cudaGetErrorString(cudaGetLastError()));
        for (int i = 3; i >= 0; --i) {                   // (a cluster lies in one group of SMs, which a number of blocks need not divide)
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1 << i);
            cfg.blockDim = dim3(kPromptThreads);
            cfg.dynamicSmemBytes = Prompt<HD>::kSmem;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 1 << i;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int fit = 0;
            if (i > 0 && cudaOccupancyMaxActiveClusters(&fit, attend_prompt_kernel<HD>, &cfg) != cudaSuccess) {
                cudaGetLastError();
                fit = 0;
            }
            resident[dev][i] = i > 0 ? fit : blm_sm_count();
        }
    }
    // A walk is shared by as many blocks as make the step shortest: its turns, each a share of the longest walk's pages and, about as long
    // as six pages, a block's beginning and end, and five more where the shares have to meet.  Heads of 128, 32 to 8 kv heads, in 1, 2, 4
    // and 8 blocks: 64 tokens alone 8.5, 14.1, 13.5, 14.8 us; 64 behind 1,000 25.8, 20.6, 16.3, 26.6; 64 behind 8,192 145, 82, 48, 32; 256
    // behind 8,192 149, 85, 50, 94.  (`pages` may be a bound far above what the step has, as in captured steps: 64 tokens alone then 14.1.)
    const long long walks = (long long)pa.a.n_kv * pa.head_groups * touched;
    long long best = (walks + resident[dev][0] - 1) / resident[dev][0] * (pages + 6);
    for (int i = 1; i < 4; ++i) {
        if (resident[dev][i] < 1) continue;
        const long long length = (walks + resident[dev][i] - 1) / resident[dev][i] * ((pages + (1 << i) - 1 >> i) + 11);
        if (length < best) { best = length; pa.ranks = 1 << i; }
    }
    const long long blocks = (long long)pa.a.n_kv * pa.head_groups * pa.ranks * most_blocks(n_tokens, pa.a.n_seqs, kPage);
    BLM_REQUIRE(blocks < 1ll << 31, "attention_q8: %d tokens of %d heads in one step", n_tokens, pa.a.n_heads);
    blm_launch_cluster(attend_prompt_kernel<HD>, pa.ranks, dim3((unsigned)blocks), dim3(kPromptThreads), Prompt<HD>::kSmem, stream, pa);
    return blm_check_launch("attention_q8");
}

template <typename T, bool VEC>
static int launch_append(const AppendArgs& a, int n_tokens, int n_seqs, int max_q_len, cudaStream_t stream) {
    const size_t smem = (size_t)kPage * (a.hd + 16 / sizeof(T)) * sizeof(T) + kAppendThreads / 32 * sizeof(float);
    const void* kernel = max_q_len == 1 ? (const void*)append_token_kernel<T, VEC> : (const void*)append_prompt_kernel<T, VEC>;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return blm_fail(BLM_CUDA_ERROR, "rope_append_q8: %s", cudaGetErrorString(cudaGetLastError()));
    if (max_q_len == 1) {
        blm_launch_dependent(append_token_kernel<T, VEC>, dim3(a.n_kv, n_seqs, 2), dim3(kAppendThreads), smem, stream, a);
    } else {
        const dim3 grid((unsigned)most_blocks(n_tokens, n_seqs, kPage), a.n_heads + 2 * a.n_kv);
        blm_launch_dependent(append_prompt_kernel<T, VEC>, grid, dim3(kAppendThreads), smem, stream, a);
    }
    return blm_check_launch("rope_append_q8");
}
}  // namespace q8

BLM_API int blm_rope_append_q8(const void* qkv, void* out, int dtype, const int* cu_seqlens, const int* slot_of_seq, const int* start_pos,
                               const int* block_table, int table_stride, const double* inv_freq, int rot, int pairing, const float* table,
                               int table_len, float turn_scale, void* pool, void* tail, void* old, int n_tokens, int n_seqs, int max_q_len,
                               int n_heads, int n_kv, int hd, int n_pages, cudaStream_t stream) {
    using namespace q8;
    if (n_seqs == 0 || max_q_len == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0, "rope_append_q8: heads of %d lanes (multiples of 16 from 16 to 256)", hd);
    BLM_REQUIRE(n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0, "rope_append_q8: %d heads do not divide into %d kv heads", n_heads, n_kv);
    BLM_REQUIRE(rot >= 0 && rot <= hd && rot % 2 == 0, "rope_append_q8: %d rotated lanes of a head of %d", rot, hd);
    BLM_REQUIRE(rot == 0 || inv_freq != nullptr, "rope_append_q8: no frequencies");
    BLM_REQUIRE(pairing >= 0 && pairing <= 2 && (pairing != PAIRS_TILED || rot % 16 == 0), "rope_append_q8: pairing %d of %d lanes", pairing, rot);
    BLM_REQUIRE(n_seqs <= 65535 && n_heads + 2 * n_kv <= 65535, "rope_append_q8: %d sequences, %d heads (at most 65535 of either)", n_seqs, n_heads + 2 * n_kv);
    BLM_REQUIRE(dtype == BLM_F32 || dtype == BLM_BF16, "rope_append_q8: dtype %d", dtype);
    const AppendArgs a{qkv, out, cu_seqlens, slot_of_seq, start_pos, block_table, table_stride, inv_freq, (const float2*)table, table ? table_len : 0,
                       turn_scale, rot, pairing, (signed char*)pool, tail, old, n_heads, n_kv, hd, n_pages, n_seqs};
    const bool vec = rot % 16 == 0;
    if (dtype == BLM_F32) return vec ? launch_append<float, true>(a, n_tokens, n_seqs, max_q_len, stream) : launch_append<float, false>(a, n_tokens, n_seqs, max_q_len, stream);
    return vec ? launch_append<__nv_bfloat16, true>(a, n_tokens, n_seqs, max_q_len, stream) : launch_append<__nv_bfloat16, false>(a, n_tokens, n_seqs, max_q_len, stream);
}

BLM_API int blm_q8_values(const void* pool, const int* pages, void* out, int dtype, int n, int n_kv, int hd, int n_pages, cudaStream_t stream) {
    using namespace q8;
    if (n == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0 && n_kv <= 65535, "q8_values: %d heads of %d lanes", n_kv, hd);
    const dim3 grid(n, n_kv, (4 * hd + 255) / 256);
    if (dtype == BLM_F32) values_kernel<<<grid, 256, 0, stream>>>((const signed char*)pool, pages, (float*)out, n_kv, hd, n_pages);
    else if (dtype == BLM_BF16) values_kernel<<<grid, 256, 0, stream>>>((const signed char*)pool, pages, (__nv_bfloat16*)out, n_kv, hd, n_pages);
    else return blm_fail(BLM_BAD_ARGUMENT, "q8_values: dtype %d", dtype);
    return blm_check_launch("q8_values");
}

// Over how many shares that meet in memory a step cuts its sequences: what the scratch holds is n_tokens * n_heads * shares * (hd + 2) float32 when there are
// several, which a second kernel merges.
BLM_API int blm_attention_q8_splits(int dtype, int n_seqs, int max_q_len, int max_kv_len, int n_heads, int n_kv, int hd, int window) {
    using namespace q8;
    if (n_seqs < 1 || n_kv < 1 || n_heads < n_kv || !tokens_take(dtype, hd, max_q_len, n_seqs, n_kv, n_heads)) return 1;
    const int splits = plan_tokens(n_seqs, n_heads, n_kv, hd, max_kv_len, window).splits;
    return splits > kClusterShares ? splits : 1;
}

BLM_API int blm_attention_q8(const void* rotated, const void* pool, const void* found, int found_by_slot, int dtype,
                             const int* block_table, int table_stride, const int* cu_seqlens, const int* slot_of_seq, const int* start_pos,
                             void* out, int n_tokens, int n_seqs, int n_heads, int n_kv, int hd, int n_pages, int window, float scale, int max_q_len,
                             int max_kv_len, float* scratch, int splits, int* status, cudaStream_t stream) {
    using namespace q8;
    if (n_tokens == 0 || n_seqs == 0) return BLM_OK;
    BLM_REQUIRE(hd >= 16 && hd <= 256 && hd % 16 == 0, "attention_q8: heads of %d lanes (multiples of 16 from 16 to 256)", hd);
    BLM_REQUIRE(n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0, "attention_q8: %d heads do not divide into %d kv heads", n_heads, n_kv);
    BLM_REQUIRE((long long)n_tokens * n_heads < (1ll << 31), "attention_q8: %d tokens of %d heads in one step", n_tokens, n_heads);
    const AttendArgs a{rotated, (const signed char*)pool, found, found_by_slot, block_table, table_stride, cu_seqlens, slot_of_seq, start_pos,
                       out, n_seqs, n_heads, n_kv, hd, n_pages, window, scale * 1.4426950408889634f};
    if (tokens_take(dtype, hd, max_q_len, n_seqs, n_kv, n_heads)) {
        const TokenPlan p = plan_tokens(n_seqs, n_heads, n_kv, hd, max_kv_len, window);
        const bool clustered = p.splits > 1 && p.splits <= kClusterShares;
        BLM_REQUIRE((clustered ? 1 : p.splits) == splits && (splits == 1 || scratch != nullptr), "attention_q8: scratch for %d shares, the step has %d", splits, p.splits);
        const TokenArgs ta{a, scratch, scratch ? scratch + (size_t)n_tokens * n_heads * splits * hd : nullptr, p.splits, p.head_tiles, p.heads_a_tile,
                           p.pages_per_split, clustered, status};
        if (hd == 64) return launch_tokens_as<64, 1>(ta, stream);
        return p.wpp == 1 ? launch_tokens_as<128, 1>(ta, stream) : launch_tokens_as<128, 2>(ta, stream);
    }
    if (dtype == BLM_BF16 && (hd == 64 || hd == 128) && max_q_len > 1) {
        const int group = n_heads / n_kv, groups = (group + 3) / 4;
        int pages = (max_kv_len + kPage - 1) / kPage;
        if (window > 0 && pages > window / kPage + 2) pages = window / kPage + 2;
        // 64-position blocks that the step touches: one sequence's are known, of several their mean
        const int from = max_kv_len > max_q_len ? max_kv_len - max_q_len : 0;
        const long long touched = n_seqs == 1 ? (from + n_tokens - 1) / kPage - from / kPage + 1 : (n_tokens + 63ll * n_seqs + 63) / kPage;
        const PromptArgs pa{a, groups, (group + groups - 1) / groups, 1, status};
        return hd == 64 ? launch_prompt<64>(pa, n_tokens, touched, pages, stream) : launch_prompt<128>(pa, n_tokens, touched, pages, stream);
    }
    if (dtype == BLM_F32) return launch_tile<float>(a, n_tokens, max_q_len, max_kv_len, stream);
    if (dtype == BLM_BF16) return launch_tile<__nv_bfloat16>(a, n_tokens, max_q_len, max_kv_len, stream);
    return blm_fail(BLM_BAD_ARGUMENT, "attention_q8: dtype %d", dtype);
}
