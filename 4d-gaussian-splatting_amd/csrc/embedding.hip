// Table lookup with scaling, and its gradient by sorted tokens.
//
//   forward    out[i, :]  = scale * table[ids[i], :]
//   backward   dtable[r, :] = scale * sum over the tokens i with ids[i] = r of dout[i, :]
//
// Both are memory-bound: the lookup writes its output and reads the rows that are asked for (most of them from L2), the
// gradient reads dout once and writes every row of dtable once, the rows that no token asks for as zeros.
//
// The gradient adds in float32 in an order that depends on the ids alone: the tokens are sorted by id (stable), and
// the sorted list together with the list of rows is walked as one sequence of T + V items - for each row its tokens,
// then the row's write - cut into shares of equal length.  A token's place in that sequence is i + id(i), so a share finds
// its first token by one search and needs no table of row starts; a share costs the same whether it holds the tokens
// of one frequent row or the zeros of many rows that nobody asked for.  A row that is cut by a share's end leaves
// partial sums in the workspace, which a last launch adds up in the shares' order.  No atomic touches a sum.
#include "fdgs_common.h"
#include <algorithm>
#include <type_traits>

// ---- element types: 16 bytes to a vector where the row is that long, else one element ----
typedef uint32_t em_u4 __attribute__((ext_vector_type(4)));
struct EmF32 { typedef float raw; static const int full = 4; typedef em_u4 wide __attribute__((aligned(4))); };
struct EmBf16 { typedef uint16_t raw; static const int full = 8; typedef em_u4 wide __attribute__((aligned(2))); };
struct EmF16 { typedef uint16_t raw; static const int full = 8; typedef em_u4 wide __attribute__((aligned(2))); };

template <class T> __device__ __forceinline__ float em_up(typename T::raw x);
template <> __device__ __forceinline__ float em_up<EmF32>(float x) { return x; }
template <> __device__ __forceinline__ float em_up<EmBf16>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
template <> __device__ __forceinline__ float em_up<EmF16>(uint16_t x) { return __half2float(__ushort_as_half(x)); }

template <class T> __device__ __forceinline__ typename T::raw em_down(float x);
template <> __device__ __forceinline__ float em_down<EmF32>(float x) { return x; }
template <> __device__ __forceinline__ uint16_t em_down<EmBf16>(float x) {   // to the nearest, halves to even
    const uint32_t b = __float_as_uint(x);
    const uint32_t r = (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
    return (uint16_t)(x != x ? 0x7FC0u : r);
}
template <> __device__ __forceinline__ uint16_t em_down<EmF16>(float x) { return __half_as_ushort(__float2half_rn(x)); }

// VEC elements at any alignment of the element's own size (gfx950 takes unaligned global accesses)
template <class T, int VEC>
struct __attribute__((packed, aligned(sizeof(typename T::raw)))) EmVec { typename T::raw x[VEC]; };

// Column of a row's vector `c` of `nv`: the last vector is moved back to end with the row, so that a width that is no
// multiple of VEC needs no narrower path (the columns it shares with its neighbour are written twice, with the same
// values).
template <int VEC>
__device__ __forceinline__ int em_col(int c, int nv, int dim) { return (VEC > 1 && c == nv - 1) ? dim - VEC : c * VEC; }

// A token's row, or `none` where it has none (negative, the padding id, or beyond the table)
__device__ __forceinline__ uint32_t em_key(const void* ids, long long i, int wide, long long padding, uint32_t none) {
    const long long id = wide ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i];
    return (id < 0 || id >= (long long)none || id == padding) ? none : (uint32_t)id;
}

// x / d for x below 2^31 by multiplication: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d) < 2^32 the quotient is
// (x * m) >> (31 + l) exactly, because the excess of m, less than 1 in 2^(31 + l) / d, adds less than 1 / d.
struct EmDiv { uint32_t d, m, s; };
static EmDiv em_div_of(uint32_t d) {
    EmDiv r;
    r.d = d;
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;                     // ceil(log2 d)
    r.s = l ? l - 1 : 0;
    r.m = d == 1 ? 0u : (uint32_t)(((1ull << (32 + r.s)) + d - 1) / d);
    return r;
}
__device__ __forceinline__ uint32_t em_div(uint32_t x, const EmDiv& v) { return v.d == 1 ? x : __umulhi(x, v.m) >> v.s; }

// Streaming store: what is written here is not read by this launch, and the table's rows are to stay in L2.
template <class T, int VEC>
__device__ __forceinline__ void em_store(typename T::raw* p, const EmVec<T, VEC>& v) {
    if constexpr (VEC == T::full) {
        __builtin_nontemporal_store(__builtin_bit_cast(em_u4, v), (typename T::wide*)p);
    } else {
        __builtin_nontemporal_store(v.x[0], p);
    }
}

// ---- forward ----
#define EF_THREADS 256
#define EF_UNROLL 4
#define EF_VECTORS (EF_THREADS * EF_UNROLL)          // of a workgroup at most

struct EmFwd {
    const void* ids; const void* table; void* out;
    long long table_stride, padding;
    int tokens, rows, dim, nv, wide, per_group, vectors; // tokens and vectors of a workgroup
    float scale;
    EmDiv by_nv;
};

// A workgroup has whole tokens, as many as make up to 512 or 1024 vectors (or, of a longer row, so many of one token): a
// thread has up to two or four vectors, all of whose ids and then all of whose rows are asked for before the first is used.
// Bound by the output's lines and, where the table does not fit an XCD's 4 MB of L2, by the rows that come from behind it:
// 300,000 x 48 floats 11.9 us (5.1 TB/s), 2,000,000 x 48 from 65,536 rows 120 us, from 8,192 rows 66 us (5.8 TB/s).
template <class T, int VEC>
__device__ __forceinline__ void ef_group(const EmFwd& a, int group, int tile, uint32_t thread) {
    typedef EmVec<T, VEC> Vec;
    typedef typename T::raw raw;
    const int tok0 = group * a.per_group, have = min(a.per_group, a.tokens - tok0);
    const int c0 = tile * a.vectors, cols = min(a.nv - c0, a.vectors);   // all of them, or a part of one row
    const uint32_t end = (uint32_t)have * (uint32_t)cols;
    auto part = [&](auto unroll) {
        constexpr int U = decltype(unroll)::value;
        Vec v[U];
        int tok[U], col[U];
        long long id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t e = u * EF_THREADS + thread;
            const uint32_t t = a.per_group > 1 ? em_div(e, a.by_nv) : 0u;
            tok[u] = e < end ? tok0 + (int)t : -1;
            col[u] = em_col<VEC>(c0 + (int)(e - t * (uint32_t)a.nv), a.nv, a.dim);
            id[u] = -1;
            if (tok[u] >= 0) {
                id[u] = a.wide ? ((const long long*)a.ids)[tok[u]] : (long long)((const int*)a.ids)[tok[u]];
                if (id[u] == a.padding) id[u] = -1;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (id[u] >= 0 && id[u] < a.rows) v[u] = *(const Vec*)((const raw*)a.table + id[u] * a.table_stride + col[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (tok[u] < 0) continue;
            const bool there = id[u] >= 0 && id[u] < a.rows;
            const float other = id[u] < 0 ? 0.0f : __builtin_nanf("");
            Vec o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.x[j] = em_down<T>(there ? em_up<T>(v[u].x[j]) * a.scale : other);
            em_store<T, VEC>((raw*)a.out + (long long)tok[u] * a.dim + col[u], o);
        }
    };
    if (a.vectors > EF_VECTORS / 2) part(std::integral_constant<int, EF_UNROLL>());
    else part(std::integral_constant<int, EF_UNROLL / 2>());
}

template <class T, int VEC>
__global__ void __launch_bounds__(EF_THREADS)
embedding_fwd_kernel(EmFwd a) { ef_group<T, VEC>(a, blockIdx.x, blockIdx.y, threadIdx.x); }

template <class T>
static int em_fwd_launch(const EmFwd& k, int vec, dim3 grid, hipStream_t s) {
    if (vec > 1) hipLaunchKernelGGL((embedding_fwd_kernel<T, T::full>), grid, dim3(EF_THREADS), 0, s, k);
    else hipLaunchKernelGGL((embedding_fwd_kernel<T, 1>), grid, dim3(EF_THREADS), 0, s, k);
    FDGS_CHECK_LAUNCH();
    return FDGS_OK;
}

static int em_full(int type) { return type == FDGS_TYPE_F32 ? EmF32::full : EmBf16::full; }
static bool em_type_ok(int t) { return t == FDGS_TYPE_F32 || t == FDGS_TYPE_BF16 || t == FDGS_TYPE_F16; }

// ---- the tokens by row: (key, token) pairs, stable ----
// The sort's launches wait more than they work: their workgroups leave most of the chip idle.  Where a lookup sorts its
// tokens for the gradient that will follow, the launches have parts of the lookup's work beside their own (16,384 tokens of 2048
// bfloat16 numbers: 29 us, 45 one after the other).
struct EmPart {
    EmFwd a;
    int first, last, type, vec;                      // workgroups' work (tokens and column tile) [first, last)
    EmDiv by_tiles;
};
__device__ __forceinline__ void ep_group(const EmPart& f, int block, int threads) {
    const int each = threads / EF_THREADS;
    const int g = f.first + block * each + (each > 1 ? (int)(threadIdx.x / EF_THREADS) : 0);
    if (g >= f.last) return;
    const int group = (int)em_div((uint32_t)g, f.by_tiles), tile = g - group * (int)f.by_tiles.d;
    const uint32_t thread = threadIdx.x % EF_THREADS;
    if (f.type == FDGS_TYPE_F32) {
        if (f.vec > 1) ef_group<EmF32, EmF32::full>(f.a, group, tile, thread);
        else ef_group<EmF32, 1>(f.a, group, tile, thread);
    } else if (f.type == FDGS_TYPE_BF16) {
        if (f.vec > 1) ef_group<EmBf16, EmBf16::full>(f.a, group, tile, thread);
        else ef_group<EmBf16, 1>(f.a, group, tile, thread);
    } else {
        if (f.vec > 1) ef_group<EmF16, EmF16::full>(f.a, group, tile, thread);
        else ef_group<EmF16, 1>(f.a, group, tile, thread);
    }
}
// One step of a sort in `blocks` workgroups, every `period`-th from the first on (an odd number: the workgroups go to the 8
// XCDs in turn), and a part of a lookup in the others.
template <class Step>
__global__ void __launch_bounds__(Step::threads)
embedding_step_kernel(Step step, int blocks, int period, EmPart part) {
    const int b = (int)blockIdx.x, round = b / period;
    if (round < blocks && round * period == b) step.run(round);
    else ep_group(part, round < blocks ? b - round - 1 : b - blocks, Step::threads);
}

// Few tokens: a token's place is the number of tokens that come before it, counted against all of them; the workgroup has
// 64 tokens, its waves divide the others.  One launch, T^2 / 64 comparisons of a wave spread over the chip; from 768 tokens for
// each digit on, a sort in LDS is quicker (gradients of rows of 8, by counting and so: 500 tokens of 500 rows 17 and 18 us,
// 2000 25 and 22; 1000 of 65,536 rows, two digits, 14 and 18, 3000 21 and 20).
#define ER_THREADS 256
#define ER_TOKENS 768                                // a sort by digits takes so long for each of its passes (at most four)

struct EmIds {
    const void* ids;
    long long padding;
    uint32_t rows;
    int tokens, wide;
    __device__ __forceinline__ uint32_t key(int i) const { return em_key(ids, i, wide, padding, rows); }
};

struct EmRank {
    static const int threads = ER_THREADS;
    EmIds in;
    uint2* sorted;
    __device__ __forceinline__ void run(int block) const {
        __shared__ __align__(16) uint32_t sk[4 * ER_TOKENS];
        __shared__ uint32_t part[4][64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tokens = in.tokens;
        const int own = block * 64;             // first token of the workgroup
        const int me = own + lane;
        const uint32_t key = me < tokens ? in.key(me) : 0xFFFFFFFFu;
        uint32_t before = 0;
        for (int j = threadIdx.x; j < (tokens + 63) / 64 * 64; j += ER_THREADS) sk[j] = j < tokens ? in.key(j) : 0xFFFFFFFFu;   // after every key
        __syncthreads();
        // blocks of 64 keys, one wave each: those before the own tokens win ties, those behind lose them
        for (int b = wave * 64; b < tokens; b += 256) {
            if (b == own) {
                for (int j = 0; j < 64; ++j) {
                    const uint32_t o = sk[b + j];
                    before += (o < key || (o == key && j < lane)) ? 1u : 0u;
                }
            } else {
                const uint32_t limit = key + (b < own ? 1u : 0u);            // o <= key, or o < key
                const uint4* q = (const uint4*)(sk + b);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint4 o = q[j];
                    before += (o.x < limit ? 1u : 0u) + (o.y < limit ? 1u : 0u) + (o.z < limit ? 1u : 0u) + (o.w < limit ? 1u : 0u);
                }
            }
        }
        part[wave][lane] = before;
        __syncthreads();
        if (wave == 0 && me < tokens) {
            const uint32_t r = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
            sorted[r] = make_uint2(key, (uint32_t)me);
        }
    }
};

// More: a workgroup sorts 4096 tokens in LDS, by digits of at most 9 bits from the lowest on.  Several such lists are merged by
// search: a token's place is its place in its own list and, in each other one, the number of tokens that come before it,
// those of equal keys among them where that list lies before its own.  Both launches take the same time whatever the ids
// are.  (Lists in buckets of neighbouring keys, whose tokens are compared with each other, make the gradient of 16,384 tokens of
// 65,536 rows of 8 21 us, not 31, where the ids are even, 71, not 34, where a few have most of the tokens, and 115, not 33,
// where one has all.)
#define EL_THREADS 1024
#define EL_WAVES (EL_THREADS / 64)
#define EL_TOKENS 4096
#define EL_PER (EL_TOKENS / EL_THREADS)
#define EL_LISTS 4
#define EX_BITS 9
#define EX_BINS (1 << EX_BITS)

// The lanes whose digit (of at most EX_BITS bits) is the lane's own, of those that are `ok`.
__device__ __forceinline__ unsigned long long ex_peers(uint32_t d, int bits, bool ok) {
    unsigned long long peers = __ballot(ok);
#pragma unroll
    for (int b = 0; b < EX_BITS; ++b) {
        if (b < bits) {
            const unsigned long long bal = __ballot((d >> b) & 1u);
            peers &= ((d >> b) & 1u) ? bal : ~bal;
        }
    }
    return peers;
}

struct EmList {
    static const int threads = EL_THREADS;
    EmIds in;
    int key_bits, passes;
    uint2* lists;
    __device__ __forceinline__ void run(int block) const {
        __shared__ uint2 ordered[EL_TOKENS];
        __shared__ __align__(16) uint16_t cnt[EL_WAVES][EX_BINS];    // a wave's count of each digit, then where its first one lies
        __shared__ uint32_t wsum[EX_BINS / 64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int from = block * EL_TOKENS, have = min(in.tokens - from, EL_TOKENS);
        const int at = wave * (64 * EL_PER) + lane;
        const unsigned long long below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
        uint2 e[EL_PER];
#pragma unroll
        for (int k = 0; k < EL_PER; ++k) {           // what is missing goes to the end: it has the largest key, and is last
            const int i = at + 64 * k;
            e[k] = i < have ? make_uint2(in.key(from + i), (uint32_t)(from + i)) : make_uint2(0xFFFFFFFFu, 0u);
        }
        int shift = 0;
        for (int pass = 0; pass < passes; ++pass) {
            const int bits = (key_bits - shift + passes - pass - 1) / (passes - pass), bins = 1 << bits;
            static_assert(sizeof(cnt) == EL_THREADS * sizeof(uint4), "cleared by one store a thread");
            ((uint4*)cnt)[threadIdx.x] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            uint32_t digit[EL_PER], rank[EL_PER];
#pragma unroll
            for (int k = 0; k < EL_PER; ++k) {
                const uint32_t d = digit[k] = (e[k].x >> shift) & (uint32_t)(bins - 1);
                const unsigned long long peers = ex_peers(d, bits, true);
                const uint32_t first = (uint32_t)__popcll(peers & below), prev = cnt[wave][d];
                rank[k] = prev + first;
                if (first == 0) cnt[wave][d] = (uint16_t)(prev + (uint32_t)__popcll(peers));
            }
            __syncthreads();
            uint32_t incl = 0, own = 0;
            if (threadIdx.x < EX_BINS) {             // eight whole waves
#pragma unroll
                for (int w = 0; w < EL_WAVES; ++w) own += cnt[w][threadIdx.x];
                incl = own;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t o = __shfl_up(incl, d);
                    if (lane >= d) incl += o;
                }
                if (lane == 63) wsum[wave] = incl;
            }
            __syncthreads();
            if (threadIdx.x < EX_BINS) {
                uint32_t g = incl - own;
#pragma unroll
                for (int w = 0; w < EX_BINS / 64; ++w) g += w < wave ? wsum[w] : 0u;
#pragma unroll
                for (int w = 0; w < EL_WAVES; ++w) {
                    const uint32_t c = cnt[w][threadIdx.x];
                    cnt[w][threadIdx.x] = (uint16_t)g;
                    g += c;
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < EL_PER; ++k) ordered[cnt[wave][digit[k]] + rank[k]] = e[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < EL_PER; ++k) e[k] = ordered[at + 64 * k];
            shift += bits;
        }
#pragma unroll
        for (int k = 0; k < EL_PER; ++k)
            if (at + 64 * k < have) lists[from + at + 64 * k] = e[k];
    }
};

struct EmMerge {
    static const int threads = 1024;
    const uint2* __restrict__ lists;
    int tokens;
    uint2* __restrict__ sorted;
    __device__ __forceinline__ void run(int block) const {
        __shared__ uint32_t keys[EL_LISTS * EL_TOKENS];
        const int i = block * threads + (int)threadIdx.x;
        const uint2 mine = i < tokens ? lists[i] : make_uint2(0u, 0u);
#pragma unroll 8
        for (int j = threadIdx.x; j < EL_LISTS * EL_TOKENS; j += threads)
            if (j < tokens) keys[j] = lists[j].x;
        __syncthreads();
        if (i >= tokens) return;
        const int own = i / EL_TOKENS;
        int before[EL_LISTS];
#pragma unroll
        for (int l = 0; l < EL_LISTS; ++l) before[l] = 0;
        // all lists step by step side by side: as many tokens come before as the largest sum of steps that reaches none behind
#pragma unroll 1
        for (int step = EL_TOKENS; step > 0; step >>= 1) {
            uint32_t key[EL_LISTS];
#pragma unroll
            for (int l = 0; l < EL_LISTS; ++l) {
                const int have = min(tokens - l * EL_TOKENS, EL_TOKENS), to = before[l] + step;
                key[l] = to <= have ? keys[l * EL_TOKENS + to - 1] : 0xFFFFFFFFu;
            }
#pragma unroll
            for (int l = 0; l < EL_LISTS; ++l)
                if (key[l] < mine.x + (l < own ? 1u : 0u)) before[l] += step;
        }
        int place = i - own * EL_TOKENS;
#pragma unroll
        for (int l = 0; l < EL_LISTS; ++l) place += l == own ? 0 : before[l];
        sorted[place] = mine;
    }
};

// Many tokens: a radix sort by digits of at most 9 bits (two passes for tables of up to 262,143 rows), two or three launches
// a pass: counts of each block of tokens, their scan, scatter.  2,000,000 tokens of 65,536 rows 43 us, 300,000 of 8,192 25 us.
#define EX_THREADS 256
#define EX_TILE(ipl) (EX_THREADS * (ipl))             // tokens that a workgroup takes at a time, ipl to a lane
#define EX_MAX_BLOCKS 1024

struct EmSort {
    EmIds ids;                                       // first pass: the tokens' ids; later passes: the pairs `in`
    const uint2* in;
    uint2* out;
    uint32_t* hist; uint32_t* totals;
    uint32_t mask;
    int tokens, per_block, nblocks, shift, bits, ngroups;        // ngroups: totals of four blocks each, 0: of all
};

template <bool FIRST>
__device__ __forceinline__ uint32_t ex_key(const EmSort& a, int i) { return FIRST ? a.ids.key(i) : a.in[i].x; }

template <bool FIRST>
struct EmHist {
    static const int threads = EX_THREADS;
    EmSort a;
    __device__ __forceinline__ void run(int block) const {
        __shared__ uint32_t h[EX_BINS];
        const int bins = 1 << a.bits;
        for (int d = threadIdx.x; d < bins; d += EX_THREADS) h[d] = 0;
        __syncthreads();
        const int begin = block * a.per_block, end = min(begin + a.per_block, a.tokens);
        for (int i = begin + threadIdx.x; i < end; i += EX_THREADS) atomicAdd(&h[(ex_key<FIRST>(a, i) >> a.shift) & a.mask], 1u);
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += EX_THREADS) a.hist[(size_t)block * bins + d] = h[d];
    }
};

// The same for four blocks of tokens in a workgroup: their counts become the places among the four of each block's first
// token, and totals [groups of four][bins] holds the four's counts.  Each workgroup of the scatter adds up the totals
// before its own by itself: a launch less, worth it while they read few counts in all (EX_READS).  Gradients of rows of 8, in a
// graph: 300,000 tokens of 8,192 rows (2.7 million counts read) 45.7 -> 42.6 us, 100,000 of 65,536 (4.9) 40.0 -> 38.4, 500,000 of
// 8,192 (7.7) 50.9 -> 49.7, 300,000 of 65,536 (11) 53.2 -> 53.6, 1,000,000 of 8,192 (31) 68.2 -> 72.3.
#define EX_READS (1 << 23)
#define EX_TOTALS 40960                              // at most: groups of four of 256 blocks and 512 bins read 2^23 of them
template <bool FIRST>
struct EmHist4 {
    static const int threads = 4 * EX_THREADS;
    EmSort a;
    __device__ __forceinline__ void run(int block) const {
        __shared__ uint32_t h[4][EX_BINS];
        const int bins = 1 << a.bits, sub = threadIdx.x / EX_THREADS, own = 4 * block + sub;
        for (int d = threadIdx.x; d < 4 * EX_BINS; d += threads) (&h[0][0])[d] = 0;
        __syncthreads();
        if (own < a.nblocks) {
            const int begin = own * a.per_block, end = min(begin + a.per_block, a.tokens);
            for (int i = begin + threadIdx.x % EX_THREADS; i < end; i += EX_THREADS) atomicAdd(&h[sub][(ex_key<FIRST>(a, i) >> a.shift) & a.mask], 1u);
        }
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += threads) {
            uint32_t sum = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (4 * block + k < a.nblocks) a.hist[(size_t)(4 * block + k) * bins + d] = sum;
                sum += h[k][d];
            }
            a.totals[(size_t)block * bins + d] = sum;
        }
    }
};

__device__ __forceinline__ uint32_t ex_scan(uint32_t v, uint32_t* wsum, uint32_t& total) {   // exclusive, 256 threads
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    uint32_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) base += wsum[w];
        total += wsum[w];
    }
    return base + incl - v;
}

// hist [blocks][bins] -> where each block's first token of each digit goes, counted from the digit's first; totals [bins].
// A workgroup has 32 digits (a line of each block's counts); 32 chunks of up to 32 blocks are scanned side by side.
#define EX_SCAN_THREADS 1024
static_assert(EX_MAX_BLOCKS <= 32 * 32, "blocks of one scan");
struct EmScan {
    static const int threads = EX_SCAN_THREADS;
    uint32_t* __restrict__ hist;
    uint32_t* __restrict__ totals;
    int nblocks, bins;
    __device__ __forceinline__ void run(int block) const {
        __shared__ uint32_t sums[32][33];
        const int d = threadIdx.x & 31, chunk = threadIdx.x >> 5, digit = block * 32 + d;
        const int each = (nblocks + 31) / 32, b0 = chunk * each;
        uint32_t v[32], s = 0;
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = k < each && b0 + k < nblocks && digit < bins ? hist[(size_t)(b0 + k) * bins + digit] : 0u;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += v[k];
        sums[chunk][d] = s;
        __syncthreads();
        uint32_t run = 0, all = 0;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            run += c < chunk ? sums[c][d] : 0u;
            all += sums[c][d];
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            if (k < each && b0 + k < nblocks && digit < bins) hist[(size_t)(b0 + k) * bins + digit] = run;
            run += v[k];
        }
        if (chunk == 0 && digit < bins) totals[digit] = all;
    }
};

template <bool FIRST, int EX_IPL>
struct EmScatter {
    static const int threads = EX_THREADS;
    EmSort a;
    __device__ __forceinline__ void run(int block) const {
        static_assert(EX_BINS == 2 * EX_THREADS, "a thread has two neighbouring digits");
        __shared__ uint32_t running[EX_BINS];            // next place of each digit for this workgroup
        __shared__ uint32_t cnt[4][EX_BINS];             // a wave's count of each digit, then where its first one lies in the tile
        __shared__ uint32_t shift_to[EX_BINS];           // from a place in the tile to the place in the output
        __shared__ uint2 ordered[EX_TILE(EX_IPL)];       // the tile in the order of its digits
        __shared__ uint32_t wsum[4];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int bins = 1 << a.bits;
        {
            uint32_t total;
            const int d = 2 * threadIdx.x;
            const bool in0 = d < bins, in1 = d + 1 < bins;
            uint32_t t0 = 0, t1 = 0, h0 = 0, h1 = 0;
            if (a.ngroups) {
                // two digits to a thread; where there are fewer than 512, several threads to the two divide the groups
                static_assert(sizeof(ordered) >= EX_THREADS * sizeof(uint4), "a sum of each thread");
                uint4* part = (uint4*)ordered;
                const int pairs = bins / 2, apart = EX_THREADS / pairs, q = threadIdx.x % pairs;
                uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll 8
                for (int g = threadIdx.x / pairs; g < a.ngroups; g += apart) {
                    const uint2 c = ((const uint2*)a.totals)[(size_t)g * pairs + q];
                    sum.x += c.x;
                    sum.y += c.y;
                    if (g < block / 4) {
                        sum.z += c.x;
                        sum.w += c.y;
                    }
                }
                part[threadIdx.x] = sum;
                __syncthreads();
                if (in0) {
                    for (int k = 0; k < apart; ++k) {
                        const uint4 c = part[threadIdx.x + k * pairs];
                        t0 += c.x;
                        t1 += c.y;
                        h0 += c.z;
                        h1 += c.w;
                    }
                }
            } else {
                t0 = in0 ? a.totals[d] : 0u;
                t1 = in1 ? a.totals[d + 1] : 0u;
            }
            if (in0) h0 += a.hist[(size_t)block * bins + d];
            if (in1) h1 += a.hist[(size_t)block * bins + d + 1];
            const uint32_t base = ex_scan(t0 + t1, wsum, total);
            running[d] = base + h0;
            running[d + 1] = base + t0 + h1;
        }
        const int begin = block * a.per_block, end = min(begin + a.per_block, a.tokens);
        const unsigned long long below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
        for (int tile = begin; tile < end; tile += EX_TILE(EX_IPL)) {
#pragma unroll
            for (int w = 0; w < 4; ++w) cnt[w][threadIdx.x] = cnt[w][threadIdx.x + EX_THREADS] = 0;
            __syncthreads();
            uint32_t key[EX_IPL], tok[EX_IPL], rank[EX_IPL];
            const int at = tile + wave * (64 * EX_IPL) + lane;
#pragma unroll
            for (int k = 0; k < EX_IPL; ++k) {
                const int i = at + 64 * k;
                if (FIRST) {
                    key[k] = i < end ? ex_key<true>(a, i) : 0xFFFFFFFFu;
                    tok[k] = (uint32_t)i;
                } else {
                    const uint2 e = i < end ? a.in[i] : make_uint2(0xFFFFFFFFu, 0u);
                    key[k] = e.x;
                    tok[k] = e.y;
                }
            }
#pragma unroll
            for (int k = 0; k < EX_IPL; ++k) {
                const bool ok = at + 64 * k < end;
                const uint32_t d = (key[k] >> a.shift) & a.mask;
                const unsigned long long peers = ex_peers(d, a.bits, ok);
                const uint32_t first = (uint32_t)__popcll(peers & below);
                const uint32_t prev = ok ? cnt[wave][d] : 0u;
                rank[k] = prev + first;
                if (ok && first == 0) cnt[wave][d] = prev + (uint32_t)__popcll(peers);
            }
            __syncthreads();
            {
                const int d = 2 * threadIdx.x;
                uint32_t c[2][4], all;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    c[0][w] = cnt[w][d];
                    c[1][w] = cnt[w][d + 1];
                }
                const uint32_t n0 = c[0][0] + c[0][1] + c[0][2] + c[0][3], n1 = c[1][0] + c[1][1] + c[1][2] + c[1][3];
                uint32_t g = ex_scan(n0 + n1, wsum, all);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    shift_to[d + h] = running[d + h] - g;
                    running[d + h] += h ? n1 : n0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        cnt[w][d + h] = g;
                        g += c[h][w];
                    }
                }
            }
            __syncthreads();
            // through LDS: written from there, the tokens of a digit are neighbours (a store of 64 lanes touches a few runs and
            // not 64 places; 13 us instead of 21 for a pass of 6 bits over 2,000,000)
#pragma unroll
            for (int k = 0; k < EX_IPL; ++k) {
                if (at + 64 * k < end) {
                    const uint32_t to = cnt[wave][(key[k] >> a.shift) & a.mask] + rank[k];
                    ordered[to] = make_uint2(key[k], tok[k]);
                }
            }
            __syncthreads();
            const int have = min(end - tile, EX_TILE(EX_IPL));
            for (int j = threadIdx.x; j < have; j += EX_THREADS) {
                const uint2 e = ordered[j];
                a.out[shift_to[(e.x >> a.shift) & a.mask] + (uint32_t)j] = e;
            }
            __syncthreads();
        }
    }
};

// ---- the walk ----
#define EW_THREADS 256
#define EW_SHARE 64                                  // items of a share at most
#define EW_ITEMS 2048                                // items of a workgroup's shares at most: their tokens lie in LDS
#define EW_BATCH 4                                   // tokens whose rows are loaded before the first is added
#define EW_SMALL FDGS_EMBEDDING_FEW                  // so few tokens are sorted by every workgroup for itself

struct EmBwd {
    const uint2* sorted;                             // (key, token)
    const void* ids; const void* dout; void* dtable;
    float* head; float* tail;                        // [shares][dim] partial sums of rows that a share's end cuts
    uint32_t* info;                                  // [shares] EW_HEAD | row: the share ends a row that began earlier
    uint8_t* fresh;                                  // [shares] 1: the row that is cut at the share's end began in it
    long long dout_stride, items, padding;           // items: rows + tokens
    int tokens, rows, dim, nv, lanes, groups, share, shares, wide;
    int walkers;                                     // the walk's groups (the join has others)
    float scale;
};
#define EW_HEAD 0x80000000u

// First sorted token whose place in the sequence (its index + its key) is not below `d`, by the whole wave.
__device__ __forceinline__ int ew_search(const uint2* __restrict__ sorted, int tokens, long long d) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = d < tokens ? (int)d : tokens;   // places grow by one at least: token d's is not below d
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const int less = __popcll(__ballot(i < hi && (long long)i + (long long)sorted[i].x < d));   // a prefix of the lanes
        if (less == 0) break;
        hi = min(hi, lo + less * step);
        lo += (less - 1) * step + 1;
    }
    return lo;
}

// A row that a share's end cuts (its first token lies before the end and its write does not) leaves partial sums: the
// shares in which it does not end leave theirs in `tail`, the one in which it ends in `head`, and a later launch adds them.
// (Letting the share in which a short row begins read on to its end saves most of the joins, but the shares of one wave
// wait for one another: 26 us instead of 17 at 300,000 tokens of 48 floats.)
// SMALL: all tokens are sorted here, no other launch is needed, and the share in which a row begins does read on.
template <class T, int VEC, bool SMALL>
__global__ void __launch_bounds__(EW_THREADS)
embedding_walk_kernel(EmBwd a) {
    typedef EmVec<T, VEC> Vec;
    typedef typename T::raw raw;
    const int cap = SMALL ? EW_SMALL : EW_ITEMS + 1;
    __shared__ uint32_t sk[cap], sp[cap];            // keys and tokens k0 <= index < k1 of the sorted list
    __shared__ uint32_t raw_key[SMALL ? EW_SMALL : 1];
    __shared__ int bound[2];
    const int span = a.groups * a.share, wave = threadIdx.x >> 6;
    const long long d0 = (long long)blockIdx.x * span;
    const long long d1 = min(d0 + span, a.items);
    int k0, k1, i0, i1;
    if (SMALL) {
        if ((int)threadIdx.x < a.tokens) raw_key[threadIdx.x] = em_key(a.ids, threadIdx.x, a.wide, a.padding, (uint32_t)a.rows);
        __syncthreads();
        if ((int)threadIdx.x < a.tokens) {
            const uint32_t key = raw_key[threadIdx.x];
            int r = 0;
            for (int j = 0; j < a.tokens; ++j) {
                const uint32_t o = raw_key[j];
                r += o < key || (o == key && j < (int)threadIdx.x) ? 1 : 0;
            }
            sk[r] = key;
            sp[r] = threadIdx.x;
        }
        k0 = i0 = 0;
        k1 = i1 = a.tokens;
    } else {
        if (wave < 2) {
            const int i = ew_search(a.sorted, a.tokens, wave ? d1 : d0);
            if ((threadIdx.x & 63) == 0) bound[wave] = i;
        }
        __syncthreads();
        i0 = bound[0];
        i1 = bound[1];                               // i1 - i0 <= span
        k0 = max(i0 - 1, 0);
        k1 = i1;                                     // k1 - k0 <= span + 1 <= cap
        for (int j = k0 + (int)threadIdx.x; j < k1; j += EW_THREADS) {
            const uint2 e = a.sorted[j];
            sk[j - k0] = e.x;
            sp[j - k0] = e.y;
        }
    }
    __syncthreads();
    const int group = threadIdx.x / a.lanes;
    const int c = blockIdx.y * a.lanes + (int)threadIdx.x - group * a.lanes;
    const long long from = d0 + (long long)group * a.share, to = min(from + a.share, d1);
    const long long share = (long long)blockIdx.x * a.groups + group;
    const bool idle = group >= a.groups || c >= a.nv;
    const raw* src = (const raw*)a.dout + em_col<VEC>(idle ? 0 : c, a.nv, a.dim);
    // All items are tokens of one row that began before them: the shares' sums are added up here and left as the last one's,
    // which spares the join all but one of them (gradient of 300,000 tokens of 48 floats, all of one row: 54 us, 127 without).
    if (!SMALL && a.groups > 1 && i1 - i0 == span && i0 > 0 && sk[i0 - 1 - k0] == sk[i1 - 1 - k0] && sk[i1 - 1 - k0] < (uint32_t)a.rows) {
        static_assert(SMALL || EW_THREADS * VEC <= EW_ITEMS, "a sum of each thread in place of the keys");
        float sum[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
        if (!idle) {
            const int p = i0 - k0 + group * a.share;
#pragma unroll 4
            for (int q = p; q < p + a.share; ++q) {
                const Vec x = *(const Vec*)(src + (long long)sp[q] * a.dout_stride);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += em_up<T>(x.x[j]);
            }
        }
        __syncthreads();
        float* sums = (float*)sk;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[threadIdx.x * VEC + j] = sum[j];
        __syncthreads();
        if (idle) return;
        if (group == 0) {
            for (int q = 1; q < a.groups; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += sums[(threadIdx.x + q * a.lanes) * VEC + j];
            float* t = a.tail + (share + a.groups - 1) * a.dim + em_col<VEC>(c, a.nv, a.dim);
#pragma unroll
            for (int j = 0; j < VEC; ++j) t[j] = sum[j];
        }
        if (c == 0) {
            a.info[share] = 0;
            a.fresh[share] = 0;
        }
        return;
    }
    if (idle) return;
    if (from >= d1) {                                // behind the last item
        if (!SMALL && c == 0) {
            a.info[share] = 0;
            a.fresh[share] = 0;
        }
        return;
    }
    auto key_at = [&](int i) { return i >= k0 && i < k1 ? sk[i - k0] : 0xFFFFFFFFu; };
    auto place = [&](int lo, int hi, long long d) {  // first token from lo on, before hi, whose place is not below d
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if ((long long)m + (long long)sk[m - k0] < d) lo = m + 1; else hi = m;
        }
        return lo;
    };
    int i = place(i0, i1, from);
    const int ie = place(i, min(i1, i + a.share), to);
    uint32_t v = (uint32_t)(from - i);               // the first row whose write may be the share's
    const uint32_t ve = (uint32_t)(to - ie);         // the first whose write is not
    const uint32_t rows = (uint32_t)a.rows;
    const int col = em_col<VEC>(c, a.nv, a.dim);
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    const bool began = i > 0 && key_at(i - 1) == v && v < rows;      // row v began in an earlier share
    const bool inside = began && v == ve;                            // and ends in a later one
    bool head = !SMALL && began;
    const uint32_t note = head && !inside ? EW_HEAD | v : 0u;
    if (SMALL && began) {                            // that share finishes it
        while (i < ie && key_at(i) == v) ++i;
        if (!inside) ++v;
    }
    bool any = !SMALL && began;                      // the row has tokens
    auto flush = [&](uint32_t row) {
        if (head) {
            float* h = a.head + share * a.dim + col;
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[j] = acc[j];
            head = false;
        } else {
            Vec o;
            const float scale = any ? a.scale : 0.0f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.x[j] = em_down<T>(acc[j] * scale);
            em_store<T, VEC>((raw*)a.dtable + (long long)row * a.dim + col, o);
        }
        any = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    };
    // Writes the rows up to `end`: the one that is being added, and behind it rows without tokens, which are zeros whatever
    // the scale is.
    auto write = [&](uint32_t end) {
        if (v >= end) return;
        flush(v);
        ++v;
        const Vec zero = {};
        raw* p = (raw*)a.dtable + (long long)v * a.dim + col;
#pragma unroll 4
        for (; v < end; ++v, p += a.dim) em_store<T, VEC>(p, zero);
    };
    // adds tokens p .. q, writing the rows that end in between; tokens without a row come last of all
    auto walk = [&](int p, int q) {
        while (p < q) {
            Vec x[EW_BATCH];
#pragma unroll
            for (int u = 0; u < EW_BATCH; ++u)
                if (p + u < q) x[u] = *(const Vec*)(src + (long long)sp[p + u - k0] * a.dout_stride);
#pragma unroll
            for (int u = 0; u < EW_BATCH; ++u) {
                if (p + u < q) {
                    const uint32_t key = sk[p + u - k0];
                    write(key);
                    any = true;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += em_up<T>(x[u].x[j]);
                }
            }
            p += EW_BATCH;
        }
    };
    int valid = ie;
    if (valid > i && key_at(valid - 1) >= rows) {
        if (key_at(i) >= rows) valid = i;
        while (valid > i && key_at(valid - 1) >= rows) --valid;
    }
    walk(i, valid);
    write(ve);
    const bool open = ie > 0 && key_at(ie - 1) == ve && ve < rows;   // a row that a later share ends in the sequence
    if (!SMALL && open) {
        float* t = a.tail + share * a.dim + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t[j] = acc[j];
    } else if (SMALL && open && !inside) {           // begun here: finished here
        int e = ie;
        while (key_at(e) == ve) ++e;
        walk(ie, e);
        flush(ve);
    }
    if (!SMALL && c == 0) {
        a.info[share] = note;
        a.fresh[share] = open && !inside ? 1 : 0;
    }
}

// ---- rows that were cut: the partial sums of the shares from the row's first token on, in order ----
// A workgroup looks at as many shares as it has groups of lanes, 4 to 16: no more, because a row of more than 16 partial sums
// takes all of it, and no two of those end within 16 shares (16,384 tokens of 100 rows of 8: 21 us, 42 with up to 256).
#define EC_SCAN(groups) ((groups) < 4 ? 4 : (groups) > 16 ? 16 : (groups))
#define EC_LONG (-2)                                 // more partial sums than two looks at the flags reach: 16

template <class T, int VEC>
__device__ __forceinline__ void ec_write(const EmBwd& a, uint32_t row, int col, const float* acc) {
    EmVec<T, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.x[j] = em_down<T>(acc[j] * a.scale);
    *(EmVec<T, VEC>*)((typename T::raw*)a.dtable + (long long)row * a.dim + col) = o;
}

template <int VEC>
__device__ __forceinline__ void ec_add(const float* p, float* acc) {
    typedef EmVec<EmF32, VEC> V;
    const V x = *(const V*)p;
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += x.x[j];
}

// The partial sums of a row from share `first` on, before the share `end` in which it ends: one of each share, but (SOME) one,
// its last share's, of a workgroup of the walk that has several shares and lies inside the row.
template <bool SOME>
struct EmSums {
    int first, head, whole, count, behind, walkers;
    __device__ __forceinline__ EmSums(int f, int end, int w) : first(f), walkers(w) {
        const int b0 = f / w, b1 = end / w;
        const bool all = !SOME || b1 - b0 < 2;
        head = all ? end - f : (b0 + 1) * w - f;
        whole = all ? 0 : b1 - b0 - 1;
        behind = b1 * w;
        count = all ? head : head + whole + end - behind;
    }
    // adds the sums from .. to, in order; tail: the column's sum of share 0
    template <int VEC>
    __device__ __forceinline__ void add(int from, int to, const float* tail, int dim, float* acc) const {
        auto run = [&](int lo, int hi, int share, int step) {    // sums lo .. hi, the first one of `share`
#pragma unroll 4
            for (int q = 0; q < hi - lo; ++q) ec_add<VEC>(tail + (long long)(share + q * step) * dim, acc);
        };
        if (!SOME || whole == 0) {
            run(from, to, first + from, 1);
        } else {
            run(from, min(to, head), first + from, 1);
            const int w0 = max(from, head), b0 = max(from, head + whole);
            run(w0, min(to, head + whole), first + head + (w0 - head + 1) * walkers - 1, walkers);
            run(b0, to, behind + b0 - head - whole, 1);
        }
    }
};

struct __attribute__((packed, aligned(1))) EmFlags8 { unsigned long long x; };

template <class T, int VEC, bool SOME>
__global__ void __launch_bounds__(EW_THREADS)
embedding_join_kernel(EmBwd a) {
    __shared__ int first_of[EC_SCAN(EW_THREADS)], end_of[EC_SCAN(EW_THREADS)];     // first and last share of the cut rows
    __shared__ uint32_t row_of[EC_SCAN(EW_THREADS)], count;
    __shared__ float sums[EW_THREADS * VEC];
    const int lane = threadIdx.x & 63;
    const int group = threadIdx.x / a.lanes;
    const int c = blockIdx.y * a.lanes + (int)threadIdx.x - group * a.lanes;
    const bool in = group < a.groups && c < a.nv;
    const int col = in ? em_col<VEC>(c, a.nv, a.dim) : 0;
    const int scan = EC_SCAN(a.groups);
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int s = blockIdx.x * scan + (int)threadIdx.x;
    if ((int)threadIdx.x < scan && s < a.shares) {
        // first share of the row that ends here: the nearest one before in which a cut row began (that row is the row: the
        // shares in between lie inside it).  Two looks at eight flags; a row that began earlier is a long one.
        const uint32_t note = a.info[s];
        const EmFlags8 f = *(const EmFlags8*)(a.fresh + s - 8);              // (what lies in front of the array is never the nearest)
        const EmFlags8 e = *(const EmFlags8*)(a.fresh + s - 16);
        if (note & EW_HEAD) {
            const uint32_t at = atomicAdd(&count, 1u);
            first_of[at] = f.x ? s - 1 - (__clzll((long long)f.x) >> 3) : e.x ? s - 9 - (__clzll((long long)e.x) >> 3) : EC_LONG;
            end_of[at] = s;
            row_of[at] = note & ~EW_HEAD;
        }
    }
    __syncthreads();
    const int n = (int)count;
    if (in) {
        for (int e = group; e < n; e += a.groups) {
            if (first_of[e] == EC_LONG) continue;
            float acc[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            ec_add<VEC>(a.head + (long long)end_of[e] * a.dim + col, acc);
            const EmSums<SOME> sum(first_of[e], end_of[e], a.walkers);
            sum.template add<VEC>(0, sum.count, a.tail + col, a.dim, acc);
            ec_write<T, VEC>(a, row_of[e], col, acc);
        }
    }
    for (int g = 0; g < n; ++g) {                    // long ones: the groups divide the shares, the first one adds up
        if (first_of[g] != EC_LONG) continue;
        const int end = end_of[g];
        const uint32_t row = row_of[g];
        int lo = 0, hi = a.tokens;                   // the row's first token, by every wave
        while (lo < hi) {
            const int step = (hi - lo + 63) / 64;
            const int i = lo + lane * step;
            const int less = __popcll(__ballot(i < hi && a.sorted[i].x < row));
            if (less == 0) break;
            hi = min(hi, lo + less * step);
            lo += (less - 1) * step + 1;
        }
        const int first = (int)(((long long)lo + (long long)row) / a.share);
        const EmSums<SOME> sum(first, end, a.walkers);
        const int each = (sum.count + a.groups - 1) / a.groups, used = (sum.count + each - 1) / each;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        if (in) sum.template add<VEC>(group * each, min((group + 1) * each, sum.count), a.tail + col, a.dim, acc);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[threadIdx.x * VEC + j] = acc[j];
        __syncthreads();
        if (in && group == 0) {
            for (int q = 1; q < used; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += sums[(threadIdx.x + q * a.lanes) * VEC + j];
            ec_add<VEC>(a.head + (long long)end * a.dim + col, acc);
            ec_write<T, VEC>(a, row, col, acc);
        }
    }
}

// ---- host: sizes, workspace, launches ----
// Where a sort's work lies in the workspace.
struct EmSortPlan { size_t other, hist, totals, bytes; };
static EmSortPlan em_sort_plan(long long tokens) {
    EmSortPlan p;
    size_t at = 0;
    auto take = [&at](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
    const bool radix = tokens > EL_TOKENS;
    p.other = take(radix ? tokens * 8 : 0);
    p.hist = take(radix ? (size_t)EX_BINS * EX_MAX_BLOCKS * 4 : 0);
    p.totals = take(radix ? EX_TOTALS * 4 : 0);
    p.bytes = at;
    return p;
}

struct EmPlan {
    int vec, nv, tiles, lanes, groups, share;
    int join_tiles, join_lanes;
    long long shares, blocks, joins;                 // blocks and joins: workgroups in x
    size_t sorted, sort, info, fresh, head, tail, bytes;   // offsets into the workspace
};

static EmPlan em_plan(long long tokens, long long rows, int dim, int type) {
    EmPlan p;
    p.vec = dim >= em_full(type) ? em_full(type) : 1;
    p.nv = (dim + p.vec - 1) / p.vec;
    p.tiles = (p.nv + EW_THREADS - 1) / EW_THREADS;
    p.lanes = (p.nv + p.tiles - 1) / p.tiles;
    p.groups = EW_THREADS / p.lanes;
    // Long shares where rows have several tokens (every share then leaves partial sums: at 2,000,000 tokens of 65,536 rows
    // walk and join take 112 us with 64 items, 115 with 32, 124 with 16), short ones where most rows have none and a long
    // share only makes the last workgroups end later (16,384 tokens of 65,536 rows of 2048: 83, 77, 73 us, 75 with 8), and
    // not so long that there are too few workgroups (300,000 tokens of 8,192 rows: 26.6, 23.9, 24.3 us, 26.0 with 8).
    const long long items = tokens + rows;
    auto workgroups = [&](int share) { return (items + (long long)p.groups * share - 1) / ((long long)p.groups * share) * p.tiles; };
    p.share = tokens > rows ? EW_SHARE : 16;
    while (p.share > 16 && workgroups(p.share) < 1024) p.share >>= 1;
    while (p.share > 8 && workgroups(p.share) < 256) p.share >>= 1;
    while (p.groups * p.share > EW_ITEMS) p.share >>= 1;
    p.blocks = (tokens + rows + (long long)p.groups * p.share - 1) / ((long long)p.groups * p.share);
    p.shares = p.blocks * p.groups;
    // at most 64 lanes to a row in the join, so that there are groups to divide the partial sums of a long one
    p.join_tiles = (p.nv + 63) / 64;
    p.join_lanes = (p.nv + p.join_tiles - 1) / p.join_tiles;
    const int scan = EC_SCAN(EW_THREADS / p.join_lanes);
    p.joins = (p.shares + scan - 1) / scan;
    size_t at = 0;
    auto take = [&at](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
    p.sorted = take(tokens * 8);
    p.sort = take(em_sort_plan(tokens).bytes);
    const bool small = tokens <= EW_SMALL;           // no row is cut
    p.info = take(small ? 0 : p.shares * 4);
    p.fresh = take(small ? 0 : p.shares + 16) + 16;
    p.head = take(small ? 0 : (size_t)p.shares * dim * 4);
    p.tail = take(small ? 0 : (size_t)p.shares * dim * 4);
    p.bytes = at > 0 ? at : 256;                      // a workspace is asked for always
    return p;
}

extern "C" size_t fdgs_embedding_bwd_workspace_bytes(int64_t num_tokens, int32_t num_rows, int32_t dim, int32_t type) {
    if (num_tokens < 0 || num_rows < 0 || dim < 1 || !em_type_ok(type)) return 0;
    return em_plan(num_tokens, num_rows, dim, type).bytes;
}

// The launches of a sort, each with its part of a lookup.
struct EmSteps {
    EmPart part;
    long long groups;                                // of the lookup, 0: none
    int whole, at;                                   // weights of the launches: of all, of those that are done
    hipStream_t s;
    template <class Step>
    int run(const Step& step, int blocks, int weight) {
        const int each = Step::threads / EF_THREADS;
        part.first = (int)(groups * at / whole);
        at += weight;
        part.last = (int)(groups * at / whole);
        const int more = (part.last - part.first + each - 1) / each;
        const int period = more >= 2 * blocks ? 3 : 1;
        hipLaunchKernelGGL((embedding_step_kernel<Step>), dim3((unsigned)(blocks + more)), dim3(Step::threads), 0, s, step, blocks, period, part);
        FDGS_CHECK_LAUNCH();
        return FDGS_OK;
    }
};

#define EM_RUN(call) do { const int rc_ = (call); if (rc_ != FDGS_OK) return rc_; } while (0)
// sorted [tokens] pairs, ws: a workspace of em_sort_plan(tokens).bytes; lookup: its workgroups run beside (NULL: none)
static int em_sort(const EmIds& in, uint2* sorted, char* ws, const EmPart* lookup, long long groups, hipStream_t s) {
    const int tokens = in.tokens;
    const EmSortPlan p = em_sort_plan(tokens);
    EmSteps steps = {};
    steps.s = s;
    steps.whole = 1;
    if (lookup) {
        steps.part = *lookup;
        steps.groups = groups;
    }
    int key_bits = 1;
    while (key_bits < 31 && (1ll << key_bits) <= (long long)in.rows) ++key_bits;       // keys 0 .. rows
    const int passes = (key_bits + EX_BITS - 1) / EX_BITS;
    if (tokens <= ER_TOKENS * passes) return steps.run(EmRank{in, sorted}, (tokens + 63) / 64, 1);
    if (tokens <= EL_TOKENS) return steps.run(EmList{in, key_bits, passes, sorted}, 1, 1);
    if (tokens <= EL_LISTS * EL_TOKENS && passes > 1) {
        uint2* lists = (uint2*)(ws + p.other);
        steps.whole = 2;
        EM_RUN(steps.run(EmList{in, key_bits, passes, lists}, (tokens + EL_TOKENS - 1) / EL_TOKENS, 1));
        return steps.run(EmMerge{lists, tokens, sorted}, (tokens + EmMerge::threads - 1) / EmMerge::threads, 1);
    }
    // a workgroup's tile takes 5 us whatever its length: short tiles while there are workgroups to be had for them
    const int ipl = tokens <= EX_MAX_BLOCKS * EX_TILE(2) / 2 ? 2 : tokens <= EX_MAX_BLOCKS * EX_TILE(4) ? 4 : 8;
    long long tiles = ((long long)tokens + EX_TILE(ipl) - 1) / EX_TILE(ipl), blocks = tiles < EX_MAX_BLOCKS ? tiles : EX_MAX_BLOCKS;
    const long long per_block = (tiles + blocks - 1) / blocks * EX_TILE(ipl);
    blocks = (tokens + per_block - 1) / per_block;
    EmSort k = {};
    k.ids = in; k.tokens = tokens;
    k.per_block = (int)per_block; k.nblocks = (int)blocks;
    k.hist = (uint32_t*)(ws + p.hist); k.totals = (uint32_t*)(ws + p.totals);
    const long long ngroups = (blocks + 3) / 4;
    const int most_bits = (key_bits + passes - 1) / passes;
    const long long counts = ngroups << most_bits;
    k.ngroups = counts <= EX_TOTALS && counts * blocks <= EX_READS ? (int)ngroups : 0;
    // The lookup goes where workgroups wait most, and in large parts (a part takes 2 us at least): to the scatters, and a little
    // of it to the scans, which leave most of the chip idle.  Sort and lookup of 2,000,000 tokens of 48 floats 152 us (one after
    // the other 163, all of it in the scatters 153, the same in every launch 164); without scans, of 300,000 tokens 33 us (a
    // quarter of it in the counts 36; with scans 37, with scans and one after the other 43).
    const int with_scan = k.ngroups ? 0 : 1, with_scatter = 5;
    steps.whole = (with_scan + with_scatter) * passes;
    for (int pass = 0; pass < passes; ++pass) {
        k.bits = (key_bits - k.shift + passes - pass - 1) / (passes - pass);           // the remaining bits, evenly
        k.mask = (1u << k.bits) - 1u;
        const bool to_first = ((passes - 1 - pass) & 1) == 0;                          // the last pass ends in `sorted`
        k.out = to_first ? sorted : (uint2*)(ws + p.other);
        k.in = to_first ? (const uint2*)(ws + p.other) : sorted;
        const int n = (int)blocks;
        if (k.ngroups) {
            EM_RUN(pass == 0 ? steps.run(EmHist4<true>{k}, k.ngroups, 0) : steps.run(EmHist4<false>{k}, k.ngroups, 0));
        } else {
            EM_RUN(pass == 0 ? steps.run(EmHist<true>{k}, n, 0) : steps.run(EmHist<false>{k}, n, 0));
            EM_RUN(steps.run(EmScan{k.hist, k.totals, k.nblocks, 1 << k.bits}, ((1 << k.bits) + 31) / 32, with_scan));
        }
        if (pass == 0) EM_RUN(ipl == 2 ? steps.run(EmScatter<true, 2>{k}, n, with_scatter) : ipl == 4 ? steps.run(EmScatter<true, 4>{k}, n, with_scatter) : steps.run(EmScatter<true, 8>{k}, n, with_scatter));
        else EM_RUN(ipl == 2 ? steps.run(EmScatter<false, 2>{k}, n, with_scatter) : ipl == 4 ? steps.run(EmScatter<false, 4>{k}, n, with_scatter) : steps.run(EmScatter<false, 8>{k}, n, with_scatter));
        k.shift += k.bits;
    }
    return FDGS_OK;
}

extern "C" size_t fdgs_embedding_sort_workspace_bytes(int64_t num_tokens) {
    return num_tokens < 0 || num_tokens > FDGS_EMBEDDING_MAX_TOKENS ? 0 : em_sort_plan(num_tokens).bytes;
}

extern "C" int fdgs_embedding_fwd(const fdgs_embedding_fwd_args* a, void* stream) {
    if (!a || a->num_tokens < 0 || a->num_rows < 0 || a->dim < 0 || !em_type_ok(a->type)) return FDGS_EINVAL;
    if (a->id_bytes != 4 && a->id_bytes != 8) return FDGS_EINVAL;
    if (a->num_tokens == 0 || a->dim == 0) return FDGS_OK;
    if (!a->ids || !a->out || (a->num_rows > 0 && !a->table)) return FDGS_EINVAL;
    if (a->num_rows > 0 && a->table_row_stride < 0) return FDGS_EINVAL;
    if (a->dim > FDGS_EMBEDDING_MAX_DIM || a->num_tokens > (a->sorted ? FDGS_EMBEDDING_MAX_TOKENS : 0x7fffffffLL)) return FDGS_ETOOLARGE;
    EmPart f = {};
    EmFwd& k = f.a;
    k.ids = a->ids; k.table = a->table; k.out = a->out;
    k.tokens = (int)a->num_tokens; k.table_stride = a->table_row_stride;
    k.padding = a->padding_id >= 0 ? a->padding_id : -1;
    k.rows = a->num_rows; k.dim = a->dim; k.wide = a->id_bytes == 8; k.scale = a->scale;
    f.type = a->type;
    f.vec = k.dim >= em_full(a->type) ? em_full(a->type) : 1;
    k.nv = (k.dim + f.vec - 1) / f.vec;
    k.by_nv = em_div_of((uint32_t)k.nv);
    // Four vectors a thread where rows come from behind L2 for long (2,000,000 x 48 floats from 12.6 MB of table, with the sort:
    // 153 us, 160 with two), else two (the kernel for 300,000 x 48 floats, launched by itself, 12.4 us, 14 with four, 17 with eight;
    // for one token 2.1, 2.7, 3.2).
    const long long size = a->type == FDGS_TYPE_F32 ? 4 : 2, row = (long long)k.dim * size;
    k.vectors = row * k.rows > (4 << 20) && row * k.tokens > (64 << 20) ? EF_VECTORS : EF_VECTORS / 2;
    k.per_group = k.nv < k.vectors ? k.vectors / k.nv : 1;
    const int tiles = (k.nv + k.vectors - 1) / k.vectors;
    const long long groups = ((long long)k.tokens + k.per_group - 1) / k.per_group;
    hipStream_t s = (hipStream_t)stream;
    const bool sort = a->sorted && a->num_tokens > EW_SMALL;     // fewer are sorted where they are added
    if (sort) {
        if (a->workspace_bytes < em_sort_plan(a->num_tokens).bytes || (a->workspace_bytes > 0 && !a->workspace)) return FDGS_EWORKSPACE;
        const EmIds in = {a->ids, k.padding, (uint32_t)a->num_rows, k.tokens, k.wide};
        f.by_tiles = em_div_of((uint32_t)tiles);
        // (in one launch of the sort there are at most 1024 workgroups of 256 threads, or as many threads, beside them)
        const bool beside = groups * tiles <= FDGS_MAX_GROUPS(EF_THREADS) - 2048;
        EM_RUN(em_sort(in, (uint2*)a->sorted, (char*)a->workspace, beside ? &f : nullptr, groups * tiles, s));
        if (beside) return FDGS_OK;
    }
    for (long long g = 0; g < groups; g += FDGS_MAX_GROUPS(EF_THREADS)) {
        const long long now = std::min(groups - g, FDGS_MAX_GROUPS(EF_THREADS)), token = g * k.per_group;
        EmFwd part = k;
        part.ids = (const char*)k.ids + token * a->id_bytes;
        part.out = (char*)k.out + token * row;
        part.tokens = (int)std::min(k.tokens - token, now * k.per_group);
        const dim3 grid((unsigned)now, (unsigned)tiles);
        if (a->type == FDGS_TYPE_F32) EM_RUN(em_fwd_launch<EmF32>(part, f.vec, grid, s));
        else if (a->type == FDGS_TYPE_BF16) EM_RUN(em_fwd_launch<EmBf16>(part, f.vec, grid, s));
        else EM_RUN(em_fwd_launch<EmF16>(part, f.vec, grid, s));
    }
    return FDGS_OK;
}

template <class T>
static int em_bwd_launch(const EmBwd& k, const EmPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)p.blocks, (unsigned)p.tiles), threads(EW_THREADS);
    if (k.tokens <= EW_SMALL) {
        if (p.vec > 1) hipLaunchKernelGGL((embedding_walk_kernel<T, T::full, true>), grid, threads, 0, s, k);
        else hipLaunchKernelGGL((embedding_walk_kernel<T, 1, true>), grid, threads, 0, s, k);
        FDGS_CHECK_LAUNCH();
        return FDGS_OK;
    }
    if (p.vec > 1) hipLaunchKernelGGL((embedding_walk_kernel<T, T::full, false>), grid, threads, 0, s, k);
    else hipLaunchKernelGGL((embedding_walk_kernel<T, 1, false>), grid, threads, 0, s, k);
    FDGS_CHECK_LAUNCH();
    EmBwd j = k;
    j.lanes = p.join_lanes;
    j.groups = EW_THREADS / p.join_lanes;
    const dim3 joins((unsigned)p.joins, (unsigned)p.join_tiles);
    if (p.vec == 1) hipLaunchKernelGGL((embedding_join_kernel<T, 1, true>), joins, threads, 0, s, j);
    else if (p.groups > 1) hipLaunchKernelGGL((embedding_join_kernel<T, T::full, true>), joins, threads, 0, s, j);
    else hipLaunchKernelGGL((embedding_join_kernel<T, T::full, false>), joins, threads, 0, s, j);
    FDGS_CHECK_LAUNCH();
    return FDGS_OK;
}

extern "C" int fdgs_embedding_bwd(const fdgs_embedding_bwd_args* a, void* stream) {
    if (!a || a->num_tokens < 0 || a->num_rows < 0 || a->dim < 0 || !em_type_ok(a->type)) return FDGS_EINVAL;
    if (a->id_bytes != 4 && a->id_bytes != 8) return FDGS_EINVAL;
    if (a->num_rows == 0 || a->dim == 0) return FDGS_OK;
    if (!a->grad_table || (a->num_tokens > 0 && (!a->ids || !a->grad_out)) || a->grad_out_row_stride < 0) return FDGS_EINVAL;
    if (a->dim > FDGS_EMBEDDING_MAX_DIM || a->num_tokens > FDGS_EMBEDDING_MAX_TOKENS) return FDGS_ETOOLARGE;
    const EmPlan p = em_plan(a->num_tokens, a->num_rows, a->dim, a->type);
    static_assert(FDGS_EMBEDDING_MAX_DIM / EmF32::full / 64 <= 65535, "column tiles in a grid's second dimension");
    if (p.shares > 0x7fffffffLL || p.blocks > FDGS_MAX_GROUPS(EW_THREADS) || p.joins > FDGS_MAX_GROUPS(EW_THREADS)) return FDGS_ETOOLARGE;
    if (!a->workspace || a->workspace_bytes < p.bytes) return FDGS_EWORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)a->workspace;
    const long long padding = a->padding_id >= 0 ? a->padding_id : -1;
    EmBwd k = {};
    k.sorted = (const uint2*)(a->sorted ? a->sorted : ws + p.sorted);
    if (a->num_tokens > EW_SMALL && !a->sorted) {
        const EmIds in = {a->ids, padding, (uint32_t)a->num_rows, (int)a->num_tokens, a->id_bytes == 8};
        EM_RUN(em_sort(in, (uint2*)(ws + p.sorted), ws + p.sort, nullptr, 0, s));
    }
    k.dout = a->grad_out; k.dtable = a->grad_table;
    k.head = (float*)(ws + p.head); k.tail = (float*)(ws + p.tail); k.fresh = (uint8_t*)(ws + p.fresh);
    k.info = (uint32_t*)(ws + p.info); k.shares = (int)p.shares;
    k.ids = a->ids; k.wide = a->id_bytes == 8; k.padding = padding;
    k.dout_stride = a->grad_out_row_stride; k.items = a->num_rows + a->num_tokens;
    k.tokens = (int)a->num_tokens; k.rows = a->num_rows; k.dim = a->dim; k.nv = p.nv; k.lanes = p.lanes; k.groups = p.groups;
    k.share = p.share; k.walkers = p.groups; k.scale = a->scale;
    if (a->type == FDGS_TYPE_F32) return em_bwd_launch<EmF32>(k, p, s);
    if (a->type == FDGS_TYPE_BF16) return em_bwd_launch<EmBf16>(k, p, s);
    return em_bwd_launch<EmF16>(k, p, s);
}
