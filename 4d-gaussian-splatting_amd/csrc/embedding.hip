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
// partial sums in the workspace, which a last launch adds up in the shares' order.  No atomics.
#include "fdgs_common.h"
#include <hip/hip_bf16.h>

// ---- element types: 16 bytes to a vector where the row is that long, else one element ----
struct EmF32 { typedef float raw; static const int full = 4; };
struct EmBf16 { typedef uint16_t raw; static const int full = 8; };
struct EmF16 { typedef uint16_t raw; static const int full = 8; };

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

// ---- forward ----
#define EF_THREADS 256
#define EF_UNROLL 4

struct EmFwd {
    const void* ids; const void* table; void* out;
    long long tokens, table_stride, padding, vectors;    // vectors: tokens * nv
    int rows, dim, nv, wide;
    float scale;
    EmDiv by_nv;
};

template <class T, int VEC>
__global__ void __launch_bounds__(EF_THREADS)
embedding_fwd_kernel(EmFwd a) {
    typedef EmVec<T, VEC> Vec;
    typedef typename T::raw raw;
    // the workgroup's first vector as (token, vector): one 64-bit division, the rest in 32 bits
    const long long first = (long long)blockIdx.x * (EF_THREADS * EF_UNROLL);
    const long long tok0 = first / a.nv;
    const uint32_t rem = (uint32_t)(first - tok0 * a.nv);
    Vec v[EF_UNROLL];
    long long at[EF_UNROLL];
    int col[EF_UNROLL];
    uint32_t key[EF_UNROLL];
    bool nan[EF_UNROLL];
#pragma unroll
    for (int u = 0; u < EF_UNROLL; ++u) {
        const uint32_t e = rem + (uint32_t)(u * EF_THREADS) + threadIdx.x;
        const uint32_t t = em_div(e, a.by_nv);
        at[u] = first + u * EF_THREADS + (int)threadIdx.x < a.vectors ? tok0 + t : -1;
        col[u] = em_col<VEC>((int)(e - t * a.by_nv.d), a.nv, a.dim);
        key[u] = (uint32_t)a.rows;
        nan[u] = false;
        if (at[u] >= 0) {
            const long long id = a.wide ? ((const long long*)a.ids)[at[u]] : (long long)((const int*)a.ids)[at[u]];
            if (id != a.padding) {
                if (id >= 0 && id < a.rows) key[u] = (uint32_t)id;
                nan[u] = id >= a.rows;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < EF_UNROLL; ++u)
        if (key[u] < (uint32_t)a.rows) v[u] = *(const Vec*)((const raw*)a.table + (long long)key[u] * a.table_stride + col[u]);
#pragma unroll
    for (int u = 0; u < EF_UNROLL; ++u) {
        if (at[u] < 0) continue;
        Vec o;
        const float other = nan[u] ? __builtin_nanf("") : 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.x[j] = em_down<T>(key[u] < (uint32_t)a.rows ? em_up<T>(v[u].x[j]) * a.scale : other);
        *(Vec*)((raw*)a.out + at[u] * a.dim + col[u]) = o;
    }
}

template <class T>
static int em_fwd_launch(const EmFwd& k0, hipStream_t s) {
    EmFwd k = k0;
    const int vec = k.dim >= T::full ? T::full : 1;
    k.nv = (k.dim + vec - 1) / vec;
    k.vectors = k.tokens * k.nv;
    k.by_nv = em_div_of((uint32_t)k.nv);
    const long long groups = (k.vectors + EF_THREADS * EF_UNROLL - 1) / (EF_THREADS * EF_UNROLL);
    if (groups > 0x7fffffffLL) return FDGS_ETOOLARGE;
    if (vec > 1) hipLaunchKernelGGL((embedding_fwd_kernel<T, T::full>), dim3((unsigned)groups), dim3(EF_THREADS), 0, s, k);
    else hipLaunchKernelGGL((embedding_fwd_kernel<T, 1>), dim3((unsigned)groups), dim3(EF_THREADS), 0, s, k);
    FDGS_CHECK_LAUNCH();
    return FDGS_OK;
}

static bool em_type_ok(int t) { return t == FDGS_TYPE_F32 || t == FDGS_TYPE_BF16 || t == FDGS_TYPE_F16; }
#define EM_MAX_DIM (1 << 24)                         // em_div's operands stay below 2^31

extern "C" int fdgs_embedding_fwd(const fdgs_embedding_fwd_args* a, void* stream) {
    if (!a || a->num_tokens < 0 || a->num_rows < 0 || a->dim < 0 || !em_type_ok(a->type)) return FDGS_EINVAL;
    if (a->id_bytes != 4 && a->id_bytes != 8) return FDGS_EINVAL;
    if (a->num_tokens == 0 || a->dim == 0) return FDGS_OK;
    if (!a->ids || !a->out || (a->num_rows > 0 && !a->table)) return FDGS_EINVAL;
    if (a->num_rows > 0 && a->table_row_stride < 0) return FDGS_EINVAL;
    if (a->dim > EM_MAX_DIM || a->num_tokens > 0x7fffffffLL) return FDGS_ETOOLARGE;
    EmFwd k = {};
    k.ids = a->ids; k.table = a->table; k.out = a->out;
    k.tokens = a->num_tokens; k.table_stride = a->table_row_stride;
    k.padding = a->padding_id >= 0 ? a->padding_id : -1;
    k.rows = a->num_rows; k.dim = a->dim; k.wide = a->id_bytes == 8; k.scale = a->scale;
    hipStream_t s = (hipStream_t)stream;
    if (a->type == FDGS_TYPE_F32) return em_fwd_launch<EmF32>(k, s);
    if (a->type == FDGS_TYPE_BF16) return em_fwd_launch<EmBf16>(k, s);
    return em_fwd_launch<EmF16>(k, s);
}

// ---- the tokens by row: (key, token) pairs, stable ----
// Few tokens: a token's place is the number of tokens that come before it, counted against all of them; the workgroup has
// 64 tokens, its waves divide the others.  T^2 / 64 comparisons of a wave spread over the chip, one launch.
#define ER_THREADS 256
#define ER_CHUNK 4096                                // keys staged in LDS at a time
#define ER_MAX_TOKENS 16384

__global__ void __launch_bounds__(ER_THREADS)
embedding_rank_kernel(const void* __restrict__ ids, int tokens, int wide, long long padding, uint32_t rows,
                      uint32_t* __restrict__ keys, uint32_t* __restrict__ perm) {
    __shared__ __align__(16) uint32_t sk[ER_CHUNK];
    __shared__ uint32_t part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int own = blockIdx.x * 64;                 // first token of the workgroup
    const int me = own + lane;
    const uint32_t key = me < tokens ? em_key(ids, me, wide, padding, rows) : 0xFFFFFFFFu;
    uint32_t before = 0;
    for (int c0 = 0; c0 < tokens; c0 += ER_CHUNK) {
        __syncthreads();
        for (int j = threadIdx.x; j < ER_CHUNK; j += ER_THREADS)
            sk[j] = c0 + j < tokens ? em_key(ids, c0 + j, wide, padding, rows) : 0xFFFFFFFFu;   // after every key
        __syncthreads();
        // blocks of 64 keys, one wave each: those before the own tokens win ties, those behind lose them
        for (int b = wave * 64; b < ER_CHUNK && c0 + b < tokens; b += 256) {
            if (c0 + b == own) {
                for (int j = 0; j < 64; ++j) {
                    const uint32_t o = sk[b + j];
                    before += (o < key || (o == key && j < lane)) ? 1u : 0u;
                }
            } else {
                const uint32_t limit = key + (c0 + b < own ? 1u : 0u);       // o <= key, or o < key
                const uint4* q = (const uint4*)(sk + b);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint4 o = q[j];
                    before += (o.x < limit ? 1u : 0u) + (o.y < limit ? 1u : 0u) + (o.z < limit ? 1u : 0u) + (o.w < limit ? 1u : 0u);
                }
            }
        }
    }
    part[wave][lane] = before;
    __syncthreads();
    if (wave == 0 && me < tokens) {
        const uint32_t r = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
        keys[r] = key;
        perm[r] = (uint32_t)me;
    }
}

// Many tokens: a radix sort by digits of at most 8 bits, three launches a pass (histogram, scan of its rows, scatter).
#define EX_THREADS 256
#define EX_IPL 8
#define EX_TILE (EX_THREADS * EX_IPL)
#define EX_BINS 256
#define EX_MAX_BLOCKS 1024

struct EmSort {
    const void* ids;                                 // first pass: the tokens' ids; later passes: keys_in
    const uint32_t* keys_in; const uint32_t* perm_in;
    uint32_t* keys_out; uint32_t* perm_out;
    uint32_t* hist; uint32_t* totals;
    long long padding;
    uint32_t rows, mask;
    int tokens, per_block, nblocks, shift, bits, wide;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t ex_key(const EmSort& a, int i) {
    return FIRST ? em_key(a.ids, i, a.wide, a.padding, a.rows) : a.keys_in[i];
}

template <bool FIRST>
__global__ void __launch_bounds__(EX_THREADS)
embedding_hist_kernel(EmSort a) {
    __shared__ uint32_t h[EX_BINS];
    for (int d = threadIdx.x; d < EX_BINS; d += EX_THREADS) h[d] = 0;
    __syncthreads();
    const int begin = blockIdx.x * a.per_block, end = min(begin + a.per_block, a.tokens);
    for (int i = begin + threadIdx.x; i < end; i += EX_THREADS) atomicAdd(&h[(ex_key<FIRST>(a, i) >> a.shift) & a.mask], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < EX_BINS; d += EX_THREADS) a.hist[(size_t)d * a.nblocks + blockIdx.x] = h[d];
}

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

__global__ void __launch_bounds__(EX_THREADS)
embedding_rowscan_kernel(uint32_t* __restrict__ hist, uint32_t* __restrict__ totals, int nblocks) {
    __shared__ uint32_t wsum[4];
    uint32_t* row = hist + (size_t)blockIdx.x * nblocks;
    uint32_t v[4], s = 0, total;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = threadIdx.x * 4 + k;
        v[k] = i < nblocks ? row[i] : 0u;
        s += v[k];
    }
    uint32_t run = ex_scan(s, wsum, total);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = threadIdx.x * 4 + k;
        if (i < nblocks) row[i] = run;
        run += v[k];
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = total;
}

template <bool FIRST>
__global__ void __launch_bounds__(EX_THREADS)
embedding_scatter_kernel(EmSort a) {
    __shared__ uint32_t running[EX_BINS];            // next place of each digit for this workgroup
    __shared__ uint32_t cnt[4][EX_BINS];             // a wave's count of each digit, then where its first one goes
    __shared__ uint32_t wsum[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bins = 1 << a.bits;
    {
        uint32_t total;
        const int d = threadIdx.x;
        const uint32_t base = ex_scan(d < bins ? a.totals[d] : 0u, wsum, total);
        running[d] = d < bins ? base + a.hist[(size_t)d * a.nblocks + blockIdx.x] : 0u;
    }
    const int begin = blockIdx.x * a.per_block, end = min(begin + a.per_block, a.tokens);
    const unsigned long long below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    for (int tile = begin; tile < end; tile += EX_TILE) {
#pragma unroll
        for (int w = 0; w < 4; ++w) cnt[w][threadIdx.x] = 0;
        __syncthreads();
        uint32_t key[EX_IPL], tok[EX_IPL], rank[EX_IPL];
        const int at = tile + wave * (64 * EX_IPL) + lane;
#pragma unroll
        for (int k = 0; k < EX_IPL; ++k) {
            const int i = at + 64 * k;
            key[k] = i < end ? ex_key<FIRST>(a, i) : 0xFFFFFFFFu;
            tok[k] = FIRST ? (uint32_t)i : (i < end ? a.perm_in[i] : 0u);
        }
#pragma unroll
        for (int k = 0; k < EX_IPL; ++k) {
            const bool ok = at + 64 * k < end;
            const uint32_t d = (key[k] >> a.shift) & a.mask;
            unsigned long long peers = __ballot(ok);  // lanes with the same digit
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                if (b < a.bits) {
                    const unsigned long long bal = __ballot((d >> b) & 1u);
                    peers &= ((d >> b) & 1u) ? bal : ~bal;
                }
            }
            const uint32_t first = (uint32_t)__popcll(peers & below);
            const uint32_t prev = ok ? cnt[wave][d] : 0u;
            rank[k] = prev + first;
            if (ok && first == 0) cnt[wave][d] = prev + (uint32_t)__popcll(peers);
        }
        __syncthreads();
        {
            const int d = threadIdx.x;
            const uint32_t c0 = cnt[0][d], c1 = cnt[1][d], c2 = cnt[2][d], c3 = cnt[3][d], g = running[d];
            cnt[0][d] = g;
            cnt[1][d] = g + c0;
            cnt[2][d] = g + c0 + c1;
            cnt[3][d] = g + c0 + c1 + c2;
            running[d] = g + c0 + c1 + c2 + c3;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EX_IPL; ++k) {
            if (at + 64 * k < end) {
                const uint32_t to = cnt[wave][(key[k] >> a.shift) & a.mask] + rank[k];
                a.keys_out[to] = key[k];
                a.perm_out[to] = tok[k];
            }
        }
        __syncthreads();
    }
}

// ---- the walk ----
#define EW_THREADS 256
#define EW_ITEMS 2048                                // items of a workgroup's shares at most: their tokens lie in LDS
#define EW_BATCH 4                                   // tokens whose rows are loaded before the first is added

struct EmBwd {
    const uint32_t* keys; const uint32_t* perm;      // sorted
    const void* dout; void* dtable;
    float* head; float* tail;                        // [shares][dim] partial sums of rows that a share's end cuts
    uint32_t* info;                                  // [shares] EW_HEAD | EW_FRESH | row of the head
    long long dout_stride, items;                    // items: rows + tokens
    int tokens, rows, dim, nv, lanes, groups, share, shares;
    float scale;
};
#define EW_HEAD 0x80000000u                          // the share ends a row that began in an earlier share
                                                     // (that row's number in the low 31 bits)

// First sorted token whose place in the sequence (its index + its key) is not below `d`, by the whole wave.
__device__ __forceinline__ int ew_search(const uint32_t* __restrict__ keys, int tokens, long long d) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = d < tokens ? (int)d : tokens;   // places grow by one at least: token d's is not below d
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const int i = lo + lane * step;
        const bool less = i < hi && (long long)i + (long long)keys[i] < d;
        const int c = __popcll(__ballot(less));      // a prefix of the lanes
        if (c == 0) break;
        const int nlo = lo + (c - 1) * step + 1;
        hi = min(hi, lo + c * step);
        lo = nlo;
    }
    return lo;
}

template <class T, int VEC>
__global__ void __launch_bounds__(EW_THREADS)
embedding_walk_kernel(EmBwd a) {
    typedef EmVec<T, VEC> Vec;
    typedef typename T::raw raw;
    __shared__ uint32_t sk[EW_ITEMS + 1], sp[EW_ITEMS];   // sk[0]: the key before the first
    __shared__ int bound[2];
    const int span = a.groups * a.share;
    const long long d0 = (long long)blockIdx.x * span;
    const long long d1 = min(d0 + span, a.items);
    const int wave = threadIdx.x >> 6;
    if (wave < 2) {
        const int i = ew_search(a.keys, a.tokens, wave ? d1 : d0);
        if ((threadIdx.x & 63) == 0) bound[wave] = i;
    }
    __syncthreads();
    const int i0 = bound[0], i1 = bound[1], have = i1 - i0;       // have <= span <= EW_ITEMS
    for (int j = threadIdx.x; j < have; j += EW_THREADS) {
        sk[j + 1] = a.keys[i0 + j];
        sp[j] = a.perm[i0 + j];
    }
    if (threadIdx.x == 0) sk[0] = i0 > 0 ? a.keys[i0 - 1] : 0xFFFFFFFFu;
    __syncthreads();
    const int group = threadIdx.x / a.lanes;
    const int c = blockIdx.y * a.lanes + (int)threadIdx.x - group * a.lanes;
    const long long from = d0 + (long long)group * a.share;
    if (group >= a.groups || c >= a.nv) return;
    if (from >= d1) {                                // behind the last item
        if (c == 0) a.info[(long long)blockIdx.x * a.groups + group] = 0;
        return;
    }
    const long long to = min(from + a.share, d1);
    int i, ie;                                       // the share's tokens, counted from i0
    {
        int lo = 0, hi = have;
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if ((long long)(i0 + m) + (long long)sk[m + 1] < from) lo = m + 1; else hi = m;
        }
        i = lo;
        hi = min(have, i + a.share);
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if ((long long)(i0 + m) + (long long)sk[m + 1] < to) lo = m + 1; else hi = m;
        }
        ie = lo;
    }
    uint32_t v = (uint32_t)(from - (i0 + i));        // the first row that the share may end
    const uint32_t ve = (uint32_t)(to - (i0 + ie));  // the first that it does not
    if (ie > i && sk[ie] >= (uint32_t)a.rows) {      // tokens without a row come last, behind the last row's end
        if (sk[i + 1] >= (uint32_t)a.rows) ie = i;
        while (ie > i && sk[ie] >= (uint32_t)a.rows) --ie;
    }
    const long long share = (long long)blockIdx.x * a.groups + group;
    const int col = em_col<VEC>(c, a.nv, a.dim);
    bool head = (i0 + i) > 0 && sk[i] == v;          // tokens of row v lie in earlier shares
    const uint32_t note = head && v < ve ? EW_HEAD | v : 0u;
    const int i_first = i;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    auto flush = [&](uint32_t row) {
        if (head) {
            float* h = a.head + share * a.dim + col;
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[j] = acc[j];
            head = false;
        } else {
            Vec o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.x[j] = em_down<T>(acc[j] * a.scale);
            *(Vec*)((raw*)a.dtable + (long long)row * a.dim + col) = o;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
    };
    const raw* src = (const raw*)a.dout + col;
    while (i < ie) {
        Vec x[EW_BATCH];
#pragma unroll
        for (int u = 0; u < EW_BATCH; ++u)
            if (i + u < ie) x[u] = *(const Vec*)(src + (long long)sp[i + u] * a.dout_stride);
#pragma unroll
        for (int u = 0; u < EW_BATCH; ++u) {
            if (i + u < ie) {
                const uint32_t key = sk[i + u + 1];
                while (v < key) { flush(v); ++v; }
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += em_up<T>(x[u].x[j]);
            }
        }
        i += EW_BATCH;
    }
    while (v < ve) { flush(v); ++v; }
    if (ie > i_first && sk[ie] == ve && ve < (uint32_t)a.rows) {   // tokens of a row that a later share ends
        float* t = a.tail + share * a.dim + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t[j] = acc[j];
    }
    if (c == 0) a.info[share] = note;
}

// ---- rows that were cut: the partial sums of the shares from the row's first token on, in order ----
#define EC_SHORT 12                                  // up to so many partial sums a group adds by itself

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

template <class T, int VEC>
__global__ void __launch_bounds__(EW_THREADS)
embedding_join_kernel(EmBwd a) {
    __shared__ int first_of[EW_THREADS];
    __shared__ float sums[EW_THREADS * VEC];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s0 = blockIdx.x * a.groups, n = min(a.groups, a.shares - s0);
    // first share of each cut row: where the row's first token lies
    for (int g = wave; g < n; g += 4) {
        const uint32_t note = a.info[s0 + g];
        int first = -1;
        if (note & EW_HEAD) {
            const uint32_t row = note & ~EW_HEAD;
            int lo = 0, hi = a.tokens;               // first token with that key, by the wave
            while (lo < hi) {
                const int step = (hi - lo + 63) / 64;
                const int i = lo + lane * step;
                const int c = __popcll(__ballot(i < hi && a.keys[i] < row));
                if (c == 0) break;
                const int nlo = lo + (c - 1) * step + 1;
                hi = min(hi, lo + c * step);
                lo = nlo;
            }
            first = (int)(((long long)lo + (long long)row) / a.share);
        }
        if (lane == 0) first_of[g] = first;
    }
    __syncthreads();
    const int group = threadIdx.x / a.lanes;
    const int c = blockIdx.y * a.lanes + (int)threadIdx.x - group * a.lanes;
    const bool in = group < a.groups && c < a.nv;
    const int col = in ? em_col<VEC>(c, a.nv, a.dim) : 0;
    if (in && group < n) {
        const int s = s0 + group, first = first_of[group];
        if (first >= 0 && s - first <= EC_SHORT) {
            float acc[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
            for (int q = first; q < s; ++q) ec_add<VEC>(a.tail + (long long)q * a.dim + col, acc);
            ec_add<VEC>(a.head + (long long)s * a.dim + col, acc);
            ec_write<T, VEC>(a, a.info[s] & ~EW_HEAD, col, acc);
        }
    }
    for (int g = 0; g < n; ++g) {                    // long ones: the groups divide the shares, the first one adds up
        const int s = s0 + g, first = first_of[g];
        if (first < 0 || s - first <= EC_SHORT) continue;
        const int each = (s - first + a.groups - 1) / a.groups;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        if (in) {
            const int end = min(first + (group + 1) * each, s);
#pragma unroll 4
            for (int q = first + group * each; q < end; ++q) ec_add<VEC>(a.tail + (long long)q * a.dim + col, acc);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[threadIdx.x * VEC + j] = acc[j];
        __syncthreads();
        if (in && group == 0) {
            for (int q = 1; q < a.groups; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += sums[(threadIdx.x + q * a.lanes) * VEC + j];
            ec_add<VEC>(a.head + (long long)s * a.dim + col, acc);
            ec_write<T, VEC>(a, a.info[s] & ~EW_HEAD, col, acc);
        }
    }
}

// ---- host: sizes, workspace, launches ----
struct EmPlan {
    int vec, nv, tiles, lanes, groups, share;
    long long shares, blocks;
    size_t keys, perm, keys2, perm2, hist, totals, info, head, tail, bytes;   // offsets into the workspace
};

static int em_full(int type) { return type == FDGS_TYPE_F32 ? EmF32::full : EmBf16::full; }

static EmPlan em_plan(long long tokens, long long rows, int dim, int type) {
    EmPlan p;
    p.vec = dim >= em_full(type) ? em_full(type) : 1;
    p.nv = (dim + p.vec - 1) / p.vec;
    p.tiles = (p.nv + EW_THREADS - 1) / EW_THREADS;
    p.lanes = (p.nv + p.tiles - 1) / p.tiles;
    p.groups = EW_THREADS / p.lanes;
    p.share = 32;
    while (p.share > 8 && (tokens + rows) * p.tiles / p.share < 4096) p.share >>= 1;   // few items: shorter shares, more of them
    while (p.groups * p.share > EW_ITEMS) p.share >>= 1;
    p.blocks = (tokens + rows + (long long)p.groups * p.share - 1) / ((long long)p.groups * p.share);
    p.shares = p.blocks * p.groups;
    size_t at = 0;
    auto take = [&at](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
    p.keys = take(tokens * 4);
    p.perm = take(tokens * 4);
    const bool radix = tokens > ER_MAX_TOKENS;
    p.keys2 = take(radix ? tokens * 4 : 0);
    p.perm2 = take(radix ? tokens * 4 : 0);
    p.hist = take(radix ? (size_t)EX_BINS * EX_MAX_BLOCKS * 4 : 0);
    p.totals = take(radix ? EX_BINS * 4 : 0);
    p.info = take(p.shares * 4);
    p.head = take((size_t)p.shares * dim * 4);
    p.tail = take((size_t)p.shares * dim * 4);
    p.bytes = at;
    return p;
}

extern "C" size_t fdgs_embedding_bwd_workspace_bytes(int64_t num_tokens, int32_t num_rows, int32_t dim, int32_t type) {
    if (num_tokens < 0 || num_rows < 0 || dim < 1 || !em_type_ok(type)) return 0;
    return em_plan(num_tokens, num_rows, dim, type).bytes;
}

// Sorted pairs end up in (ws + p.keys, ws + p.perm).
static int em_sort(const fdgs_embedding_bwd_args* a, const EmPlan& p, char* ws, hipStream_t s) {
    const int tokens = (int)a->num_tokens;
    const long long padding = a->padding_id >= 0 ? a->padding_id : -1;
    const int wide = a->id_bytes == 8;
    if (tokens <= ER_MAX_TOKENS) {
        hipLaunchKernelGGL(embedding_rank_kernel, dim3((tokens + 63) / 64), dim3(ER_THREADS), 0, s, a->ids, tokens, wide, padding,
                           (uint32_t)a->num_rows, (uint32_t*)(ws + p.keys), (uint32_t*)(ws + p.perm));
        FDGS_CHECK_LAUNCH();
        return FDGS_OK;
    }
    int key_bits = 1;
    while (key_bits < 31 && (1ll << key_bits) <= (long long)a->num_rows) ++key_bits;   // keys 0 .. num_rows
    const int passes = (key_bits + 7) / 8;
    long long tiles = ((long long)tokens + EX_TILE - 1) / EX_TILE, blocks = tiles < EX_MAX_BLOCKS ? tiles : EX_MAX_BLOCKS;
    const long long per_block = (tiles + blocks - 1) / blocks * EX_TILE;
    blocks = (tokens + per_block - 1) / per_block;
    EmSort k = {};
    k.ids = a->ids; k.wide = wide; k.padding = padding; k.rows = (uint32_t)a->num_rows; k.tokens = tokens;
    k.per_block = (int)per_block; k.nblocks = (int)blocks;
    k.hist = (uint32_t*)(ws + p.hist); k.totals = (uint32_t*)(ws + p.totals);
    for (int pass = 0; pass < passes; ++pass) {
        k.bits = (key_bits - k.shift + passes - pass - 1) / (passes - pass);           // the remaining bits, evenly
        k.mask = (1u << k.bits) - 1u;
        const bool to_first = ((passes - 1 - pass) & 1) == 0;                          // the last pass ends in keys / perm
        k.keys_out = (uint32_t*)(ws + (to_first ? p.keys : p.keys2));
        k.perm_out = (uint32_t*)(ws + (to_first ? p.perm : p.perm2));
        k.keys_in = (const uint32_t*)(ws + (to_first ? p.keys2 : p.keys));
        k.perm_in = (const uint32_t*)(ws + (to_first ? p.perm2 : p.perm));
        const dim3 grid((unsigned)blocks), threads(EX_THREADS);
        if (pass == 0) hipLaunchKernelGGL(embedding_hist_kernel<true>, grid, threads, 0, s, k);
        else hipLaunchKernelGGL(embedding_hist_kernel<false>, grid, threads, 0, s, k);
        FDGS_CHECK_LAUNCH();
        hipLaunchKernelGGL(embedding_rowscan_kernel, dim3(1u << k.bits), threads, 0, s, k.hist, k.totals, k.nblocks);
        FDGS_CHECK_LAUNCH();
        if (pass == 0) hipLaunchKernelGGL(embedding_scatter_kernel<true>, grid, threads, 0, s, k);
        else hipLaunchKernelGGL(embedding_scatter_kernel<false>, grid, threads, 0, s, k);
        FDGS_CHECK_LAUNCH();
        k.shift += k.bits;
    }
    return FDGS_OK;
}

template <class T>
static int em_bwd_launch(const EmBwd& k, const EmPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)p.blocks, (unsigned)p.tiles), threads(EW_THREADS);
    if (p.vec > 1) {
        hipLaunchKernelGGL((embedding_walk_kernel<T, T::full>), grid, threads, 0, s, k);
        FDGS_CHECK_LAUNCH();
        if (k.tokens > 0) hipLaunchKernelGGL((embedding_join_kernel<T, T::full>), grid, threads, 0, s, k);
    } else {
        hipLaunchKernelGGL((embedding_walk_kernel<T, 1>), grid, threads, 0, s, k);
        FDGS_CHECK_LAUNCH();
        if (k.tokens > 0) hipLaunchKernelGGL((embedding_join_kernel<T, 1>), grid, threads, 0, s, k);
    }
    FDGS_CHECK_LAUNCH();
    return FDGS_OK;
}

extern "C" int fdgs_embedding_bwd(const fdgs_embedding_bwd_args* a, void* stream) {
    if (!a || a->num_tokens < 0 || a->num_rows < 0 || a->dim < 0 || !em_type_ok(a->type)) return FDGS_EINVAL;
    if (a->id_bytes != 4 && a->id_bytes != 8) return FDGS_EINVAL;
    if (a->num_rows == 0 || a->dim == 0) return FDGS_OK;
    if (!a->grad_table || (a->num_tokens > 0 && (!a->ids || !a->grad_out)) || a->grad_out_row_stride < 0) return FDGS_EINVAL;
    if (a->dim > EM_MAX_DIM || a->num_tokens > FDGS_EMBEDDING_MAX_TOKENS) return FDGS_ETOOLARGE;
    const EmPlan p = em_plan(a->num_tokens, a->num_rows, a->dim, a->type);
    if (p.shares > 0x7fffffffLL || p.tiles > 65535) return FDGS_ETOOLARGE;
    if (!a->workspace || a->workspace_bytes < p.bytes) return FDGS_EWORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)a->workspace;
    if (a->num_tokens > 0) {
        const int rc = em_sort(a, p, ws, s);
        if (rc != FDGS_OK) return rc;
    }
    EmBwd k = {};
    k.keys = (const uint32_t*)(ws + p.keys); k.perm = (const uint32_t*)(ws + p.perm);
    k.dout = a->grad_out; k.dtable = a->grad_table;
    k.head = (float*)(ws + p.head); k.tail = (float*)(ws + p.tail); k.info = (uint32_t*)(ws + p.info);
    k.dout_stride = a->grad_out_row_stride; k.items = a->num_rows + a->num_tokens;
    k.tokens = (int)a->num_tokens; k.rows = a->num_rows; k.dim = a->dim; k.nv = p.nv; k.lanes = p.lanes; k.groups = p.groups;
    k.share = p.share; k.shares = (int)p.shares; k.scale = a->scale;
    if (a->type == FDGS_TYPE_F32) return em_bwd_launch<EmF32>(k, p, s);
    if (a->type == FDGS_TYPE_BF16) return em_bwd_launch<EmBf16>(k, p, s);
    return em_bwd_launch<EmF16>(k, p, s);
}
