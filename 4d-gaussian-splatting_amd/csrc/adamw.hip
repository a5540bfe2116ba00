// AdamW over many tensors in one launch (moments in float32 or in 8 bits, parameters in float32 or in
// bfloat16), and the 8-bit moments' conversions.
//
//   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
//   p = (1 - lr wd) p - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Memory-bound.  Bytes per element: float32 parameters 28 with float32 moments, 16 with 8-bit ones; bfloat16
// parameters 26 and 14 (parameter, the 16 bits it drops, gradient, moments).  A wave takes a block of 256 consecutive
// elements, four to a lane, which is also the 8-bit moments' block: its exponent is a reduction inside the wave, with
// no LDS and no barrier.  Loads and stores are 4 elements wide at any alignment of the element's own size (gfx950
// takes unaligned global accesses), so tensors packed back to back need no slower path.
//
// The products and sums are not contracted to fused multiply-adds: which code an 8-bit moment gets then depends on
// the formula alone and not on the compiler's choices, and the same step is the same bits on every replica.
#include "moment8.h"
#include <type_traits>

#define AW_MAX 40                                // tensors whose records fill 4 KB of kernel arguments
// A wave has one block (with two the step over 2,000,000 Gaussians with 8-bit moments, and their read-out, takes 3 % longer),
// a workgroup eight of them (97 bfloat16 tensors: 184 us, 192 with four, 185 with sixteen, with which 8-bit moments lose 4 to 10 %).
#define AW_THREADS 512
#define AW_PER_GROUP (AW_THREADS / 64 * M8_BLOCK)

struct AwTensor {
    void* p; const void* g; void* m; void* v;
    int16_t* low; uint8_t* me; uint8_t* ve;
    long long n, gstride;
    int glen;
    float step_size, inv_root, decay;
    uint32_t key, pad;
};
struct AwStep {
    float b1, omb1, b2, omb2, eps;
};
template <class Record, int MAX>
struct AwPart {
    Record t[MAX];
    int start[MAX];                              // first workgroup of each tensor
    int num;
};
// The one that workgroup `b` works on (scalar; six steps for 40 tensors.  Comparing with every start is more work than
// the waiting it saves: 8 % for the 8-bit step over 2,000,000 Gaussians, a lane each through vector loads 2 %.)
template <class Ints>
__device__ __forceinline__ int aw_find(Ints start, int num, int b) {
    int lo = 0, hi = num;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start[m] <= b) lo = m; else hi = m;
    }
    return lo;
}

// Where the records of a launch lie: in its arguments, or (more tensors than these hold) the last ones there and the others in a
// table in device memory that small launches before it have filled from theirs, 1.5 us each, the first of them up to 5.  60 float32 tensors of 5,000
// elements: 6.5 us (8.4 in two launches over arguments), 100: 9.4 (11.1 with all records in the table); 211 bfloat16 tensors
// with 8-bit moments and their read-out 181 (250 in six launches and five).
template <class Record, int MAX>
struct AwInArgs {
    AwPart<Record, MAX> part;
    __device__ __forceinline__ const Record& find(int b, int& first) const {
        const int i = aw_find(part.start, part.num, b);
        first = part.start[i];
        return part.t[i];
    }
};
// (The table is read through the constant address space: nothing in the launch writes it, so a record is loaded once and into
// scalar registers like the arguments.  As ordinary memory the 8-bit step reads it again behind every store: 131 us, not 94, for
// 40,000,000 elements.)
template <class Record, int MAX>
struct AwInBoth {
    AwPart<Record, MAX> part;
    int n;
    const Record* t;
    const int* start;
    typedef const __attribute__((address_space(4))) int* Ints;
    __device__ __forceinline__ Record find(int b, int& first) const {
        if (b >= part.start[0]) {
            const int i = aw_find(part.start, part.num, b);
            first = part.start[i];
            return part.t[i];
        }
        const Ints starts = (Ints)(uintptr_t)start;
        const int i = aw_find(starts, n, b);
        first = starts[i];
        int words[sizeof(Record) / 4];
        const Ints from = (Ints)(uintptr_t)(t + i);
#pragma unroll
        for (int k = 0; k < (int)(sizeof(Record) / 4); ++k) words[k] = from[k];
        return __builtin_bit_cast(Record, words);
    }
};
static_assert(sizeof(AwStep) + sizeof(AwInBoth<AwTensor, AW_MAX>) <= 4096, "kernel arguments of one launch");
template <class Record, int MAX>
__global__ void __launch_bounds__(256)
list_table_kernel(AwPart<Record, MAX> part, Record* table, int* start) {
    // one load a thread: the arguments are far away (with four after one another a fill took 4.8 us)
    struct __attribute__((packed, aligned(4))) W4 { uint32_t x[4]; };
    static_assert(MAX * sizeof(Record) <= 256 * sizeof(W4) && MAX * sizeof(Record) % sizeof(W4) == 0 && MAX <= 256, "one load a thread");
    const int i = threadIdx.x;
    const W4 x = i < (int)(MAX * sizeof(Record) / sizeof(W4)) ? ((const W4*)part.t)[i] : W4{};
    const int first = i < MAX ? part.start[i] : 0;
    uint32_t* to = (uint32_t*)table;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * i + j < part.num * (int)(sizeof(Record) / 4)) to[4 * i + j] = x.x[j];
    if (i < part.num) start[i] = first;
}
static size_t list_table_bytes(int num, size_t record) { return (size_t)num * (record + sizeof(int)) + 512; }

// Runs `launch(source, workgroups)` for all the records that `next(record, workgroups)` gives (false: no more): in one launch
// where the arguments hold them all or there is a workspace for the others, else in as many launches as it takes.
template <class Record, int MAX, class Next, class Launch>
static int list_launch(int count, void* workspace, size_t bytes, hipStream_t s, Next next, Launch launch) {
    const bool table = count > MAX && workspace && bytes >= list_table_bytes(count, sizeof(Record));
    Record* records = (Record*)(((uintptr_t)workspace + 255) / 256 * 256);
    int* starts = (int*)(records + count);
    AwInBoth<Record, MAX> both;
    AwPart<Record, MAX>& part = both.part;
    int blocks = 0, filled = 0, groups = 0;
    part.num = 0;
    for (Record r; next(r, groups); blocks += groups) {
        if (part.num == MAX) {
            if (table) {
                hipLaunchKernelGGL((list_table_kernel<Record, MAX>), dim3(1), dim3(256), 0, s, part, records + filled, starts + filled);
                filled += MAX;
            } else {
                launch(AwInArgs<Record, MAX>{part}, blocks);
                blocks = 0;
            }
            FDGS_CHECK_LAUNCH();
            part.num = 0;
        }
        part.t[part.num] = r;
        part.start[part.num++] = blocks;
    }
    if (part.num == 0) return FDGS_OK;
    both.n = filled;
    both.t = records;
    both.start = starts;
    if (filled) launch(both, blocks);
    else launch(AwInArgs<Record, MAX>{part}, blocks);
    FDGS_CHECK_LAUNCH();
    return FDGS_OK;
}

struct __attribute__((packed, aligned(4))) aw_f4 { float x[4]; };
struct __attribute__((packed, aligned(2))) aw_h4 { uint32_t x[2]; };   // four 16-bit numbers, two to a word
struct __attribute__((packed, aligned(1))) aw_b8 { uint32_t x[2]; };
struct __attribute__((packed, aligned(2))) aw_w4 { uint32_t x[4]; };

// Streaming accesses for what only the optimizer touches (moments, residuals) and for the gradient, which is used up:
// they leave the caches to the parameters, which the next forward pass reads.  At 300,000 Gaussians 108 -> 99 us.
typedef uint32_t aw_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t aw_u2 __attribute__((ext_vector_type(2)));
typedef aw_u4 aw_u4_at4 __attribute__((aligned(4)));
typedef aw_u2 aw_u2_at2 __attribute__((aligned(2)));
typedef uint32_t aw_u1_at1 __attribute__((aligned(1)));
__device__ __forceinline__ aw_f4 aw_take(const float* p) { return __builtin_bit_cast(aw_f4, __builtin_nontemporal_load((const aw_u4_at4*)p)); }
__device__ __forceinline__ aw_h4 aw_take(const uint16_t* p) { return __builtin_bit_cast(aw_h4, __builtin_nontemporal_load((const aw_u2_at2*)p)); }
__device__ __forceinline__ uint32_t aw_take(const uint8_t* p) { return __builtin_nontemporal_load((const aw_u1_at1*)p); }
__device__ __forceinline__ void aw_put(float* p, const aw_f4& x) { __builtin_nontemporal_store(__builtin_bit_cast(aw_u4, x), (aw_u4_at4*)p); }
__device__ __forceinline__ void aw_put(uint16_t* p, const aw_h4& x) { __builtin_nontemporal_store(__builtin_bit_cast(aw_u2, x), (aw_u2_at2*)p); }
__device__ __forceinline__ void aw_put(uint8_t* p, uint32_t x) { __builtin_nontemporal_store(x, (aw_u1_at1*)p); }

// float32 -> bfloat16 to the nearest, halves away from zero, and the signed 16 bits between the two: the pair is the
// float32 value again exactly, and (unlike rounding halves to even) the difference always fits: it is the pattern's low half.
__device__ __forceinline__ void aw_split(float w, uint16_t& hi, int16_t& lo) {
    const uint32_t b = __float_as_uint(w);
    const bool nan = w != w;
    hi = (uint16_t)(nan ? 0x7FC0u : (b + 0x8000u) >> 16);
    lo = (int16_t)(nan ? 0u : b);
}
// The weight: pattern plus residual, as far as the two belong together.  A zero has no residual below it and an infinity none above
// it; one that is written from outside (a mask, a reset) beside another weight's residual stays what it is instead of the NaN that the
// plain sum would make of it.
__device__ __forceinline__ float aw_weight(uint32_t hi, int lo) {     // hi: the pattern in the upper half, zeros below
    const int size = (int)(hi & 0x7FFFFFFFu), most = size > 0x7F800000 ? size : 0x7F800000;
    int w = size + lo;
    w = w > 0 ? w : 0;
    w = w < most ? w : most;
    return __uint_as_float((uint32_t)w | (hi & 0x80000000u));
}
__device__ __forceinline__ float aw_join(uint16_t hi, int16_t lo) { return aw_weight((uint32_t)hi << 16, lo); }
__device__ __forceinline__ void aw_split4(const float* w, aw_h4& h, aw_h4& l) {
    if (__ballot(__builtin_isunordered(w[0], w[1]) || __builtin_isunordered(w[2], w[3])) == 0) {     // no NaN in the wave
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t a = __float_as_uint(w[2 * j]), b = __float_as_uint(w[2 * j + 1]);
            h.x[j] = __builtin_amdgcn_perm(b + 0x8000u, a + 0x8000u, 0x07060302u);
            l.x[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint16_t h0, h1;
            int16_t l0, l1;
            aw_split(w[2 * j], h0, l0);
            aw_split(w[2 * j + 1], h1, l1);
            h.x[j] = h0 | ((uint32_t)h1 << 16);
            l.x[j] = (uint16_t)l0 | ((uint32_t)(uint16_t)l1 << 16);
        }
    }
}
__device__ __forceinline__ void aw_join4(const aw_h4& h, const aw_h4& l, float* w) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        w[2 * j] = aw_weight(h.x[j] << 16, (int)(l.x[j] << 16) >> 16);
        w[2 * j + 1] = aw_weight(h.x[j] & 0xFFFF0000u, (int)l.x[j] >> 16);
    }
}
__device__ __forceinline__ float aw_bf16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }

// The update, every operation correctly rounded.  (With the chip's root and reciprocal, 1.6 units of 2^-24 off each, the step over
// 2,000,000 Gaussians with 8-bit moments and their read-out takes 512 us, not 522; which form the moments have is no reason for
// another rounding.)
__device__ __forceinline__ float aw_update(float w, float m, float v, const AwStep& k, const AwTensor& t) {
#pragma clang fp contract(off)
    const float denom = sqrtf(v) * t.inv_root + k.eps;
    return w * t.decay - (m * t.step_size) / denom;
}

template <bool BF16>
__device__ __forceinline__ float aw_grad(const void* g, long long i) {
    return BF16 ? aw_bf16(((const uint16_t*)g)[i]) : ((const float*)g)[i];
}
// Four gradient elements from element i on in rows of L elements, S apart: a column slice of a wider array.
template <bool BF16>
__device__ __forceinline__ void aw_grad_rows(const AwTensor& t, long long i, int valid, float* out) {
    long long row;
    int col;
    if (t.n <= 0xFFFFFFFFLL) {                   // a 32-bit division where the index allows it
        const uint32_t r = (uint32_t)i / (uint32_t)t.glen;
        row = r;
        col = (int)((uint32_t)i - r * (uint32_t)t.glen);
    } else {
        row = i / t.glen;
        col = (int)(i - row * t.glen);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        out[j] = j < valid ? aw_grad<BF16>(t.g, row * t.gstride + col) : 0.0f;
        if (++col == t.glen) { col = 0; ++row; }
    }
}

// A lane's four elements of a block as they lie in memory.
template <bool BF16, bool EIGHT>
struct AwLane {
    float g[4], w[4], m[4], v[4];                // m, v: float32 moments only
    uint32_t cm, cv;                             // 8-bit moments' codes
    int em, ev;                                  // and their block's exponents
};

// WHOLE: the block has 256 elements.  Else a lane has `valid` (0 to 4) of its four and the rest are zeros.
template <bool BF16, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void aw_load(const AwTensor& t, long long block, int valid, AwLane<BF16, EIGHT>& x) {
    const uint32_t o = 4u * (threadIdx.x & 63);  // the block is the wave's: its address is scalar, the lane's part 32 bits
    if (t.glen != 0) {
        aw_grad_rows<BF16>(t, block + o, WHOLE ? 4 : valid, x.g);
    } else if (WHOLE) {
        if (BF16) {
            const aw_h4 g = aw_take((const uint16_t*)t.g + block + o);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x.g[2 * j] = __uint_as_float(g.x[j] << 16);
                x.g[2 * j + 1] = __uint_as_float(g.x[j] & 0xFFFF0000u);
            }
        } else {
            const aw_f4 g = aw_take((const float*)t.g + block + o);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.g[j] = g.x[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x.g[j] = j < valid ? aw_grad<BF16>(t.g, block + o + j) : 0.0f;
    }
    if (EIGHT) {
        x.em = t.me[block / M8_BLOCK];
        x.ev = t.ve[block / M8_BLOCK];
    }
    if (WHOLE) {
        if (BF16) {
            const aw_h4 h = *(const aw_h4*)((const uint16_t*)t.p + block + o), l = aw_take((const uint16_t*)t.low + block + o);
            aw_join4(h, l, x.w);
        } else {
            const aw_f4 p = *(const aw_f4*)((const float*)t.p + block + o);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.w[j] = p.x[j];
        }
        if (EIGHT) {
            x.cm = aw_take((const uint8_t*)t.m + block + o);
            x.cv = aw_take((const uint8_t*)t.v + block + o);
        } else {
            const aw_f4 m = aw_take((const float*)t.m + block + o), v = aw_take((const float*)t.v + block + o);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x.m[j] = m.x[j]; x.v[j] = v.x[j]; }
        }
        return;
    }
    x.cm = x.cv = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool ok = j < valid;
        const long long i = block + o + j;
        if (BF16) x.w[j] = ok ? aw_join(((const uint16_t*)t.p)[i], t.low[i]) : 0.0f;
        else x.w[j] = ok ? ((const float*)t.p)[i] : 0.0f;
        if (EIGHT) {
            x.cm |= (ok ? (uint32_t)((const uint8_t*)t.m)[i] : 0u) << (8 * j);
            x.cv |= (ok ? (uint32_t)((const uint8_t*)t.v)[i] : 0u) << (8 * j);
        } else {
            x.m[j] = ok ? ((const float*)t.m)[i] : 0.0f;
            x.v[j] = ok ? ((const float*)t.v)[i] : 0.0f;
        }
    }
}

template <bool BF16, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void aw_finish(const AwStep& k, const AwTensor& t, long long block, int valid, AwLane<BF16, EIGHT>& x) {
    const uint32_t lane = threadIdx.x & 63, o = 4 * lane;
    float b1 = k.b1, b2 = k.b2;
    if (EIGHT) {
        const int em = __builtin_amdgcn_readfirstlane(x.em), ev = __builtin_amdgcn_readfirstlane(x.ev);
        const int bm = m8_base<true>(em), bv = m8_base<false>(ev);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.m[j] = __uint_as_float(m8_decode<true>((x.cm >> (8 * j)) & 255u, bm));
            x.v[j] = __uint_as_float(m8_decode<false>((x.cv >> (8 * j)) & 255u, bv));
        }
        if (em == 255) b1 = __builtin_nanf("");  // the block stands for NaN
        if (ev == 255) b2 = __builtin_nanf("");
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma clang fp contract(off)
        x.m[j] = x.m[j] * b1 + x.g[j] * k.omb1;
        x.v[j] = x.v[j] * b2 + (x.g[j] * x.g[j]) * k.omb2;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.w[j] = aw_update(x.w[j], x.m[j], x.v[j], k, t);
    uint32_t cm = 0, cv = 0;
    if (EIGHT) {
        uint32_t tm = 0, tv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = __float_as_uint(x.m[j]) & 0x7FFFFFFFu, b = __float_as_uint(x.v[j]) & 0x7FFFFFFFu;
            if (WHOLE || j < valid) {
                tm = a > tm ? a : tm;
                tv = b > tv ? b : tv;
            }
        }
        const uint32_t e2 = m8_wave_max2((tm >> 23) | ((tv >> 23) << 16));
        const int em = (int)(e2 & 0xFFFFu), ev = (int)(e2 >> 16);
        const int bm = m8_base<true>(em), bv = m8_base<false>(ev);
        // the hash's first product, once: the elements follow one another
        const uint32_t x0 = ((uint32_t)block + o + m8_key(t.key, block)) * M8_C1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t h = m8_hash(x0 + (uint32_t)j * M8_C1);
            cm |= m8_encode<true>(__float_as_uint(x.m[j]) & 0x7FFFFFFFu, m8_noise_m(h), bm) << (8 * j);
            cv |= m8_encode<false>(__float_as_uint(x.v[j]) & 0x7FFFFFFFu, m8_noise_v(h), bv) << (8 * j);
        }
        cm |= m8_signs(x.m);
        cm = em == 255 ? 0u : cm;
        cv = ev == 255 ? 0u : cv;
        if (lane == 0) {
            t.me[block / M8_BLOCK] = (uint8_t)em;
            t.ve[block / M8_BLOCK] = (uint8_t)ev;
        }
    }
    if (WHOLE) {
        if (BF16) {
            aw_h4 h, l;
            aw_split4(x.w, h, l);
            *(aw_h4*)((uint16_t*)t.p + block + o) = h;
            aw_put((uint16_t*)t.low + block + o, l);
        } else {
            aw_f4 p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p.x[j] = x.w[j];
            *(aw_f4*)((float*)t.p + block + o) = p;
        }
        if (EIGHT) {
            aw_put((uint8_t*)t.m + block + o, cm);
            aw_put((uint8_t*)t.v + block + o, cv);
        } else {
            aw_f4 m, v;
#pragma unroll
            for (int j = 0; j < 4; ++j) { m.x[j] = x.m[j]; v.x[j] = x.v[j]; }
            aw_put((float*)t.m + block + o, m);
            aw_put((float*)t.v + block + o, v);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j >= valid) break;
        const long long i = block + o + j;
        if (BF16) {
            uint16_t hi;
            int16_t lo;
            aw_split(x.w[j], hi, lo);
            ((uint16_t*)t.p)[i] = hi;
            t.low[i] = lo;
        } else {
            ((float*)t.p)[i] = x.w[j];
        }
        if (EIGHT) {
            ((uint8_t*)t.m)[i] = (uint8_t)(cm >> (8 * j));
            ((uint8_t*)t.v)[i] = (uint8_t)(cv >> (8 * j));
        } else {
            ((float*)t.m)[i] = x.m[j];
            ((float*)t.v)[i] = x.v[j];
        }
    }
}

template <bool BF16, bool EIGHT, class Source>
__global__ void __launch_bounds__(AW_THREADS)
adamw_kernel(AwStep k, Source source) {
    int first;
    const AwTensor& t = source.find((int)blockIdx.x, first);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long block = (long long)((int)blockIdx.x - first) * AW_PER_GROUP + wave * M8_BLOCK;
    AwLane<BF16, EIGHT> x;
    if (block + M8_BLOCK <= t.n) {
        aw_load<BF16, EIGHT, true>(t, block, 4, x);
        aw_finish<BF16, EIGHT, true>(k, t, block, 4, x);
        return;
    }
    if (block >= t.n) return;
    const long long left = t.n - (block + 4 * (threadIdx.x & 63));
    const int valid = left >= 4 ? 4 : left > 0 ? (int)left : 0;
    aw_load<BF16, EIGHT, false>(t, block, valid, x);
    aw_finish<BF16, EIGHT, false>(k, t, block, valid, x);
}

extern "C" int fdgs_adamw_step(const fdgs_adamw_args* a, void* stream) {
    if (!a || a->num_tensors < 0 || (a->num_tensors > 0 && !a->tensors)) return FDGS_EINVAL;
    const bool bf16 = a->param_type == FDGS_TYPE_BF16, eight = a->state_bits == 8;
    if (!bf16 && a->param_type != FDGS_TYPE_F32) return FDGS_EINVAL;
    if (!eight && a->state_bits != 32) return FDGS_EINVAL;
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 && a->eps >= 0.0)) return FDGS_EINVAL;
    long long total = 0;                         // workgroups
    for (int i = 0; i < a->num_tensors; ++i) {   // all of them before the first launch: no step is half done
        const fdgs_adamw_tensor& s = a->tensors[i];
        if (s.numel < 0 || s.step < 1 || s.grad_row_len < 0) return FDGS_EINVAL;
        if (s.grad_row_len > 0 && s.grad_row_stride < s.grad_row_len) return FDGS_EINVAL;
        if (s.numel == 0) continue;
        total += (s.numel - 1) / AW_PER_GROUP + 1;
        if (total > FDGS_MAX_GROUPS(AW_THREADS)) return FDGS_ETOOLARGE;
        if (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq || (bf16 && !s.residual)) return FDGS_EINVAL;
        if (eight && (!s.exp_avg_exponents || !s.exp_avg_sq_exponents)) return FDGS_EINVAL;
    }
    AwStep k;
    k.b1 = (float)a->beta1; k.omb1 = (float)(1.0 - a->beta1);
    k.b2 = (float)a->beta2; k.omb2 = (float)(1.0 - a->beta2);
    k.eps = (float)a->eps;
    int i = 0, step = 0;
    double correct1 = 1.0;
    float inv_root = 1.0f;
    auto next = [&](AwTensor& t, int& groups) {
        while (i < a->num_tensors && a->tensors[i].numel == 0) ++i;
        if (i == a->num_tensors) return false;
        const fdgs_adamw_tensor& s = a->tensors[i++];
        groups = (int)((s.numel + AW_PER_GROUP - 1) / AW_PER_GROUP);
        t.p = s.param; t.g = s.grad; t.m = s.exp_avg; t.v = s.exp_avg_sq;
        t.low = s.residual; t.me = s.exp_avg_exponents; t.ve = s.exp_avg_sq_exponents;
        t.n = s.numel; t.gstride = s.grad_row_stride; t.glen = s.grad_row_len;
        if (s.step != step) {                    // most tensors of a list have the same count
            step = s.step;
            correct1 = 1.0 - pow(a->beta1, (double)step);
            inv_root = (float)(1.0 / sqrt(1.0 - pow(a->beta2, (double)step)));
        }
        t.step_size = (float)(s.lr / correct1);
        t.inv_root = inv_root;
        t.decay = (float)(1.0 - s.lr * s.weight_decay);
        t.key = s.round_key; t.pad = 0;
        return true;
    };
    hipStream_t st = (hipStream_t)stream;
    auto launch = [&](const auto& source, int blocks) {
        typedef std::remove_cv_t<std::remove_reference_t<decltype(source)>> Source;
        const dim3 grid((unsigned)blocks), threads(AW_THREADS);
        if (bf16 && eight) hipLaunchKernelGGL((adamw_kernel<true, true, Source>), grid, threads, 0, st, k, source);
        else if (bf16) hipLaunchKernelGGL((adamw_kernel<true, false, Source>), grid, threads, 0, st, k, source);
        else if (eight) hipLaunchKernelGGL((adamw_kernel<false, true, Source>), grid, threads, 0, st, k, source);
        else hipLaunchKernelGGL((adamw_kernel<false, false, Source>), grid, threads, 0, st, k, source);
    };
    return list_launch<AwTensor, AW_MAX>(a->num_tensors, a->workspace, a->workspace_bytes, st, next, launch);
}

extern "C" size_t fdgs_adamw_workspace_bytes(int32_t num_tensors) {
    return num_tensors > AW_MAX ? list_table_bytes(num_tensors, sizeof(AwTensor)) : 0;
}

// ---- 8-bit moments to values and back ----
#define M8_MAX 92                                // tensors whose records fill 4 KB of kernel arguments
struct M8Tensor { uint8_t* codes; uint8_t* exps; void* value; long long n; uint32_t key; int is_signed; };
static_assert(sizeof(AwInBoth<M8Tensor, M8_MAX>) + 8 <= 4096, "kernel arguments of one launch");

// What a lane takes at a time: as many codes as make 16 bytes of values, a wave's stores being neighbours (8 codes for two
// stores of float32: 116,000,000 elements 150 us, not 101).  Ordinary loads: with streaming ones the next step finds the codes
// evicted (2,000,000 Gaussians: 3 us less here, 17 more there).
template <bool BF16>
struct M8Some {
    static constexpr int n = BF16 ? 8 : 4;
    uint32_t c[n / 4];
    int e;
    __device__ __forceinline__ void load(const M8Tensor& t, long long i) {
        if (BF16) {
            const aw_b8 x = *(const aw_b8*)(t.codes + i);
            c[0] = x.x[0];
            c[n / 4 - 1] = x.x[1];
        } else {
            c[0] = *(const aw_u1_at1*)(t.codes + i);
        }
        e = t.exps[i / M8_BLOCK];
    }
    template <bool SIGNED>
    __device__ __forceinline__ void store(const M8Tensor& t, long long i) const {
        const int base = m8_base<SIGNED>(e);
        uint32_t b[n];
#pragma unroll
        for (int j = 0; j < n; ++j) {
            b[j] = m8_decode<SIGNED>((c[j / 4] >> (8 * (j & 3))) & 255u, base);
            b[j] = e == 255 ? 0x7FC00000u : b[j];
        }
        if (BF16) {                              // four significant bits: bfloat16 holds them exactly
            aw_w4 h;
#pragma unroll
            for (int j = 0; j < 4; ++j) h.x[j] = (b[(2 * j) % n] >> 16) | (b[(2 * j + 1) % n] & 0xFFFF0000u);
            *(aw_w4*)((uint16_t*)t.value + i) = h;
        } else {
            aw_f4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f.x[j] = __uint_as_float(b[j]);
            *(aw_f4*)((float*)t.value + i) = f;
        }
    }
};

#define M8_PER_GROUP 4096                        // elements per workgroup (422 moments of 211 tensors: 49 us; 8192: 51, 16384: 55)
template <bool BF16, bool SIGNED>
__device__ __forceinline__ void m8_unpack_group(const M8Tensor& t, long long first) {
    constexpr int n = M8Some<BF16>::n, rounds = M8_PER_GROUP / (256 * n);
    const long long base = first + n * (int)threadIdx.x;
    if (first + M8_PER_GROUP <= t.n) {           // all loads before the first use (2,000,000 Gaussians: 160 -> 123 us)
        M8Some<BF16> x[rounds];
#pragma unroll
        for (int u = 0; u < rounds; ++u) x[u].load(t, base + u * (256 * n));
#pragma unroll
        for (int u = 0; u < rounds; ++u) x[u].template store<SIGNED>(t, base + u * (256 * n));
        return;
    }
#pragma unroll 1
    for (long long i = base; i < t.n && i < first + M8_PER_GROUP; i += 256 * n) {
        if (i + n <= t.n) {
            M8Some<BF16> x;
            x.load(t, i);
            x.template store<SIGNED>(t, i);
            continue;
        }
        const int e = t.exps[i / M8_BLOCK], at = m8_base<SIGNED>(e);
        for (long long j = i; j < t.n; ++j) {
            const uint32_t b = e == 255 ? 0x7FC00000u : m8_decode<SIGNED>(t.codes[j], at);
            if (BF16) ((uint16_t*)t.value)[j] = (uint16_t)(b >> 16);
            else ((float*)t.value)[j] = __uint_as_float(b);
        }
    }
}

template <bool BF16, class Source>
__global__ void __launch_bounds__(256)
moment8_unpack_kernel(Source source) {
    int group;
    const M8Tensor& t = source.find((int)blockIdx.x, group);
    const long long first = (long long)((int)blockIdx.x - group) * M8_PER_GROUP;
    if (t.is_signed) m8_unpack_group<BF16, true>(t, first);
    else m8_unpack_group<BF16, false>(t, first);
}

// A lane's four values of block b to codes.  116,000,000 elements: 101 us (5.8 TB/s); 185 with loads and bytes one at a time.
template <bool SIGNED>
__device__ __forceinline__ void m8_pack4(bool nearest, const M8Tensor& t, long long b, const float* x) {
    const int lane = threadIdx.x & 63;
    const long long i = b + 4 * lane;
    uint32_t top = 0, codes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        top = a > top ? a : top;
    }
    const int e = (int)m8_wave_max2(top >> 23), base = m8_base<SIGNED>(e);
    const uint32_t x0 = ((uint32_t)i + m8_key(t.key, i)) * M8_C1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t h = nearest ? 0x80008000u : m8_hash(x0 + (uint32_t)j * M8_C1);
        codes |= m8_encode<SIGNED>(__float_as_uint(x[j]) & 0x7FFFFFFFu, SIGNED ? m8_noise_m(h) : m8_noise_v(h), base) << (8 * j);
    }
    if (SIGNED) codes |= m8_signs(x);
    codes = e == 255 ? 0u : codes;
    if (lane == 0) t.exps[b / M8_BLOCK] = (uint8_t)e;
    if (i + 4 <= t.n) {
        *(aw_u1_at1*)(t.codes + i) = codes;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < t.n) t.codes[i + j] = (uint8_t)(codes >> (8 * j));
    }
}

#define M8_WAVE_BLOCKS (M8_PER_GROUP / 4 / M8_BLOCK)
template <class Source>
__global__ void __launch_bounds__(256)
moment8_pack_kernel(int nearest, Source source) {
    int first;
    const M8Tensor& t = source.find((int)blockIdx.x, first);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long base = (long long)((int)blockIdx.x - first) * M8_PER_GROUP + wave * (M8_PER_GROUP / 4);
    const float* value = (const float*)t.value + 4 * (int)(threadIdx.x & 63);
    float x[M8_WAVE_BLOCKS][4];
#pragma unroll
    for (int u = 0; u < M8_WAVE_BLOCKS; ++u) {   // all loads before the first use
        const long long b = base + u * M8_BLOCK;
        if (b + M8_BLOCK <= t.n) {
            const aw_f4 f = *(const aw_f4*)(value + b);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][j] = f.x[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][j] = b + 4 * (int)(threadIdx.x & 63) + j < t.n ? value[b + j] : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < M8_WAVE_BLOCKS; ++u) {
        const long long b = base + u * M8_BLOCK;
        if (b >= t.n) return;                    // the whole wave
        if (t.is_signed) m8_pack4<true>(nearest != 0, t, b, x[u]);
        else m8_pack4<false>(nearest != 0, t, b, x[u]);
    }
}

static int moment8_launch(const fdgs_moment8_args* a, void* stream, bool pack) {
    if (!a || a->num_tensors < 0 || (a->num_tensors > 0 && !a->tensors)) return FDGS_EINVAL;
    const bool bf16 = a->value_type == FDGS_TYPE_BF16;
    if ((bf16 && pack) || (!bf16 && a->value_type != FDGS_TYPE_F32)) return FDGS_EINVAL;
    long long total = 0;                         // workgroups
    for (int i = 0; i < a->num_tensors; ++i) {
        const fdgs_moment8_tensor& s = a->tensors[i];
        if (s.numel < 0) return FDGS_EINVAL;
        if (s.numel == 0) continue;
        if (!s.codes || !s.exponents || !s.value) return FDGS_EINVAL;
        total += (s.numel - 1) / M8_PER_GROUP + 1;
        if (total > FDGS_MAX_GROUPS(256)) return FDGS_ETOOLARGE;
    }
    int i = 0;
    auto next = [&](M8Tensor& t, int& groups) {
        while (i < a->num_tensors && a->tensors[i].numel == 0) ++i;
        if (i == a->num_tensors) return false;
        const fdgs_moment8_tensor& s = a->tensors[i++];
        groups = (int)((s.numel + M8_PER_GROUP - 1) / M8_PER_GROUP);
        t.codes = s.codes; t.exps = s.exponents; t.value = s.value;
        t.n = s.numel; t.key = s.round_key; t.is_signed = s.is_signed != 0;
        return true;
    };
    hipStream_t st = (hipStream_t)stream;
    auto launch = [&](const auto& source, int blocks) {
        typedef std::remove_cv_t<std::remove_reference_t<decltype(source)>> Source;
        const dim3 grid((unsigned)blocks), threads(256);
        if (pack) hipLaunchKernelGGL((moment8_pack_kernel<Source>), grid, threads, 0, st, (int)(a->nearest != 0), source);
        else if (bf16) hipLaunchKernelGGL((moment8_unpack_kernel<true, Source>), grid, threads, 0, st, source);
        else hipLaunchKernelGGL((moment8_unpack_kernel<false, Source>), grid, threads, 0, st, source);
    };
    return list_launch<M8Tensor, M8_MAX>(a->num_tensors, a->workspace, a->workspace_bytes, st, next, launch);
}

extern "C" size_t fdgs_moment8_workspace_bytes(int32_t num_tensors) {
    return num_tensors > M8_MAX ? list_table_bytes(num_tensors, sizeof(M8Tensor)) : 0;
}

extern "C" int fdgs_moment8_unpack(const fdgs_moment8_args* a, void* stream) { return moment8_launch(a, stream, false); }
extern "C" int fdgs_moment8_pack(const fdgs_moment8_args* a, void* stream) { return moment8_launch(a, stream, true); }
