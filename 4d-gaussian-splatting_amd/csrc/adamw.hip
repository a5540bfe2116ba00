// AdamW over many tensors in one launch per 40 tensors (moments in float32 or in 8 bits, parameters in float32 or in
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

#define AW_MAX 40                                // tensors per launch: their records fill 4 KB of kernel arguments
#define AW_PER_WAVE 512                          // two blocks of 256 per wave
#define AW_PER_GROUP 2048                        // elements per workgroup of four waves

struct AwTensor {
    void* p; const void* g; void* m; void* v;
    int16_t* low; uint8_t* me; uint8_t* ve;
    long long n, gstride;
    int glen;
    float step_size, inv_root, decay;
    uint32_t key, pad;
};
struct AwPart {
    int num;
    float b1, omb1, b2, omb2, eps;
    int start[AW_MAX];                           // first workgroup of each tensor
    AwTensor t[AW_MAX];
};
static_assert(sizeof(AwPart) <= 4096, "kernel arguments of one launch");

struct __attribute__((packed, aligned(4))) aw_f4 { float x[4]; };
struct __attribute__((packed, aligned(2))) aw_h4 { uint16_t x[4]; };
struct __attribute__((packed, aligned(1))) aw_b4 { uint32_t x; };

// float32 -> bfloat16 to the nearest, halves away from zero, and the signed 16 bits between the two: the pair is the
// float32 value again exactly, and (unlike rounding halves to even) the difference always fits.
__device__ __forceinline__ void aw_split(float w, uint16_t& hi, int16_t& lo) {
    const uint32_t b = __float_as_uint(w);
    const bool nan = w != w;
    const uint32_t h = (b + 0x8000u) >> 16;
    hi = (uint16_t)(nan ? 0x7FC0u : h);
    lo = (int16_t)(nan ? 0u : b - (h << 16));
}
__device__ __forceinline__ float aw_join(uint16_t hi, int16_t lo) {
    return __uint_as_float(((uint32_t)hi << 16) + (uint32_t)(int)lo);
}
__device__ __forceinline__ float aw_bf16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }

__device__ __forceinline__ void aw_one(float& w, float g, float& m, float& v, const AwPart& k, const AwTensor& t) {
#pragma clang fp contract(off)
    m = m * k.b1 + g * k.omb1;
    v = v * k.b2 + (g * g) * k.omb2;
    const float denom = sqrtf(v) * t.inv_root + k.eps;
    w = w * t.decay - (m * t.step_size) / denom;
}

// The tensor that workgroup `b` works on: one look at every tensor's first workgroup, a lane each.
__device__ __forceinline__ int aw_find(const int* start, int num, int b) {
    const int lane = threadIdx.x & 63;
    const int s = lane < num ? start[lane] : 0x7FFFFFFF;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(s <= b)) - 1);
}

template <bool BF16, bool EIGHT>
struct AwLane {                                  // a lane's four elements of a block
    float w[4], g[4], m[4], v[4];
};

// Gradient element i: i itself, or (rows of L elements, S apart) its place in a column slice of a wider array.
template <bool BF16>
__device__ __forceinline__ float aw_grad(const void* g, long long i) {
    return BF16 ? aw_bf16(((const uint16_t*)g)[i]) : ((const float*)g)[i];
}
template <bool BF16>
__device__ __forceinline__ void aw_grad4(const AwTensor& t, long long i, int valid, float* out) {
    if (t.glen == 0) {
        if (valid == 4) {
            if (BF16) {
                const aw_h4 x = *(const aw_h4*)((const uint16_t*)t.g + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] = aw_bf16(x.x[j]);
            } else {
                const aw_f4 x = *(const aw_f4*)((const float*)t.g + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] = x.x[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = j < valid ? aw_grad<BF16>(t.g, i + j) : 0.0f;
        }
        return;
    }
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

template <bool BF16, bool EIGHT>
__device__ __forceinline__ void aw_load(const AwTensor& t, long long i, int valid, int em, int ev, AwLane<BF16, EIGHT>& x) {
    aw_grad4<BF16>(t, i, valid, x.g);
    uint32_t cm = 0, cv = 0;
    if (valid == 4) {
        if (BF16) {
            const aw_h4 h = *(const aw_h4*)((const uint16_t*)t.p + i), l = *(const aw_h4*)(t.low + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.w[j] = aw_join(h.x[j], (int16_t)l.x[j]);
        } else {
            const aw_f4 p = *(const aw_f4*)((const float*)t.p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.w[j] = p.x[j];
        }
        if (EIGHT) {
            cm = ((const aw_b4*)((const uint8_t*)t.m + i))->x;
            cv = ((const aw_b4*)((const uint8_t*)t.v + i))->x;
        } else {
            const aw_f4 m = *(const aw_f4*)((const float*)t.m + i), v = *(const aw_f4*)((const float*)t.v + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x.m[j] = m.x[j]; x.v[j] = v.x[j]; }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool ok = j < valid;
            if (BF16) x.w[j] = ok ? aw_join(((const uint16_t*)t.p)[i + j], t.low[i + j]) : 0.0f;
            else x.w[j] = ok ? ((const float*)t.p)[i + j] : 0.0f;
            if (EIGHT) {
                cm |= (ok ? (uint32_t)((const uint8_t*)t.m)[i + j] : 0u) << (8 * j);
                cv |= (ok ? (uint32_t)((const uint8_t*)t.v)[i + j] : 0u) << (8 * j);
            } else {
                x.m[j] = ok ? ((const float*)t.m)[i + j] : 0.0f;
                x.v[j] = ok ? ((const float*)t.v)[i + j] : 0.0f;
            }
        }
    }
    if (EIGHT) {
        const int bm = m8_base<true>(em), bv = m8_base<false>(ev);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.m[j] = m8_decode<true>((cm >> (8 * j)) & 255u, em, bm);
            x.v[j] = m8_decode<false>((cv >> (8 * j)) & 255u, ev, bv);
        }
    }
}

template <bool BF16, bool EIGHT>
__device__ __forceinline__ void aw_finish(const AwPart& k, const AwTensor& t, long long block, int valid, AwLane<BF16, EIGHT>& x) {
    const int lane = threadIdx.x & 63;
    const long long i = block + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) aw_one(x.w[j], x.g[j], x.m[j], x.v[j], k, t);
    uint32_t cm = 0, cv = 0;
    if (EIGHT) {
        uint32_t tm = 0, tv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = __float_as_uint(x.m[j]) & 0x7FFFFFFFu, b = __float_as_uint(x.v[j]) & 0x7FFFFFFFu;
            if (j < valid) {
                tm = a > tm ? a : tm;
                tv = b > tv ? b : tv;
            }
        }
        const uint32_t e2 = m8_wave_max2((tm >> 23) | ((tv >> 23) << 16));
        const int em = (int)(e2 & 0xFFFFu), ev = (int)(e2 >> 16);
        const int bm = m8_base<true>(em), bv = m8_base<false>(ev);
        const uint32_t key = m8_key(t.key, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t h = m8_hash((uint32_t)i + j, key);
            cm |= m8_encode<true>(x.m[j], m8_noise_m(h), em, bm) << (8 * j);
            cv |= m8_encode<false>(x.v[j], m8_noise_v(h), ev, bv) << (8 * j);
        }
        if (lane == 0) {
            t.me[block / M8_BLOCK] = (uint8_t)em;
            t.ve[block / M8_BLOCK] = (uint8_t)ev;
        }
    }
    if (valid == 4) {
        if (BF16) {
            aw_h4 h, l;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int16_t lo;
                aw_split(x.w[j], h.x[j], lo);
                l.x[j] = (uint16_t)lo;
            }
            *(aw_h4*)((uint16_t*)t.p + i) = h;
            *(aw_h4*)(t.low + i) = l;
        } else {
            aw_f4 p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p.x[j] = x.w[j];
            *(aw_f4*)((float*)t.p + i) = p;
        }
        if (EIGHT) {
            ((aw_b4*)((uint8_t*)t.m + i))->x = cm;
            ((aw_b4*)((uint8_t*)t.v + i))->x = cv;
        } else {
            aw_f4 m, v;
#pragma unroll
            for (int j = 0; j < 4; ++j) { m.x[j] = x.m[j]; v.x[j] = x.v[j]; }
            *(aw_f4*)((float*)t.m + i) = m;
            *(aw_f4*)((float*)t.v + i) = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= valid) break;
            if (BF16) {
                uint16_t hi;
                int16_t lo;
                aw_split(x.w[j], hi, lo);
                ((uint16_t*)t.p)[i + j] = hi;
                t.low[i + j] = lo;
            } else {
                ((float*)t.p)[i + j] = x.w[j];
            }
            if (EIGHT) {
                ((uint8_t*)t.m)[i + j] = (uint8_t)(cm >> (8 * j));
                ((uint8_t*)t.v)[i + j] = (uint8_t)(cv >> (8 * j));
            } else {
                ((float*)t.m)[i + j] = x.m[j];
                ((float*)t.v)[i + j] = x.v[j];
            }
        }
    }
}

template <bool BF16, bool EIGHT>
__global__ void __launch_bounds__(256)
adamw_kernel(AwPart k) {
    const int ti = aw_find(k.start, k.num, (int)blockIdx.x);
    const AwTensor& t = k.t[ti];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long base = (long long)((int)blockIdx.x - k.start[ti]) * AW_PER_GROUP + wave * AW_PER_WAVE;
    AwLane<BF16, EIGHT> x[2];
    if (base + AW_PER_WAVE <= t.n) {             // both blocks whole: all loads before the first use
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long long b = base + u * M8_BLOCK;
            const int em = EIGHT ? t.me[b / M8_BLOCK] : 0, ev = EIGHT ? t.ve[b / M8_BLOCK] : 0;
            aw_load<BF16, EIGHT>(t, b + 4 * lane, 4, em, ev, x[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) aw_finish<BF16, EIGHT>(k, t, base + u * M8_BLOCK, 4, x[u]);
        return;
    }
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
        const long long b = base + u * M8_BLOCK;
        if (b >= t.n) return;
        const long long left = t.n - (b + 4 * lane);
        const int valid = left >= 4 ? 4 : left > 0 ? (int)left : 0;
        const int em = EIGHT ? t.me[b / M8_BLOCK] : 0, ev = EIGHT ? t.ve[b / M8_BLOCK] : 0;
        aw_load<BF16, EIGHT>(t, b + 4 * lane, valid, em, ev, x[0]);
        aw_finish<BF16, EIGHT>(k, t, b, valid, x[0]);
    }
}

extern "C" int fdgs_adamw_step(const fdgs_adamw_args* a, void* stream) {
    if (!a || a->num_tensors < 0 || (a->num_tensors > 0 && !a->tensors)) return FDGS_EINVAL;
    const bool bf16 = a->param_type == FDGS_TYPE_BF16, eight = a->state_bits == 8;
    if (!bf16 && a->param_type != FDGS_TYPE_F32) return FDGS_EINVAL;
    if (!eight && a->state_bits != 32) return FDGS_EINVAL;
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 && a->eps >= 0.0)) return FDGS_EINVAL;
    for (int i = 0; i < a->num_tensors; ++i) {   // all of them before the first launch: no step is half done
        const fdgs_adamw_tensor& s = a->tensors[i];
        if (s.numel < 0 || s.step < 1 || s.grad_row_len < 0) return FDGS_EINVAL;
        if (s.grad_row_len > 0 && s.grad_row_stride < s.grad_row_len) return FDGS_EINVAL;
        if (s.numel == 0) continue;
        if ((s.numel - 1) / AW_PER_GROUP >= 0x7fffffffLL / AW_MAX) return FDGS_ETOOLARGE;
        if (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq || (bf16 && !s.residual)) return FDGS_EINVAL;
        if (eight && (!s.exp_avg_exponents || !s.exp_avg_sq_exponents)) return FDGS_EINVAL;
    }
    AwPart k;
    k.b1 = (float)a->beta1; k.omb1 = (float)(1.0 - a->beta1);
    k.b2 = (float)a->beta2; k.omb2 = (float)(1.0 - a->beta2);
    k.eps = (float)a->eps;
    for (int i = 0; i < a->num_tensors;) {
        int blocks = 0;
        k.num = 0;
        for (; i < a->num_tensors && k.num < AW_MAX; ++i) {
            const fdgs_adamw_tensor& s = a->tensors[i];
            if (s.numel == 0) continue;
            k.start[k.num] = blocks;
            blocks += (int)((s.numel + AW_PER_GROUP - 1) / AW_PER_GROUP);
            AwTensor& t = k.t[k.num++];
            t.p = s.param; t.g = s.grad; t.m = s.exp_avg; t.v = s.exp_avg_sq;
            t.low = s.residual; t.me = s.exp_avg_exponents; t.ve = s.exp_avg_sq_exponents;
            t.n = s.numel; t.gstride = s.grad_row_stride; t.glen = s.grad_row_len;
            t.step_size = (float)(s.lr / (1.0 - pow(a->beta1, (double)s.step)));
            t.inv_root = (float)(1.0 / sqrt(1.0 - pow(a->beta2, (double)s.step)));
            t.decay = (float)(1.0 - s.lr * s.weight_decay);
            t.key = s.round_key; t.pad = 0;
        }
        if (k.num == 0) break;
        const dim3 grid((unsigned)blocks), threads(256);
        hipStream_t st = (hipStream_t)stream;
        if (bf16 && eight) hipLaunchKernelGGL((adamw_kernel<true, true>), grid, threads, 0, st, k);
        else if (bf16) hipLaunchKernelGGL((adamw_kernel<true, false>), grid, threads, 0, st, k);
        else if (eight) hipLaunchKernelGGL((adamw_kernel<false, true>), grid, threads, 0, st, k);
        else hipLaunchKernelGGL((adamw_kernel<false, false>), grid, threads, 0, st, k);
        FDGS_CHECK_LAUNCH();
    }
    return FDGS_OK;
}

// ---- 8-bit moments to values and back ----
#define M8_MAX 64                                // tensors per launch
struct M8Tensor { uint8_t* codes; uint8_t* exps; void* value; long long n; uint32_t key; int is_signed; };
struct M8Part {
    int num, nearest;
    int start[M8_MAX];
    M8Tensor t[M8_MAX];
};
static_assert(sizeof(M8Part) <= 4096, "kernel arguments of one launch");

template <bool BF16, bool SIGNED>
__device__ __forceinline__ void m8_unpack_block(const M8Tensor& t, long long b) {
    const int lane = threadIdx.x & 63;
    const long long i = b + 4 * lane;
    if (i >= t.n) return;
    const int e = t.exps[b / M8_BLOCK], base = m8_base<SIGNED>(e);
    if (i + 4 <= t.n) {
        const uint32_t c = ((const aw_b4*)(t.codes + i))->x;
        if (BF16) {                              // four significant bits: bfloat16 holds them exactly
            aw_h4 h;
#pragma unroll
            for (int j = 0; j < 4; ++j) h.x[j] = (uint16_t)(__float_as_uint(m8_decode<SIGNED>((c >> (8 * j)) & 255u, e, base)) >> 16);
            *(aw_h4*)((uint16_t*)t.value + i) = h;
        } else {
            aw_f4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f.x[j] = m8_decode<SIGNED>((c >> (8 * j)) & 255u, e, base);
            *(aw_f4*)((float*)t.value + i) = f;
        }
    } else {
        for (long long j = i; j < t.n; ++j) {
            const float f = m8_decode<SIGNED>(t.codes[j], e, base);
            if (BF16) ((uint16_t*)t.value)[j] = (uint16_t)(__float_as_uint(f) >> 16);
            else ((float*)t.value)[j] = f;
        }
    }
}

template <bool BF16>
__global__ void __launch_bounds__(256)
moment8_unpack_kernel(M8Part k) {
    const int ti = aw_find(k.start, k.num, (int)blockIdx.x);
    const M8Tensor& t = k.t[ti];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long base = (long long)((int)blockIdx.x - k.start[ti]) * AW_PER_GROUP + wave * AW_PER_WAVE;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (t.is_signed) m8_unpack_block<BF16, true>(t, base + u * M8_BLOCK);
        else m8_unpack_block<BF16, false>(t, base + u * M8_BLOCK);
    }
}

template <bool SIGNED>
__device__ __forceinline__ void m8_pack_block(const M8Part& k, const M8Tensor& t, long long b) {
    const int lane = threadIdx.x & 63;
    const long long i = b + 4 * lane;
    if (b >= t.n) return;                        // the whole wave
    float x[4];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = i + j < t.n ? ((const float*)t.value)[i + j] : 0.0f;
        const uint32_t a = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        top = a > top ? a : top;
    }
    const int e = (int)m8_wave_max2(top >> 23), base = m8_base<SIGNED>(e);
    const uint32_t key = m8_key(t.key, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (i + j >= t.n) break;
        const uint32_t h = k.nearest ? 0x80008000u : m8_hash((uint32_t)i + j, key);
        t.codes[i + j] = (uint8_t)m8_encode<SIGNED>(x[j], SIGNED ? m8_noise_m(h) : m8_noise_v(h), e, base);
    }
    if (lane == 0) t.exps[b / M8_BLOCK] = (uint8_t)e;
}

__global__ void __launch_bounds__(256)
moment8_pack_kernel(M8Part k) {
    const int ti = aw_find(k.start, k.num, (int)blockIdx.x);
    const M8Tensor& t = k.t[ti];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long base = (long long)((int)blockIdx.x - k.start[ti]) * AW_PER_GROUP + wave * AW_PER_WAVE;
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
        if (t.is_signed) m8_pack_block<true>(k, t, base + u * M8_BLOCK);
        else m8_pack_block<false>(k, t, base + u * M8_BLOCK);
    }
}

static int moment8_launch(const fdgs_moment8_args* a, void* stream, bool pack) {
    if (!a || a->num_tensors < 0 || (a->num_tensors > 0 && !a->tensors)) return FDGS_EINVAL;
    const bool bf16 = a->value_type == FDGS_TYPE_BF16;
    if ((bf16 && pack) || (!bf16 && a->value_type != FDGS_TYPE_F32)) return FDGS_EINVAL;
    for (int i = 0; i < a->num_tensors; ++i) {
        const fdgs_moment8_tensor& s = a->tensors[i];
        if (s.numel < 0) return FDGS_EINVAL;
        if (s.numel == 0) continue;
        if (!s.codes || !s.exponents || !s.value) return FDGS_EINVAL;
        if ((s.numel - 1) / AW_PER_GROUP >= 0x7fffffffLL / M8_MAX) return FDGS_ETOOLARGE;
    }
    M8Part k;
    k.nearest = a->nearest != 0;
    for (int i = 0; i < a->num_tensors;) {
        int blocks = 0;
        k.num = 0;
        for (; i < a->num_tensors && k.num < M8_MAX; ++i) {
            const fdgs_moment8_tensor& s = a->tensors[i];
            if (s.numel == 0) continue;
            k.start[k.num] = blocks;
            blocks += (int)((s.numel + AW_PER_GROUP - 1) / AW_PER_GROUP);
            M8Tensor& t = k.t[k.num++];
            t.codes = s.codes; t.exps = s.exponents; t.value = s.value;
            t.n = s.numel; t.key = s.round_key; t.is_signed = s.is_signed != 0;
        }
        if (k.num == 0) break;
        const dim3 grid((unsigned)blocks), threads(256);
        hipStream_t st = (hipStream_t)stream;
        if (pack) hipLaunchKernelGGL(moment8_pack_kernel, grid, threads, 0, st, k);
        else if (bf16) hipLaunchKernelGGL(moment8_unpack_kernel<true>, grid, threads, 0, st, k);
        else hipLaunchKernelGGL(moment8_unpack_kernel<false>, grid, threads, 0, st, k);
        FDGS_CHECK_LAUNCH();
    }
    return FDGS_OK;
}

extern "C" int fdgs_moment8_unpack(const fdgs_moment8_args* a, void* stream) { return moment8_launch(a, stream, false); }
extern "C" int fdgs_moment8_pack(const fdgs_moment8_args* a, void* stream) { return moment8_launch(a, stream, true); }
