// rp_optim.hip — an AdamW step over many tensors at once, its states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2            (t = steps of this tensor so far, this one included)
//   w = w (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in f32, every product, sum, quotient and root rounded on its own, in this order.
//
// States in 8 bits: blocks of 256 consecutive elements of a tensor (a tensor's last block is
// padded with zeros) share one scale, a power of two held as its biased exponent e, so scaling is exact.
//   m:       e4m3, |m| 2^(134 - e): e is the exponent of the block's largest |m|, which lands in [128, 256)
//   sqrt(v): unsigned, 5 bits of exponent (bias 31) and 3 of mantissa, sqrt(v) 2^(126 - e): the largest
//            lands in [0.5, 1). The root is held, not v: it spans half the binades (2^-33 .. 1 below the
//            largest), and the update divides by it.
// Rounding to a code is stochastic: the 20 mantissa bits that are dropped are first added to 16 random
// bits (a hash of seed, step, tensor and element). With b2 = 0.999 a step changes v by 0.1 % while two
// codes lie 6 to 12 % apart: rounding to the nearest would keep every v where its largest gradient
// put it; rounded at random the expected root is the exact one (and v, its square, larger by the rounding's variance: under 0.0125 %
// of v a step).
// One m is not rounded at random. The least code of m stands for 2^-17 to 2^-16 of the block's largest, far over the
// least root's 2^-33: an m below it would now and then become one that its root, held well, turns into a step of
// many lr. But whatever the gradients are they leave |m| <= B sqrt(v) (Cauchy and Schwarz on the two sums), with
// B^2 = (1 - b1)^2 / ((1 - b2) (1 - b1^2 / b2)), B = 7.3 with the usual betas. Where the least code is more than B root it is
// not taken and m becomes 0. Such an element, its root under 2^-19 or so of the block's largest m, then moves by its
// current gradient's share of m alone, at (1 - b1) of its pace. Without the rule a steady gradient of 1e-7 beside one of 1
// made steps of 190 lr, one of 1e-9 steps of 12000 lr (eps = 0).
// A block that holds a NaN or an infinity gets e = 255 and stands for NaN from then on.
#include <cmath>
#include <new>
#include <vector>

#include "rp_common.h"

using namespace rpd;

struct rp_adamw {
    int device = -1;
    int32_t tensors = 0, bits = 32, grad_type = RP_F32, each = 1;
    int64_t items = 0, blocks = 0;
    // what the caller keeps; a block's states start at 256 elements times its number
    void *m = nullptr, *v = nullptr;
    uint8_t *m_scale = nullptr, *v_scale = nullptr;
    int32_t* steps = nullptr;
    DevBuf table, list, scalars, done;
};

namespace {

constexpr int kBlock = 256;     // elements under one scale: 4 for each lane of a wave
// blocks of one tensor that one wave takes: one while the chip holds a wave for each (8192), four beyond. A wave's blocks follow each
// other, each with its loads' latency: 1 MB in tensors of 16 KB takes 5.0 us a step with one block, 6.8 with four
constexpr int kWaves = 8192, kItemBlocks = 4;
constexpr int64_t kMaxItems = (1 << 26) - 4;  // a wave each: a grid has fewer than 2^32 threads

struct Tensor {
    float* w;
    const void* g;
    uint16_t* copy;
    int64_t n, first_block;
    int32_t vec, pad;  // vec: w, g and copy are aligned for four elements at a time
};
struct Item {
    uint32_t tensor, block;  // block: within its tensor
};
struct Scalars {
    float by, rs;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t key;
    int32_t active;
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x9E3779B1u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

struct Numbers {
    double lr, b1, b2;
    uint32_t seed_lo, seed_hi;
};
// what the update of tensor t scales by in its step k
__device__ __forceinline__ Scalars scalars_of(const Numbers& x, int32_t t, int32_t k) {
    return {(float)(x.lr / (1.0 - pow(x.b1, (double)k))), (float)(1.0 / sqrt(1.0 - pow(x.b2, (double)k))),
            mix(mix(mix(mix(x.seed_lo) ^ x.seed_hi) ^ (uint32_t)k) ^ (uint32_t)t), 1};
}

// one thread a tensor: its step count goes up
__global__ void adamw_begin_kernel(Scalars* __restrict__ sc, int32_t* __restrict__ steps, int32_t T, const uint8_t* __restrict__ active, Numbers x) {
    const int32_t t = (int32_t)(blockIdx.x * blockDim.x + threadIdx.x);
    if (t >= T) return;
    Scalars s{0.f, 0.f, 0u, 0};
    if (!active || active[t]) s = scalars_of(x, t, ++steps[t]);
    sc[t] = s;
}

__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exponent_of(uint32_t bits) {  // 255: not finite
    const int e = (int)(bits >> 23);
    return e == 255 ? 255 : max(e, 30);
}
// A code c stands for the float whose top bits it is (sign apart), times a power of two: subnormal
// codes come out right by the arithmetic of subnormal floats.
__device__ __forceinline__ float decode_m(uint32_t c, int e) {
    const float x = __uint_as_float((c & 127u) << 20) * 0x1p120f * power(e - 134);
    return e == 255 ? __uint_as_float(0x7fc00000u) : (c & 128u) ? -x : x;
}
__device__ __forceinline__ float decode_root(uint32_t c, int e) {
    const float x = __uint_as_float(c << 20) * 0x1p96f * power(e - 126);
    return e == 255 ? __uint_as_float(0x7fc00000u) : x;
}
// most: B root (a NaN, as of an infinite B and a root of 0, keeps nothing back)
__device__ __forceinline__ uint32_t encode_m(float m, int e, uint32_t rnd, float most) {
    if (e == 255) return 0u;
    const float least = power(e - 143);  // what code 1 stands for
    const uint32_t t = __float_as_uint(fabsf(m) * power(134 - e) * 0x1p-120f), sign = __float_as_uint(m) >> 31 << 7;
    return fabsf(m) < least && most < least ? sign : ((t + rnd) >> 20) | sign;
}
__device__ __forceinline__ uint32_t encode_root(float r, int e, uint32_t rnd) {
    if (e == 255) return 0u;
    return (__float_as_uint(r * power(126 - e) * 0x1p-96f) + rnd) >> 20;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
    return x;
}

// rounded to nearest even, two at a time (one instruction); a NaN stays one
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

struct StepArgs {
    const Tensor* tensors;
    const Item* items;
    const Scalars* scalars;
    int64_t n_items;
    int32_t each;  // blocks of an item
    void *m, *v;
    uint8_t *m_scale, *v_scale;
    float b1, c1, b2, c2, eps, keep, bound;  // c = 1 - b, keep = 1 - lr decay, bound: B above
    // for one launch
    Numbers x;
    int32_t* steps;
    const uint8_t* active;
    int32_t T;
    uint32_t* done;  // blocks that have read their counts, 0 between launches
};

// One wave an item: up to `each` blocks of one tensor, lane l holding elements 4 l .. 4 l + 3 of a block. Every byte is read and written
// once, which bounds it: 512 tensors of 16384 and 262144 (71 million), copies written: 0.40 ms in 32 bits (2.14 GB, 5.3 TB/s), 0.26 ms in
// 8 (1.30 GB, 5.1 TB/s).
template <int BITS, bool GRAD16>
__device__ __forceinline__ void step_item(const StepArgs& a, const Item& it, const Scalars& sc) {
    const int lane = threadIdx.x & 63;
    const Tensor ts = a.tensors[it.tensor];
    const int64_t nb = (ts.n + kBlock - 1) / kBlock;
    for (int64_t b = it.block; b < min(nb, (int64_t)it.block + a.each); ++b) {
        const int64_t at = b * kBlock + lane * 4, state = (ts.first_block + b) * kBlock + lane * 4;
        const int64_t left = ts.n - at;
        float w[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {0.f, 0.f, 0.f, 0.f}, m[4], v[4], root[4];
        if (ts.vec && left >= 4) {
            const float4 x = *reinterpret_cast<const float4*>(ts.w + at);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            if constexpr (GRAD16) {
                const uint2 y = *reinterpret_cast<const uint2*>((const uint16_t*)ts.g + at);
                g[0] = __uint_as_float(y.x << 16), g[1] = __uint_as_float(y.x & 0xffff0000u);
                g[2] = __uint_as_float(y.y << 16), g[3] = __uint_as_float(y.y & 0xffff0000u);
            } else {
                const float4 y = *reinterpret_cast<const float4*>((const float*)ts.g + at);
                g[0] = y.x, g[1] = y.y, g[2] = y.z, g[3] = y.w;
            }
        } else {
            for (int k = 0; k < 4; ++k)
                if (k < left) {
                    w[k] = ts.w[at + k];
                    g[k] = GRAD16 ? __uint_as_float((uint32_t)((const uint16_t*)ts.g)[at + k] << 16) : ((const float*)ts.g)[at + k];
                }
        }
        if constexpr (BITS == 32) {
            const float4 x = *reinterpret_cast<const float4*>((const float*)a.m + state);
            const float4 y = *reinterpret_cast<const float4*>((const float*)a.v + state);
            m[0] = x.x, m[1] = x.y, m[2] = x.z, m[3] = x.w;
            v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
        } else {
            const uint32_t cm = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.m + state);
            const uint32_t cv = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.v + state);
            const int em = a.m_scale[ts.first_block + b], ev = a.v_scale[ts.first_block + b];
            for (int k = 0; k < 4; ++k) {
                m[k] = decode_m(cm >> (8 * k) & 255u, em);
                const float r = decode_root(cv >> (8 * k) & 255u, ev);
                v[k] = r * r;
            }
        }
        for (int k = 0; k < 4; ++k) {
            m[k] = m[k] * a.b1 + g[k] * a.c1;
            v[k] = v[k] * a.b2 + g[k] * g[k] * a.c2;
            root[k] = sqrtf(v[k]);
            w[k] = w[k] * a.keep - m[k] / (root[k] * sc.rs + a.eps) * sc.by;
        }
        if (ts.vec && left >= 4) {
            *reinterpret_cast<float4*>(ts.w + at) = make_float4(w[0], w[1], w[2], w[3]);
            if (ts.copy)
                *reinterpret_cast<uint2*>(ts.copy + at) = make_uint2(to_bf16(w[0], w[1]), to_bf16(w[2], w[3]));
        } else {
            for (int k = 0; k < 4; ++k)
                if (k < left) {
                    ts.w[at + k] = w[k];
                    if (ts.copy) ts.copy[at + k] = (uint16_t)to_bf16(w[k], 0.f);
                }
        }
        if constexpr (BITS == 32) {
            *reinterpret_cast<float4*>((float*)a.m + state) = make_float4(m[0], m[1], m[2], m[3]);
            *reinterpret_cast<float4*>((float*)a.v + state) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint32_t mm = 0u, rr = 0u;
            for (int k = 0; k < 4; ++k) {
                if (k >= left) m[k] = root[k] = 0.f;
                mm = max(mm, __float_as_uint(m[k]) & 0x7fffffffu);
                rr = max(rr, __float_as_uint(root[k]) & 0x7fffffffu);
            }
            const int em = exponent_of(wave_max(mm)), ev = exponent_of(wave_max(rr));
            const uint32_t high = (uint32_t)(at >> 32), key = high ? mix(sc.key + high) : sc.key;
            uint32_t cm = 0u, cv = 0u;
            for (int k = 0; k < 4; ++k) {
                const uint32_t rnd = mix((uint32_t)(at + k) ^ key);
                cm |= encode_m(m[k], em, (rnd >> 16 << 4) + 8u, root[k] * a.bound) << (8 * k);
                cv |= encode_root(root[k], ev, ((rnd & 0xffffu) << 4) + 8u) << (8 * k);
            }
            *reinterpret_cast<uint32_t*>((uint8_t*)a.m + state) = cm;
            *reinterpret_cast<uint32_t*>((uint8_t*)a.v + state) = cv;
            if (lane == 0) {
                a.m_scale[ts.first_block + b] = (uint8_t)em;
                a.v_scale[ts.first_block + b] = (uint8_t)ev;
            }
        }
    }
}

template <int BITS, bool GRAD16>
__global__ void __launch_bounds__(256) adamw_step_kernel(StepArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= a.n_items) return;
    const Item it = a.items[item];
    const Scalars sc = a.scalars[it.tensor];
    if (sc.active) step_item<BITS, GRAD16>(a, it, sc);
}

// Short lists, whose step is bound by its two launches: every wave works out its tensor's scalars, and the block that is the last to have
// read the counts raises them, once its first wave has done its own work. 256 blocks of the state: 4.7 against 7.3 us a step (5.0 where a
// graph replays the two); 1024, with four times the turns at the one counter: 7.0 against 7.2 (5.3).
constexpr int64_t kOneLaunch = 768;  // items
constexpr int kOneTensors = 256;      // four a lane
template <int BITS, bool GRAD16>
__global__ void __launch_bounds__(256) adamw_one_kernel(StepArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    Item it{0u, 0u};
    int32_t k = 0;
    bool active = false;
    if (item < a.n_items) {
        it = a.items[item];
        k = a.steps[it.tensor];
        active = !a.active || a.active[it.tensor];
    }
    asm volatile("" ::"v"(k) : "memory");  // the count has arrived
    __syncthreads();
    uint32_t before = 0u;
    if (threadIdx.x == 0) before = atomicAdd(a.done, 1u);
    if (active) step_item<BITS, GRAD16>(a, it, scalars_of(a.x, (int32_t)it.tensor, k + 1));
    if (threadIdx.x >= 64 || (uint32_t)__builtin_amdgcn_readfirstlane((int)before) != gridDim.x - 1) return;
    int32_t counts[kOneTensors / 64];
#pragma unroll
    for (int i = 0; i < kOneTensors / 64; ++i) {
        const int t = i * 64 + (int)threadIdx.x;
        counts[i] = t < a.T && (!a.active || a.active[t]) ? a.steps[t] : -1;
    }
#pragma unroll
    for (int i = 0; i < kOneTensors / 64; ++i)
        if (counts[i] >= 0) a.steps[i * 64 + threadIdx.x] = counts[i] + 1;
    if (threadIdx.x == 0) *a.done = 0u;
}

// the states in 8 bits as the values they stand for: one wave a block, further ones beyond the 2^22 of the largest grid (an axis of a grid
// has fewer than 2^32 threads)
constexpr int64_t kValuesGrid = 1 << 20;
__global__ void __launch_bounds__(256)
adamw_values_kernel(const uint32_t* __restrict__ m, const uint32_t* __restrict__ v, const uint8_t* __restrict__ m_scale,
                    const uint8_t* __restrict__ v_scale, int64_t blocks, float4* __restrict__ out_m, float4* __restrict__ out_root) {
    for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < blocks; b += (int64_t)gridDim.x * 4) {
        const int64_t i = b * 64 + (threadIdx.x & 63);
        const uint32_t cm = m[i], cv = v[i];
        const int em = m_scale[b], ev = v_scale[b];
        out_m[i] = make_float4(decode_m(cm & 255u, em), decode_m(cm >> 8 & 255u, em), decode_m(cm >> 16 & 255u, em), decode_m(cm >> 24, em));
        out_root[i] = make_float4(decode_root(cv & 255u, ev), decode_root(cv >> 8 & 255u, ev), decode_root(cv >> 16 & 255u, ev),
                                  decode_root(cv >> 24, ev));
    }
}

}  // namespace

extern "C" {

int rp_adamw_create(int device, int32_t n_tensors, const int64_t* numels, float* const* params, const void* const* grads,
                    int32_t grad_type, uint16_t* const* copies, int32_t state_bits, void* exp_avg, void* exp_avg_sq,
                    uint8_t* exp_avg_scale, uint8_t* root_scale, int32_t* steps, rp_adamw** out) {
    if (!out) return fail(RP_ERR_INVALID, "NULL out");
    *out = nullptr;
    if (n_tensors <= 0 || !numels || !params || !grads) return fail(RP_ERR_INVALID, "no tensors");
    if (grad_type != RP_F32 && grad_type != RP_BF16) return fail(RP_ERR_INVALID, "grad_type must be RP_F32 or RP_BF16");
    if (state_bits != 32 && state_bits != 8) return fail(RP_ERR_INVALID, "state_bits must be 32 or 8");
    if (!exp_avg || !exp_avg_sq || !steps || (state_bits == 8 && (!exp_avg_scale || !root_scale)))
        return fail(RP_ERR_INVALID, "NULL state");
    if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) return fail(RP_ERR_INVALID, "states must be 16-byte aligned");
    rp_adamw* h = nullptr;
    try {
        std::vector<Tensor> ts((size_t)n_tensors);
        std::vector<Item> items;
        int64_t first = 0, all = 0;
        for (int32_t t = 0; t < n_tensors; ++t)
            all += (std::min<int64_t>(std::max<int64_t>(numels[t], 0), (int64_t)1 << 38) + kBlock - 1) / kBlock;
        const int each = all <= kWaves ? 1 : kItemBlocks;
        for (int32_t t = 0; t < n_tensors; ++t) {
            const int64_t n = numels[t];
            if (n < 0 || n > ((int64_t)1 << 38)) return fail(RP_ERR_INVALID, "tensor %d: bad size", (int)t);
            if (n && (!params[t] || !grads[t] || (copies && !copies[t]))) return fail(RP_ERR_INVALID, "tensor %d: NULL", (int)t);
            const size_t gs = grad_type == RP_BF16 ? 2 : 4;
            if (((uintptr_t)params[t] & 3) || ((uintptr_t)grads[t] & (gs - 1)) || (copies && ((uintptr_t)copies[t] & 1)))
                return fail(RP_ERR_INVALID, "tensor %d: not aligned to its elements", (int)t);
            Tensor& x = ts[(size_t)t];
            x.w = params[t], x.g = grads[t], x.copy = copies ? copies[t] : nullptr, x.n = n, x.first_block = first, x.pad = 0;
            x.vec = !((uintptr_t)x.w & 15) && !((uintptr_t)x.g & (4 * gs - 1)) && !((uintptr_t)x.copy & 7);
            const int64_t nb = (n + kBlock - 1) / kBlock;
            if ((int64_t)items.size() + (nb + each - 1) / each > kMaxItems) return fail(RP_ERR_UNSUPPORTED, "too many elements");
            for (int64_t b = 0; b < nb; b += each) items.push_back({(uint32_t)t, (uint32_t)b});
            first += nb;
        }
        h = new rp_adamw;
        h->device = device, h->tensors = n_tensors, h->bits = state_bits, h->grad_type = grad_type;
        h->items = (int64_t)items.size(), h->blocks = first, h->each = each;
        h->m = exp_avg, h->v = exp_avg_sq, h->m_scale = exp_avg_scale, h->v_scale = root_scale, h->steps = steps;
        DeviceGuard guard;
        int rc = guard.enter(device);
        if (!rc) rc = h->table.ensure(sizeof(Tensor) * ts.size(), device);
        if (!rc) rc = h->list.ensure(sizeof(Item) * std::max<size_t>(items.size(), 1), device);
        if (!rc) rc = h->scalars.ensure(sizeof(Scalars) * ts.size(), device);
        if (!rc) rc = h->done.ensure(4, device);
        if (!rc) {
            const uint32_t zero = 0u;
            hipError_t e = hipMemcpy(h->done.p, &zero, 4, hipMemcpyHostToDevice);
            if (e == hipSuccess) e = hipMemcpy(h->table.p, ts.data(), sizeof(Tensor) * ts.size(), hipMemcpyHostToDevice);
            if (e == hipSuccess && !items.empty())
                e = hipMemcpy(h->list.p, items.data(), sizeof(Item) * items.size(), hipMemcpyHostToDevice);
            if (e != hipSuccess) rc = fail(RP_ERR_HIP, "hipMemcpy: %s", hipGetErrorString(e));
        }
        if (rc) {
            delete h;
            return rc;
        }
    } catch (const std::bad_alloc&) {
        delete h;
        return fail(RP_ERR_NOMEM, "out of host memory");
    }
    *out = h;
    return RP_OK;
}

int rp_adamw_step(rp_adamw* h, double lr, double beta1, double beta2, double eps, double weight_decay, uint64_t seed,
                  const uint8_t* active, void* stream) {
    if (!h) return fail(RP_ERR_INVALID, "NULL handle");
    if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0))
        return fail(RP_ERR_INVALID, "lr, eps and weight_decay must not be negative, the betas lie in [0, 1)");
    DeviceGuard guard;
    int rc = guard.enter(h->device);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    // no bound where b1^2 >= b2: gradients can leave any m then
    const double bound = beta1 * beta1 < beta2 ? (1.0 - beta1) / sqrt((1.0 - beta2) * (1.0 - beta1 * beta1 / beta2)) : INFINITY;
    const Numbers x{lr, beta1, beta2, (uint32_t)seed, (uint32_t)(seed >> 32)};
    const StepArgs a{(const Tensor*)h->table.p, (const Item*)h->list.p, (const Scalars*)h->scalars.p, h->items, h->each, h->m, h->v, h->m_scale,
                     h->v_scale, (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps,
                     (float)(1.0 - lr * weight_decay), (float)bound, x, h->steps, active, h->tensors, (uint32_t*)h->done.p};
    const dim3 grid((unsigned)((h->items + 3) / 4)), block(256);
    const bool g16 = h->grad_type == RP_BF16;
    if (h->items && h->items <= kOneLaunch && h->tensors <= kOneTensors) {
        if (h->bits == 32 && g16) hipLaunchKernelGGL((adamw_one_kernel<32, true>), grid, block, 0, st, a);
        else if (h->bits == 32) hipLaunchKernelGGL((adamw_one_kernel<32, false>), grid, block, 0, st, a);
        else if (g16) hipLaunchKernelGGL((adamw_one_kernel<8, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((adamw_one_kernel<8, false>), grid, block, 0, st, a);
        HIP_TRY(hipGetLastError());
        return RP_OK;
    }
    hipLaunchKernelGGL(adamw_begin_kernel, dim3((unsigned)((h->tensors + 63) / 64)), dim3(64), 0, st, (Scalars*)h->scalars.p,
                       h->steps, h->tensors, active, x);
    HIP_TRY(hipGetLastError());
    if (!h->items) return RP_OK;
    if (h->bits == 32 && g16) hipLaunchKernelGGL((adamw_step_kernel<32, true>), grid, block, 0, st, a);
    else if (h->bits == 32) hipLaunchKernelGGL((adamw_step_kernel<32, false>), grid, block, 0, st, a);
    else if (g16) hipLaunchKernelGGL((adamw_step_kernel<8, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((adamw_step_kernel<8, false>), grid, block, 0, st, a);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

int rp_adamw_values(rp_adamw* h, float* exp_avg, float* root, void* stream) {
    if (!h || !exp_avg || !root) return fail(RP_ERR_INVALID, "NULL handle or output");
    if (h->bits != 8) return fail(RP_ERR_INVALID, "the states are held in 32 bits");
    if (((uintptr_t)exp_avg | (uintptr_t)root) & 15) return fail(RP_ERR_INVALID, "outputs must be 16-byte aligned");
    if (!h->blocks) return RP_OK;
    DeviceGuard guard;
    int rc = guard.enter(h->device);
    if (rc) return rc;
    hipLaunchKernelGGL(adamw_values_kernel, dim3((unsigned)std::min(kValuesGrid, (h->blocks + 3) / 4)), dim3(256), 0, (hipStream_t)stream,
                       (const uint32_t*)h->m, (const uint32_t*)h->v, h->m_scale, h->v_scale, h->blocks, (float4*)exp_avg, (float4*)root);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

int rp_adamw_destroy(rp_adamw* h) {
    delete h;
    return RP_OK;
}

}  // extern "C"
