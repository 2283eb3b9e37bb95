// rp_adapt.hip — low-rank adapters of many requests beside the dense projection, and their gradients.
//
// The dense projection Y = X C^T (rp_dense.hip) has one frozen matrix C for every row. Here row i also
// has an adapter a = ids[i] of rank R (none where ids[i] is outside 0..G-1), G of them in two banks
// `down` (G x R x m) and `up` (G x R x p), both with the long axis contiguous:
//
//   hidden_i = down[a] x_i,                 y_i = C x_i + scale[a] up[a]^T hidden_i
//   t_i = scale[a] up[a] dy_i,              dx_i = C^T dy_i + down[a]^T t_i
//   d_down[a] = sum_i t_i x_i^T,            d_up[a] = scale[a] sum_i hidden_i dy_i^T
//
// so both directions are made of three products over rows that share an adapter, whatever the bank:
//   shrink  H = Z W^T      (n x q, R x q -> n x R)
//   expand  O += H W       (n x R, R x q -> n x q)
//   outer   dW = H^T Z     (per adapter, over its rows)
#include <type_traits>

#include "rp_common.h"

using namespace rpd;

namespace {

// rows that one block groups (up to 700 adapters, whose counts by 16 waves fit its LDS), else three launches: a call of 6225 rows 60 us, 70
// with three; 16384 rows grouped in 22 us and in 17.5
constexpr int kSmallRows = 8192;
// An axis of a grid has fewer than 2^32 threads: blocks of the largest grids fill rows of 2^20 (up to 512 threads a block; a multiple of 8,
// so block i runs on XCD i % 8 in every row)
constexpr int64_t kGridRow = 1 << 20;
dim3 grid_of(int64_t blocks, unsigned z = 1) { return dim3((unsigned)std::min(blocks, kGridRow), (unsigned)((blocks + kGridRow - 1) / kGridRow), z); }
__device__ __forceinline__ unsigned block_of_grid() { return blockIdx.y * gridDim.x + blockIdx.x; }
constexpr int kMaxRank = 128, kMaxAdapters = 16383;  // a wave's counts of all groups fit 64 KB of LDS

// rounded to nearest even, two at a time (one instruction); a NaN stays one
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ void store_as(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_as(uint16_t* p, float x) { *p = (uint16_t)to_bf16(x, 0.f); }

// ------------------------------------------------------------------------------------------
// Rows grouped by adapter: a stable counting sort of the ids (rows without an adapter come last, as
// group G), one wave a chunk of rows. Lanes that hold the same id find each other by a ballot for each
// bit of the id, so a lane's rank is a population count and the order never depends on timing.
struct Groups {
    int32_t* perm;    // sorted position -> row
    int32_t* sid;     // sorted position -> group (0 .. G)
    int32_t* start;   // group -> first sorted position; G + 2 entries
    int4* tiles;      // {group, first sorted position, rows, 0}: at most tile_rows rows of one group (G included)
    int4* chunks;     // {group, first sorted position, rows, its partial sums' number or -1}: at most chunk_rows rows (none where the
                      // group has none), group < G
    int32_t* tile0;   // group -> its first tile; G + 1 entries
    int32_t* chunk0;  // group -> its first chunk; G + 1 entries
    int32_t* multi0;  // group -> the first of its partial sums, where it has more than one chunk; G + 1 entries
    int32_t* number;  // {tiles, chunks}
    int32_t* hist;    // (G + 1) x n_chunks counts, then first positions
};

__device__ __forceinline__ int group_of(int32_t id, int G) { return id >= 0 && id < G ? id : G; }

// the lanes (of `live` ones) that hold the same g
__device__ __forceinline__ uint64_t same_lanes(int g, bool live, int bits) {
    uint64_t m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool on = (g >> b) & 1;
        const uint64_t v = __ballot(on);
        m &= on ? v : ~v;
    }
    return m;
}

// LDS that the lanes of one wave share: what was written before is read after
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// counts the ids of rows [r0, r1) by group into cnt (this wave's alone, zero before)
__device__ __forceinline__ void count_rows(const int32_t* __restrict__ ids, int64_t r0, int64_t r1, int G, int bits, int32_t* cnt) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = r0; r < r1; r += 64) {
        const bool live = r + lane < r1;
        const int g = live ? group_of(ids[r + lane], G) : 0;
        const uint64_t m = same_lanes(g, live, bits);
        if (live && __ffsll((unsigned long long)m) - 1 == lane) cnt[g] += __popcll(m);
        wave_sync();
    }
}

// gives every row of [r0, r1) its position, next[g] being the first free one of this wave's rows of group g
__device__ __forceinline__ void place_rows(const int32_t* __restrict__ ids, int64_t r0, int64_t r1, int G, int bits, int32_t* next,
                                           const Groups& o) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = r0; r < r1; r += 64) {
        const bool live = r + lane < r1;
        const int g = live ? group_of(ids[r + lane], G) : 0;
        const uint64_t m = same_lanes(g, live, bits);
        if (live) {
            const int at = next[g] + __popcll(m & ((1ull << lane) - 1));
            o.perm[at] = (int32_t)(r + lane);
            o.sid[at] = g;
        }
        wave_sync();  // every lane has read next before its leader moves it
        if (live && __ffsll((unsigned long long)m) - 1 == lane) next[g] += __popcll(m);
        wave_sync();
    }
}

// exclusive prefix sum over the block's threads; total: of all of them
template <typename I>
__device__ __forceinline__ I block_scan(I x, uint64_t* sums, I& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    I s = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const I y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 63) sums[w] = (uint64_t)s;
    __syncthreads();
    I before = 0;
    total = 0;
    for (int k = 0; k < nw; ++k) {
        const I y = (I)sums[k];
        if (k < w) before += y;
        total += y;
    }
    return before + s - x;
}

// one block: from each group's first position (first(g), g <= G + 1) its tiles and chunks
template <typename F>
__device__ __forceinline__ void list_groups(const F& first, int G, int tile_rows, int chunk_rows, uint64_t* sums, const Groups& o) {
    int t0 = 0, c0 = 0, p0 = 0;
    for (int base = 0; base <= G; base += blockDim.x) {
        const int g = base + threadIdx.x;
        const int s = g <= G ? first(g) : 0, rows = g <= G ? first(g + 1) - s : 0;
        const int nt = (rows + tile_rows - 1) / tile_rows, nc = g < G ? max(1, (rows + chunk_rows - 1) / chunk_rows) : 0;
        int tt, tc, tp;
        const int t = t0 + block_scan(nt, sums, tt), c = c0 + block_scan(nc, sums, tc);
        const int p = p0 + block_scan(nc > 1 ? nc : 0, sums, tp);
        if (g <= G) {
            o.start[g] = s;
            o.tile0[g] = t;
            o.chunk0[g] = c;
            o.multi0[g] = p;
            if (g == G) o.start[G + 1] = s + rows;
        }
        t0 += tt, c0 += tc, p0 += tp;
    }
    if (threadIdx.x == 0) o.number[0] = t0, o.number[1] = c0;
    __syncthreads();
    for (int g = threadIdx.x >> 6; g <= G; g += blockDim.x >> 6) {  // a wave a group
        const int s = o.start[g], rows = o.start[g + 1] - s, nc = g < G ? max(1, (rows + chunk_rows - 1) / chunk_rows) : 0;
        for (int k = threadIdx.x & 63; k * tile_rows < rows; k += 64)
            o.tiles[o.tile0[g] + k] = make_int4(g, s + k * tile_rows, min(tile_rows, rows - k * tile_rows), 0);
        for (int k = threadIdx.x & 63; k < nc; k += 64)
            o.chunks[o.chunk0[g] + k] = make_int4(g, s + k * chunk_rows, min(chunk_rows, rows - k * chunk_rows),
                                                nc > 1 ? o.multi0[g] + k : -1);
    }
}

// Rows whose width is no multiple of the kernels' step, copied to rows that are, zeros behind: block `block` of `blocks`
struct Pad {
    const void* from;
    void* to;  // or NULL: nothing to do
    int64_t ld, rows;
    int width, padded, size;  // size: bytes of an element
};
// E elements (16 bytes) of a row from its element c on, zeros behind its end
template <typename T>
__device__ __forceinline__ uint4 load_of_row(const T* row, int c, int width) {
    constexpr int E = 16 / (int)sizeof(T);
    T x[E];
    if (c + E <= width) {
        __builtin_memcpy(x, row + c, 16);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = c + e < width ? row[c + e] : T(0);
    }
    uint4 y;
    __builtin_memcpy(&y, x, 16);
    return y;
}
constexpr int pad_threads(int64_t chunks, int threads) { return chunks <= 64 ? 64 : chunks <= 256 ? 256 : threads; }  // of a row
// 16 bytes a thread, loaded from wherever they begin: an element at a time 255 MB of bf16 took 303 us
template <typename T>
__device__ __forceinline__ void pad_rows_of(const Pad& p, int64_t block, int64_t blocks) {
    constexpr int E = 16 / (int)sizeof(T);
    const int chunks = p.padded / E, each = pad_threads(chunks, blockDim.x), per = blockDim.x / each, lane = threadIdx.x % each;
    for (int64_t r = block * per + threadIdx.x / each; r < p.rows; r += blocks * per) {
        const T* from = (const T*)p.from + r * p.ld;
        uint4* to = (uint4*)((T*)p.to + r * p.padded);
        for (int c = lane; c < chunks; c += each) to[c] = load_of_row(from, c * E, p.width);
    }
}
__device__ __forceinline__ void pad_rows(const Pad& p, int64_t block, int64_t blocks) {
    if (!p.to) return;
    if (p.size == 2) pad_rows_of<uint16_t>(p, block, blocks);
    else pad_rows_of<float>(p, block, blocks);
}
__global__ void __launch_bounds__(256) pad_kernel(Pad p, Pad q) {
    pad_rows(p, blockIdx.x, gridDim.x);
    pad_rows(q, blockIdx.x, gridDim.x);
}

// few rows: one block does it all, its waves' counts in LDS as cnt[wave][group]; other blocks pad rows meanwhile
__global__ void __launch_bounds__(1024)
group_small_kernel(const int32_t* __restrict__ ids, int n, int G, int bits, int tile_rows, int chunk_rows, Groups o, Pad p, Pad q) {
    extern __shared__ int32_t lds_groups[];
    __shared__ uint64_t sums[16];
    if (blockIdx.x) {
        pad_rows(p, blockIdx.x - 1, gridDim.x - 1);
        pad_rows(q, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, nt = blockDim.x, nw = nt >> 6;
    int32_t* cnt = lds_groups;             // nw x (G + 1): the wave's rows of a group, then the first of them
    int32_t* first = cnt + nw * (G + 1);   // G + 2, and G + 1 each of the lists' first entries
    int32_t *tile0 = first + G + 2, *chunk0 = tile0 + G + 1, *multi0 = chunk0 + G + 1;
    for (int i = tid; i < nw * (G + 1); i += nt) cnt[i] = 0;
    const int each = (n + nt - 1) / nt * 64, r0 = w * each;
    int g[kSmallRows / 1024], at[kSmallRows / 1024];  // the lane's rows' groups, and their places among the wave's rows of these
#pragma unroll
    for (int k = 0; k < kSmallRows / 1024; ++k) g[k] = k * 64 < each && r0 + k * 64 + lane < n ? group_of(ids[r0 + k * 64 + lane], G) : -1;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSmallRows / 1024; ++k) {
        if (k * 64 >= each) break;
        const uint64_t m = same_lanes(max(g[k], 0), g[k] >= 0, bits);
        const int before = g[k] >= 0 ? cnt[w * (G + 1) + g[k]] : 0;
        at[k] = before + __popcll(m & ((1ull << lane) - 1));
        wave_sync();  // every lane has read the count before its first lane moves it
        if (g[k] >= 0 && __ffsll((unsigned long long)m) - 1 == lane) cnt[w * (G + 1) + g[k]] = before + __popcll(m);
        wave_sync();
    }
    __syncthreads();
    int row0 = 0;
    uint64_t list0 = 0;  // tiles, chunks and partial sums so far, 21 bits each
    for (int base = 0; base <= G; base += nt) {
        const int h = base + tid;
        int rows = 0, total;
        if (h <= G)
            for (int k = 0; k < nw; ++k) rows += cnt[k * (G + 1) + h];
        int s = row0 + block_scan(rows, sums, total);
        const int nt_ = (rows + tile_rows - 1) / tile_rows, nc = h < G ? max(1, (rows + chunk_rows - 1) / chunk_rows) : 0;
        const uint64_t lists = h <= G ? (uint64_t)nt_ | (uint64_t)nc << 21 | (uint64_t)(nc > 1 ? nc : 0) << 42 : 0;
        uint64_t all;
        const uint64_t l = list0 + block_scan(lists, sums, all);
        if (h <= G) {
            first[h] = o.start[h] = s;
            tile0[h] = (int)(l & 0x1fffff), chunk0[h] = (int)(l >> 21 & 0x1fffff), multi0[h] = o.multi0[h] = (int)(l >> 42);
            if (h == G) first[G + 1] = o.start[G + 1] = n;
            for (int k = 0; k < nw; ++k) {
                const int c = cnt[k * (G + 1) + h];
                cnt[k * (G + 1) + h] = s;
                s += c;
            }
        }
        row0 += total, list0 += all;
    }
    if (tid == 0) o.number[0] = (int)(list0 & 0x1fffff), o.number[1] = (int)(list0 >> 21 & 0x1fffff);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSmallRows / 1024; ++k)
        if (k * 64 < each && g[k] >= 0) {
            const int to = cnt[w * (G + 1) + g[k]] + at[k];
            o.perm[to] = r0 + k * 64 + lane;
            o.sid[to] = g[k];
        }
    for (int h = w; h <= G; h += nw) {  // a wave a group
        const int s = first[h], rows = first[h + 1] - s, nc = h < G ? max(1, (rows + chunk_rows - 1) / chunk_rows) : 0;
        for (int k = lane; k * tile_rows < rows; k += 64)
            o.tiles[tile0[h] + k] = make_int4(h, s + k * tile_rows, min(tile_rows, rows - k * tile_rows), 0);
        for (int k = lane; k < nc; k += 64)
            o.chunks[chunk0[h] + k] = make_int4(h, s + k * chunk_rows, min(chunk_rows, rows - k * chunk_rows), nc > 1 ? multi0[h] + k : -1);
    }
}

// up to 64 rows: a row's place is the number of those before it, a group's first row the number of rows of lower ones. Each adapter has one
// chunk; there is no list of tiles.
__device__ __forceinline__ void group_few(const int32_t* __restrict__ ids, int n, int G, int32_t* g, const Groups& o) {
    const int tid = threadIdx.x;
    if (tid < 64) g[tid] = tid < n ? group_of(ids[tid], G) : G + 1;
    __syncthreads();
    if (tid < n) {
        int to = 0;
        for (int i = 0; i < n; ++i) to += g[i] < g[tid] || (g[i] == g[tid] && i < tid);
        o.perm[to] = tid;
        o.sid[to] = g[tid];
    }
    for (int h = tid; h <= G + 1; h += blockDim.x) {
        int first = 0, rows = 0;
        for (int i = 0; i < n; ++i) first += g[i] < h, rows += g[i] == h;
        o.start[h] = first;
        if (h < G) o.chunks[h] = make_int4(h, first, rows, -1), o.multi0[h] = 0;
    }
    if (tid == 0) o.number[0] = 0, o.number[1] = G;
}

// many rows: counts of each wave's rows (4 waves a block) to hist[group][chunk]
__global__ void __launch_bounds__(256)
group_count_kernel(const int32_t* __restrict__ ids, int64_t n, int G, int bits, int64_t each, int n_chunks, Groups o) {
    extern __shared__ int32_t lds_groups[];
    int32_t* cnt = lds_groups + (threadIdx.x >> 6) * (G + 1);
    const int lane = threadIdx.x & 63, chunk = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    for (int g = lane; g <= G; g += 64) cnt[g] = 0;
    wave_sync();
    const int64_t r0 = min(n, chunk * each);
    count_rows(ids, r0, min(n, r0 + each), G, bits, cnt);
    if (chunk < n_chunks)
        for (int g = lane; g <= G; g += 64) o.hist[(int64_t)g * n_chunks + chunk] = cnt[g];
}

// one block: exclusive prefix sums of hist in its order, 4096 entries at a time and the next ones on their way, and the lists
__global__ void __launch_bounds__(1024) group_scan_kernel(int64_t n, int G, int n_chunks, int tile_rows, int chunk_rows, Groups o) {
    __shared__ uint64_t sums[16];
    const int all = (G + 1) * n_chunks;
    const auto load = [&](int i) {
        int4 x = make_int4(0, 0, 0, 0);
        if (i + 4 <= all) x = *reinterpret_cast<const int4*>(o.hist + i);
        else if (i < all) x = make_int4(o.hist[i], i + 1 < all ? o.hist[i + 1] : 0, i + 2 < all ? o.hist[i + 2] : 0, 0);
        return x;
    };
    int before = 0, total;
    int4 x = load(threadIdx.x * 4);
    for (int i = threadIdx.x * 4; i - (int)threadIdx.x * 4 < all; i += 4096) {
        const int4 next = load(i + 4096);  // on its way meanwhile
        int s = before + block_scan(x.x + x.y + x.z + x.w, sums, total);
        const int4 y = make_int4(s, s + x.x, s + x.x + x.y, s + x.x + x.y + x.z);
        if (i + 4 <= all) {
            *reinterpret_cast<int4*>(o.hist + i) = y;
        } else {
            if (i < all) o.hist[i] = y.x;
            if (i + 1 < all) o.hist[i + 1] = y.y;
            if (i + 2 < all) o.hist[i + 2] = y.z;
        }
        before += total, x = next;
    }
    __syncthreads();
    list_groups([&](int g) { return g <= G ? o.hist[(int64_t)g * n_chunks] : (int)n; }, G, tile_rows, chunk_rows, sums, o);
}

__global__ void __launch_bounds__(256)
group_place_kernel(const int32_t* __restrict__ ids, int64_t n, int G, int bits, int64_t each, int n_chunks, Groups o) {
    extern __shared__ int32_t lds_groups[];
    int32_t* next = lds_groups + (threadIdx.x >> 6) * (G + 1);
    const int lane = threadIdx.x & 63, chunk = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (chunk >= n_chunks) return;
    for (int g = lane; g <= G; g += 64) next[g] = o.hist[(int64_t)g * n_chunks + chunk];
    wave_sync();
    const int64_t r0 = min(n, chunk * each);
    place_rows(ids, r0, min(n, r0 + each), G, bits, next, o);
}

// ------------------------------------------------------------------------------------------
// Matrix instructions. 16 x 16 tiles; a lane's operand is 16 bytes of a row of each side (row = lane &
// 15, 16-byte chunk = lane >> 4), so 64 bytes of a row are one step of the contraction: 32 bf16 in one
// instruction, 16 f32 in four (element e of every lane's chunk in instruction e: a permutation of the
// step, the same on both sides). D[i][j], i a row of `a`, j a row of `b`: lane l holds j = l & 15, i = 4 (l >> 4) + e.
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));


__device__ __forceinline__ void put4(float* p, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void put4(uint16_t* p, f32x4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(to_bf16(x[0], x[1]), to_bf16(x[2], x[3]));
}

template <typename T>
__device__ __forceinline__ f32x4 mma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    }
}

// x = hi + mid + low exactly, each a bf16 (8 bits of the 24 at a time, cut off): an f32 factor against
// bf16 ones in three matrix instructions without a rounding. An infinity is hi alone.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& low) {
    hi = __float_as_uint(x) & 0xffff0000u;
    const float h = __uint_as_float(hi), y = h == x ? 0.f : x - h;
    mid = __float_as_uint(y) & 0xffff0000u;
    low = __float_as_uint(y - __uint_as_float(mid)) & 0xffff0000u;
}
// What mid and low are multiplied by: bf16 values with the largest finite one for an infinity or a NaN. Against an infinity itself a mid or
// low of 0 would make a NaN; hi, which has it, is 0 only where x is (or under 2^-133), and a mid or low that is not 0 has the sign of hi. Under
// what one box varies by: gradients of 16384 x 16384 -> 1024 703 us, 707 without; 1777 x 4096 -> 4096 of rank 64 100 to 103, 101 to 103 without.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t finite(uint32_t x) {
    const u16x2 y = __builtin_elementwise_min(__builtin_bit_cast(u16x2, x & 0x7fff7fffu), u16x2{0x7f7f, 0x7f7f});
    return (__builtin_bit_cast(uint32_t, y) & 0x7fff7fffu) | (x & 0x80008000u);
}
__device__ __forceinline__ uint4 finite(uint4 x) { return make_uint4(finite(x.x), finite(x.y), finite(x.z), finite(x.w)); }
// the upper halves of a (low half of the result) and b
__device__ __forceinline__ uint32_t pack_high(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t pack_low(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

// 16 bytes that nothing reads again soon, past the caches: they leave the room to what does
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_anywhere __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 load_once(const void* p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_anywhere*>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store_once(void* p, uint4 x) {
    __builtin_nontemporal_store(u32x4{x.x, x.y, x.z, x.w}, reinterpret_cast<u32x4*>(p));
}

// The factor that the expand reads: `parts` pieces of scale[a] H[i][r] for every row, each of its ranks padded with zeros to 64
// bytes. bf16: the pieces of split3; f32: the value itself.
__host__ __device__ __forceinline__ int padded_rank(int R, int size) { return size == 2 ? (R + 31) / 32 * 32 : (R + 15) / 16 * 16; }
template <typename T>
__host__ __device__ constexpr int pieces() { return sizeof(T) == 2 ? 3 : 1; }

struct ShrinkArgs {
    const void* Z;
    int64_t ldz, kp;
    const void* W;
    int G, R;
    const float* scale;  // or NULL: 1
    float* H;            // or NULL; n x R
    int scaled;          // H takes the scale too
    void* S;             // or NULL; n x pieces x padded rank
    f32x4* part;
};

// a lane's four ranks of one row of a tile (place i of the tile's 16 x 16 sums, KT of them along the ranks) to H and to the pieces
template <typename T, int KT>
__device__ __forceinline__ void shrink_finish(const ShrinkArgs& a, const Groups& o, int4 tile, int i, f32x4 x) {
    const int R = a.R, rp = padded_rank(R, sizeof(T));
    const int l = i & 63, row = i / (64 * KT) * 16 + (l & 15), r = (i >> 6) % KT * 16 + 4 * (l >> 4);
    if (row >= tile.z) return;
    const int64_t to = o.perm[tile.y + row];
    f32x4 y = x * (a.scale ? a.scale[tile.x] : 1.f);
    if (a.H) {
        float* h = a.H + to * R + r;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (r + e < R) h[e] = a.scaled ? y[e] : x[e];
    }
    if (!a.S || r >= rp) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r + e >= R) y[e] = 0.f;
    if constexpr (sizeof(T) == 2) {
        uint32_t v[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split3(y[e], v[0][e], v[1][e], v[2][e]);
        uint16_t* d = (uint16_t*)a.S + to * 3 * rp + r;
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            *reinterpret_cast<uint2*>(d + u * rp) = make_uint2(pack_high(v[u][0], v[u][1]), pack_high(v[u][2], v[u][3]));
            if (KT == 1) *reinterpret_cast<uint2*>(d + u * rp + 16) = make_uint2(0, 0);  // ranks 16 .. 31
        }
    } else {
        *reinterpret_cast<f32x4*>((float*)a.S + to * rp + r) = y;
    }
}

// H[i][r] = (scaled ? scale[a] : 1) sum_q Z[i][q] W[a][r][q], zeros for rows without an adapter, and its pieces. A block takes a tile
// of 16 RT rows of one group; its four waves split the contraction and add up in LDS in their order. Bound by reading Z once where
// there are many rows: the wave holds 16 RT x 16 KT of H, so W (from L2) is read once for 16 RT rows, and there is nothing between
// the loads and the matrix instructions (65536 x 16384 by rank 16 in bf16: 0.39 ms, 5.5 TB/s). Where there are few, by how much of
// its row a compute unit can take in: the contraction is then split over the grid too, and shrink_join_kernel adds up.
template <typename T, int RT, int KT>
__global__ void __launch_bounds__(256)
shrink_kernel(ShrinkArgs a, Groups o) {
    constexpr int NW = 4;
    __shared__ f32x4 red[NW][RT * KT][64];
    if ((int)blockIdx.x >= o.number[0]) return;
    const int4 tile = o.tiles[blockIdx.x];
    const int g = tile.x, pos = tile.y, rows = tile.z, R = a.R;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, q = lane >> 4;
    if (g == a.G) {
        if (a.H && blockIdx.y == 0)
            for (int i = tid; i < rows * R; i += 64 * NW) a.H[(int64_t)o.perm[pos + i / R] * R + i % R] = 0.f;
        return;
    }
    const T* __restrict__ Z = (const T*)a.Z;
    const T* __restrict__ W = (const T*)a.W;
    const int64_t kp = a.kp;
    const char* z[RT];
    const char* b[KT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
        z[t] = reinterpret_cast<const char*>(Z + o.perm[pos + min(t * 16 + c, rows - 1)] * a.ldz) + q * 16;
#pragma unroll
    for (int j = 0; j < KT; ++j)
        b[j] = reinterpret_cast<const char*>(W + ((int64_t)g * R + min(j * 16 + c, R - 1)) * kp) + q * 16;
    f32x4 acc[RT][KT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < KT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t lines = kp * (int64_t)sizeof(T) / 128;  // 128 bytes of a row: two steps
    const int64_t s0 = lines * blockIdx.y / gridDim.y, s1 = lines * (blockIdx.y + 1) / gridDim.y, each = (s1 - s0 + NW - 1) / NW;
    const int64_t l1 = min(s1, s0 + (w + 1) * each);
    for (int64_t l = s0 + w * each; l < l1; ++l) {
        uint4 zf[2][RT], bf[2][KT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < RT; ++t) zf[h][t] = *reinterpret_cast<const uint4*>(z[t] + l * 128 + h * 64);
#pragma unroll
            for (int j = 0; j < KT; ++j) bf[h][j] = *reinterpret_cast<const uint4*>(b[j] + l * 128 + h * 64);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < KT; ++j) acc[t][j] = mma<T>(bf[h][j], zf[h][t], acc[t][j]);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < KT; ++j) red[w][t * KT + j][lane] = acc[t][j];
    __syncthreads();
    for (int i = tid; i < RT * KT * 64; i += 64 * NW) {
        const f32x4* p = &red[0][0][0] + i;
        f32x4 x = p[0];
#pragma unroll
        for (int k = 1; k < NW; ++k) x += p[k * RT * KT * 64];
        if (gridDim.y == 1) shrink_finish<T, KT>(a, o, tile, i, x);
        else a.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (RT * KT * 64) + i] = x;
    }
}

// the splits' sums of tiles of 16 rows, in order
template <typename T, int KT>
__global__ void __launch_bounds__(64 * KT) shrink_join_kernel(ShrinkArgs a, Groups o, int splits) {
    if ((int)blockIdx.x >= o.number[0]) return;
    const int4 tile = o.tiles[blockIdx.x];
    if (tile.x == a.G) return;
    const int i = threadIdx.x;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < splits; ++k) x += a.part[((int64_t)k * gridDim.x + blockIdx.x) * (KT * 64) + i];
    shrink_finish<T, KT>(a, o, tile, i, x);
}

// D[g][r][c] (+ partial sums) = (mul ? mul[g] : 1) sum over rows i of adapter g of H[i][r] Z[i][c]. A block takes 16
// KT ranks by 128 (bf16) or 64 (f32) columns over a chunk of one group's rows, a wave every fourth step of them, its lanes
// reading 16 bytes of neighbouring columns of each row, aligned or not: no LDS for Z, which is read once (per 16 KT ranks) and bounds the kernel
// (16384 x 16384 and 16384 x 1024 in bf16, rank 16: 0.11 ms, 5.2 TB/s).
//   bf16: 32 rows a step, lane (c, q) rows 8 q .. 8 q + 7, columns 8 c .. 8 c + 7: 8 x 8 values turned round in
//         registers (a byte permutation for two values), so column j of every lane is one matrix operand. H is split exactly
//         into three bf16.
//   f32:  4 rows a matrix instruction, lane (c, q) row q, columns 4 c .. 4 c + 3.
struct OuterArgs {
    const void* Z;
    int64_t ldz, qp, q, wide;  // qp: columns of the partial sums' rows; wide: readable ones of Z
    int R;
    const float *mul, *H;
    float* D;
    int64_t ldd, sdd;
    float* part;
    int vec;  // rows of D and of the partial sums are 16-byte aligned
};

constexpr int kMaxChunk = 2048;

template <typename T, int KT>
__global__ void __launch_bounds__(256, KT == 1 ? 4 : 2) outer_kernel(OuterArgs a0, OuterArgs a1, int blocks0, int blocks, Groups o) {
    constexpr int NC = sizeof(T) == 2 ? 8 : 4;  // columns of a lane
    constexpr int RS = sizeof(T) == 2 ? 8 : 4;  // rows of a lane in a step of 4 RS rows
    __shared__ int32_t list[kMaxChunk];
    __shared__ float red[4][NC][64][4];
    const unsigned id = block_of_grid();
    const int which = (int)(id / (unsigned)blocks), block = (int)(id % (unsigned)blocks);
    if (which >= o.number[1]) return;
    const bool second = block >= blocks0;  // both banks' gradients in one launch
    const OuterArgs& a = second ? a1 : a0;
    const int4 chunk = o.chunks[which];
    const int g = chunk.x, rows = chunk.z;
    for (int i = threadIdx.x; i < rows; i += 256) list[i] = o.perm[chunk.y + i];
    __syncthreads();
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
    const int64_t col0 = (int64_t)(block - (second ? blocks0 : 0)) * (16 * NC), col = col0 + c * NC;
    // a lane whose columns reach past the readable ones takes the last of these: `shift` of them are its neighbour's
    const int64_t from = min(col, a.wide - NC);
    const int shift = (int)(col - from);
    const T* __restrict__ Z = (const T*)a.Z + from;
    const float* __restrict__ H = a.H;
    const int64_t ldz = a.ldz;
    const int r0 = blockIdx.z * 16 * KT, R = a.R;
    f32x4 acc[KT][NC];
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[k][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](int i0, uint4 (&z)[RS], float (&h)[KT][RS]) {
#pragma unroll
        for (int j = 0; j < RS; ++j) {
            const int i = i0 + (sizeof(T) == 2 ? q * RS + j : j * 4 + q);
            const int64_t row = list[min(i, rows - 1)];
            z[j] = load_once(Z + row * ldz);
#pragma unroll
            for (int k = 0; k < KT; ++k) h[k][j] = H[row * R + min(r0 + k * 16 + c, R - 1)];
        }
    };
    auto add = [&](int i0, uint4 (&z)[RS], float (&h)[KT][RS]) {
        if (i0 + 4 * RS > rows) {  // what lies behind the last row counts nothing, whatever it is
#pragma unroll
            for (int j = 0; j < RS; ++j)
                if (i0 + (sizeof(T) == 2 ? q * RS + j : j * 4 + q) >= rows) {
                    z[j] = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < KT; ++k) h[k][j] = 0.f;
                }
        }
        if constexpr (sizeof(T) == 2) {
            uint4 hp[KT][3];
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                uint32_t p[3][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) split3(h[k][j], p[0][j], p[1][j], p[2][j]);
#pragma unroll
                for (int s = 0; s < 3; ++s)
                    hp[k][s] = make_uint4(pack_high(p[s][0], p[s][1]), pack_high(p[s][2], p[s][3]), pack_high(p[s][4], p[s][5]),
                                          pack_high(p[s][6], p[s][7]));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const auto word = [&](int i) { return j / 2 == 0 ? z[i].x : j / 2 == 1 ? z[i].y : j / 2 == 2 ? z[i].z : z[i].w; };
                const auto pair = [&](int i) { return j & 1 ? pack_high(word(i), word(i + 1)) : pack_low(word(i), word(i + 1)); };
                const uint4 zc = make_uint4(pair(0), pair(2), pair(4), pair(6)), zf = finite(zc);
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int s = 0; s < 3; ++s) acc[k][j] = mma<T>(hp[k][s], s ? zf : zc, acc[k][j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = __uint_as_float(j == 0 ? z[i].x : j == 1 ? z[i].y : j == 2 ? z[i].z : z[i].w);
#pragma unroll
                    for (int k = 0; k < KT; ++k) acc[k][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(h[k][i], v, acc[k][j], 0, 0, 0);
                }
        }
    };
    if (rows) {
        uint4 z[RS];
        float h[KT][RS];
        for (int i0 = w * 4 * RS; i0 < rows; i0 += 16 * RS) {
            load(i0, z, h);
            add(i0, z, h);
        }
    }
    const float s = a.mul && rows ? a.mul[g] : 1.f;
    float* out = chunk.w >= 0 ? a.part + (int64_t)chunk.w * R * a.qp : a.D + g * a.sdd;
    const int64_t ld = chunk.w >= 0 ? a.qp : a.ldd;
    // the four waves' sums, in order, 16 ranks at a time; a thread then has four neighbouring columns of a rank
#pragma unroll
    for (int k = 0; k < KT; ++k) {
        if (k) __syncthreads();
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (j >= shift) *reinterpret_cast<f32x4*>(red[w][j - shift][lane]) = acc[k][j];
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < 16 * 4 * NC; i += 256) {
            const int quad = i % (4 * NC), rank = i / (4 * NC), r = r0 + k * 16 + rank, j0 = quad * 4 % NC;
            const int at_lane = (rank >> 2) * 16 + quad * 4 / NC;
            const int64_t at = col0 + quad * 4;
            if (r >= R || at >= a.q) continue;
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = (red[0][j0 + e][at_lane][rank & 3] + red[1][j0 + e][at_lane][rank & 3] + red[2][j0 + e][at_lane][rank & 3] +
                        red[3][j0 + e][at_lane][rank & 3]) * s;
            float* d = out + r * ld + at;
            if (a.vec && at + 4 <= a.q) {
                *reinterpret_cast<f32x4*>(d) = x;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < a.q) d[e] = x[e];
            }
        }
    }
}

// adapters whose rows were cut into chunks: the partial sums in order
__global__ void __launch_bounds__(256) outer_join_kernel(OuterArgs a0, OuterArgs a1, int blocks0, Groups o, int chunk_rows) {
    const int g = blockIdx.z, r = blockIdx.y;
    const int rows = o.start[g + 1] - o.start[g], nc = (rows + chunk_rows - 1) / chunk_rows;
    if (nc <= 1) return;
    const bool second = (int)blockIdx.x >= blocks0;
    const OuterArgs& a = second ? a1 : a0;
    const int64_t c = (int64_t)(blockIdx.x - (second ? blocks0 : 0)) * 256 + threadIdx.x;
    if (c >= a.q) return;
    float s = 0.f;
    const float* p = a.part + ((int64_t)o.multi0[g] * a.R + r) * a.qp + c;
    for (int k = 0; k < nc; ++k) s += p[(int64_t)k * a.R * a.qp];
    a.D[g * a.sdd + r * a.ldd + c] = s;
}

// ------------------------------------------------------------------------------------------
// The shared product with the adapters' expand: O[i][c] = sum_k A[i][k] B[c][k] + sum_r (scale[a] H[i][r]) W[a][r][c].
//
// BM x BN tiles, WM x WN waves; rows are taken in the order of the adapters (gathered by the loads, scattered by the
// stores, at no cost), so few tiles hold more than one or two. The main loop stages 128 bytes of every row of A and of B
// at a time by loads that go to LDS directly. Whole lines: with 64 bytes a stage every line crossed from L2 twice (its other
// half had left the L1 by the next stage): 1.10 against 1.25 PFLOP/s at 65536 x 16384 -> 1024. A stage is multiplied in two
// halves, each half's operands read into registers during the half before; in the middle all waves meet once, the next stage
// having landed. LDS is five slots of one operand's stage, taken in turn (A, B, A, B, ..): when a stage has been read, B of the stage
// after the next and A of the one behind that start into its slots, so A, which comes from HBM, is two stages ahead, and all
// 160 KB are used (two whole stages of each: 1.28 against 1.38 PFLOP/s; a third would not fit). A thread's loads are spread over
// the half's matrix instructions.
// After the loop the pieces of the rows' H (exact in three bf16) and the adapter's W take the slots' place, 64 bytes of ranks
// at a time, and are multiplied into registers of their own, from where only the adapter's rows are added: a value that is
// not finite in one adapter reaches no other's rows. The result goes through LDS so that rows are stored 128 bytes at a
// time (16 rows a store otherwise: a tenth longer at 16384 x 1024 -> 16384 with bf16 out).
// Measured: 65536 x 16384 -> 1024 1.61 to 1.68 ms with rank 16, 1.34 PFLOP/s, matrix units busy 0.72 of the time; 16384 x 1024 -> 16384 with bf16
// out 0.60 to 0.62 ms, busy half of it: 16 stages a tile, and a unit holds one tile, whose first loads, adapters (0.05 ms in all) and stores (0.05
// ms) nothing overlaps. Blocks that go from tile to tile and load the next one's first stage behind the stores need more than the 256
// registers that a tile of 256 x 256 leaves nothing of: what is spilled made it 0.92 ms.
struct GemmArgs {
    const char *A, *B;
    int64_t lda, ldb;  // bytes
    int64_t M;
    int N, steps;  // stages of 128 bytes of a row
    void* out;
    int64_t ldo;
    int vec, stream;  // rows of out are 16-byte aligned; out is larger than the caches
    const char* S;  // the rows' factors (ShrinkArgs)
    const char* W;
    int64_t ldw;    // bytes between ranks
    int G, R;
    unsigned m_tiles, n_tiles, splits, per_xcd;
    float* part;  // without the expand: partial sums, splits x M x ldp
    int64_t ldp;
};

// EXPAND: with the adapters' part; else rows are taken as they lie and `o` is not read. lds: 5 slots.
template <typename T, typename O, int BM, int BN, int WM, int WN, bool EXPAND>
__device__ __forceinline__ void gemm_tile(const GemmArgs& a, const Groups& o, unsigned block, uint4* lds) {
    constexpr int NT = 64 * WM * WN, MT = BM / WM / 16, NN = BN / WN / 16, SL = BM * 8;  // SL: chunks of a slot
    constexpr int PL = BM * 8 / NT, PB = BN * 8 / NT;  // loads of a thread for a stage of A and of B
    // hi, mid and low of H, for a result in bf16 too: where the product and the adapters' part cancel, low is not below its rounding
    constexpr int PARTS = pieces<T>(), KR = 64 / (int)sizeof(T);
    static_assert(PL == 4 && (PB == 4 || PB == 2), "the waits below count these loads");
    static_assert(2 * (PARTS * BM * 4 + BN * 4) <= 4 * SL, "adapters take four slots' place");
    static_assert(WM * WN * MT * 16 * 8 <= 4 * SL && NN == 4, "so do the stores, 64 columns a wave");
    static_assert(NT >= BM && BM * 3 <= SL * 4, "a row a thread; the fifth slot holds the tables");
    int32_t* sid = reinterpret_cast<int32_t*>(lds + 4 * SL);  // after the main loop: the tile's rows' groups,
    int32_t* rows = sid + BM;                                 // where they are,
    int32_t* ends = rows + BM;                                // and where in the tile their group ends
    // XCD x (block i runs on XCD i % 8) takes a run of tiles; tiles go down 8 row tiles, then along the columns, so the
    // tiles that run at the same time on an XCD share their rows of A and of B in its L2
    const unsigned tiles = a.m_tiles * a.n_tiles, id = (block & 7u) * a.per_xcd + (block >> 3);
    if ((block >> 3) >= a.per_xcd || id >= tiles * a.splits) return;
    const unsigned split = id / tiles, t = id % tiles, band = t / (8u * a.n_tiles), in = t % (8u * a.n_tiles);
    const unsigned high = min(8u, a.m_tiles - band * 8u), mt = band * 8u + in % high, nt = in / high;
    const int64_t m0 = (int64_t)mt * BM;
    const int n0 = (int)nt * BN, live = (int)min((int64_t)BM, a.M - m0);
    const int k0 = (int)((int64_t)a.steps * split / a.splits), steps = (int)((int64_t)a.steps * (split + 1) / a.splits) - k0;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w / WN, wn = w % WN, fr = lane & 15, fq = lane >> 4;
    const auto row_of = [&](int i) { return EXPAND ? (int64_t)o.perm[m0 + i] : m0 + i; };
    const int first = EXPAND ? o.sid[m0] : a.G, first_end = EXPAND ? (int)min((int64_t)live, o.start[first + 1] - m0) : 0;
    // 16-byte chunk c of row r of a slot lies at r * 8 + (c ^ (r & 7)): lanes that read one chunk of 16 rows hit all banks
    const int srow = tid >> 3, sxc = (tid & 7) ^ (srow & 7);
    const char* ga[PL];
    const char* gb[PB];
#pragma unroll
    for (int i = 0; i < PL; ++i) ga[i] = a.A + row_of(min(i * (NT / 8) + srow, live - 1)) * a.lda + sxc * 16 + (int64_t)k0 * 128;
#pragma unroll
    for (int i = 0; i < PB; ++i) gb[i] = a.B + min(n0 + i * (NT / 8) + srow, a.N - 1) * a.ldb + sxc * 16 + (int64_t)k0 * 128;
    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)reinterpret_cast<uintptr_t>(lds + 64 * w));
    // Loads to LDS as inline asm: the compiler does not see what they write, so it puts no wait for all of them before an LDS
    // read; the waits are below. No output register is involved. M0 holds the wave's destination, and the hardware asks for an instruction between
    // its write and the load: the s_nop, 0.1 % at 65536 x 16384 -> 1024, 1.3 % at 16384 x 1024 -> 16384 (the address formed there instead: 1.8 % more
    // and 1.2 % less; the sum taken into M0 itself: 1.3 and 0.3 %).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the clobber keeps the compiler's own uses safe
    auto to_lds = [&](const char* from, int chunk) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds0 + (uint32_t)chunk * 16u) : "m0");
    };
#pragma clang diagnostic pop
    auto load_a = [&](int kt, int i, int slot) { to_lds(ga[i] + (int64_t)kt * 128, slot * SL + i * NT); };
    auto load_b = [&](int kt, int i, int slot) { to_lds(gb[i] + (int64_t)kt * 128, slot * SL + i * NT); };
    const int ra = wm * MT * 16 + fr, rb = wn * NN * 16 + fr;
    const int a0 = ra * 8 + (fq ^ (ra & 7)), a1 = ra * 8 + ((4 + fq) ^ (ra & 7));  // a lane's chunk of the two halves
    const int b0 = rb * 8 + (fq ^ (rb & 7)), b1 = rb * 8 + ((4 + fq) ^ (rb & 7));
    uint4 fa[2][MT], fb[2][NN];
    f32x4 acc[MT][NN];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
        for (int ni = 0; ni < NN; ++ni) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};
    // x is multiplied while y is read (rd) from pa and pb, and B of stage next (>= 0) starts into slot sb, A of the stage behind it
    // into slot sa; a row of tiles at a time, in this order
    auto half = [&](uint4 (&xa)[MT], uint4 (&xb)[NN], uint4 (&ya)[MT], uint4 (&yb)[NN], const uint4* pa, const uint4* pb, bool rd,
                    int next, int sb, int sa) {
        constexpr int RD = (MT + NN + MT - 1) / MT, LD = (PL + PB) / MT;
#pragma unroll
        for (int mi = 0; mi < MT; ++mi) {
            if (rd)
#pragma unroll
                for (int r = mi * RD; r < (mi + 1) * RD; ++r) {
                    if (r < NN) yb[r < NN ? r : 0] = pb[r * 128];
                    else if (r < NN + MT) ya[r >= NN && r < NN + MT ? r - NN : 0] = pa[(r - NN) * 128];
                }
            if (next >= 0)
#pragma unroll
                for (int d = mi * LD; d < (mi + 1) * LD; ++d) {
                    if (d < PB) load_b(next, d < PB ? d : 0, sb);
                    else if (next + 1 < steps) load_a(next + 1, d >= PB ? d - PB : 0, sa);
                }
#pragma unroll
            for (int ni = 0; ni < NN; ++ni) acc[mi][ni] = mma<T>(xb[ni], xa[mi], acc[mi][ni]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // KR ranks of an adapter, 64 bytes of each row's pieces and of each column of W: `fetch` starts the pieces to LDS (those of
    // other adapters' rows come along and are not used) and W into registers, `place` turns it round into LDS. Two blocks lie in LDS,
    // so the next is fetched while one is multiplied, and the first during the last half stage of the main loop.
    constexpr int EW = BN * KR / NT, BLOCK = PARTS * BM * 4 + BN * 4, FP = PARTS * BM * 4 / NT;
    constexpr int WC = EW * (int)sizeof(T) / 16;  // chunks of W a thread
    static_assert(WC * 16 == EW * (int)sizeof(T) && (PL + PB) % MT == 0, "whole chunks, whole rows of tiles");
    const int wi = tid % BN, we = __builtin_amdgcn_readfirstlane(tid / BN * EW);
    T wx[EW];
    auto F = [](int r) { return (4 - ((r >> 2) & 3)) & 3; };  // chunk c of a row r of 64 bytes lies at r * 4 + (c ^ F(r)): all banks
    const int rp = padded_rank(a.R, sizeof(T));
    auto fetch = [&](int g, int r0, int buf, auto row_at) {
#pragma unroll
        for (int i = 0; i < FP; ++i) {
            const int k = i * NT + tid, u = k / (BM * 4), r = (k >> 2) % BM, ch = (k & 3) ^ F(r);
            to_lds(a.S + (((int64_t)row_at(r) * pieces<T>() + u) * rp + r0) * (int)sizeof(T) + ch * 16, buf * BLOCK + i * NT);
        }
        const char* base = a.W + (int64_t)g * a.R * a.ldw + (int64_t)min(n0 + wi, a.N - 1) * (int)sizeof(T);
#pragma unroll
        for (int e = 0; e < EW; ++e) wx[e] = *reinterpret_cast<const T*>(base + min(r0 + we + e, a.R - 1) * a.ldw);
    };
    auto place = [&](int r0, int buf) {
        uint4* sw = lds + buf * BLOCK + PARTS * BM * 4;
#pragma unroll
        for (int k = 0; k < WC; ++k) {
            constexpr int E = 16 / (int)sizeof(T);
            T y[E];
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = r0 + we + k * E + e < a.R ? wx[k * E + e] : T(0);
            uint4 z;
            __builtin_memcpy(&z, y, 16);
            sw[wi * 4 + ((we / E + k) ^ F(wi))] = z;
        }
    };
#pragma unroll
    for (int i = 0; i < PL; ++i) load_a(0, i, 0);
#pragma unroll
    for (int i = 0; i < PB; ++i) load_b(0, i, 1);
    if (steps > 1) {
#pragma unroll
        for (int i = 0; i < PL; ++i) load_a(1, i, 2);
#pragma unroll
        for (int i = 0; i < PB; ++i) load_b(1, i, 3);
    }
    if (steps > 2)
#pragma unroll
        for (int i = 0; i < PL; ++i) load_a(2, i, 4);
    if (steps > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PL + PB) : "memory");  // the first stage
    else if (steps > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PL + PB) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int ni = 0; ni < NN; ++ni) fb[0][ni] = lds[SL + b0 + ni * 128];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) fa[0][mi] = lds[a0 + mi * 128];
    // in the middle of a stage: this wave's reads of it are in registers, the next one has landed (of what it has started, A of
    // the stage behind that may still be on its way); then so it is for every wave
    auto meet = [&](bool more) {
        if (more) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    int kt = 0, sa = 0, sb = 1;  // slots of stage kt
    for (; kt + 1 < steps; ++kt) {
        const int na = sb == 4 ? 0 : sb + 1, nb = na == 4 ? 0 : na + 1;
        half(fa[0], fb[0], fa[1], fb[1], lds + sa * SL + a1, lds + sb * SL + b1, true, -1, 0, 0);
        meet(kt + 2 < steps);
        half(fa[1], fb[1], fa[0], fb[0], lds + na * SL + a0, lds + nb * SL + b0, true, kt + 2 < steps ? kt + 2 : -1, sa, sb);
        sa = na, sb = nb;
    }
    half(fa[0], fb[0], fa[1], fb[1], lds + sa * SL + a1, lds + sb * SL + b1, true, -1, 0, 0);
    meet(false);
    if (EXPAND && tid < BM) {
        const int i = min(tid, live - 1), g = o.sid[m0 + i];
        sid[tid] = tid < live ? g : a.G;
        rows[tid] = o.perm[m0 + i];
        ends[tid] = (int)min((int64_t)live, o.start[g + 1] - m0);
    }
    if (EXPAND && first < a.G) fetch(first, 0, 0, [&](int r) { return o.perm[m0 + min(r, live - 1)]; });
    half(fa[1], fb[1], fa[0], fb[0], lds, lds, false, -1, 0, 0);
    // 128 bytes of columns of the wave's rows at a time: written to LDS as the lanes hold them, read as rows
    auto store = [&](auto* out, int64_t ldo, bool vec) {
        using V = std::remove_pointer_t<decltype(out)>;
        constexpr int E = 16 / (int)sizeof(V), NP = 128 / (int)sizeof(V) / 16;  // values of a chunk; tiles in 128 bytes
        char* mine = reinterpret_cast<char*>(lds + w * MT * 16 * 8);
#pragma unroll
        for (int n = 0; n < NN; n += NP) {
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int r = mi * 16 + fr, at = j * 16 + 4 * fq;  // its first column
                    put4(reinterpret_cast<V*>(mine + r * 128 + ((at / E) ^ (r & 7)) * 16) + at % E, acc[mi][n + j]);
                }
            wave_sync();
            const int c = n0 + wn * NN * 16 + n * 16 + (lane & 7) * E;
#pragma unroll
            for (int i = 0; i < MT * 2; ++i) {
                const int r = i * 8 + (lane >> 3), row = wm * MT * 16 + r;
                const uint4 x = *reinterpret_cast<const uint4*>(mine + r * 128 + ((lane & 7) ^ (r & 7)) * 16);
                if (row >= live || c >= a.N) continue;
                V* d = out + (EXPAND ? (int64_t)rows[row] : m0 + row) * ldo + c;
                if (vec && c + E <= a.N) {
                    if (a.stream) store_once(d, x);
                    else *reinterpret_cast<uint4*>(d) = x;
                } else {
                    V v[E];
                    __builtin_memcpy(v, &x, 16);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (c + e < a.N) d[e] = v[e];
                }
            }
            wave_sync();
        }
    };
    // the adapters of the tile's rows, one after the other (rows without one come last), KR ranks at a time
    if (EXPAND) {
        int g = first, p0 = 0, p1 = first_end, r0 = 0, buf = 0;
        while (g < a.G) {
            place(r0, buf);
            meet(false);  // this block has landed for every wave, and the one before has been read
            int g1 = g, q0 = p0, q1 = p1, r1 = r0 + KR;
            if (r1 >= a.R) {
                r1 = 0, q0 = p1;
                g1 = q0 < live ? __builtin_amdgcn_readfirstlane(sid[q0]) : a.G;
                if (g1 < a.G) q1 = __builtin_amdgcn_readfirstlane(ends[q0]);
            }
            if (g1 < a.G) fetch(g1, r1, buf ^ 1, [&](int r) { return rows[r]; });
            const uint4* st = lds + buf * BLOCK;
            const uint4* sw = st + PARTS * BM * 4;
#pragma unroll
            for (int ni = 0; ni < NN; ++ni) {
                fb[0][ni] = sw[(rb + ni * 16) * 4 + (fq ^ F(rb + ni * 16))];
                if constexpr (PARTS > 1) fb[1][ni] = finite(fb[0][ni]);  // here: between the products it spills 9 to 11 registers
            }
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) {
                const int r = ra + mi * 16;
                if (r - fr + 16 <= p0 || r - fr >= p1) continue;  // none of the 16 rows
                f32x4 x[NN];
#pragma unroll
                for (int ni = 0; ni < NN; ++ni) x[ni] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < PARTS; ++u) {
                    const uint4 h = st[(u * BM + r) * 4 + (fq ^ F(r))];
#pragma unroll
                    for (int ni = 0; ni < NN; ++ni) x[ni] = mma<T>(fb[u ? 1 : 0][ni], h, x[ni]);
                }
                if (r >= p0 && r < p1)
#pragma unroll
                    for (int ni = 0; ni < NN; ++ni) acc[mi][ni] += x[ni];
            }
            g = g1, p0 = q0, p1 = q1, r0 = r1, buf ^= 1;
        }
    }
    // lane: row ra + 16 mi, columns rb - fr + 16 ni + 4 fq + e
    __syncthreads();  // the buffers have been read by all
    if constexpr (EXPAND) store((O*)a.out, a.ldo, a.vec);
    else store(a.part + (int64_t)split * a.M * a.ldp, a.ldp, true);
}

template <typename T, typename O, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) gemm_kernel(GemmArgs a, Groups o) {
    __shared__ uint4 lds[5 * BM * 8];
    gemm_tile<T, O, BM, BN, WM, WN, true>(a, o, block_of_grid(), lds);
}


// ------------------------------------------------------------------------------------------
// Few rows (up to 64): everything is read once and little is computed, so the contraction is cut over the chip and
// joined, and what counts is how much is on its way. One launch forms the sums of both products over x:
//  * 128 rows of C by all rows over up to 8 lines (128 bytes) of the contraction: the rows' lines go to LDS directly, a line a wave,
//    each wave loads its 16 rows of C into registers, all at once, and everyone waits once;
//  * 16 KT ranks of one adapter by its rows (16 at a time) over a range of lines: the 8 waves take an eighth each and add up in LDS.
// Bound by reading C and the used adapters' down: 64 x 16384 -> 1024 with 38 of 64 adapters of rank 16 in use takes 18 us and reads 73 MB (4.1 TB/s),
// 54 of them C and down, the rest X, which each XCD reads whole for its eighth of C (17), and once more for the adapters. A second launch adds the
// ranges, in order, and expands: a lane four columns of one row. No sort: the rows of an adapter are found by comparing up to 64 ids, a
// lane an id. Replayed in a graph, against the launches of more rows: 21 and 26 us there, 10 and 15 us at 16 x 4096 -> 1024.
constexpr int kFewRows = 64, kFewWaves = 8, kFewLines = 8;
// of results up to the width that the join's grid (256 columns a block) can cover
bool few_rows(int64_t n, int64_t width) { return n <= kFewRows && width <= (int64_t)65535 * 256; }

struct FewArgs {
    const char *X, *C, *W;  // W: the bank contracted with x
    int64_t ldx, kp;        // bytes of a row of X, and of C and W
    int width;              // of a row of X
    int n, p, pp, G, R, c_blocks, c_lines, c_splits, r_blocks, r_splits;
    const int32_t* ids;
    float *part, *part_h;  // c_splits x n x pp (p padded to a multiple of 4), r_splits x n x R
};

// ODD: rows of X end inside a line, and begin anywhere: they are loaded into registers, without what lies behind their end. One more block
// groups the rows where the gradients of the banks are to come.
template <typename T, int NT, int KT, bool ODD>
__global__ void __launch_bounds__(64 * kFewWaves, 4) few_sums_kernel(FewArgs a, Groups o) {
    constexpr int XL = 16 * NT * 8;  // chunks of a line of all rows
    constexpr int E = 16 / (int)sizeof(T), LE = 128 / (int)sizeof(T);  // elements of a chunk, of a line
    __shared__ uint4 lds[kFewLines * (XL > KT * 64 ? XL : KT * 64)];
    __shared__ int members[17];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, q = lane >> 4;
    const int lines = (int)(a.kp / 128);
    int id = blockIdx.x;
    if (id == a.c_blocks * a.c_splits + a.n * a.r_blocks * a.r_splits) {
        group_few(a.ids, a.n, a.G, reinterpret_cast<int32_t*>(lds), o);
        return;
    }
    if (id < a.c_blocks * a.c_splits) {
        const int split = id / a.c_blocks, l0 = split * a.c_lines, count = min(a.c_lines, lines - l0), c0 = id % a.c_blocks * 128 + w * 16;
        if (w < count) {
            const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)reinterpret_cast<uintptr_t>(lds + w * XL));
            const int r = lane >> 3, ch = (lane & 7) ^ (r & 7);  // chunk ch of row r lies at r * 8 + (ch ^ (r & 7))
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                const char* row = a.X + min(i * 8 + r, a.n - 1) * a.ldx;
                if constexpr (ODD) {
                    lds[w * XL + i * 64 + lane] = load_of_row((const T*)row, (l0 + w) * LE + ch * E, a.width);
                    continue;
                }
                const char* from = row + (int64_t)(l0 + w) * 128 + ch * 16;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the clobber keeps the compiler's own uses safe
                asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to + (uint32_t)i * 1024u) : "memory", "m0");
#pragma clang diagnostic pop
            }
        }
        const char* pc = a.C + min(c0 + c, a.p - 1) * a.kp + (int64_t)l0 * 128 + q * 16;
        uint4 f[kFewLines][2];
#pragma unroll
        for (int l = 0; l < kFewLines; ++l)
            if (l < count)
#pragma unroll
                for (int h = 0; h < 2; ++h) f[l][h] = *reinterpret_cast<const uint4*>(pc + l * 128 + h * 64);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the wave's line of x has landed too
        __syncthreads();
        f32x4 acc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int l = 0; l < kFewLines; ++l) {
            if (l >= count) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[j] = mma<T>(f[l][h], lds[l * XL + (j * 16 + c) * 8 + ((4 * h + q) ^ (c & 7))], acc[j]);
        }
        const int col = c0 + 4 * q;
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (j * 16 + c < a.n && col < a.pp)
                *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.n + j * 16 + c) * a.pp + col) = acc[j];
        return;
    }
    id -= a.c_blocks * a.c_splits;
    const int split = id % a.r_splits, k = id / a.r_splits, row = k / a.r_blocks, r0 = k % a.r_blocks * 16 * KT;
    const int g = lane < a.n ? group_of(a.ids[lane], a.G) : a.G, mine = __builtin_amdgcn_readlane(g, row);
    if (mine == a.G) return;
    const uint64_t same = __ballot(g == mine);
    const int before = __popcll(same & ((1ull << row) - 1)), at = __popcll(same & ((1ull << lane) - 1)) - before;
    if (before % 16) return;  // the block of an earlier row takes this one
    if (w == 0) {
        if ((same >> lane & 1) && at >= 0 && at < 16) members[at] = lane;
        if (lane == 0) members[16] = min(16, (int)__popcll(same) - before);
    }
    __syncthreads();
    const int count = members[16];
    const char *pa[KT], *pb = a.X + members[min(c, count - 1)] * a.ldx;
#pragma unroll
    for (int i = 0; i < KT; ++i) pa[i] = a.W + ((int64_t)mine * a.R + min(r0 + i * 16 + c, a.R - 1)) * a.kp + q * 16;
    const int l0 = (int)((int64_t)lines * split / a.r_splits), l1 = (int)((int64_t)lines * (split + 1) / a.r_splits);
    f32x4 acc[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto add = [&](int l, auto count_of_lines) {
        constexpr int N = decltype(count_of_lines)::value * 2;  // half lines
        uint4 fa[N][KT], fb[N];
#pragma unroll
        for (int h = 0; h < N; ++h) {
            // four lines: all inside the row
            if constexpr (ODD && N == 2) fb[h] = load_of_row((const T*)pb, l * LE + h * 4 * E + q * E, a.width);
            else if constexpr (ODD) __builtin_memcpy(&fb[h], (const T*)pb + l * LE + h * 4 * E + q * E, 16);
            else fb[h] = *reinterpret_cast<const uint4*>(pb + (int64_t)l * 128 + h * 64 + q * 16);
#pragma unroll
            for (int i = 0; i < KT; ++i) fa[h][i] = *reinterpret_cast<const uint4*>(pa[i] + (int64_t)l * 128 + h * 64);
        }
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
            for (int i = 0; i < KT; ++i) acc[i] = mma<T>(fa[h][i], fb[h], acc[i]);
    };
    const int each = (l1 - l0 + kFewWaves - 1) / kFewWaves, e1 = min(l1, l0 + (w + 1) * each);
    int l = l0 + w * each;
    for (const int inside = ODD ? min(e1, a.width / LE) : e1; l + 4 <= inside; l += 4) add(l, std::integral_constant<int, 4>{});
    for (; l < e1; ++l) add(l, std::integral_constant<int, 1>{});
    f32x4(*red)[KT][64] = reinterpret_cast<f32x4(*)[KT][64]>(lds);
#pragma unroll
    for (int i = 0; i < KT; ++i) red[w][i][lane] = acc[i];
    __syncthreads();
    if (w >= KT || c >= count) return;
    f32x4 x = red[0][w][lane];
#pragma unroll
    for (int i = 1; i < kFewWaves; ++i) x += red[i][w][lane];
    const int r = r0 + w * 16 + 4 * q;
    float* h = a.part_h + ((int64_t)split * a.n + members[c]) * a.R + r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r + e < a.R) h[e] = x[e];
}

template <typename T, typename O>
__global__ void __launch_bounds__(64)
few_join_kernel(FewArgs a, const T* __restrict__ up, int64_t wp, const float* __restrict__ scale, O* __restrict__ Y, int64_t ldy,
                float* __restrict__ hidden) {
    __shared__ float h[kMaxRank];
    const int row = blockIdx.x, lane = threadIdx.x, g = group_of(a.ids[row], a.G);
    const int col = (blockIdx.y * 64 + lane) * 4;
    f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
    if (col < a.pp)
#pragma unroll 8
        for (int k = 0; k < a.c_splits; ++k) y += *reinterpret_cast<const f32x4*>(a.part + ((int64_t)k * a.n + row) * a.pp + col);
    if (g < a.G || hidden) {
        const float s = g < a.G && scale ? scale[g] : 1.f;
        for (int r = lane; r < a.R; r += 64) {
            float x = 0.f;
            if (g < a.G)
#pragma unroll 4
                for (int k = 0; k < a.r_splits; ++k) x += a.part_h[((int64_t)k * a.n + row) * a.R + r];
            h[r] = x * s;
            if (hidden && blockIdx.y == 0) hidden[(int64_t)row * a.R + r] = x;
        }
    }
    __syncthreads();
    if (col >= a.p) return;
    if (g < a.G) {
        const T* __restrict__ u = up + (int64_t)g * a.R * wp + col;  // columns up to the padded width are there
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int r = 0; r < a.R; ++r) {
            f32x4 v;
            if constexpr (sizeof(T) == 2) {
                const uint2 b = *reinterpret_cast<const uint2*>(u + r * wp);
                v = f32x4{__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                          __uint_as_float(b.y & 0xffff0000u)};
            } else {
                v = *reinterpret_cast<const f32x4*>(u + r * wp);
            }
            const float f = h[r];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(f, v[e], x[e]);
        }
        y += x;
    }
    O* d = Y + row * ldy + col;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < a.p) store_as(d + e, y[e]);
}

// ------------------------------------------------------------------------------------------
// Some rows (over 64, but too few tiles for the chip): the product over splits of the contraction and, in blocks of the same launch, the
// shrink over ranges of it, since neither needs the other; few_join_kernel adds both up and expands.
template <typename T, int KT, int BN>
__global__ void __launch_bounds__(256, 2) some_sums_kernel(GemmArgs g, ShrinkArgs s, Groups o, float* part_h, int r_blocks, int r_splits, int64_t n) {
    __shared__ uint4 lds[5 * 128 * 8];
    const unsigned products = g.per_xcd * 8;
    if (blockIdx.x < products) {
        gemm_tile<T, float, 128, BN, BN == 128 ? 2 : 4, BN == 128 ? 2 : 1, false>(g, o, blockIdx.x, lds);
        return;
    }
    const int id = (int)(blockIdx.x - products), split = id % r_splits, k = id / r_splits, r0 = k % r_blocks * 16 * KT;
    if (k / r_blocks >= o.number[0]) return;
    const int4 tile = o.tiles[k / r_blocks];
    if (tile.x == s.G) return;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, q = lane >> 4;
    const char* z = reinterpret_cast<const char*>((const T*)s.Z + o.perm[tile.y + min(c, tile.z - 1)] * s.ldz) + q * 16;
    const char* b[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j)
        b[j] = reinterpret_cast<const char*>((const T*)s.W + ((int64_t)tile.x * s.R + min(r0 + j * 16 + c, s.R - 1)) * s.kp) + q * 16;
    const int lines = (int)(s.kp * (int64_t)sizeof(T) / 128);
    const int l0 = (int)((int64_t)lines * split / r_splits), l1 = (int)((int64_t)lines * (split + 1) / r_splits), each = (l1 - l0 + 3) / 4;
    const int e1 = min(l1, l0 + (w + 1) * each);
    f32x4 acc[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto add = [&](int l, auto count_of_lines) {
        constexpr int N = decltype(count_of_lines)::value * 2;  // half lines
        uint4 zf[N], bf[N][KT];
#pragma unroll
        for (int h = 0; h < N; ++h) {
            zf[h] = *reinterpret_cast<const uint4*>(z + (int64_t)l * 128 + h * 64);
#pragma unroll
            for (int j = 0; j < KT; ++j) bf[h][j] = *reinterpret_cast<const uint4*>(b[j] + (int64_t)l * 128 + h * 64);
        }
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
            for (int j = 0; j < KT; ++j) acc[j] = mma<T>(bf[h][j], zf[h], acc[j]);
    };
    int l = l0 + w * each;
    for (; l + 4 <= e1; l += 4) add(l, std::integral_constant<int, 4>{});
    for (; l < e1; ++l) add(l, std::integral_constant<int, 1>{});
    f32x4(*red)[KT][64] = reinterpret_cast<f32x4(*)[KT][64]>(lds);
#pragma unroll
    for (int j = 0; j < KT; ++j) red[w][j][lane] = acc[j];
    __syncthreads();
    if (w >= KT || c >= tile.z) return;
    const f32x4 x = red[0][w][lane] + red[1][w][lane] + red[2][w][lane] + red[3][w][lane];
    const int r = r0 + w * 16 + 4 * q;
    float* h = part_h + (split * n + o.perm[tile.y + c]) * s.R + r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r + e < s.R) h[e] = x[e];
}

int64_t padded(int64_t w, int32_t dtype) {
    const int64_t step = dtype == RP_BF16 ? 64 : 32;
    return (w + step - 1) / step * step;
}

// the arguments both directions share
int check_shared(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t G, int32_t R) {
    if (dtype != RP_F32 && dtype != RP_BF16) return fail(RP_ERR_INVALID, "dtype must be RP_F32 or RP_BF16");
    if (n < 0 || m <= 0 || p <= 0 || G <= 0 || R <= 0) return fail(RP_ERR_INVALID, "bad shape");
    if (R > kMaxRank) return fail(RP_ERR_UNSUPPORTED, "rank %d is over %d", (int)R, kMaxRank);
    if (n > INT32_MAX || m > INT32_MAX - 512 || p > INT32_MAX - 512 || G > kMaxAdapters)
        return fail(RP_ERR_UNSUPPORTED, "n, m, p or the number of adapters too large");
    return RP_OK;
}

int check_operand(const char* name, const void* p, int64_t ld, int64_t width, int32_t dtype) {
    if (!p) return fail(RP_ERR_INVALID, "NULL %s", name);
    if (ld < width) return fail(RP_ERR_INVALID, "%s: row stride %lld is under its width %lld", name, (long long)ld,
                                (long long)width);
    if (((uintptr_t)p & 15) || (ld * (dtype == RP_BF16 ? 2 : 4)) % 16)
        return fail(RP_ERR_INVALID, "%s must have 16-byte aligned rows", name);
    return RP_OK;
}

// rows that are copied to padded ones first may lie anywhere
int check_rows(const char* name, const void* p, int64_t ld, int64_t width, int32_t dtype) {
    if (padded(width, dtype) == width) return check_operand(name, p, ld, width, dtype);
    if (!p) return fail(RP_ERR_INVALID, "NULL %s", name);
    if (ld < width || ((uintptr_t)p & (dtype == RP_BF16 ? 1 : 3)))
        return fail(RP_ERR_INVALID, "%s: row stride under its width, or not aligned to its elements", name);
    return RP_OK;
}

// a product with its expand for few rows: O (n x p) = X C^T + the adapters' part, hidden = the rows' H or NULL (p = 0: H alone)
struct FewCut {
    int c_blocks, c_lines, c_splits, r_blocks, r_splits;
};
FewCut few_cut(int64_t n, int64_t p, int R, int64_t line_bytes) {
    FewCut f;
    const int64_t lines = line_bytes / 128;
    f.c_blocks = (int)((p + 127) / 128), f.r_blocks = (R + (R <= 16 ? 15 : 31)) / (R <= 16 ? 16 : 32);
    // 8 lines a block, fewer where that leaves under 256 blocks; an adapter's lines over about 512 blocks, none with less than two a wave
    f.c_lines = (int)std::max<int64_t>(2, std::min<int64_t>(kFewLines, lines * f.c_blocks / 256));
    f.c_splits = p ? (int)((lines + f.c_lines - 1) / f.c_lines) : 0;
    f.r_splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(1, n * f.r_blocks), lines / (2 * kFewWaves), 16}));
    return f;
}
size_t few_bytes(int64_t n, int64_t p, int R, int64_t line_bytes) {
    const FewCut f = few_cut(n, p, R, line_bytes);
    return ((size_t)4 * n * ((size_t)f.c_splits * ((p + 3) / 4 * 4) + (size_t)f.r_splits * R) + 255) & ~(size_t)255;
}
int64_t few_blocks(const FewCut& f, int64_t n) { return (int64_t)f.c_blocks * f.c_splits + n * f.r_blocks * f.r_splits; }

template <typename T, typename O>
int launch_few(const T* X, int64_t ldx, int64_t width, const T* C, int64_t kp, int64_t n, int64_t p, const T* W, const T* U, int64_t wp, int G, int R,
               const float* scale, const int32_t* ids, const Groups* groups, O* out, int64_t ldo, float* hidden, char* ws, hipStream_t st) {
    constexpr int64_t es = sizeof(T);
    FewArgs a{};
    a.X = (const char*)X, a.C = (const char*)C, a.W = (const char*)W, a.ldx = ldx * es, a.kp = kp * es, a.width = (int)width;
    a.n = (int)n, a.p = (int)p, a.pp = (int)((p + 3) / 4 * 4), a.G = G, a.R = R, a.ids = ids;
    const FewCut f = few_cut(n, p, R, a.kp);
    a.c_blocks = f.c_blocks, a.c_lines = f.c_lines, a.c_splits = f.c_splits, a.r_blocks = f.r_blocks, a.r_splits = f.r_splits;
    a.part = (float*)ws, a.part_h = a.part + (int64_t)a.c_splits * n * a.pp;
    const Groups o = groups ? *groups : Groups{};
    const dim3 grid((unsigned)(few_blocks(f, n) + (groups ? 1 : 0))), block(64 * kFewWaves);
    const int nt = n <= 16 ? 1 : n <= 32 ? 2 : 4;
    const auto launch = [&](auto k_tiles, auto odd) {
        constexpr int KT = decltype(k_tiles)::value;
        constexpr bool ODD = decltype(odd)::value;
        if (nt == 1) hipLaunchKernelGGL((few_sums_kernel<T, 1, KT, ODD>), grid, block, 0, st, a, o);
        else if (nt == 2) hipLaunchKernelGGL((few_sums_kernel<T, 2, KT, ODD>), grid, block, 0, st, a, o);
        else hipLaunchKernelGGL((few_sums_kernel<T, 4, KT, ODD>), grid, block, 0, st, a, o);
    };
    using std::integral_constant, std::true_type, std::false_type;
    if (R <= 16) kp == width ? launch(integral_constant<int, 1>{}, false_type{}) : launch(integral_constant<int, 1>{}, true_type{});
    else kp == width ? launch(integral_constant<int, 2>{}, false_type{}) : launch(integral_constant<int, 2>{}, true_type{});
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((few_join_kernel<T, O>), dim3((unsigned)n, (unsigned)std::max<int64_t>(1, (p + 255) / 256)), dim3(64), 0, st, a, U, wp,
                       scale, out, ldo, hidden);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

// Everything a call lays out in its workspace and launches, from its sizes alone.
struct Plan {
    int bits, tile_rows, chunk_rows, kt;  // kt: shrink's rank tiles (1, 2, 4 or 8)
    bool small;                                  // one block groups the rows
    bool some;                                   // too few tiles for the chip (Tiling::few)
    int64_t each;                                // else rows of a wave that counts
    int n_chunks;
    int64_t max_tiles, max_chunks, max_parts;
    size_t perm, sid, start, tiles, chunks, tile0, chunk0, multi0, number, hist, pieces, t, part, shrink, pad_x, pad_dy, bytes;
};

// Tiles of a product: 128 x 128, two on a compute unit, or 256 x 256, one. What a round of 256 units takes, in twentieths of a small tile's
// time beside another: 40 for two small tiles a unit, 25 for one (20 in f32, where the matrix instructions alone bind), 60 for a large
// one (76). The cheaper kind is taken. Whole calls in us, small and large: bf16, rank 64, from 4096 to 4096: 103 and 129 at 1777 rows, 141
// and 132 at 2304, 220 and 242 at 5000; f32, rank 8 and 16: 415 and 520 at 3000 x 2000 -> 2900, 2098 and 2010 at 8192 x 4096 -> 4096.
// Results of up to 64 columns take tiles of 128 x 64: 24203 x 2368 -> 21 in f32 131 us, 199 with 128 x 128; -> 64 in bf16 70 and 74.
// Small tiles that leave much of the chip idle are split over the contraction (`few`), for up to 512 blocks of 8 stages and more (256 of
// 2 in f32, where two on a unit take twice as long: 27 and 31 us of sums at 1003 x 4001 -> 200), and the adapters' part is left to the
// join: where the part of the time that is idle (0.6 us a stage for a block alone, 1.75 in f32) is more than the partial sums take.
// Whole and split: 61 and 45 us at 2100 x 4096 -> 1024, 66 and 69 at 3900 rows, 29 and 37 at 3900 x 512, 38 and 28 at 300 x 2000 -> 2900;
// f32 279 and 40 at 1003 x 4001 -> 200, 94 and 100 at 3900 x 1024 -> 1024.
struct Tiling {
    bool big, narrow, few;
    unsigned m_tiles, n_tiles, splits;
};
Tiling tiling(int64_t M, int64_t N, int64_t row_bytes, int es) {
    Tiling t;
    const auto tiles_of = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
    const int64_t left = tiles_of(128) % 512;
    const int64_t small = tiles_of(128) / 512 * 40 + (left > 256 ? 40 : left == 0 ? 0 : es == 2 ? 25 : 20);
    t.big = N > 64 && (tiles_of(256) + 255) / 256 * (es == 2 ? 60 : 76) < small;
    const int64_t b = t.big ? 256 : 128, tiles = std::max<int64_t>(1, tiles_of(b)), stages = row_bytes / 128;
    t.narrow = !t.big && N <= 64;
    t.m_tiles = (unsigned)((M + b - 1) / b), t.n_tiles = (unsigned)((N + b - 1) / b);
    const int64_t splits = es == 2 ? std::min<int64_t>({512 / tiles, stages / 8, 16}) : std::min<int64_t>({256 / tiles, stages / 2, 32});
    t.splits = (unsigned)std::max<int64_t>(1, splits);
    const double idle = 1 - (double)tiles / (es == 2 ? 320 : 256);  // in bf16 two blocks on a unit have 1.25 times the rate of one
    t.few = !t.big && (double)stages * (es == 2 ? 0.6 : 1.75) * (t.narrow ? 0.5 : 1) * idle > 0.028 * (double)(tiles * t.splits);
    if (!t.few) t.splits = 1;
    return t;
}

// the shrink beside a split product: about 512 blocks, none with less than two lines a wave
struct SomeCut {
    int r_blocks, r_splits;
};
SomeCut some_cut(int64_t tiles, int R, int64_t row_bytes) {
    SomeCut c;
    c.r_blocks = (R + (R <= 16 ? 15 : 31)) / (R <= 16 ? 16 : 32);
    c.r_splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(1, tiles * c.r_blocks), row_bytes / 128 / 8, 16}));
    return c;
}
size_t some_bytes(const Tiling& t, int64_t tiles, int64_t n, int64_t p, int R, int64_t row_bytes) {
    return (size_t)4 * n * ((size_t)t.splits * ((p + 3) / 4 * 4) + (size_t)some_cut(tiles, R, row_bytes).r_splits * R);
}

// of the shrink of few rows: about 1024 blocks, none with less than two lines a wave (whole calls of 1777 x 4096 -> 4096 and 4000 x 16384 ->
// 1024: 103 and 196 us, 104 and 203 unsplit)
int shrink_splits(int64_t tiles, int64_t row_bytes) {
    return (int)std::max<int64_t>(1, std::min<int64_t>({1024 / std::max<int64_t>(1, tiles), row_bytes / 128 / 8, 32}));
}

Plan plan_for(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t G, int R, int what) {
    Plan l;
    const int es = dtype == RP_BF16 ? 2 : 4;
    const int64_t mk = padded(m, dtype), pk = padded(p, dtype);
    l.bits = 1;
    while ((G >> l.bits) != 0) ++l.bits;
    l.kt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
    const int rt = l.kt <= 4 ? 4 : 2;
    Tiling g = what == RP_ADAPT_PROJECT ? tiling(n, p, mk * es, es) : tiling(n, m, pk * es, es);
    l.some = g.few;
    // many rows: as many of them as registers hold under one read of the adapter (65536 x 16384 -> 1024: 2.06 ms, 2.16 with 16); few: 16,
    // for more blocks (16384 x 4096: 164 us, 172 with 64), and beside a split product, whose blocks take 16
    const bool many = n >= 512 * 16 * rt && !l.some;
    l.tile_rows = many ? 16 * rt : 16;
    // chunks of rows for the banks' gradients: long, unless that leaves under 2048 blocks (16384 x 16384, 16 adapters: the partial sums
    // joined in 11 us, 17 with 512 rows)
    l.chunk_rows = (int)std::max<int64_t>(512, std::min<int64_t>(kMaxChunk, n * ((m + 127) / 128) / 2048 / 64 * 64));
    l.small = n <= kSmallRows && G <= 700;
    // rows of a wave: 256 at least, which is fewer than 128 waves under 32768 rows, then 128 waves and more, of up to 2048 rows, unless the
    // counts to scan become more than a million (4 million rows, 32 adapters: 0.10 ms, 0.70 with 128 waves)
    l.each = std::min<int64_t>(2048, std::max<int64_t>(256, (n / 128 + 63) / 64 * 64));
    while ((n + l.each - 1) / l.each * (G + 1) > (1 << 20)) l.each *= 2;
    l.n_chunks = l.small ? 0 : (int)std::max<int64_t>(1, (n + l.each - 1) / l.each);  // one without rows too: the lists come from its counts
    l.max_tiles = n / l.tile_rows + std::min(n, G + 1);
    l.max_chunks = n / l.chunk_rows + G;
    l.max_parts = 2 * (n / l.chunk_rows);
    size_t at = 0;
    const auto take = [&](size_t b) {
        const size_t r = at;
        at = (at + b + 255) & ~(size_t)255;
        return r;
    };
    l.perm = take(4 * n), l.sid = take(4 * n), l.start = take(4 * (G + 2));
    l.tiles = take(16 * l.max_tiles), l.chunks = take(16 * l.max_chunks);
    l.tile0 = take(4 * (G + 1)), l.chunk0 = take(4 * (G + 1)), l.multi0 = take(4 * (G + 1)), l.number = take(8);
    l.hist = take((size_t)4 * l.n_chunks * (G + 1));
    l.t = l.part = at;
    // the rows' factors, for the products that have an expand
    const size_t factors = (size_t)n * (dtype == RP_BF16 ? 3 : 1) * padded_rank(R, es) * es;
    l.pieces = take(what == RP_ADAPT_GRADIENTS ? 0 : factors);
    if (what == RP_ADAPT_PROJECT) {
        l.part = take(l.some ? some_bytes(g, l.max_tiles, n, p, R, mk * es) : 0);
    } else {
        l.t = take((size_t)4 * n * R);
        size_t part = (size_t)4 * l.max_parts * R * (mk + pk);
        // with or without dX, t is summed in one order: the banks' gradients are the same bits
        if (what != RP_ADAPT_GRADIENTS_DX) g.splits = 0;
        if (l.some) part = std::max(part, some_bytes(g, l.max_tiles, n, m, R, pk * es));
        if (few_rows(n, m)) part = std::max(part, few_bytes(n, what == RP_ADAPT_GRADIENTS_DX ? m : 0, R, pk * es));
        l.part = take(part);
    }
    const int splits = l.tile_rows > 16 ? 1 : shrink_splits(l.max_tiles, (what == RP_ADAPT_PROJECT ? mk : pk) * es);
    l.shrink = take(splits > 1 ? (size_t)splits * l.max_tiles * l.kt * 1024 : 0);
    l.pad_x = take(mk != m && (what == RP_ADAPT_PROJECT || m < 16 / es) ? (size_t)n * mk * es : 0);  // for the gradients only if narrow
    l.pad_dy = take(what != RP_ADAPT_PROJECT && pk != p ? (size_t)n * pk * es : 0);
    l.bytes = at;
    return l;
}

Groups groups_of(const Plan& l, char* ws) {
    Groups o;
    o.perm = (int32_t*)(ws + l.perm), o.sid = (int32_t*)(ws + l.sid), o.start = (int32_t*)(ws + l.start);
    o.tiles = (int4*)(ws + l.tiles), o.chunks = (int4*)(ws + l.chunks);
    o.tile0 = (int32_t*)(ws + l.tile0), o.chunk0 = (int32_t*)(ws + l.chunk0), o.multi0 = (int32_t*)(ws + l.multi0);
    o.number = (int32_t*)(ws + l.number), o.hist = (int32_t*)(ws + l.hist);
    return o;
}

// X as the kernels read it: itself, or a padded copy made by the call's first launch
template <typename T>
Pad pad_of(const T*& X, int64_t& ldx, int64_t n, int64_t width, void* to) {
    Pad p{};
    const int64_t kp = padded(width, sizeof(T) == 2 ? RP_BF16 : RP_F32);
    if (kp == width || n == 0) return p;
    p = Pad{X, to, ldx, n, (int)width, (int)kp, (int)sizeof(T)};
    X = (const T*)to, ldx = kp;
    return p;
}
unsigned pad_blocks(const Pad& p, const Pad& q, int threads) {
    const auto need = [&](const Pad& x) {
        const int each = pad_threads((int64_t)x.padded * x.size / 16, threads);
        return x.to ? (x.rows + threads / each - 1) / (threads / each) : 0;
    };
    return (unsigned)std::min<int64_t>(std::max(need(p), need(q)), 2048);
}

int launch_groups(const Plan& l, const Groups& o, const int32_t* ids, int64_t n, int G, const Pad& p, const Pad& q, hipStream_t st) {
    if (l.small) {
        const unsigned waves = n <= 256 ? 4 : 16;
        const size_t lds = 4 * ((waves + 4) * (G + 1) + 1);
        hipLaunchKernelGGL(group_small_kernel, dim3(1 + pad_blocks(p, q, (int)waves * 64)), dim3(64 * waves), lds, st, ids,
                           (int)n, G, l.bits, l.tile_rows, l.chunk_rows, o, p, q);
    } else {
        if (const unsigned blocks = pad_blocks(p, q, 256)) {
            hipLaunchKernelGGL(pad_kernel, dim3(blocks), dim3(256), 0, st, p, q);
            HIP_TRY(hipGetLastError());
        }
        const int waves = G < 4000 ? 4 : 1;
        const dim3 grid((unsigned)((l.n_chunks + waves - 1) / waves)), block(64 * waves);
        const size_t lds = (size_t)4 * waves * (G + 1);
        hipLaunchKernelGGL(group_count_kernel, grid, block, lds, st, ids, n, G, l.bits, l.each, l.n_chunks, o);
        HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(group_scan_kernel, dim3(1), dim3(1024), 0, st, n, G, l.n_chunks, l.tile_rows, l.chunk_rows, o);
        HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(group_place_kernel, grid, block, lds, st, ids, n, G, l.bits, l.each, l.n_chunks, o);
    }
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

template <typename T>
int launch_shrink(const Plan& l, const ShrinkArgs& a, const Groups& o, hipStream_t st) {
    if (l.tile_rows > 16) {
        const dim3 grid((unsigned)l.max_tiles), block(256);
        if (l.kt == 1) hipLaunchKernelGGL((shrink_kernel<T, 4, 1>), grid, block, 0, st, a, o);
        else if (l.kt == 2) hipLaunchKernelGGL((shrink_kernel<T, 4, 2>), grid, block, 0, st, a, o);
        else if (l.kt == 4) hipLaunchKernelGGL((shrink_kernel<T, 4, 4>), grid, block, 0, st, a, o);
        else hipLaunchKernelGGL((shrink_kernel<T, 2, 8>), grid, block, 0, st, a, o);
        HIP_TRY(hipGetLastError());
        return RP_OK;
    }
    const int splits = shrink_splits(l.max_tiles, a.kp * (int64_t)sizeof(T));
    const dim3 grid((unsigned)l.max_tiles, (unsigned)splits), block(256), tiles((unsigned)l.max_tiles), lanes(64 * l.kt);
    if (l.kt == 1) hipLaunchKernelGGL((shrink_kernel<T, 1, 1>), grid, block, 0, st, a, o);
    else if (l.kt == 2) hipLaunchKernelGGL((shrink_kernel<T, 1, 2>), grid, block, 0, st, a, o);
    else if (l.kt == 4) hipLaunchKernelGGL((shrink_kernel<T, 1, 4>), grid, block, 0, st, a, o);
    else hipLaunchKernelGGL((shrink_kernel<T, 1, 8>), grid, block, 0, st, a, o);
    HIP_TRY(hipGetLastError());
    if (splits == 1) return RP_OK;
    if (l.kt == 1) hipLaunchKernelGGL((shrink_join_kernel<T, 1>), tiles, lanes, 0, st, a, o, splits);
    else if (l.kt == 2) hipLaunchKernelGGL((shrink_join_kernel<T, 2>), tiles, lanes, 0, st, a, o, splits);
    else if (l.kt == 4) hipLaunchKernelGGL((shrink_join_kernel<T, 4>), tiles, lanes, 0, st, a, o, splits);
    else hipLaunchKernelGGL((shrink_join_kernel<T, 8>), tiles, lanes, 0, st, a, o, splits);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

int64_t outer_columns(int64_t q, int es) { return (q + 256 / es - 1) / (256 / es); }  // blocks of 128 (bf16) or 64 columns

template <typename T>
int launch_outer(const Plan& l, const OuterArgs& a, const OuterArgs& b, const Groups& o, int64_t n, int G, hipStream_t st) {
    const int64_t qa = outer_columns(a.q, sizeof(T)), qb = outer_columns(b.q, sizeof(T)), blocks = (qa + qb) * l.max_chunks;
    const int kt = a.R <= 16 ? 1 : a.R <= 32 ? 2 : 4;
    const dim3 grid = grid_of(blocks, (unsigned)((a.R + 16 * kt - 1) / (16 * kt))), block(256);
    if (kt == 1) hipLaunchKernelGGL((outer_kernel<T, 1>), grid, block, 0, st, a, b, (int)qa, (int)(qa + qb), o);
    else if (kt == 2) hipLaunchKernelGGL((outer_kernel<T, 2>), grid, block, 0, st, a, b, (int)qa, (int)(qa + qb), o);
    else hipLaunchKernelGGL((outer_kernel<T, 4>), grid, block, 0, st, a, b, (int)qa, (int)(qa + qb), o);
    HIP_TRY(hipGetLastError());
    if (n > l.chunk_rows) {  // else no adapter has two chunks
        const unsigned ja = (unsigned)((a.q + 255) / 256), jb = (unsigned)((b.q + 255) / 256);
        hipLaunchKernelGGL(outer_join_kernel, dim3(ja + jb, (unsigned)a.R, (unsigned)G), dim3(256), 0, st, a, b, (int)ja, o, l.chunk_rows);
        HIP_TRY(hipGetLastError());
    }
    return RP_OK;
}

int64_t tiles_per_xcd(const Tiling& t) { return ((int64_t)t.m_tiles * t.n_tiles * t.splits + 7) / 8; }
void place_tiles(GemmArgs& a, const Tiling& t) {
    a.m_tiles = t.m_tiles, a.n_tiles = t.n_tiles, a.splits = t.splits, a.per_xcd = (unsigned)tiles_per_xcd(t);
}

template <typename T, typename O>
int launch_gemm(GemmArgs a, const Groups& o, hipStream_t st) {
    const Tiling t = tiling(a.M, a.N, (int64_t)a.steps * 128, sizeof(T));
    place_tiles(a, t);
    const dim3 grid = grid_of((int64_t)a.per_xcd * 8);
    if (t.big) hipLaunchKernelGGL((gemm_kernel<T, O, 256, 256, 2, 4>), grid, dim3(512), 0, st, a, o);
    else if (t.narrow) hipLaunchKernelGGL((gemm_kernel<T, O, 128, 64, 4, 1>), grid, dim3(256), 0, st, a, o);
    else hipLaunchKernelGGL((gemm_kernel<T, O, 128, 128, 2, 2>), grid, dim3(256), 0, st, a, o);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

template <typename T, typename O>
GemmArgs gemm_args(const T* A, int64_t lda, const T* B, int64_t kp, int64_t M, int64_t N, O* out, int64_t ldo, const char* S,
                   const T* W, int64_t wp, int G, int R, void* part) {
    GemmArgs a{};
    a.A = (const char*)A, a.B = (const char*)B, a.lda = lda * (int64_t)sizeof(T), a.ldb = kp * (int64_t)sizeof(T);
    a.M = M, a.N = (int)N, a.steps = (int)(kp * (int64_t)sizeof(T) / 128), a.out = out, a.ldo = ldo;
    a.vec = !((uintptr_t)out & 15) && ldo * sizeof(O) % 16 == 0;
    // beyond half of the 256 MB last-level cache: 537 MB of dX written through it cost the next pass's outer products 45 of 156 us
    a.stream = M * N * (int64_t)sizeof(O) > (128 << 20);
    a.S = S, a.W = (const char*)W, a.ldw = wp * (int64_t)sizeof(T), a.G = G, a.R = R, a.part = (float*)part;
    return a;
}

// the product and the shrink of some rows in one launch, then the join; H: without the scale, or NULL. p = 0: H alone.
template <typename T, typename O>
int launch_some(const Plan& l, const T* X, int64_t ldx, const T* C, int64_t kp, int64_t n, int64_t p, const T* W, const T* U, int64_t wp, int G,
                int R, const float* scale, const int32_t* ids, const Groups& o, O* out, int64_t ldo, float* H, char* ws, hipStream_t st) {
    GemmArgs g = gemm_args<T, float>(X, ldx, C, kp, n, p, (float*)nullptr, 0, nullptr, U, wp, G, R, ws);
    Tiling t = tiling(n, p, kp * (int64_t)sizeof(T), sizeof(T));
    if (!p) t.splits = 0;
    place_tiles(g, t);
    const SomeCut c = some_cut(l.max_tiles, R, kp * (int64_t)sizeof(T));
    g.ldp = (p + 3) / 4 * 4;
    float* part_h = g.part + t.splits * n * g.ldp;
    const ShrinkArgs s{X, ldx, kp, W, G, R, nullptr, nullptr, 0, nullptr, nullptr};
    const dim3 grid(g.per_xcd * 8 + (unsigned)(l.max_tiles * c.r_blocks * c.r_splits)), block(256);
    if (R <= 16 && t.narrow) hipLaunchKernelGGL((some_sums_kernel<T, 1, 64>), grid, block, 0, st, g, s, o, part_h, c.r_blocks, c.r_splits, n);
    else if (R <= 16) hipLaunchKernelGGL((some_sums_kernel<T, 1, 128>), grid, block, 0, st, g, s, o, part_h, c.r_blocks, c.r_splits, n);
    else if (t.narrow) hipLaunchKernelGGL((some_sums_kernel<T, 2, 64>), grid, block, 0, st, g, s, o, part_h, c.r_blocks, c.r_splits, n);
    else hipLaunchKernelGGL((some_sums_kernel<T, 2, 128>), grid, block, 0, st, g, s, o, part_h, c.r_blocks, c.r_splits, n);
    HIP_TRY(hipGetLastError());
    FewArgs a{};
    a.n = (int)n, a.p = (int)p, a.pp = (int)g.ldp, a.G = G, a.R = R, a.ids = ids;
    a.c_splits = (int)t.splits, a.r_splits = c.r_splits, a.part = g.part, a.part_h = part_h;
    hipLaunchKernelGGL((few_join_kernel<T, O>), dim3((unsigned)n, (unsigned)std::max<int64_t>(1, (p + 255) / 256)), dim3(64), 0, st, a, U, wp,
                       scale, out, ldo, H);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

// The arguments both directions share, and that each launch of the call fits: fewer than 2^31 blocks of the product and of the outer
// products, and of the others fewer than 2^32 threads.
int check_call(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t G, int32_t R, int what) {
    if (const int rc = check_shared(dtype, n, m, p, G, R)) return rc;
    if (what < RP_ADAPT_PROJECT || what > RP_ADAPT_GRADIENTS_DX) return fail(RP_ERR_INVALID, "what must be one of RP_ADAPT_*");
    const int es = dtype == RP_BF16 ? 2 : 4;
    const bool forward = what == RP_ADAPT_PROJECT;
    const int64_t width = forward ? p : m, made = what == RP_ADAPT_GRADIENTS ? 0 : width, row_bytes = padded(forward ? m : p, dtype) * es;
    const bool few = few_rows(n, width);
    int64_t outer = 0, product = 0, threads = 0;
    if (few) threads = (few_blocks(few_cut(n, made, R, row_bytes), n) + 1) * 64 * kFewWaves;
    if (!few || !forward) {
        const Plan l = plan_for(dtype, n, m, p, G, R, what);
        if (!forward) outer = (outer_columns(m, es) + outer_columns(p, es)) * l.max_chunks;
        if (!few) {
            const SomeCut c = some_cut(l.max_tiles, R, row_bytes);
            if (made) product = tiles_per_xcd(tiling(n, width, row_bytes, es)) * 8;
            threads = (l.some ? product + l.max_tiles * c.r_blocks * c.r_splits : l.max_tiles) * 256;
        }
    }
    if (std::max(outer, product) >= (int64_t)1 << 31 || threads >= (int64_t)1 << 32)
        return fail(RP_ERR_UNSUPPORTED, "too many rows, columns or adapters for one launch");
    return RP_OK;
}

int64_t workspace_of(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t G, int32_t R, int what) {
    if (what == RP_ADAPT_PROJECT && few_rows(n, p)) return (int64_t)few_bytes(n, p, R, padded(m, dtype) * (dtype == RP_BF16 ? 2 : 4));
    return (int64_t)plan_for(dtype, n, m, p, G, R, what).bytes;
}

template <typename T>
int project(const T* X, int64_t ldx, int64_t n, int64_t m, const T* C, int64_t p, const T* down, const T* up, int G, int R,
            const float* scale, const int32_t* ids, float* Y, int64_t ldy, float* hidden, char* ws, hipStream_t st) {
    constexpr int32_t dt = sizeof(T) == 2 ? RP_BF16 : RP_F32;
    const int64_t mk = padded(m, dt), pk = padded(p, dt);
    if (few_rows(n, p))
        return launch_few<T, float>(X, ldx, m, C, mk, n, p, down, up, pk, G, R, scale, ids, nullptr, Y, ldy, hidden, ws, st);
    const Plan l = plan_for(dt, n, m, p, G, R, RP_ADAPT_PROJECT);
    const Groups o = groups_of(l, ws);
    const Pad pad = pad_of(X, ldx, n, m, ws + l.pad_x);
    int rc = launch_groups(l, o, ids, n, G, pad, Pad{}, st);
    if (!rc && l.some)
        return launch_some<T, float>(l, X, ldx, C, mk, n, p, down, up, pk, G, R, scale, ids, o, Y, ldy, hidden, ws + l.part, st);
    if (!rc) rc = launch_shrink<T>(l, ShrinkArgs{X, ldx, mk, down, G, R, scale, hidden, 0, ws + l.pieces, (f32x4*)(ws + l.shrink)}, o, st);
    if (!rc) rc = launch_gemm<T, float>(gemm_args<T, float>(X, ldx, C, mk, n, p, Y, ldy, ws + l.pieces, up, pk, G, R, ws + l.part), o, st);
    return rc;
}

template <typename T>
OuterArgs outer_args(const T* Z, int64_t ldz, int64_t qp, int64_t q, int64_t wide, int R, const float* mul, const float* H, float* D, int64_t ldd,
                     int64_t sdd, char* part) {
    OuterArgs a{Z, ldz, qp, q, wide, R, mul, H, D, ldd, sdd, (float*)part, 0};
    a.vec = !((uintptr_t)D & 15) && ldd % 4 == 0 && sdd % 4 == 0;
    return a;
}

template <typename T>
int gradients(const T* dY, int64_t lddy, const T* X, int64_t ldx, int64_t n, int64_t m, int64_t p, const T* Ct, const T* down,
              const T* up, int G, int R, const float* scale, const int32_t* ids, const float* hidden, T* dX, int64_t lddx,
              float* d_down, int64_t ldd, int64_t sdd, float* d_up, int64_t ldu, int64_t sdu, char* ws, hipStream_t st) {
    constexpr int32_t dt = sizeof(T) == 2 ? RP_BF16 : RP_F32;
    const int64_t mk = padded(m, dt), pk = padded(p, dt);
    const Plan l = plan_for(dt, n, m, p, G, R, dX ? RP_ADAPT_GRADIENTS_DX : RP_ADAPT_GRADIENTS);
    const Groups o = groups_of(l, ws);
    float* t = (float*)(ws + l.t);
    const bool few = n && few_rows(n, m), some = n && !few && l.some, bare = few || some || n == 0;
    // The outer products take rows of any alignment, and so do the few rows' sums: X is copied only if narrower than a lane's load, dY
    // for the products of more rows. 7981 x 15997 in bf16, all launches: 92 us, 162 with a padded copy of X.
    constexpr int64_t lane = 16 / sizeof(T);
    const Pad px = m < lane ? pad_of(X, ldx, n, m, ws + l.pad_x) : Pad{};
    const Pad py = p < lane || !few ? pad_of(dY, lddy, n, p, ws + l.pad_dy) : Pad{};
    const int64_t dy_wide = py.to ? pk : p;
    int rc = RP_OK;
    // with few rows, or some, t holds up dy without the scale, which the outer product takes on
    if (few) {
        if (px.to || py.to) {
            hipLaunchKernelGGL(pad_kernel, dim3(pad_blocks(px, py, 256)), dim3(256), 0, st, px, py);
            HIP_TRY(hipGetLastError());
        }
        rc = launch_few<T, T>(dY, lddy, dy_wide, Ct, pk, n, dX ? m : 0, up, down, mk, G, R, scale, ids, &o, dX, lddx, t, ws + l.part, st);
    } else {
        rc = launch_groups(l, o, ids, n, G, px, py, st);
    }
    if (!rc && some)
        rc = launch_some<T, T>(l, dY, lddy, Ct, pk, n, dX ? m : 0, up, down, mk, G, R, scale, ids, o, dX, lddx, t, ws + l.part, st);
    if (!rc && !bare) rc = launch_shrink<T>(l, ShrinkArgs{dY, lddy, pk, up, G, R, scale, t, 1, dX ? ws + l.pieces : nullptr,
                                                                   (f32x4*)(ws + l.shrink)}, o, st);
    if (!rc) {
        const OuterArgs a = outer_args<T>(X, ldx, mk, m, px.to ? mk : m, R, bare ? scale : nullptr, t, d_down, ldd, sdd, ws + l.part);
        const OuterArgs b = outer_args<T>(dY, lddy, pk, p, dy_wide, R, scale, hidden, d_up, ldu, sdu, ws + l.part + 4 * l.max_parts * R * mk);
        rc = launch_outer<T>(l, a, b, o, n, G, st);
    }
    if (!rc && dX && !bare)
        rc = launch_gemm<T, T>(gemm_args<T, T>(dY, lddy, Ct, pk, n, m, dX, lddx, ws + l.pieces, down, mk, G, R, ws + l.part), o, st);
    return rc;
}

}  // namespace

extern "C" {

int64_t rp_adapt_workspace_bytes(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t adapters, int32_t rank,
                                 int32_t what) {
    if (check_call(dtype, n, m, p, adapters, rank, what)) return -1;
    return workspace_of(dtype, n, m, p, adapters, rank, what);
}

int rp_adapt_project_device(int device, const void* X, int64_t ldx, int32_t dtype, int64_t n, int64_t m, const void* C,
                            int64_t p, const void* down, const void* up, int64_t adapters, int32_t rank, const float* scale,
                            const int32_t* ids, float* Y, int64_t ldy, float* hidden, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    int rc = check_call(dtype, n, m, p, adapters, rank, RP_ADAPT_PROJECT);
    if (rc) return rc;
    const int64_t mk = padded(m, dtype), pk = padded(p, dtype);
    if ((rc = check_rows("X", X, ldx, m, dtype)) || (rc = check_operand("C", C, mk, mk, dtype)) ||
        (rc = check_operand("down", down, mk, mk, dtype)) || (rc = check_operand("up", up, pk, pk, dtype)))
        return rc;
    if (!ids || !Y) return fail(RP_ERR_INVALID, "NULL ids or Y");
    if (ldy < p) return fail(RP_ERR_INVALID, "Y: row stride %lld is under p=%lld", (long long)ldy, (long long)p);
    if (n == 0) return RP_OK;
    const int64_t need = workspace_of(dtype, n, m, p, adapters, rank, RP_ADAPT_PROJECT);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need)
        return fail(RP_ERR_INVALID, "workspace must be 256-byte aligned and hold %lld bytes", (long long)need);
    DeviceGuard guard;
    if ((rc = guard.enter(device))) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RP_BF16)
        return project<uint16_t>((const uint16_t*)X, ldx, n, m, (const uint16_t*)C, p, (const uint16_t*)down,
                                 (const uint16_t*)up, (int)adapters, rank, scale, ids, Y, ldy, hidden,
                                 (char*)workspace, st);
    return project<float>((const float*)X, ldx, n, m, (const float*)C, p, (const float*)down, (const float*)up, adapters,
                          rank, scale, ids, Y, ldy, hidden,
                                 (char*)workspace, st);
}

int rp_adapt_gradients_device(int device, const void* dY, int64_t lddy, const void* X, int64_t ldx, int32_t dtype, int64_t n,
                              int64_t m, int64_t p, const void* Ct, const void* down, const void* up, int64_t adapters,
                              int32_t rank, const float* scale, const int32_t* ids, const float* hidden, void* dX,
                              int64_t lddx, float* d_down, int64_t d_down_row, int64_t d_down_adapter, float* d_up,
                              int64_t d_up_row, int64_t d_up_adapter, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    int rc = check_call(dtype, n, m, p, adapters, rank, dX ? RP_ADAPT_GRADIENTS_DX : RP_ADAPT_GRADIENTS);
    if (rc) return rc;
    const int64_t mk = padded(m, dtype), pk = padded(p, dtype);
    if (n && ((rc = check_rows("dY", dY, lddy, p, dtype)) || (rc = check_rows("X", X, ldx, m, dtype)))) return rc;
    if ((rc = check_operand("down", down, mk, mk, dtype)) || (rc = check_operand("up", up, pk, pk, dtype))) return rc;
    if (!Ct != !dX) return fail(RP_ERR_INVALID, "Ct and dX go together");
    if (Ct && ((rc = check_operand("Ct", Ct, pk, pk, dtype)))) return rc;
    if (dX && lddx < m) return fail(RP_ERR_INVALID, "dX: row stride %lld is under m=%lld", (long long)lddx, (long long)m);
    if (!d_down || !d_up || (n && (!ids || !hidden))) return fail(RP_ERR_INVALID, "NULL ids, hidden, d_down or d_up");
    if (d_down_row < m || d_down_adapter < d_down_row * rank || d_up_row < p || d_up_adapter < d_up_row * rank)
        return fail(RP_ERR_INVALID, "d_down or d_up: strides under the shape");
    const int64_t need = workspace_of(dtype, n, m, p, adapters, rank, dX ? RP_ADAPT_GRADIENTS_DX : RP_ADAPT_GRADIENTS);
    if (need && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need))
        return fail(RP_ERR_INVALID, "workspace must be 256-byte aligned and hold %lld bytes", (long long)need);
    DeviceGuard guard;
    if ((rc = guard.enter(device))) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RP_BF16)
        return gradients<uint16_t>((const uint16_t*)dY, lddy, (const uint16_t*)X, ldx, n, m, p, (const uint16_t*)Ct,
                                   (const uint16_t*)down, (const uint16_t*)up, (int)adapters, rank, scale, ids, hidden, (uint16_t*)dX,
                                   lddx, d_down, d_down_row, d_down_adapter, d_up, d_up_row, d_up_adapter, (char*)workspace, st);
    return gradients<float>((const float*)dY, lddy, (const float*)X, ldx, n, m, p, (const float*)Ct, (const float*)down,
                            (const float*)up, adapters, rank, scale, ids, hidden, (float*)dX, lddx, d_down, d_down_row,
                            d_down_adapter, d_up, d_up_row, d_up_adapter, (char*)workspace, st);
}

}  // extern "C"
