// gfx950 (CDNA4) kernels for several sequences over paged caches, and for the scores of rows
// of logits: a code object of its own, loaded by the host runtime beside kernels.hip's and
// compiled with the same flags (expressions round as written).
//
// A paged cache is [pages][key heads][page][dh]: token t of a sequence lies in slot t % page of
// page table[t / page]. The bits of a sequence's attention and eviction depend on the sequence
// alone, not on the batch around it or on how the launch is cut. (Log probabilities add a row up in
// an order that goes by the rows' number and alignment.)

#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "batch.h"

#define KERNEL extern "C" __global__

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8_4 __attribute__((ext_vector_type(8), aligned(8)));  // at a multiple of four

static constexpr float NEG_INF = -__builtin_inff();

// Memory that the compiler is to know as global, or as LDS (where it cannot tell, a store holds
// up both kinds of loads).
#define GLOBAL_MEM __attribute__((address_space(1)))
#define LDS_MEM __attribute__((address_space(3)))

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}
// Sums and maxima over a row of 16 lanes (in every lane): lane pairs, quads, then the mirrored
// lane of eight and of sixteen.
__device__ __forceinline__ float row_sum(float x) {
    x += dpp<0xB1>(x);
    x += dpp<0x4E>(x);
    x += dpp<0x141>(x);
    return x + dpp<0x140>(x);
}
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));
    return fmaxf(x, dpp<0x140>(x));
}
// The same over lanes 16 (32) apart, by register lane swaps.
__device__ __forceinline__ float sum16(float v) {
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float sum32(float v) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float max16(float v) {
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float max32(float v) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float wave_sum(float v) { return sum32(sum16(row_sum(v))); }
__device__ __forceinline__ float wave_max(float v) { return max32(max16(row_max(v))); }

__device__ __forceinline__ int lanes_below(uint64_t mask) {  // set bits below this lane
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// fp16 mode's rounding of what an operation writes (the fp32 value rounds: the register is
// opaque, so the compiler does not fold the product before it into the conversion).
__device__ __forceinline__ float r16(float v) {
    asm volatile("" : "+v"(v));
    return (float)(_Float16)v;
}

// Row of a sequence's token t under key head h, over [pages][kh][page].
__device__ __forceinline__ uint32_t row_of(const SeqsDev& s, int b, uint32_t t, int h, int kh, int page) {
    uint32_t pg = t / (uint32_t)page;
    return (s.table[(int64_t)b * s.width + pg] * (uint32_t)kh + (uint32_t)h) * (uint32_t)page + (t - pg * (uint32_t)page);
}

// ---------------------------------------------------------------------------------------
// store: the new tokens' keys and values into the pages
// ---------------------------------------------------------------------------------------

// Rows of new tokens lie one sequence after another; a row's sequence is found by bisection of
// the batch's row offsets. One thread an element: a row of 64 floats is one wave's store of 256
// bytes. A slot's noted weight starts at zero, its position is the token's. Bound by the launch and
// its chain of reads (offset, length, table, row): 1.5 to 5 us from one sequence to 64.
template <typename T>
__device__ __forceinline__ void store_body(const PStoreArgs& a) {
    const int64_t per = (int64_t)a.kh * a.dh, total = (int64_t)a.rows * per;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        uint32_t row = (uint32_t)(i / per);
        int e = (int)(i - row * per), h = e / a.dh, d = e - h * a.dh;
        int lo = a.each ? (int)row : 0, hi = a.each ? lo + 1 : a.s.n;  // first[lo] <= row < first[hi]
        while (hi - lo > 1) {
            int mid = (lo + hi) >> 1;
            if (a.s.first[mid] <= row) lo = mid;
            else hi = mid;
        }
        uint32_t behind = a.each ? 1 : a.s.first[lo + 1] - row;  // 1: the newest
        uint32_t to = row_of(a.s, lo, a.s.len[lo] - behind, h, a.kh, a.page);
        ((T*)a.k)[(int64_t)to * a.dh + d] = (T)a.ksrc[i];
        ((T*)a.v)[(int64_t)to * a.dh + d] = (T)a.vsrc[i];
        if (d == 0) {
            if (a.mass) a.mass[to] = 0.0f;
            if (a.born) a.born[to] = a.s.seen[lo] - behind;
        }
    }
}
KERNEL void __launch_bounds__(256) slm_paged_store(PStoreArgs a) { store_body<float>(a); }
KERNEL void __launch_bounds__(256) slm_paged_store16(PStoreArgs a) { store_body<_Float16>(a); }

// ---------------------------------------------------------------------------------------
// attend: one new token a sequence
// ---------------------------------------------------------------------------------------

// y_g = sum_t softmax_t(scale · q_g·k_t) v_t for the query heads g of one key head. A workgroup
// takes one superblock of SLM_PG_KEYS slots, its waves 64 keys each (32 of fp32 heads above 64);
// for each head a wave has the maximum m, l = sum 2^(x - m) and o = sum 2^(x - m) v of
// x = (scale · log2 e) q·k over its keys, the workgroup those of the superblock, and
// slm_paged_join_* adds the superblocks up. No visible key: m = -inf; one at least: m >= -FLT_MAX.
//
// A superblock is where a long cache is cut for the chip's 256 compute units and where bits are
// fixed: 12000 tokens of one sequence are 47 workgroups a key head. Heads of one key head follow
// each other in the grid: their rows are one page's (the heads slowest: 62 -> 103 us for 64 x 2500
// tokens of 12 heads).
//
// What bounds it is the reading of keys and values (fp32, 64 sequences of up to 2500 tokens, 12
// heads of 64: 346 MB in 61 us, 5.6 TB/s; two of 100003, 4 key heads: 410 MB in 81 us, 5.0; fp16,
// 24 of up to 6000, 4 key heads: 55 MB in 14.4 us, 3.8, where four workgroups a compute unit are
// all there are), and for short caches its chain: batch, table, rows, keys, scores, values, sums
// (one sequence of 37 tokens 4.8 us). So a wave issues all of its keys and values (32 KB of
// fp32) at once, straight into registers, as soon as it has its rows' addresses: 16 lanes read
// a row, each 4 of every 64 elements. A row's dot product is then in 16 lanes, and 16 rows'
// are brought to one lane each by adding and halving (15 additions, not 64): the softmax
// works on a key a lane. A key's weight goes back to the 16 lanes that hold its value by a lane
// broadcast within the row.
extern __shared__ __attribute__((aligned(16))) char lds_[];  // (read and written 8 and 16 bytes at once)

template <int J>
__device__ __forceinline__ uint32_t bcast(uint32_t x) {  // lane J of each row of 16, to the row
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x150 + J, 0xF, 0xF, true);
}
template <int J>
__device__ __forceinline__ float bcast(float x) { return __uint_as_float(bcast<J>(__float_as_uint(x))); }

// J = 0 .. N - 1 as constants.
template <int N, int J = 0, typename F>
__device__ __forceinline__ void each(F f) {
    if constexpr (J < N) {
        f(std::integral_constant<int, J>());
        each<N, J + 1>(f);
    }
}

// Sums over rows of 16 lanes of N values a lane: value c % N to lane c.
template <int N>
__device__ __forceinline__ float scatter_sum(float (&s)[N], int c) {
    auto halve = [&](auto n, auto ctrl, int bit) {
        constexpr int H = decltype(n)::value / 2;
#pragma unroll
        for (int j = 0; j < H; j++) {
            float keep = c & bit ? s[j + H] : s[j], give = c & bit ? s[j] : s[j + H];
            s[j] = keep + dpp<decltype(ctrl)::value>(give);
        }
    };
    using std::integral_constant;
    if constexpr (N == 16) halve(integral_constant<int, 16>(), integral_constant<int, 0x128>(), 8);
    else
#pragma unroll
        for (int j = 0; j < N; j++) s[j] += dpp<0x128>(s[j]);
    // (the partners: lane 7 - i of eight, 3 - i of four, then the neighbour)
    if constexpr (N >= 8) halve(integral_constant<int, 8>(), integral_constant<int, 0x141>(), 4);
    else
#pragma unroll
        for (int j = 0; j < N; j++) s[j] += dpp<0x141>(s[j]);
    halve(integral_constant<int, 4>(), integral_constant<int, 0x1B>(), 2);
    halve(integral_constant<int, 2>(), integral_constant<int, 0xB1>(), 1);
    return s[0];
}

__device__ __forceinline__ void lds_barrier() {  // (loads from memory stay in flight)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Slots of a sequence that a call looks at: all where positions are given, else those before
// the gap.
__device__ __forceinline__ uint32_t looks(const PAttnArgs& a, uint32_t len) {
    return a.born ? len : (int64_t)len > a.gap ? (uint32_t)(len - a.gap) : 0;
}

// M = max m_z and L = sum l_z 2^(m_z - M) over nz superblocks for one head, by a wave: lane z % 64
// adds z in order, the lanes as one tree. (Up to 512 superblocks are read once, all at once.)
__device__ __forceinline__ float2 join_ml(const float2* ml, int nz) {
    const int lane = threadIdx.x & 63;
    float2 v = make_float2(NEG_INF, 0.0f);
    if (lane < nz) v = ml[lane];
    if (nz <= 64) {
        float m = wave_max(v.x);
        return make_float2(m, wave_sum(v.y * __builtin_amdgcn_exp2f(v.x - (m == NEG_INF ? 0.0f : m))));
    }
    float2 q[7];
#pragma unroll
    for (int i = 0; i < 7; i++) q[i] = lane + 64 * i + 64 < nz ? ml[lane + 64 * i + 64] : make_float2(NEG_INF, 0.0f);
    float m = v.x;
#pragma unroll
    for (int i = 0; i < 7; i++) m = fmaxf(m, q[i].x);
    for (int z = lane + 512; z < nz; z += 64) m = fmaxf(m, ml[z].x);
    m = wave_max(m);
    const float ms = m == NEG_INF ? 0.0f : m;
    float l = v.y * __builtin_amdgcn_exp2f(v.x - ms);
#pragma unroll
    for (int i = 0; i < 7; i++) l = fmaf(q[i].y, __builtin_amdgcn_exp2f(q[i].x - ms), l);
    for (int z = lane + 512; z < nz; z += 64) {
        float2 p = ml[z];
        l = fmaf(p.y, __builtin_amdgcn_exp2f(p.x - ms), l);
    }
    return make_float2(m, wave_sum(l));
}

// Sums over the four rows of 16 lanes of four values a lane: value r to row r. (A swap of half
// waves, or of the odd rows, puts two values' partners side by side: one addition for both.)
__device__ __forceinline__ float scatter_rows(f4 v) {
    auto add = [](auto p) { return __uint_as_float(p[0]) + __uint_as_float(p[1]); };
    float a = add(__builtin_amdgcn_permlane32_swap(__float_as_uint(v.x), __float_as_uint(v.z), false, false));
    float b = add(__builtin_amdgcn_permlane32_swap(__float_as_uint(v.y), __float_as_uint(v.w), false, false));
    return add(__builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false));
}

__device__ __forceinline__ float scatter_rows_max(f4 v) {  // the same of maxima
    auto most = [](auto p) { return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])); };
    float a = most(__builtin_amdgcn_permlane32_swap(__float_as_uint(v.x), __float_as_uint(v.z), false, false));
    float b = most(__builtin_amdgcn_permlane32_swap(__float_as_uint(v.y), __float_as_uint(v.w), false, false));
    return most(__builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false));
}

// GM: the query heads a key head, 1 to 4 exactly, on the vector units; or 16: any number, through the
// matrix unit. Measured, 8 sequences of 12000 tokens, 4 heads on each of 4 key heads: exactly 47 us
// (fp32, 64), 94 (128), 27 (fp16, 64), 54 (fp16, 128), by the matrix unit 49, 115, 33, 72; 16 heads on
// one of 64 exactly, four at a time, 31, by the matrix unit 22. GM 16 (9 sequences of up to 7777, 8 heads
// on each of 2 fp16 key heads of 128: 17 us, 1.9 TB/s, one workgroup a compute unit): the products
// are 16x16x4, fp32; the heads are the rows of both, whatever their number: a score
// tile is 16 heads by 16 keys, a lane eight or sixteen bytes of every 32 or 16 elements of key c
// of the tile; the weights go by way of LDS to where a value product wants them, which takes the
// values as they lie.
//
// fp16 keys always go through the matrix unit (16x16x32): its products are exact and its sums
// fp32, so fp32 queries are cut into three fp16 parts (q = q0 + 2^-11 q1 + 2^-22 q2, 33 bits, about
// each head's own power of two), which are rows of one product for four heads: 4·part + head. A
// score's parts are then in three rows of 16 lanes, and one exchange adds them and hands every lane
// its key's. What the parts cannot say is made from the query and the key themselves.
template <typename T, int NT, int GM>
__device__ __forceinline__ void attn_body(const PAttnArgs& a) {
    constexpr int QP = 64 * NT + 8;  // halves from one row of a query part to the next
    constexpr bool HALF = sizeof(T) == 2, MANY = GM > 4;
    constexpr int KS = HALF || NT == 1 ? 16 : 8, NW = 64 / KS, DP = 64 * NT, THREADS = 64 * NW;
    typedef std::conditional_t<HALF, h4, f4> V4;
    using std::integral_constant;
    const int item = blockIdx.x / a.kh, h = blockIdx.x % a.kh;
    const uint4 it = ((const uint4*)a.s.items)[item];
    const uint32_t b = it.x, len = it.z, base = it.y * SLM_PG_KEYS;
    if (b == SLM_NO_SEQ) return;
    const uint32_t most = looks(a, len);
    // (direct: a sequence that sees nothing still gets its zeros)
    if (base >= most && !(it.y == 0 && a.direct)) return;
    const int G = GM <= 4 ? GM : a.heads / a.kh, dh = a.dh;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane >> 4, c = lane & 15;
    constexpr int QS = MANY ? DP + 4 : DP;            // floats from one query to the next
    constexpr int CH = MANY ? 64 : DP;                // elements whose values are added up at once
    float* sq = (float*)lds_;                         // [G][QS], or the three parts: [G in fours][12][QP] halves
    float* so = sq + (HALF ? (G + 3) / 4 * 6 * QP : G * QS);  // [NW][G][CH]
    float* swm = so + NW * G * CH;                    // [NW][G][2]
    float* sml = swm + NW * G * 2;                    // [G][2]
    float* sw = sml + ((G * 2 + 3) & ~3);             // [NW][G][4 * KS], for GM 16
    float* ss = sw + (MANY ? G * SLM_PG_KEYS : 0);    // [G][SLM_PG_KEYS], with direct and mass_out

    // this lane's key: the one whose score it will have
    const int mine = w * (4 * KS) + (HALF || MANY ? KS * r + (c & (KS - 1)) : 4 * (c & (KS - 1)) + r);
    const bool some = base + w * (4 * KS) < most;     // the wave has a key to look at
    bool sees = base + mine < most;
    uint32_t row = 0;
    if (some) {
        row = row_of(a.s, b, min(base + mine, len - 1), h, a.kh, a.page);
        if (a.born && sees) sees = (uint64_t)a.born[row] + (uint64_t)a.gap < a.s.seen[b];
    }
    const uint64_t at = (uint64_t)row * (uint32_t)dh;  // where its row starts, in values
    // the queries, on their way to LDS
    constexpr int QN = (DP * (GM <= 4 ? GM : 16) + THREADS - 1) / THREADS;
    float q[QN];
#pragma unroll
    for (int u = 0; u < QN; u++) {
        int i = tid + u * THREADS, g = i / DP, d = i % DP;
        q[u] = g < G && d < dh ? a.q[((int64_t)b * a.heads + h * G + g) * dh + d] : 0.0f;
    }
    // values: the lane's four of every 64 elements of its row of 16's keys (past the head size: the
    // last four again, of no effect)
    V4 v[KS][NT];
    auto load_rows = [&](const void* from, V4 (&to)[KS][NT]) {
        each<KS>([&](auto j) {
            uint64_t o = (uint64_t)bcast<j>((uint32_t)(at >> 32)) << 32 | bcast<j>((uint32_t)at);
#pragma unroll
            for (int i = 0; i < NT; i++) to[j][i] = *(const V4*)((const T*)from + o + min(64 * i + 4 * c, dh - 4));
        });
    };
    // keys: like the values, or as the matrix unit takes them, 16 keys a tile
    constexpr int TILES = KS / 4, NK = HALF ? 2 * NT : MANY ? 4 * NT : NT;
    std::conditional_t<HALF, h8, f4> k[HALF || MANY ? TILES : KS][NK];
    auto k_start = [&](int i) { return max(0, min(32 * i + 8 * r, dh - 8)); };
    auto tile_lane = [&](int t) { return ((16 * t + c) / KS << 4) | ((16 * t + c) & (KS - 1)); };  // of key c's row
    if (some) {
        if constexpr (HALF) {
            // the four tiles' rows, from the lanes that have them
            auto p = __builtin_amdgcn_permlane16_swap(row, row, false, false);
            auto even = __builtin_amdgcn_permlane32_swap(p[0], p[0], false, false);
            auto odd = __builtin_amdgcn_permlane32_swap(p[1], p[1], false, false);
            const uint32_t rows[4] = {even[0], odd[0], even[1], odd[1]};
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const T* from = (const T*)a.k + (uint64_t)rows[t] * (uint32_t)dh;
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    if (dh >= 8) {
                        k[t][i] = *(const h8_4*)(from + k_start(i));
                    } else {
                        h4 x = *(const h4*)from;
                        k[t][i] = h8{x.x, x.y, x.z, x.w, 0, 0, 0, 0};
                    }
                }
            }
        } else if constexpr (MANY) {
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                const T* from = (const T*)a.k + (uint64_t)__shfl(row, tile_lane(t)) * (uint32_t)dh;
#pragma unroll
                for (int i = 0; i < NK; i++) k[t][i] = *(const f4*)(from + min(16 * i + 4 * r, dh - 4));
            }
        } else {
            load_rows(a.k, k);
        }
        if (NT < 4) load_rows(a.v, v);  // (the largest heads have room for one of the two in registers)
    }
    __shared__ __attribute__((aligned(16))) float q_unit[16];  // of fp16 keys: each head's power of two
    if constexpr (HALF) {
        // A head's queries are cut with its largest number in [2^13, 2^14), by a power of two that its scores
        // get back: what another head of the key head holds has no part in it.
        __shared__ uint32_t q_top[16];
        if (tid < 16) q_top[tid] = 0;
        lds_barrier();
#pragma unroll
        for (int u = 0; u < QN; u++) {
            const int g = (64 * w + u * THREADS) / DP;  // (a wave's 64 elements are one head's)
            if (g >= G) continue;
            float m = fabsf(q[u]);
            m = wave_max(m <= FLT_MAX ? m : 0.0f);
            if (lane == 0) atomicMax(&q_top[g], __float_as_uint(m));
        }
        lds_barrier();
        auto exponent = [&](int g) { return max((int)(q_top[g] >> 23) - 127 - 13, -126); };
        if (tid < 16) q_unit[tid] = __uint_as_float((uint32_t)(127 + exponent(tid)) << 23);
#pragma unroll
        for (int u = 0; u < QN; u++) {
            int i = tid + u * THREADS, g = i / DP, d = i % DP;
            if (g >= G) continue;
            _Float16* to = (_Float16*)sq + ((g >> 2) * 12 + (g & 3)) * QP + d;
            const float whole = q[u] * __uint_as_float((uint32_t)(127 - exponent(g)) << 23);
            float x = whole;
#pragma unroll
            for (int k = 0; k < 3; k++) {
                _Float16 part = (_Float16)x;
                to[4 * k * QP] = part;
                x = (x - (float)part) * 2048.0f;
            }
            // What the parts leave (x 2^-33) is less than fp32's rounding of the element, but where that is far
            // below the head's largest: a NaN then has the head's scores made element by element.
            if (fabsf(x) > 512.0f * fabsf(whole) || (whole == 0.0f && q[u] != 0.0f)) to[0] = (_Float16)__builtin_nanf("");
        }
    } else {
#pragma unroll
        for (int u = 0; u < QN; u++) {
            int i = tid + u * THREADS;
            if (i < G * DP) sq[i / DP * QS + i % DP] = q[u];
        }
    }
    const bool all = __ballot(sees) == ~0ull, any = __ballot(sees) != 0;
    lds_barrier();
    // what lies past the head size becomes zeros (of fp16 keys, what another lane has already)
    if (dh < DP && some) {
#pragma unroll
        for (int i = 0; i < NK; i++) {
            if constexpr (HALF) {
                const int twice = 32 * i + 8 * r - k_start(i);
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (twice >= 8 || e < twice) k[t][i][e] = 0;
            } else if (MANY ? 16 * i + 4 * r >= dh : 64 * i + 4 * c >= dh) {
#pragma unroll
                for (int j = 0; j < (MANY ? TILES : KS); j++) k[j][i] = V4{};
            }
        }
    }

    // A score over fp16 keys that the parts cannot say (an infinite or NaN key or query, a query whose
    // elements' sizes lie far apart): head g's and this lane's key's, element by element in fp32, read again.
    auto by_element = [&](int g) {
        const float* from = a.q + ((int64_t)b * a.heads + h * G + g) * dh;
        const T* key = (const T*)a.k + (uint64_t)row * (uint32_t)dh;
        float z = 0.0f;
#pragma unroll 1
        for (int d = 0; d < dh; d += 4) {
            const V4 x = *(const V4*)(key + d);
#pragma unroll
            for (int e = 0; e < 4; e++) z = fmaf(from[d + e], (float)x[e], z);
        }
        return z;
    };

    float p[MANY ? 1 : GM];
    auto scores = [&](auto gx, int g0, float* out) {  // gx heads from g0: their weights
        constexpr int GX = decltype(gx)::value;
        float x[GX];
#pragma unroll
        for (int g = 0; g < GX; g++) x[g] = NEG_INF;
        if (some) {
            if constexpr (HALF) {
                const _Float16* rows = (const _Float16*)sq + ((g0 >> 2) * 12 + (c < 12 ? c : c - 12)) * QP;
                f4 acc[4] = {};
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    h8 q = *(const h8_4*)(rows + k_start(i));
#pragma unroll
                    for (int t = 0; t < 4; t++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q, k[t][i], acc[t], 0, 0, 0);
                }
                // row r has the queries' part r: part 1 is in 2^-11ths, part 2 in 2^-22ths, there is no part 3
                const float unit = r == 0 ? 1.0f : r == 1 ? 0x1p-11f : r == 2 ? 0x1p-22f : 0.0f;
                uint32_t odd = 0;
#pragma unroll
                for (int g = 0; g < GX; g++) {
                    x[g] = scatter_rows(f4{acc[0][g] * unit, acc[1][g] * unit, acc[2][g] * unit, acc[3][g] * unit});
                    odd |= fabsf(x[g]) <= FLT_MAX ? 0 : 1u << g;
                    x[g] *= q_unit[g0 + g];
                }
                if (__ballot(odd != 0)) {
#pragma unroll 1
                    for (int n = 0; n < GX; n++) {
                        const float z = by_element(g0 + n);
#pragma unroll
                        for (int g = 0; g < GX; g++)
                            if (g == n && (odd >> g & 1)) x[g] = z;
                    }
                }
#pragma unroll
                for (int g = 0; g < GX; g++) x[g] *= a.scale;
            } else if constexpr (!MANY) {
#pragma unroll
                for (int g = 0; g < GX; g++) {
                    float s[KS];
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        f4 q = *(const f4*)(sq + (g0 + g) * DP + 64 * i + 4 * c);
#pragma unroll
                        for (int j = 0; j < KS; j++) {
                            s[j] = i ? fmaf(q.x, k[j][i].x, s[j]) : q.x * k[j][i].x;
                            s[j] = fmaf(q.y, k[j][i].y, s[j]);
                            s[j] = fmaf(q.z, k[j][i].z, s[j]);
                            s[j] = fmaf(q.w, k[j][i].w, s[j]);
                        }
                    }
                    x[g] = scatter_sum<KS>(s, c) * a.scale;
                }
            }
#pragma unroll
            for (int g = 0; g < GX; g++)
                if (!sees) x[g] = NEG_INF;
        }
        // maxima and sums of the heads in one reduction: head r's in row r
        f4 heads = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
        for (int g = 0; g < GX; g++) heads[g] = x[g];
        float mr = GX == 1 ? wave_max(x[0]) : row_max(scatter_rows_max(heads));
        if (any) mr = fmaxf(mr, -FLT_MAX);
        heads = f4{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < GX; g++) {
            const float m = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mr), 16 * g));
            out[g] = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(x[g] - m);
            heads[g] = c < KS ? out[g] : 0.0f;
        }
        const float lr = GX == 1 ? wave_sum(heads[0]) : row_sum(scatter_rows(heads));
        if (c == 0 && r < GX) *(float2*)(swm + (w * G + g0 + r) * 2) = make_float2(mr, lr);
#pragma unroll
        for (int g = 0; g < GX; g++) {
            if (a.mass_out && c < KS) {
                if (a.direct) ((LDS_MEM float*)ss)[(g0 + g) * SLM_PG_KEYS + mine] = x[g];
                else ((GLOBAL_MEM float*)a.sc)[((int64_t)item * a.heads + h * G + g0 + g) * SLM_PG_KEYS + mine] = x[g];
            }
        }
    };
    float wgt[MANY ? KS : 1];  // head c's weights for the row's keys
    if constexpr (!MANY) {
        scores(integral_constant<int, GM>(), 0, p);
    } else {
        float* sp = sw + w * G * (4 * KS);
        if constexpr (HALF) {
            auto four = [&](auto gx, int g0) {
                float e[decltype(gx)::value];
                scores(gx, g0, e);
#pragma unroll
                for (int g = 0; g < decltype(gx)::value; g++) sp[(g0 + g) * (4 * KS) + KS * r + c] = e[g];
            };
            for (int g0 = 0; G <= 8 && g0 < G; g0 += 4) {
                if (G - g0 >= 4) four(integral_constant<int, 4>(), g0);
                else if (G - g0 == 3) four(integral_constant<int, 3>(), g0);
                else if (G - g0 == 2) four(integral_constant<int, 2>(), g0);
                else four(integral_constant<int, 1>(), g0);
            }
        }
        // The heads are the rows: of fp32 keys, and of fp16 keys with more than eight heads, in three products
        // (8 x 12000 tokens, 16 heads on one of 128: 28.9 us, four at a time 30.2; of 256 43 and 44.6. The
        // border is from when this LDS lay off 16 bytes and 8 heads on each of two of 128 took 46 us as rows
        // and 44.5 four at a time; they now would take 36 as rows, and take 40; of 64, 24 either way).
        if (!HALF || G > 8) {
            f4 acc[TILES] = {};
            if constexpr (HALF) {
                // the queries' smallest part first: each one's sums are 2^-11 of the next's unit
                auto add = [&](int part, f4 (&to)[TILES]) {
                    const _Float16* q = (const _Float16*)sq + ((min(c, G - 1) >> 2) * 12 + 4 * part + (min(c, G - 1) & 3)) * QP;
#pragma unroll
                    for (int i = 0; i < NK; i++) {
                        h8 x = *(const h8_4*)(q + k_start(i));
#pragma unroll
                        for (int t = 0; t < TILES; t++) to[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, k[t][i], to[t], 0, 0, 0);
                    }
                };
                if (some) {
                    uint32_t odd = 0;
#pragma unroll
                    for (int part = 2; part >= 0; part--) {
                        add(part, acc);
#pragma unroll
                        for (int t = 0; t < TILES; t++)
#pragma unroll
                            for (int n = 0; n < 4; n++) {
                                if (part) acc[t][n] *= 0x1p-11f;
                                else odd |= fabsf(acc[t][n]) <= FLT_MAX ? 0 : 1u << (4 * t + n);
                            }
                    }
                    const f4 unit = *(const f4*)(q_unit + 4 * r);
#pragma unroll
                    for (int t = 0; t < TILES; t++) acc[t] *= unit;
                    if (__ballot(odd != 0)) {
#pragma unroll 1
                        for (int g = 0; g < G; g++) {
                            const float z = by_element(g);
#pragma unroll
                            for (int t = 0; t < TILES; t++) {
                                const float y = __shfl(z, tile_lane(t));
#pragma unroll
                                for (int n = 0; n < 4; n++)
                                    if (4 * r + n == g && (odd >> (4 * t + n) & 1)) acc[t][n] = y;
                            }
                        }
                    }
                }
            } else if (some) {
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    if (16 * i >= dh) break;
                    const f4 q1 = *(const f4*)(sq + min(c, G - 1) * QS + 16 * i + 4 * r);
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int t = 0; t < TILES; t++)
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(q1[e], k[t][i][e], acc[t], 0, 0, 0);
                }
            }
            // row r has heads 4r .. 4r + 3, a lane the tiles' key c
#pragma unroll
            for (int t = 0; t < TILES; t++) acc[t] *= a.scale;
            if (!all) {
#pragma unroll
                for (int t = 0; t < TILES; t++)
                    if (!__shfl((int)sees, tile_lane(t))) acc[t] = f4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
            }
            float m[4], l[4];
            f4 e[TILES];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                m[n] = NEG_INF;
#pragma unroll
                for (int t = 0; t < TILES; t++) m[n] = fmaxf(m[n], acc[t][n]);
            }
#pragma unroll
            for (int n = 0; n < 4; n++) {
                m[n] = row_max(m[n]);
                if (any) m[n] = fmaxf(m[n], -FLT_MAX);
            }
#pragma unroll
            for (int n = 0; n < 4; n++) {
                l[n] = 0.0f;
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    e[t][n] = m[n] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(acc[t][n] - m[n]);
                    l[n] += e[t][n];
                }
            }
#pragma unroll
            for (int n = 0; n < 4; n++) l[n] = row_sum(l[n]);
            const int key = w * (4 * KS) + c;  // of tile 0
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const int g = 4 * r + n;
                if (g >= G) continue;
#pragma unroll
                for (int t = 0; t < TILES; t++) sp[g * (4 * KS) + 16 * t + c] = e[t][n];
                if (c == 0) *(float2*)(swm + (w * G + g) * 2) = make_float2(m[n], l[n]);
                if (!a.mass_out) continue;
                LDS_MEM float* near = (LDS_MEM float*)ss + g * SLM_PG_KEYS + key;
                GLOBAL_MEM float* far = (GLOBAL_MEM float*)a.sc + ((int64_t)item * a.heads + h * G + g) * SLM_PG_KEYS + key;
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    if (a.direct) near[16 * t] = acc[t][n];
                    else far[16 * t] = acc[t][n];
                }
            }
        }
        // (a wave's own writes: in order before these reads)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < KS; j += 4) {
            f4 x = *(const f4*)(sp + min(c, G - 1) * (4 * KS) + KS * r + j);
#pragma unroll
            for (int e = 0; e < 4; e++) wgt[j + e] = x[e];
        }
    }
    if (NT == 4 && some) load_rows(a.v, v);
    if (some && !all) {  // what is not seen may hold anything
        uint32_t seen = sees;
        each<KS>([&](auto j) {
            if (!bcast<j>(seen)) {
#pragma unroll
                for (int i = 0; i < NT; i++) v[j][i] = V4{};
            }
        });
    }
    each<DP / CH>([&](auto part) {  // elements CH·part on
        if constexpr (MANY) {
            f4 acc[4] = {};  // element 64·part + 4c + e of heads 4r .. 4r + 3
            if (some) {
                auto wide = [&](int j) {
                    f4 x;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = (float)v[j][part][e];
                    return x;
                };
                f4 x = wide(0);
                each<KS>([&](auto j) {
                    // (the next four are widened while these are multiplied)
                    f4 next = wide(j + 1 < KS ? j + 1 : j);
                    if (HALF) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(wgt[j], x[e], acc[e], 0, 0, 0);
                    x = next;
                });
            }
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (4 * r + n < G)
                    *(f4*)(so + (w * G + 4 * r + n) * CH + 4 * c) = f4{acc[0][n], acc[1][n], acc[2][n], acc[3][n]};
        } else {
            f4 o[GM][NT];
#pragma unroll
            for (int g = 0; g < GM; g++)
#pragma unroll
                for (int i = 0; i < NT; i++) o[g][i] = f4{0, 0, 0, 0};
            if (some)
                each<KS>([&](auto j) {
#pragma unroll
                    for (int g = 0; g < GM; g++) {
                        float w1 = bcast<j>(p[g]);
#pragma unroll
                        for (int i = 0; i < NT; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[g][i][e] = j ? fmaf(w1, (float)v[j][i][e], o[g][i][e]) : w1 * (float)v[j][i][e];
                    }
                });
#pragma unroll
            for (int g = 0; g < GM; g++)
#pragma unroll
                for (int i = 0; i < NT; i++) so[(w * G + g) * CH + 64 * i + 4 * c + r] = scatter_rows(o[g][i]);
        }
        lds_barrier();
        // the superblock's, from its waves' in order: four elements a thread
        for (int i = tid; i < G * (CH / 4); i += THREADS) {
            const int g = i / (CH / 4), in = i % (CH / 4) * 4, d = CH * part + in;
            if (d >= dh) continue;
            float m = NEG_INF, l = 0.0f;
            float2 ml[NW];
            f4 o = {0, 0, 0, 0};
#pragma unroll
            for (int k2 = 0; k2 < NW; k2++) ml[k2] = *(const float2*)(swm + (k2 * G + g) * 2);
#pragma unroll
            for (int k2 = 0; k2 < NW; k2++) m = fmaxf(m, ml[k2].x);
            const float ms = m == NEG_INF ? 0.0f : m;
#pragma unroll
            for (int k2 = 0; k2 < NW; k2++) {
                float f = __builtin_amdgcn_exp2f(ml[k2].x - ms);
                f4 z = *(const f4*)(so + (k2 * G + g) * CH + in);
                l = fmaf(ml[k2].y, f, l);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = fmaf(z[e], f, o[e]);
            }
            const int head = h * G + g;
            if (a.direct) {
                float* y = a.y + ((int64_t)b * a.heads + head) * dh + d;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float z = m == NEG_INF ? 0.0f : o[e] / l;
                    y[e] = a.r16 ? r16(z) : z;
                }
                if (d == 0) *(LDS_MEM f2*)(sml + 2 * g) = f2{m, l};
            } else {
                *(f4*)(a.po + ((int64_t)item * a.heads + head) * dh + d) = o;
                if (d == 0) *(GLOBAL_MEM f2*)(a.ml + 2 * ((int64_t)head * a.items + item)) = f2{m, l};
            }
        }
        if (part + 1 < DP / CH) lds_barrier();  // (the next elements' sums go where these lie)
    });
    if (!a.direct || !a.mass_out) return;
    lds_barrier();
    if (NT > 1 && tid >= SLM_PG_KEYS) return;
    const uint32_t t = base + tid;
    if (t >= len) return;
    float add = 0.0f;
    for (int g = 0; g < G; g++)
        if (sml[2 * g] != NEG_INF) add += __builtin_amdgcn_exp2f(ss[g * SLM_PG_KEYS + tid] - sml[2 * g]) / sml[2 * g + 1];
    uint32_t slot = row_of(a.s, b, t, h, a.kh, a.page);
    a.mass_out[slot] = a.mass[slot] + add;
}

#define PAGED_ATTN(name, T, NT, GM) \
    KERNEL void __launch_bounds__(sizeof(T) == 2 || NT == 1 ? 256 : 512) name(PAttnArgs a) { attn_body<T, NT, GM>(a); }
#define PAGED_ATTNS(name, T, NT)       \
    PAGED_ATTN(name##_1, T, NT, 1)     \
    PAGED_ATTN(name##_2, T, NT, 2)     \
    PAGED_ATTN(name##_3, T, NT, 3)     \
    PAGED_ATTN(name##_4, T, NT, 4)     \
    PAGED_ATTN(name##_16, T, NT, 16)
PAGED_ATTNS(slm_paged_attn_1, float, 1)
PAGED_ATTNS(slm_paged_attn_2, float, 2)
PAGED_ATTNS(slm_paged_attn_4, float, 4)
PAGED_ATTNS(slm_paged_attn16_1, _Float16, 1)
PAGED_ATTNS(slm_paged_attn16_2, _Float16, 2)
PAGED_ATTNS(slm_paged_attn16_4, _Float16, 4)

// y = sum_z o_z 2^(m_z - M) / L: a workgroup a (sequence, head), superblock z in group z % KG of
// dh / 4 threads, a group in order, then the groups in order. Behind them, with mass_out, four
// waves a (superblock, key head): mass_out = mass + sum_g 2^(x_g - M_g) / L_g. Sixteen waves a
// workgroup, or four where that still leaves every superblock a group of its own: the same sums.
// Bound by its chain (4.1 us for 64 x 12 heads of 10 superblocks), for long caches by the noted weights
// (two of 100003 tokens, 12 heads: 11 us for 18 MB). Measured, the whole call: 64 sequences of
// 1066 tokens 32 us with four waves, 34 with sixteen; one of 51200 fp16 tokens, 12 heads of 256 on 4,
// 70 with four, 67 with sixteen. (Joined by the workgroup that is last to be done instead of a
// launch: 6 to 12 us slower, by the fence that every workgroup then needs.)
template <int THREADS>
__device__ __forceinline__ void join_body(const PAttnArgs& a) {
    __shared__ f4 so[THREADS];
    __shared__ float2 sml[THREADS / 256][16];
    const int tid = threadIdx.x, H = a.heads, dh = a.dh;
    if ((int)blockIdx.x < a.s.n * H) {
        const int b = blockIdx.x / H, head = blockIdx.x % H;
        const int nz = (int)((looks(a, a.s.len[b]) + SLM_PG_KEYS - 1) / SLM_PG_KEYS);
        const int64_t z0 = a.s.ifirst[b];
        const float2* ml = (const float2*)a.ml + (int64_t)head * a.items + z0;
        const int cols = dh / 4, KG = THREADS / cols, c = tid % cols, zg = tid / cols;
        const float* po = a.po + (z0 * H + head) * dh + 4 * c;
        const bool mine = zg < KG && zg < nz;
        f4 v = {0, 0, 0, 0};
        float mz = NEG_INF;
        if (mine) {  // (the first of its superblocks, on its way while the sums are made)
            v = *(const f4*)(po + (int64_t)zg * H * dh);
            mz = ml[zg].x;
        }
        const float2 ML = join_ml(ml, nz);
        const float ms = ML.x == NEG_INF ? 0.0f : ML.x;
        f4 o = {0, 0, 0, 0};
        if (mine) {
            float wz = __builtin_amdgcn_exp2f(mz - ms);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = v[e] * wz;
#pragma unroll 4
            for (int z = zg + KG; z < nz; z += KG) {
                wz = __builtin_amdgcn_exp2f(ml[z].x - ms);
                v = *(const f4*)(po + (int64_t)z * H * dh);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = fmaf(v[e], wz, o[e]);
            }
        }
        so[tid] = o;
        __syncthreads();
        if (tid < dh) {
            float s = 0.0f;
            const int ng = min(nz, KG);
#pragma unroll 8
            for (int k = 0; k < ng; k++) s += ((const float*)so)[k * dh + tid];
            float y = ML.x == NEG_INF ? 0.0f : s / ML.y;
            a.y[((int64_t)b * H + head) * dh + tid] = a.r16 ? r16(y) : y;
        }
        return;
    }
    const int pair = ((int)blockIdx.x - a.s.n * H) * (THREADS / 256) + (tid >> 8);
    const int item = pair / a.kh, h = pair % a.kh, G = H / a.kh;
    const int part = tid >> 8, w = (tid >> 6) & 3, key = tid & 255;
    uint4 it = {SLM_NO_SEQ, 0, 0, 0};
    if (item < a.items) it = ((const uint4*)a.s.items)[item];
    const uint32_t b = it.x, len = it.z, t = it.y * SLM_PG_KEYS + key;
    const bool live = b != SLM_NO_SEQ;
    const int nz = live ? (int)((looks(a, len) + SLM_PG_KEYS - 1) / SLM_PG_KEYS) : 0;
    const bool seen = (int)it.y < nz;
    float x[4];
    uint32_t slot = 0;
    float old = 0.0f;
    if (live && t < len) {
        slot = row_of(a.s, b, t, h, a.kh, a.page);
        old = a.mass[slot];
    }
    const float* sc = a.sc + ((int64_t)item * H + h * G) * SLM_PG_KEYS + key;
#pragma unroll
    for (int g = 0; g < 4; g++) x[g] = seen && g < G ? sc[g * SLM_PG_KEYS] : 0.0f;
    if (seen) {
        const int64_t z0 = a.s.ifirst[b];
        for (int g = w; g < G; g += 4) {
            float2 ML = join_ml((const float2*)a.ml + (int64_t)(h * G + g) * a.items + z0, nz);
            if ((tid & 63) == 0) sml[part][g] = ML;
        }
    }
    __syncthreads();
    float add = 0.0f;
    auto take = [&](int g, float xg) {
        float2 ML = sml[part][g];
        if (ML.x != NEG_INF) add += __builtin_amdgcn_exp2f(xg - ML.x) / ML.y;
    };
    if (seen) {
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (g < G) take(g, x[g]);
        for (int g = 4; g < G; g++) take(g, sc[g * SLM_PG_KEYS]);
    }
    if (live && t < len) a.mass_out[slot] = old + add;
}
KERNEL void __launch_bounds__(256) slm_paged_join_4(PAttnArgs a) { join_body<256>(a); }
KERNEL void __launch_bounds__(1024) slm_paged_join_16(PAttnArgs a) { join_body<1024>(a); }

// ---------------------------------------------------------------------------------------
// evict: which slots stay, then the moves
// ---------------------------------------------------------------------------------------

// A slot's rank as a number: the newest above all, then by weight (NaN below all, -0 as 0).
__device__ __forceinline__ uint32_t mass_key(float m, uint32_t born, uint32_t recent, uint32_t seen) {
    if ((uint64_t)born + recent >= seen) return 0xffffffffu;
    if (m != m) return 0;
    uint32_t u = __float_as_uint(m + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or0(uint32_t x) {  // 0 where the lane has no such neighbour
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, true);
}
// Inclusive prefix sums over a wave: within rows of 16, then the rows' last lanes to those behind.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += dpp_or0<0x111, 0xF>(x);
    x += dpp_or0<0x112, 0xF>(x);
    x += dpp_or0<0x114, 0xF>(x);
    x += dpp_or0<0x118, 0xF>(x);
    x += dpp_or0<0x142, 0xA>(x);
    x += dpp_or0<0x143, 0xC>(x);
    return x;
}
// Exclusive prefix sum over a workgroup of sixteen waves. s: 16 words of LDS of this call's own.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* s) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t incl = wave_scan(x);
    if (lane == 63) s[w] = incl;
    __syncthreads();
    uint32_t before = wave_scan(lane < 16 ? s[lane] : 0);
    return (w ? __builtin_amdgcn_readlane(before, w - 1) : 0) + incl - x;
}

// Keys and values of rows from[] to rows to[], V at a time, by the workgroup: a power of two of
// lanes a row, and `step` rows at once, four times over.
template <typename V>
__device__ __forceinline__ void move_rows(const PEvictArgs& a, const uint32_t* to, const uint32_t* from, uint32_t n) {
    const uint32_t vecs = (uint32_t)(a.dh * a.unit) / sizeof(V);
    const int lg = vecs <= 1 ? 0 : 32 - __clz(vecs - 1);
    const uint32_t c = threadIdx.x & ((1u << lg) - 1), r0 = threadIdx.x >> lg, step = blockDim.x >> lg;
    if (c >= vecs) return;
    V* k = (V*)a.k + c;
    V* v = (V*)a.v + c;
    for (uint32_t r = r0; r < n; r += 4 * step) {
        V kv[4], vv[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            int64_t f = (int64_t)from[min(r + u * step, n - 1)] * vecs;
            kv[u] = k[f];
            vv[u] = v[f];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (r + u * step >= n) break;
            int64_t t = (int64_t)to[r + u * step] * vecs;
            k[t] = kv[u];
            v[t] = vv[u];
        }
    }
}

// A workgroup of 1024 a (sequence, key head). The slots' keys are read once, into LDS (up to
// `room` of them; those of longer sequences are read again each time). The keep-th largest is
// found by rounds of counting digits (11, 11 and 10 bits), fewer where a round's digit leaves no
// key to be told from another. Then the slots that stay, a bit each, 64 a wave at a time; from
// the words' counts, added up, which of the first `keep` are left and which of those behind move
// there. Few moves (SLM_MOVES_HERE) are made here, more by a launch of their own.
//
// Bound by the chain of its steps, a barrier each (one sequence of 1040 tokens, 4 heads: 7 us; 32
// of up to 4200, 4 heads, of which up to 199 move: 12.5; 12 of 16384, 12 heads: 22), and past `room` by one
// compute unit's reading of the weights, five to eight times over: one sequence of 36000 tokens cut
// to 30000 takes 43 us, of 40000 149. Measured for the moves: 32 sequences, up to 250 moves, here
// 15.9 us against 18.9 by a launch; one sequence, 500 moves, 14.1 here, 12.8 by a launch; 900,
// 17.1 and 13.4; but 32 sequences, 500 moves, 21.7 and 24.2.
KERNEL void __launch_bounds__(1024) slm_paged_select(PEvictArgs a) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t red[6][16];
    __shared__ uint32_t pick[3][3];
    uint32_t* keys = (uint32_t*)lds_;                         // [room]
    uint64_t* stays = (uint64_t*)(keys + a.room);             // [room / 64]: the slots that stay, a bit each
    uint32_t* counts = (uint32_t*)(stays + a.room / 64);      // [room / 64]: what comes before a word's
    const int h = blockIdx.x % a.kh, b = blockIdx.x / a.kh, tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t len = a.s.len[b], seen = a.s.seen[b];
    const bool over = len > a.keep, held = len <= a.room;
    if (!over && tid == 0 && a.count) a.count[blockIdx.x] = 0;
    if (!over && a.in_place) return;

    auto row = [&](uint32_t t) { return row_of(a.s, b, t, h, a.kh, a.page); };
    auto key_at = [&](uint32_t r) { return mass_key(a.mass[r], a.born[r], a.recent, seen); };
    auto key_of = [&](uint32_t t) { return held ? keys[t] : key_at(row(t)); };
    auto front = [&](uint32_t t0) -> uint64_t {  // the slots of t0's 64 that are among the first `keep`
        return a.keep <= t0 ? 0 : a.keep - t0 >= 64 ? ~0ull : (1ull << (a.keep - t0)) - 1;
    };
    auto there = [&](uint32_t t0) -> uint64_t {  // ... that hold a token
        return len <= t0 ? 0 : len - t0 >= 64 ? ~0ull : (1ull << (len - t0)) - 1;
    };
    if (over) {
        auto count = [&](uint32_t k) { atomicAdd(&hist[k >> 21], 1u); };
        hist[2 * tid] = hist[2 * tid + 1] = 0;
        __syncthreads();
        if (held && a.vec) {  // four slots of a page at once, four times over
            for (uint32_t t0 = 4 * tid; t0 < len; t0 += 16384) {
                f4 m[4];
                uint4 p[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    uint32_t r = row(min(t0 + 4096 * u, (len - 1) & ~3u));
                    m[u] = *(const f4*)(a.mass + r);
                    p[u] = *(const uint4*)(a.born + r);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    uint32_t t = t0 + 4096 * u;
                    if (t >= len) break;
                    uint4 k = {mass_key(m[u].x, p[u].x, a.recent, seen), mass_key(m[u].y, p[u].y, a.recent, seen),
                               mass_key(m[u].z, p[u].z, a.recent, seen), mass_key(m[u].w, p[u].w, a.recent, seen)};
                    *(uint4*)(keys + t) = k;
                    count(k.x);
                    if (t + 1 < len) count(k.y);
                    if (t + 2 < len) count(k.z);
                    if (t + 3 < len) count(k.w);
                }
            }
        } else {
            for (uint32_t t = tid; t < len; t += 1024) {
                uint32_t k = key_at(row(t));
                if (held) keys[t] = k;
                count(k);
            }
        }
        __syncthreads();
    }
    // the first `need` of the keys that are `prefix` from bit `shift` up stay, and all above
    uint32_t prefix = 0, need = a.keep;
    int shift = 32;
    bool ties = over;  // ... and some such keys go
    for (int round = 0; round < 3 && ties; round++) {
        const int bits = round == 2 ? 10 : 11;
        if (round) {
            for (uint32_t t = tid; t < len; t += 1024) {
                uint32_t k = key_of(t);
                if (k >> shift == prefix) atomicAdd(&hist[(k >> (shift - bits)) & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
        }
        shift -= bits;
        // the digit at which the count from above reaches `need`: each thread two bins, from above
        uint32_t h1 = hist[2047 - 2 * tid], h0 = hist[2046 - 2 * tid];
        hist[2047 - 2 * tid] = hist[2046 - 2 * tid] = 0;
        uint32_t before = block_scan(h1 + h0, red[round]);
        if (before < need && before + h1 + h0 >= need) {
            bool first = before + h1 >= need;
            pick[round][0] = 2047 - 2 * tid - (first ? 0 : 1);
            pick[round][1] = need - before - (first ? 0 : h1);
            pick[round][2] = (first ? h1 : h0) > pick[round][1];
        }
        __syncthreads();
        prefix = (prefix << bits) | pick[round][0];
        need = pick[round][1];
        ties = pick[round][2] != 0;
    }
    // the lists of slots left and of slots that move there: in memory, or few of them in LDS
    uint32_t* list = a.moves + (int64_t)blockIdx.x * 2 * a.most;
    uint32_t *to = hist, *from = hist + SLM_MOVES_HERE;
    uint32_t moves = 0;
    if (over && held) {
        const uint32_t words = (len + 63) / 64;
        if (ties) {  // equal keys: the lower slots stay
            for (uint32_t q = w; q < words; q += 16) {
                uint64_t em = __ballot(64 * q + lane < len && keys[64 * q + lane] == prefix);
                if (lane == 0) counts[q] = __popcll(em);
            }
            __syncthreads();
            uint32_t before = block_scan(tid < words ? counts[tid] : 0, red[3]);
            if (tid < words) counts[tid] = before;
            __syncthreads();
        }
        // (the compute unit's sixteen waves share one scalar unit: what can be a lane's work is)
#pragma unroll 2
        for (uint32_t q = w; q < words; q += 16) {
            const uint32_t t = 64 * q + lane, k = keys[min(t, len - 1)] >> shift;
            uint64_t m = __ballot(k >= prefix);
            if (ties) {
                uint64_t em = __ballot(k == prefix && t < len);
                m = __ballot(k > prefix || (k == prefix && counts[q] + lanes_below(em) < need));
            }
            if (lane == 0) stays[q] = m;
        }
        __syncthreads();
        // a thread a word: holes below, movers above, both counts in one word (neither passes 2^16)
        ulonglong2* both = (ulonglong2*)keys;  // (the keys have done their work)
        uint32_t n = 0;
        if (tid < words) {
            uint64_t in = there(64 * tid), m = stays[tid] & in, f = front(64 * tid);
            both[tid] = make_ulonglong2(~m & f & in, m & ~f);
            n = __popcll(~m & f & in) | __popcll(m & ~f) << 16;
        }
        uint32_t before = block_scan(n, red[4]);
        if (tid < words) counts[tid] = before;
        if (tid == words - 1) pick[0][0] = (before + n) >> 16;
        __syncthreads();
        moves = pick[0][0];
        auto write = [&](auto* to, auto* from) {
#pragma unroll 2
            for (uint32_t q = w; q < words; q += 16) {
                const ulonglong2 m = both[q];
                const uint32_t c = counts[q];
                const uint32_t hole = (uint32_t)(lane < 32 ? m.x : m.x >> 32) >> (lane & 31) & 1;
                const uint32_t mover = (uint32_t)(lane < 32 ? m.y : m.y >> 32) >> (lane & 31) & 1;
                if (hole) to[(c & 0xffff) + lanes_below(m.x)] = 64 * q + lane;
                if (mover) from[(c >> 16) + lanes_below(m.y)] = 64 * q + lane;
            }
        };
        if (a.count) write((GLOBAL_MEM uint32_t*)list, (GLOBAL_MEM uint32_t*)(list + a.most));
        else write((LDS_MEM uint32_t*)to, (LDS_MEM uint32_t*)from);
    } else if (over) {
        // too many for LDS: a wave a run of whole 64s of slots, their keys read again each time
        const uint32_t run = (len + 1024 - 1) / 1024 * 64, lo = min(len, w * run), hi = min(len, lo + run);
        uint32_t tie0 = 0;
        auto stay = [&](uint32_t t0, uint32_t& tie) -> uint64_t {
            const bool in = t0 + lane < hi;
            uint32_t k = in ? key_of(t0 + lane) >> shift : 0;
            uint64_t em = __ballot(in && k == prefix);
            uint64_t m = __ballot(in && (k > prefix || (k == prefix && (!ties || tie + lanes_below(em) < need))));
            tie += __popcll(em);
            return m;
        };
        auto sum_before = [&](uint32_t n, uint32_t* s, uint32_t* all) {  // over the waves before this one
            uint32_t v = block_scan(lane == 0 ? n : 0, s);
            __syncthreads();
            *all = 0;
            for (int i = 0; i < 16; i++) *all += s[i];
            return (uint32_t)__builtin_amdgcn_readfirstlane(v);
        };
        uint32_t all;
        if (ties) {
            uint32_t n = 0;
            for (uint32_t t0 = lo; t0 < hi; t0 += 64) n += __popcll(__ballot(t0 + lane < hi && key_of(t0 + lane) >> shift == prefix));
            tie0 = sum_before(n, red[3], &all);
        }
        uint32_t holes = 0, movers = 0, tie = tie0;
        for (uint32_t t0 = lo; t0 < hi; t0 += 64) {
            uint64_t m = stay(t0, tie);
            holes += __popcll(~m & front(t0) & there(t0));
            movers += __popcll(m & ~front(t0));
        }
        uint32_t hole0 = sum_before(holes, red[4], &all), mover0 = sum_before(movers, red[5], &moves);
        tie = tie0;
        for (uint32_t t0 = lo; t0 < hi; t0 += 64) {
            uint64_t m = stay(t0, tie), f = front(t0), hm = ~m & f & there(t0), mm = m & ~f;
            if (__builtin_amdgcn_inverse_ballot_w64(hm)) {
                if (a.count) ((GLOBAL_MEM uint32_t*)list)[hole0 + lanes_below(hm)] = t0 + lane;
                else ((LDS_MEM uint32_t*)to)[hole0 + lanes_below(hm)] = t0 + lane;
            }
            if (__builtin_amdgcn_inverse_ballot_w64(mm)) {
                if (a.count) ((GLOBAL_MEM uint32_t*)list)[a.most + mover0 + lanes_below(mm)] = t0 + lane;
                else ((LDS_MEM uint32_t*)from)[mover0 + lanes_below(mm)] = t0 + lane;
            }
            hole0 += __popcll(hm);
            mover0 += __popcll(mm);
            if (!a.in_place && (m & f) >> lane & 1) {
                uint32_t r = row(t0 + lane);
                a.mass_out[r] = a.mass[r];
                a.born_out[r] = a.born[r];
            }
        }
    }
    if (over) {
        if (a.count) {
            if (tid == 0) a.count[blockIdx.x] = moves;
        } else {
            // rows of all the moves first, then their keys and values, four loads of each in flight
            __syncthreads();
            for (uint32_t i = tid; i < 2 * moves; i += 1024) {
                uint32_t at = i < moves ? i : SLM_MOVES_HERE + i - moves;
                hist[at] = row(hist[at]);
            }
            __syncthreads();
            for (uint32_t i = tid; i < moves; i += 1024) {
                a.mass_out[to[i]] = a.mass[from[i]];
                a.born_out[to[i]] = a.born[from[i]];
            }
            if (a.dh * a.unit % 16 == 0) move_rows<f4>(a, to, from, moves);
            else move_rows<h4>(a, to, from, moves);
        }
        if (a.in_place || !held) return;
    }
    // mass and born of what stays where it is, into the buffers for them
    const uint32_t end = min(len, a.keep);
    if (a.vec) {
#pragma unroll 2
        for (uint32_t t = 4 * tid; t < end; t += 4096) {
            uint32_t r = row(t);
            uint32_t m = over ? (uint32_t)(stays[t / 64] >> (t % 64)) & 15 : 15;
            if (end - t < 4) m &= (1u << (end - t)) - 1;
            f4 mass = *(const f4*)(a.mass + r);
            uint4 born = *(const uint4*)(a.born + r);
            if (m == 15) {
                *(f4*)(a.mass_out + r) = mass;
                *(uint4*)(a.born_out + r) = born;
                continue;
            }
            if (m & 1) a.mass_out[r] = mass.x, a.born_out[r] = born.x;
            if (m & 2) a.mass_out[r + 1] = mass.y, a.born_out[r + 1] = born.y;
            if (m & 4) a.mass_out[r + 2] = mass.z, a.born_out[r + 2] = born.z;
            if (m & 8) a.mass_out[r + 3] = mass.w, a.born_out[r + 3] = born.w;
        }
    } else {
        for (uint32_t t = tid; t < end; t += 1024) {
            if (over && !(stays[t / 64] >> (t % 64) & 1)) continue;
            uint32_t r = row(t);
            a.mass_out[r] = a.mass[r];
            a.born_out[r] = a.born[r];
        }
    }
}

// The moves of a (sequence, key head), SLM_MOVES_WG of them a workgroup. Bound by memory: 12
// sequences of 12 heads of 64, 467 MB read and written in 101 us, 4.6 TB/s.
template <typename V>
__device__ __forceinline__ void move_body(const PEvictArgs& a, uint32_t blocks) {
    __shared__ uint32_t to[SLM_MOVES_WG], from[SLM_MOVES_WG];
    const uint32_t pair = blockIdx.x / blocks, r0 = blockIdx.x % blocks * SLM_MOVES_WG, total = a.count[pair];
    if (r0 >= total) return;
    const int h = pair % a.kh, b = pair / a.kh;
    const uint32_t n = min(total - r0, (uint32_t)SLM_MOVES_WG), i = threadIdx.x;
    const uint32_t* list = a.moves + (int64_t)pair * 2 * a.most + r0;
    if (i < n) {
        uint32_t t = row_of(a.s, b, list[i], h, a.kh, a.page), f = row_of(a.s, b, list[a.most + i], h, a.kh, a.page);
        to[i] = t;
        from[i] = f;
        a.mass_out[t] = a.mass[f];
        a.born_out[t] = a.born[f];
    }
    __syncthreads();
    move_rows<V>(a, to, from, n);
}
KERNEL void __launch_bounds__(256) slm_paged_move16(PMoveArgs a) { move_body<f4>(a.e, a.blocks); }
KERNEL void __launch_bounds__(256) slm_paged_move8(PMoveArgs a) { move_body<h4>(a.e, a.blocks); }

// ---------------------------------------------------------------------------------------
// logprobs
// ---------------------------------------------------------------------------------------

// A logit's rank as a number: NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t logit_key(float x) {
    if (x != x) return 0;
    uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float logit_of(uint32_t key) {  // (a number, not a NaN's key)
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// Part of a row's sums: its maximum m, the count c of logits equal to it, and over the others
// S = sum e^(x-m) and E = sum e^(x-m) (x-m); so log L = log c + log1p(S / c) keeps its digits
// where one token has nearly all the probability. A NaN is in S.
template <typename C>
struct Sums {
    float m;
    C c;
    float S, E;
    __device__ __forceinline__ void raise(float to) {  // the same sum about a maximum `to` >= m
        if (!(to > m)) return;
        if (m > NEG_INF) {
            float d = m - to, f = __builtin_amdgcn_exp2f(d * 1.44269504f), all = (float)c + S;
            E = f * fmaf(fmaxf(d, -1e4f), all, E);
            S = f * all;
        }
        c = 0;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {  // x <= m, or a NaN; m > -inf
        float d = x - m, e = __builtin_amdgcn_exp2f(d * 1.44269504f);
        const bool top = x == m;
        S += top ? 0.0f : e;
        c += top;
        E = fmaf(e, fmaxf(d, -1e4f), E);  // (e^-1e4 is 0: an impossible token adds nothing)
    }
};
typedef Sums<uint32_t> LaneSum;
typedef Sums<float> RowSum;

// The largest t (to 16 bits: a bound is all it is for) such that at least `want` of the wave's 64
// keys are >= t: by its bits from above, a ballot each; two wants at once.
__device__ __forceinline__ void wave_nth(uint32_t key, int want0, int want1, uint32_t& t0, uint32_t& t1) {
    t0 = t1 = 0;
    for (int bit = 31; bit >= 16; bit--) {
        uint32_t c0 = t0 | (1u << bit), c1 = t1 | (1u << bit);
        if (__popcll(__ballot(key >= c0)) >= want0) t0 = c0;
        if (__popcll(__ballot(key >= c1)) >= want1) t1 = c1;
    }
}

// A workgroup of W waves a row, in panels of W·2048 logits that a wave holds in registers while
// it adds them up: the row is read once. The alternatives are those of largest rank (key, then
// the lower index), found without a second look at the row: `top` logits at least as large as
// a bound T exist if every wave has ceil(top / W) lanes whose own maximum reaches it (the least
// over the waves of that lane's maximum), or one wave has `top` of them (the most over the
// waves): T is the larger of the two, from the first panel. Whatever reaches T goes into the
// wave's list, which is cut to its `top` best when more than 64 are in it (T rises with it);
// about 5·top of a row of 32000 reach T. Of what the lists hold at the end, those that reach a
// second bound of the same kind are ranked by counting the better ones.
//
// With SPLIT a row goes to `parts` workgroups, which leave their sums and alternatives to
// slm_logprobs_join.
//
// Bound by reading the logits where there are many (1021 rows of 65003: 265 MB in 55 us, 4.8
// TB/s), else by its chain: read, maxima, bound, lists, ranks (256 rows of 32000, 5 alternatives:
// one workgroup a compute unit, 11 to 12 us; one row of 32000 with 20: 7.5 and 4 us for its join).
template <int W, bool SPLIT>
__device__ __forceinline__ void logprobs_body(const LogpArgs& a) {
    __shared__ uint64_t list[W][128], fin[W * 64];
    __shared__ uint32_t cnts[W], bound[W][2], nfin;
    __shared__ __attribute__((aligned(16))) float sums[W][4];
    const int part = SPLIT ? blockIdx.x % a.parts : 0;
    const int64_t row = SPLIT ? blockIdx.x / a.parts : blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), top = a.top;
    const float* x = a.x + row * a.n;
    // whole 16 bytes from the last such address at or before the row's first logit
    const int a0 = (int)(((uintptr_t)x >> 2) & 3), end = (int)a.n + a0;
    const float* xa = x - a0;
    const int fair = (top + W - 1) / W;
    const float given = SPLIT ? 0.0f : x[a.ids ? a.ids[row] : a.few[row]];
    const int begin = SPLIT ? part * a.span : 0, stop = SPLIT ? min(end, begin + a.span) : end;
    if (tid == 0) nfin = 0;

    auto threshold = [&](uint32_t key) -> uint32_t {
        uint32_t t0, t1;
        wave_nth(key, top, fair, t0, t1);
        if (lane == 0) {
            bound[w][0] = t0;
            bound[w][1] = t1;
        }
        __syncthreads();
        uint32_t most = bound[0][0], least = bound[0][1];
#pragma unroll
        for (int i = 1; i < W; i++) {
            most = max(most, bound[i][0]);
            least = min(least, bound[i][1]);
        }
        __syncthreads();
        return max(most, least);
    };

    LaneSum mine{NEG_INF, 0, 0.0f, 0.0f};
    uint64_t least = 0;  // what a logit's rank must pass to be listed
    float least_x = NEG_INF;
    int cnt = 0;
    auto cut = [&]() {  // the list's `top` best, best first
        uint64_t e0 = lane < cnt ? list[w][lane] : 0, e1 = lane + 64 < cnt ? list[w][lane + 64] : 0;
        int r0 = 0, r1 = 0;
        for (int i = 0; i < cnt; i++) {
            uint64_t o = list[w][i];
            r0 += o > e0;
            r1 += o > e1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (e0 && r0 < top) list[w][r0] = e0;
        if (e1 && r1 < top) list[w][r1] = e1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (cnt >= top) {
            cnt = top;
            least = list[w][top - 1];
            least = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(least >> 32)) << 32 |
                    (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)least);
            least_x = least >> 32 ? logit_of((uint32_t)(least >> 32)) : NEG_INF;
        }
    };

    for (int p0 = begin; p0 < stop; p0 += W * 2048) {
        f4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            int at = p0 + ((j >> 2) * W + w) * 1024 + (j & 3) * 256 + lane * 4;
            if (at >= a0 && at + 4 <= end) {
                v[j] = *(const f4*)(xa + at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[j][e] = at + e >= a0 && at + e < end ? xa[at + e] : NEG_INF;
            }
        }
        float m = NEG_INF;
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += 4) {  // (the first half while the second is on its way)
            float m4 = NEG_INF;
#pragma unroll
            for (int j = j0; j < j0 + 4; j++) m4 = fmaxf(fmaxf(m4, fmaxf(v[j].x, v[j].y)), fmaxf(v[j].z, v[j].w));
            m = fmaxf(m, m4);
            mine.raise(m4);
            if (mine.m > NEG_INF) {
#pragma unroll
                for (int j = j0; j < j0 + 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mine.add(v[j][e]);
            } else {
#pragma unroll
                for (int j = j0; j < j0 + 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mine.S += v[j][e] == NEG_INF ? 0.0f : v[j][e];  // (a NaN)
            }
        }
        if (top) {
            if (p0 == begin) {
                // (a lane of nothing but NaNs and -infinities bounds nothing)
                uint32_t t = threshold(m > NEG_INF ? logit_key(m) : 0);
                least = t ? ((uint64_t)t << 32) - 1 : 0;
                least_x = t ? logit_of(t) : NEG_INF;
            }
            if (__ballot(m >= least_x)) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float m4 = fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w));
                    if (!__ballot(!(m4 < least_x))) continue;
                    int at = p0 + ((j >> 2) * W + w) * 1024 + (j & 3) * 256 + lane * 4 - a0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (!__ballot(!(v[j][e] < least_x))) continue;
                        uint64_t r = (uint64_t)logit_key(v[j][e]) << 32 | (0xffffffffu - (uint32_t)(at + e));
                        bool in = at + e >= 0 && at + e < (int)a.n && r > least;
                        uint64_t mask = __ballot(in);
                        if (!mask) continue;
                        if (in) list[w][cnt + lanes_below(mask)] = r;
                        cnt += __popcll(mask);
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                        if (cnt > 64) cut();
                    }
                }
            }
        }
    }

    // the row's sums: the wave's, then the waves' (a lane of each row of 16 for each)
    RowSum s{mine.m, (float)mine.c, mine.S, mine.E};
    float m = wave_max(s.m);
    s.raise(m);
    s.c = wave_sum(s.c);
    s.S = wave_sum(s.S);
    s.E = wave_sum(s.E);
    if (lane == 0) {
        *(f4*)sums[w] = f4{m, s.c, s.S, s.E};
        cnts[w] = cnt;
    }
    __syncthreads();
    s = RowSum{NEG_INF, 0.0f, 0.0f, 0.0f};
    int total = 0;
    if ((lane & 15) < W) {
        f4 q = *(const f4*)sums[lane & 15];
        s = RowSum{q.x, q.y, q.z, q.w};
        total = cnts[lane & 15];
    }
    m = row_max(s.m);
    s.raise(m);
    s.c = row_sum(s.c);
    s.S = row_sum(s.S);
    s.E = row_sum(s.E);
    total = (int)row_sum((float)total);
    // no logit above -inf (and no NaN): no token is possible
    const bool none = m == NEG_INF && s.S == 0.0f;
    auto log_sum = [&] { return logf(s.c) + log1pf(s.S / s.c); };
    if (SPLIT) {
        if (tid == 0) *(f4*)(a.part_sums + 4 * (row * a.parts + part)) = f4{m, s.c, s.S, s.E};
    } else if (w == 0) {
        const float logl = log_sum();
        if (lane == 0) {
            a.lp[row] = none ? NEG_INF : (given - m) - logl;
            if (a.ent) a.ent[row] = none ? 0.0f : (m - m) + logl - s.E / (s.c + s.S);
        }
    }
    if (!top) return;
    uint64_t e = lane < cnt ? list[w][lane] : 0;
    if (total > 128) {
        uint32_t t = threshold((uint32_t)(e >> 32));
        if ((uint32_t)(e >> 32) < t) e = 0;
    }
    {  // a wave's share of the places at once
        uint64_t mask = __ballot(e != 0);
        uint32_t at = 0;
        if (lane == 0 && mask) at = atomicAdd(&nfin, (uint32_t)__popcll(mask));
        at = (uint32_t)__builtin_amdgcn_readfirstlane(at) + lanes_below(mask);
        if (e) fin[at] = e;
    }
    __syncthreads();
    const int n = nfin;
    uint64_t* listed = SPLIT ? a.part_top + (row * a.parts + part) * top : nullptr;
    if (SPLIT && tid >= n && tid < top) listed[tid] = 0;  // (a part of fewer logits)
    if (64 * w >= n) return;
    e = tid < n ? fin[tid] : 0;
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < n; i++) r += fin[i] > e;
    if (SPLIT) {
        if (tid < n && r < top) listed[r] = e;
    } else if (tid < n && r < top) {
        uint32_t key = (uint32_t)(e >> 32), id = 0xffffffffu - (uint32_t)e;
        a.top_ids[row * top + r] = id;
        a.top_lp[row * top + r] = none ? NEG_INF : ((key ? logit_of(key) : __builtin_nanf("")) - m) - log_sum();
    }
}
KERNEL void __launch_bounds__(256) slm_logprobs_4(LogpArgs a) { logprobs_body<4, false>(a); }
KERNEL void __launch_bounds__(1024) slm_logprobs_16(LogpArgs a) { logprobs_body<16, false>(a); }
KERNEL void __launch_bounds__(256) slm_logprobs_split(LogpArgs a) { logprobs_body<4, true>(a); }

// A row's parts (at most 64) together: a workgroup a row. Of the parts' alternatives only those
// that reach the best part's last one can be among the row's.
KERNEL void __launch_bounds__(256) slm_logprobs_join(LogpArgs a) {
    __shared__ uint64_t fin[64 * SLM_TOP_MAX];
    __shared__ uint32_t nfin;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, top = a.top, parts = a.parts;
    const float* x = a.x + row * a.n;
    const float given = x[a.ids ? a.ids[row] : a.few[row]];
    if (tid == 0) nfin = 0;
    RowSum s{NEG_INF, 0.0f, 0.0f, 0.0f};
    if (lane < parts) {
        f4 q = *(const f4*)(a.part_sums + 4 * (row * parts + lane));
        s = RowSum{q.x, q.y, q.z, q.w};
    }
    const uint64_t* listed = a.part_top + row * parts * top;
    uint64_t e[64 * SLM_TOP_MAX / 256], last = 0;
    if (top) {
        if (lane < parts) last = listed[lane * top + top - 1];
#pragma unroll
        for (int u = 0; u < 64 * SLM_TOP_MAX / 256; u++) e[u] = tid + 256 * u < parts * top ? listed[tid + 256 * u] : 0;
    }
    const float m = wave_max(s.m);
    s.raise(m);
    s.c = wave_sum(s.c);
    s.S = wave_sum(s.S);
    s.E = wave_sum(s.E);
    const bool none = m == NEG_INF && s.S == 0.0f;
    const float logl = logf(s.c) + log1pf(s.S / s.c);
    if (tid == 0) {
        a.lp[row] = none ? NEG_INF : (given - m) - logl;
        if (a.ent) a.ent[row] = none ? 0.0f : (m - m) + logl - s.E / (s.c + s.S);
    }
    if (!top) return;
    for (int o = 32; o; o >>= 1) {
        uint64_t v = (uint64_t)__shfl_xor((unsigned long long)last, o);
        if (v > last) last = v;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 64 * SLM_TOP_MAX / 256; u++) {
        if (256 * u >= parts * top) break;
        const bool in = e[u] != 0 && e[u] >= last;
        uint64_t mask = __ballot(in);
        uint32_t at = 0;
        if (lane == 0 && mask) at = atomicAdd(&nfin, (uint32_t)__popcll(mask));
        at = (uint32_t)__builtin_amdgcn_readfirstlane(at) + lanes_below(mask);
        if (in) fin[at] = e[u];
    }
    __syncthreads();
    const int n = nfin;
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = fin[i];
        int r = 0;
#pragma unroll 8
        for (int k = 0; k < n; k++) r += fin[k] > mine;
        if (r < top) {
            uint32_t key = (uint32_t)(mine >> 32), id = 0xffffffffu - (uint32_t)mine;
            a.top_ids[row * top + r] = id;
            a.top_lp[row * top + r] = none ? NEG_INF : ((key ? logit_of(key) : __builtin_nanf("")) - m) - logl;
        }
    }
}
