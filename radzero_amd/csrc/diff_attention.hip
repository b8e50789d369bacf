// radzero_hip — differential attention: the difference of two softmax maps over the same values.
//
//   s_m[i][j] = scale * q_m[i] . k_m[j],  m = 1, 2 (the halves of a head's row);  hidden keys count for nothing
//   o[i] = sum_j (softmax(s_1[i])[j] - lambda softmax(s_2[i])[j]) v[j]
//   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
//   out[i] = out_scale * o[i] / sqrt(mean(o[i]^2) + eps) * w      (or out_scale * o[i] without a norm weight)
//
// One pass over the keys: each map keeps its own reference maximum m, sum l and sum of values O, all fp32; the maps meet when both sums are known.
//
// A wave owns 32 query rows (query-major, the heads that share a key head beside each other, so that one tile of keys serves all of them) and computes
// everything transposed on 32x32 MFMAs: S^T = K Q^T puts a query in a column = in a lane, so that its maximum, its sum and every rescale are
// that lane's own; P^T then is the B operand of O^T = V^T P^T as it stands in the registers, and one fragment of V^T serves both maps.
//   16-bit: 32x32x16, V^T fragments by transposing LDS reads, weights rounded to the type as any such product's operands are;  fp32: the same from three bf16
//   parts of every operand (rows), or 32x32x2, whose V^T fragments are plain reads of a row (keys).
// Three ways to share the work:
//   rows  4 waves x 32 rows on the same key tiles (16-bit: double-buffered in LDS, filled by LDS-DMA): many queries.  Bound by the matrix unit and the
//         exponentials, whose times add on a SIMD: bf16, 4 x 5330 tokens, 6 heads of 64: 539 us, 970 TFLOP/s executed (12 d per query and key)
//   keys  4 waves on the same 32 rows, every wave its own key tiles, joined in LDS: few queries over many keys.  Bound by HBM: 16 heads over 4 key heads, 8
//         caches of 18432 .. 32768 tokens, bf16: 91 us, 4.6 TB/s
//   few   a handful of rows without the matrix unit: fp32, 8 x 4 key heads x 8192 tokens: 58 us, 4.6 TB/s
// Each may also split the keys over workgroups; partial (O, m, l) then go through the workspace and a second kernel joins them.
#include <atomic>
#include <type_traits>

#include "rz_common.h"
#include "rz_kernels.h"

namespace rz {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 16-byte operand chunk: 8 elements of K per 32x32x16 step, or 4 of them as four 32x32x2 steps
template <typename T> struct Op;
template <> struct Op<bf16_t> {
    typedef bf16x8 chunk;
    static __device__ __forceinline__ f32x16 mma(chunk a, chunk b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Op<f16_t> {
    typedef f16x8 chunk;
    static __device__ __forceinline__ f32x16 mma(chunk a, chunk b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Op<float> {
    typedef f32x4 chunk;
    static __device__ __forceinline__ f32x16 mma(chunk a, chunk b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// x = hi + mid + lo exactly, three bf16 of 8 bits each: hi cut off (nothing overflows), mid rounded (its rest is 8 bits of either sign, below 2^-16 |x|).  A part
// below 2^-126 is lost; an infinity becomes NaN.
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&c)[3]) {
    u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint32_t x0 = __float_as_uint(x[e]), x1 = __float_as_uint(x[e + 1]);
        const float r0 = x[e] - __uint_as_float(x0 & 0xffff0000u), r1 = x[e + 1] - __uint_as_float(x1 & 0xffff0000u);
        const uint32_t mid = __builtin_bit_cast(uint32_t, bf16x2{(bf16_t)r0, (bf16_t)r1});
        w[0][e / 2] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
        w[1][e / 2] = mid;
        w[2][e / 2] = __builtin_amdgcn_perm(__float_as_uint(r1 - __uint_as_float(mid & 0xffff0000u)), __float_as_uint(r0 - __uint_as_float(mid << 16)), 0x07060302u);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) c[k] = __builtin_bit_cast(bf16x8, w[k]);
}

// 32 keys' weights as the product with the values takes them, and this lane's share of their sum
template <typename T, int PLANES> struct Weights {
    typename Op<T>::chunk w[1][2];
    __device__ __forceinline__ float set(const f32x16& p) {
#pragma unroll
        for (int u = 0; u < 2; ++u) w[0][u] = pack8<T>(p[8 * u], p[8 * u + 1], p[8 * u + 2], p[8 * u + 3], p[8 * u + 4], p[8 * u + 5], p[8 * u + 6], p[8 * u + 7]);
        // the sum of the rounded weights (they then add up to one), two of them to an instruction
        float t[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if constexpr (std::is_same<T, bf16_t>::value)
                    t[u] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{w[0][u][e], w[0][u][e + 1]}, bf16x2{(bf16_t)1.f, (bf16_t)1.f}, t[u], false);
                else
                    t[u] = __builtin_amdgcn_fdot2(f16x2{w[0][u][e], w[0][u][e + 1]}, f16x2{(f16_t)1.f, (f16_t)1.f}, t[u], false);
            }
        return t[0] + t[1];
    }
};
__device__ __forceinline__ float sum16(const f32x16& p) {
    float t[2] = {p[0], p[1]};
#pragma unroll
    for (int e = 2; e < 16; ++e) t[e & 1] += p[e];
    return t[0] + t[1];
}
template <> struct Weights<float, 1> {
    f32x16 w;
    __device__ __forceinline__ float set(const f32x16& p) {
        w = p;
        return sum16(p);
    }
};
template <> struct Weights<bf16_t, 3> {
    bf16x8 w[3][2];
    __device__ __forceinline__ float set(const f32x16& p) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8];
            bf16x8 c[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[8 * u + e];
            split8(x, c);
#pragma unroll
            for (int k = 0; k < 3; ++k) w[k][u] = c[k];
        }
        return sum16(p);
    }
};

// the larger of a lane and the lane 32 away, the sum of the two (both hold the same query)
__device__ __forceinline__ float pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS by 32-bit address: a fragment's place is a lane's constant XOR a constant of the step, plus an offset the instruction carries
template <typename V> __device__ __forceinline__ V lds_read(uint32_t at) { return *(const __attribute__((address_space(3))) V*)at; }
__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }
// A lane number that the compiler takes to be new: what is computed from it is computed where it stands, and does not hold registers across the loop.
__device__ __forceinline__ int fresh(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

template <typename T, int D> struct Shape {
    static constexpr int RB = 2 * D * (int)sizeof(T);          // bytes of a key's row: both maps' halves; the same for its values
    static constexpr int CH = RB / 16;                         // 16-byte chunks of a row
    static constexpr int NT = D * (int)sizeof(T) / 32;         // 32-byte steps of a score product
    static constexpr int NC = 2 * D / 32;                      // 32-column blocks of the values
    // LDS images: chunk c of row r stands at c ^ swz(r).  Scores read 32 rows x one chunk, 16 different rows must not meet in a bank (256 bytes):
    // with 128-byte rows two of them share the banks.  Transposing reads take 4 rows x 64 bytes at a time, fp32 reads 2 rows 4 apart x 128 bytes.
    static __device__ __forceinline__ int swz_k(int r) { return RB == 128 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int swz_v(int r) {
        if constexpr (sizeof(T) == 4) return ((r >> 2) & 1) << 3;
        else return RB == 128 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
    }
};

// How a workgroup shares the work.  MAPS: maps of a wave.  Two share a fragment of the values; head dim 128 would need 256 registers for both O, so there
// two waves take a map each.  BN: keys of a tile, 64 where the tile buffers of two workgroups fit the LDS, 32 for long rows.
// PLANES: fp32 products as 6 of the 9 of three bf16 parts each (what is left out is below 2^-22 |a||b|): 192 cycles of the matrix unit for 16 terms where
// 32x32x2 takes 512.  The parts are made once per tile, on the way to LDS.  The keys form, bound by HBM, keeps 32x32x2.
template <typename T, int D, bool KEYS> struct Form {
    static constexpr int PLANES = sizeof(T) == 4 && !KEYS ? 3 : 1;
    typedef typename std::conditional<PLANES == 3, bf16_t, T>::type M;         // what the matrix unit takes
    static constexpr int RB = Shape<M, D>::RB;
    static constexpr int MAPS = D == 128 ? 1 : 2;
    static constexpr int W = KEYS ? (RB <= 256 ? 4 : 2) : 4;   // keys: as many private double buffers of 32 keys as 128 KB hold
    static constexpr int BR = KEYS ? 32 : 32 * W * MAPS / 2;   // query rows
    static constexpr int BN = KEYS || PLANES == 3 ? 32 : RB <= 256 ? 64 : 32;
    static constexpr int TILE = PLANES * BN * RB, BUF = 2 * TILE;                // keys, then values
    static constexpr int NC = Shape<M, D>::NC;
    static constexpr int kTiles = PLANES == 3 ? BUF + 16 : 2 * BUF * (KEYS ? W : 1);
    // what the waves exchange at the end: keys, every wave's O, maxima and sums; one map per wave, the second maps' O
    static constexpr int kJoin = KEYS ? W * (2 * 2 * D * 32 + 64) * 4 : MAPS == 1 ? W / 2 * 2 * D * 32 * 4 : 0;
    static constexpr int kLds = kTiles > kJoin ? kTiles : kJoin;
    // workgroups that a CU holds: LDS, and 512 registers of a SIMD lane (two waves of the 16-bit forms, one of fp32; one more with 64-column values)
    static constexpr int kWaves = (sizeof(T) == 4 ? 1 : 2) + (D == 32);
    static constexpr int kPerCu = kWaves * 4 / W < 160 * 1024 / kLds ? kWaves * 4 / W : 160 * 1024 / kLds;
    static_assert(kLds <= 160 * 1024 && kPerCu >= 1, "LDS");
    static_assert(!KEYS || MAPS == 2, "one map per wave: rows only");
};

// Units of work: a block of query rows of a key head.  The first `full` of them run whole.  The rest, too few for the chip's places, lie end to end as one line of
// units * blocks blocks of keys, which `ranges` workgroups share evenly: a workgroup's stretch is at most a unit long and ends in one unit or goes on in the next.
// With lengths (`shared`) each unit is cut into as many pieces as its sequence's length earns it instead; those of one cut lie beside each other, row blocks
// innermost: they read the same keys.
struct Args {
    rz_diff_attention_args a;
    int group, rows, row_blocks;                               // heads per key head, query rows per key head, their blocks
    int units, full, cus;
    int blocks, ranges, each, more;                            // blocks of a unit, of 64 keys (keys form: as many as it has pieces); a workgroup's stretch: `each`, one more for the first `more` of them
    bool shared;
    int splits, least;                                         // shared: pieces of a unit on average, keys of a piece at least
    float c, up;                                               // scale * log2(e); f16_up
    int part_rows, slots;                                      // rows of a unit in the workspace, its places for pieces
    float* ws;
};
// workspace, floats: [slot][row] x {O1[2D], O2[2D]}, then m1, m2, l1, l2 of every row
__host__ __device__ inline int64_t parts(const Args& x) { return (int64_t)x.slots * x.part_rows; }
constexpr int kMostSplits = 64;                                // the join reads a row's pieces by one wave
__device__ __forceinline__ int range_begin(const Args& x, int g) { return g * x.each + min(g, x.more); }
__device__ __forceinline__ int range_of(const Args& x, int block) {
    const int wide = x.more * (x.each + 1);
    return block < wide ? block / (x.each + 1) : x.more + (block - wide) / x.each;
}

// a value that is the same in all lanes, into a scalar register (divisions run on the vector unit)
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The lengths of a batch of at most 64 share its batch * splits pieces per unit: lane b holds sequence b's.  1 + [its length / (the sum of all / (pieces - batch))]
// never add up to more, and no piece is longer than that share.  4 lengths of 7427 .. 11882: 85 -> 82 us; 8 of 18432 .. 32768, one query each: 97 -> 92 us.
struct Lengths {
    int n, splits, first;                                      // keys, pieces of each unit, the first piece
    __device__ __forceinline__ Lengths(const Args& x, int lane) {
        n = lane < x.a.batch ? min(max(x.a.kv_lens_dev[lane], 0), x.a.n_k) : 0;
        const uint32_t t = (uint32_t)(n + 63) >> 6;
        uint32_t sum = t;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const uint32_t most = (uint32_t)x.a.batch * (uint32_t)(x.splits - 1), share = max((sum + most - 1) / most, 1u);
        splits = lane < x.a.batch ? min(1 + (int)(t / share), min(max(n / x.least, 1), kMostSplits)) : 0;
        int end = splits * x.a.kv_heads * x.row_blocks;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(end, o, 64);
            if (lane >= o) end += below;
        }
        first = end - splits * x.a.kv_heads * x.row_blocks;
    }
};

struct Work {
    int rb, hk, b, n;                                          // row block, key head, sequence, its keys
    int lo, hi, of;                                            // the piece: [lo, hi) of `of` equal parts of the keys that the unit sees
    int slot, range, from, to;                                 // where it goes in the workspace; what is left of the workgroup's stretch
    bool any;
    __device__ __forceinline__ void unit(const Args& x, int u) {
        hk = scalar(u / x.row_blocks);
        rb = x.row_blocks - 1 - (u - hk * x.row_blocks);       // causal: the longest first
    }
    __device__ __forceinline__ void place(const Args& x, int u) {
        const int per_batch = x.a.kv_heads * x.row_blocks;
        b = scalar(u / per_batch);
        n = x.a.kv_lens_dev ? min(max(scalar(x.a.kv_lens_dev[b]), 0), x.a.n_k) : x.a.n_k;
        unit(x, u - b * per_batch);
    }
    __device__ __forceinline__ void next(const Args& x) {      // the stretch as far as it lies in one unit
        const int t = scalar(from / x.blocks);
        lo = from - t * x.blocks;
        hi = min(x.blocks, lo + to - from);
        of = x.blocks;
        slot = range + t;                                      // ascends by one at least from piece to piece; those of a unit are neighbours
        from += hi - lo;
        place(x, x.full + t);
    }
    __device__ __forceinline__ Work(const Args& x, int lane) {
        const int id = blockIdx.x;
        any = true;
        lo = slot = range = from = to = 0, hi = of = 1;
        if (x.shared) {
            const int per_batch = x.a.kv_heads * x.row_blocks;
            const Lengths all(x, lane);
            const int end = __builtin_amdgcn_readlane(all.first, 63) + __builtin_amdgcn_readlane(all.splits, 63) * per_batch;      // lanes behind the batch: no pieces
            any = id < end;
            if (!any) return;
            slot = xcd_remap(id, end);
            b = __popcll(__ballot(all.first <= slot && all.splits > 0)) - 1;         // first ascends, every sequence has a piece
            n = __builtin_amdgcn_readlane(all.n, b);
            of = __builtin_amdgcn_readlane(all.splits, b);
            const int local = slot - __builtin_amdgcn_readlane(all.first, b);
            lo = scalar(local / per_batch);
            hi = lo + 1;
            unit(x, local - lo * per_batch);
        } else if (id < x.full && x.a.causal && x.full == x.units) {
            // The longest first, a key head always on the same XCD if their number allows, and every second round over the CUs backwards: a CU that began with a long
            // unit goes on with a short one.  14 x 512 tokens, 12 heads of 32 over 4: 33.7 -> 28.2 us; 8192 tokens, 16 heads of 64 over 4: 564 -> 423 us.
            const int round = scalar(id / x.cus), i = id - round * x.cus, heads = x.a.kv_heads * x.a.batch;
            const int at = (round & 1) && (round + 1) * x.cus <= x.units && x.cus % 8 == 0 ? round * x.cus + x.cus - 8 - (i & ~7) + (i & 7) : id;
            const int t = scalar(at / heads);
            place(x, (at - t * heads) * x.row_blocks + t);
        } else if (id < x.full) {
            place(x, xcd_remap(id, x.full));
        } else {
            range = xcd_remap(id - x.full, x.ranges);
            from = range_begin(x, range);
            to = range_begin(x, range + 1);
            next(x);
        }
    }
    // the first key of part p: whole blocks of 64
    __device__ __forceinline__ int key(int p, int end) const {
        const int blocks = (end + 63) >> 6;
        return min(end, 64 * (blocks == of ? p : scalar((int)((double)blocks * p / of))));
    }
};

// lambda of query head h, by the whole wave
__device__ __forceinline__ float head_lambda(const rz_diff_attention_args& a, int h, int lane) {
    const float* p = a.lambda_qk_dev + (int64_t)h * a.lambda_head_stride;
    const int d = a.head_dim;
    float x1 = 0.f, x2 = 0.f;
    for (int e = lane; e < d; e += 64) {
        x1 = fmaf(p[e], p[d + e], x1);
        x2 = fmaf(p[2 * d + e], p[3 * d + e], x2);
    }
    return expf(wave_sum(x1)) - expf(wave_sum(x2)) + a.lambda_init;
}

// Steps of f16 end at 2^-24: what a smaller weight is rounded by, 2^-25 at most, is lost alike for all keys of a flat tail (65535 keys of weight 2^-25.05 beside one of 1: all of
// their 1.9e-3 of the sum).  The weight of a row's first reference is 2^up, so that n keys lose 2^(log2 n - 25 - up) = 2^-13 of its sum at most, a quarter of the rounding of the
// result; what is left of 2^16 is for maxima that grow.  Up to 4096 keys: 0.  10 at most: beyond 2^22 keys of one wave, n 2^-35.
// A constant 8 would cost rows whose scores spread widely more turns of the slow path (8 x 1370 tokens, 6 heads of 64, scores of deviation 4.5: 112 -> 144 us).
inline float f16_up(int n_k) {
    int up = 0;
    while (up < 10 && n_k > 4096 << up) ++up;
    return (float)up;
}

// bits of the keys below `n` (any n)
__device__ __forceinline__ uint64_t below(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// ---- one wave's 32 query rows ---------------------------------------------------------------------------------------------------
template <typename T, int D, int MAPS, int PLANES> struct Wave {             // T: what the matrix unit takes
    typedef Shape<T, D> S;
    typedef typename Op<T>::chunk chunk;
    typedef Weights<T, PLANES> W;
    static constexpr int NT = S::NT, NC = S::NC, RB = S::RB;
    static constexpr int PLANE = 32 * RB;   // bytes from one part of a tile to the next (PLANES == 3: tiles of 32 keys)

    chunk q[PLANES][MAPS][NT];
    f32x16 o[MAPS][NC];
    float m[MAPS], l[MAPS];                 // reference of the scores in log2 units: their maximum so far or an earlier one, less `up` (-inf: no key yet), this lane's share of the sum
    float c;                          // scale * log2(e)
    float up;                         // f16: the key of the reference has weight 2^up
    int h;                            // which half of every 8 keys the lane holds
    bool started;                     // every row has a reference maximum (wave-uniform)

    template <typename Q> __device__ __forceinline__ void init(const Args& x, const Q* qrow) {      // qrow: the first of the wave's maps
        c = x.c, up = std::is_same<T, f16_t>::value ? x.up : 0.f;
        started = false;
#pragma unroll
        for (int y = 0; y < MAPS; ++y) {
            m[y] = -INFINITY, l[y] = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (PLANES == 3) {
                    const f32x4* p = reinterpret_cast<const f32x4*>(qrow + (y * NT + t) * 16 + h * 8);
                    const f32x4 a = p[0], b = p[1];
                    chunk c[3];
                    split8({a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}, c);
#pragma unroll
                    for (int k = 0; k < 3; ++k) q[k][y][t] = c[k];
                } else q[0][y][t] = *reinterpret_cast<const chunk*>((const char*)qrow + (y * NT + t) * 32 + h * 16);
            }
#pragma unroll
            for (int cb = 0; cb < NC; ++cb)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[y][cb][e] = 0.f;
        }
    }

    // c + a b of fp32 operands in parts, the smallest products first
    static __device__ __forceinline__ f32x16 mma(const chunk (&a)[PLANES], const chunk (&b)[PLANES], f32x16 c) {
#pragma unroll
        for (int i = PLANES - 1; i >= 0; --i)
#pragma unroll
            for (int k = i; k >= 0; --k) c = Op<T>::mma(a[k], b[i - k], c);
        return c;
    }

    // S^T of the 32 keys at kt (k_lane() of their LDS image): register e is key 8 (e / 4) + 4 h + e % 4 of them
    static __device__ __forceinline__ uint32_t k_lane(int lane) {
        const int r = lane & 31;
        return r * RB + (((lane >> 5) ^ S::swz_k(r)) << 4);
    }
    __device__ __forceinline__ f32x16 scores(uint32_t kt, int y) const {
        f32x16 s = {};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            chunk k[PLANES], x[PLANES];
#pragma unroll
            for (int i = 0; i < PLANES; ++i) k[i] = lds_read<chunk>((kt ^ ((y * NT + t) << 5)) + i * PLANE), x[i] = q[i][y][t];
            s = mma(k, x, s);
        }
        return s;
    }

    // hides keys, and where `need` (a row's first keys, or weights that outgrew the reference) takes the maximum anew; O and l follow it
    __device__ __forceinline__ void recentre(f32x16& s, int y, uint32_t seen, bool need) {
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = (seen >> (8 * (e / 4) + e % 4)) & 1 ? s[e] : -INFINITY;
            mx = fmaxf(mx, s[e]);
        }
        const float top = pair_max(mx) * c - up, mn = need ? fmaxf(m[y], top) : m[y];
        if (__any(mn > m[y])) {
            const float f = m[y] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[y] - mn);            // m == mn: 1
            l[y] *= f;
#pragma unroll
            for (int cb = 0; cb < NC; ++cb)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[y][cb][e] *= f;
            m[y] = mn;
        }
    }

    __device__ __forceinline__ void exponentials(f32x16& s, float reference) const {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, -reference));
    }
    // a hidden key's weight to +0, whatever it is
    static __device__ __forceinline__ void hide(f32x16& p, uint32_t seen) {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = __uint_as_float(__float_as_uint(p[e]) & (uint32_t)__builtin_amdgcn_sbfe((int)seen, 8 * (e / 4) + e % 4, 1));
    }
    // The weights of 32 keys without a maximum: one that outgrows the reference shows in the sum, which 16 finite weights of f16 keep below 2^20 (rounding one beyond 65504
    // gives an infinity).  False: some row's did.
    // One run of instructions from the matrix products to what reads them: with a branch between, the fp32 kernels came out without the wait states they need.
    static constexpr float kMost = std::is_same<T, f16_t>::value ? 1048576.f : 32768.f;
    template <bool HIDE> __device__ __forceinline__ bool straight(uint32_t kt, uint32_t seen, W (&p)[MAPS], float (&t)[MAPS], bool& fine) const {
        f32x16 s[MAPS];
#pragma unroll
        for (int y = 0; y < MAPS; ++y) s[y] = scores(kt, y);
        fine = true;
#pragma unroll
        for (int y = 0; y < MAPS; ++y) {
            exponentials(s[y], m[y]);
            if constexpr (HIDE) hide(s[y], seen);
            t[y] = p[y].set(s[y]);
            fine = fine && t[y] <= kMost;
        }
        return !__any(!fine);
    }

    // O^T += V^T P^T, the values of 32 keys at vt (v_lane() of their LDS image)
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ s16x4 tr(uint32_t at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at); }
    static __device__ __forceinline__ uint32_t v_lane(int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 4) {
            const int col = lane & 31;
            return 4 * h * RB + (((col >> 2) ^ S::swz_v(4 * h)) << 4) + (col & 3) * 4;
        } else {
            // a transposing read gives lane x of 16 column x of 4 rows; the lanes of a group point at those rows, 4 lanes (32 bytes) each
            const int x = lane & 15, sub = (lane >> 4) & 1, r0 = 4 * h + (x >> 2);
            return r0 * RB + (((sub * 2 + ((x & 3) >> 1)) ^ S::swz_v(x >> 2)) << 4) + (x & 1) * 8;
        }
    }
    __device__ __forceinline__ void values(uint32_t vt, const W (&p)[MAPS]) {
        // fp32: the 32 keys' products are summed by themselves and join O once.  12 roundings at the size of O for every 32 keys (three parts), or 16 (32x32x2), would cost a
        // decimal over 3500 keys, and 65536 values of 1 + 2^-12 in two waves came out 2.1e-4 off.
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int cb = 0; cb < NC; ++cb) {
                f32x16 t[MAPS] = {};
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = lds_read<float>((vt ^ ((cb & 1) << 7)) + (cb >> 1) * 256 + (8 * (e / 4) + e % 4) * RB);
#pragma unroll
                    for (int y = 0; y < MAPS; ++y) t[y] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[y].w[e], t[y], 0, 0, 0);
                }
#pragma unroll
                for (int y = 0; y < MAPS; ++y)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[y][cb][e] += t[y][e];
            }
        } else if constexpr (PLANES == 3) {
#pragma unroll
            for (int cb = 0; cb < NC; ++cb) {
                f32x16 t[MAPS] = {};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t at = (vt ^ ((cb & 3) << 6)) + (cb >> 2) * 256 + 16 * u * RB;
                    chunk v[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) v[i] = __builtin_bit_cast(chunk, __builtin_shufflevector(tr(at + i * PLANE), tr(at + i * PLANE + 8 * RB), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int y = 0; y < MAPS; ++y) {
                        const chunk w[3] = {p[y].w[0][u], p[y].w[1][u], p[y].w[2][u]};
                        t[y] = mma(v, w, t[y]);
                    }
                }
#pragma unroll
                for (int y = 0; y < MAPS; ++y)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[y][cb][e] += t[y][e];
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int cb = 0; cb < NC; ++cb) {
                    const uint32_t at = (vt ^ ((cb & 3) << 6)) + (cb >> 2) * 256 + 16 * u * RB;
                    const chunk v = __builtin_bit_cast(chunk, __builtin_shufflevector(tr(at), tr(at + 8 * RB), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int y = 0; y < MAPS; ++y) o[y][cb] = Op<T>::mma(v, p[y].w[0][u], o[y][cb]);
                }
        }
    }

    // 32 keys that stand in LDS at kt, vt.  bits: those that somebody may see; rest: how many of them at most this lane's query sees (its causal end or length);
    // all: every query of the wave sees every key; odd: bit j = key j's values were not all finite (take_odd)
    __device__ __forceinline__ void block(uint32_t kt, uint32_t vt, uint32_t bits, int rest, bool all, uint32_t odd) {
        W p[MAPS];
        float t[MAPS];
        auto mine = [&] { return (bits & (uint32_t)below(rest)) >> (4 * h); };
        bool done = false, fine = true;
        if (started) done = all ? straight<false>(kt, 0, p, t, fine) : straight<true>(kt, mine(), p, t, fine);
        if (!done) {
            // Hardly ever taken: one map after the other, on fragments read anew.  What the path above holds is not kept for this one (registers).  A row is centred
            // anew for its own sake alone: its result does not depend on the rows beside it.
            bool need = !fine;
#pragma unroll
            for (int y = 0; y < MAPS; ++y) need = need || m[y] == -INFINITY;
            for (bool more = true; more;) {
                need = pair_max(need ? 1.f : 0.f) > 0.f;
                const uint32_t again = (uint32_t)fresh((int)kt);
                started = true;
                bool over = false;
#pragma unroll
                for (int y = 0; y < MAPS; ++y) {
                    __builtin_amdgcn_sched_barrier(0);
                    f32x16 s = scores(again, y);
                    recentre(s, y, mine(), need);
                    exponentials(s, m[y] == -INFINITY ? 0.f : m[y]);
                    t[y] = p[y].set(s);
                    over = over || !(t[y] <= kMost);
                    started = started && __all(m[y] > -INFINITY);
                }
                __builtin_amdgcn_sched_barrier(0);
                over = over && !need;                                      // seen while another row's first keys were: once more, for it
                more = __any(over);
                need = need || over;
            }
        }
        if (odd && mine() & odd >> (4 * h)) t[0] = __builtin_nanf("");
#pragma unroll
        for (int y = 0; y < MAPS; ++y) l[y] += t[y];
        values(vt, p);
    }
};

// LDS-DMA of 16 bytes per lane to 1 KB at `lds` (wave-uniform), from a uniform address plus a lane's offset, or from a lane's address.  Written in assembly: the
// compiler takes every LDS read behind its own builtin to depend on the copy and would wait for the next tile before it reads this one.  The copies have no
// output register; whoever reads the tile waits for all of them first (landed()).  One wait state between the write of m0 and its use.
__device__ __forceinline__ uint32_t lds_offset(char* lds) { return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds); }
__device__ __forceinline__ void lds_dma(char* lds, const char* base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_offset(lds)), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_dma(char* lds, const char* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_offset(lds)), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Fills LDS rows [0, ROWS) x RB bytes with keys j0 ..; wave w of W.  Keys that nobody may see (bits 0: hidden, or behind the last) are replaced by the first that
// somebody does: their weights are 0, and 0 * (what a hidden place holds) would not be.
template <typename T, int D, int ROWS, int W, bool VALUES> struct Stage {
    typedef Shape<T, D> S;
    static constexpr int per = 1024 / S::RB, N = ROWS * S::RB / 1024 / W;  // rows of one LDS-DMA instruction (1 KB), instructions of a wave
    static_assert(S::RB <= 1024 && ROWS * S::RB % (1024 * W) == 0, "tile and waves do not fit");
    const char* src;
    int64_t stride;
    int w;
    uint32_t in;                                                           // a lane's row, from the first of its instruction
    bool near;                                                             // every such offset fits 32 bits
    static __device__ __forceinline__ int swz(int r) { return VALUES ? S::swz_v(r) : S::swz_k(r); }

    __device__ __forceinline__ void init(const void* p, int64_t bytes, int wave, int lane) {
        src = (const char*)p, stride = bytes, w = wave;
        in = (uint32_t)(lane / S::CH) * (uint32_t)stride;
        near = stride >= 0 && stride < (1 << 28);
    }
    __device__ __forceinline__ void fill(char* lds, int j0, uint64_t bits, int lane) const {
        lane = fresh(lane);
        const int sub = lane / S::CH, cp = lane % S::CH ^ swz(sub);        // a row's XOR is that of its instruction's first row and its own place behind it
        if (near && bits == (ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1)) {        // every key: a uniform address and a lane's offset
            const char* base = src + (j0 + w * N * per) * stride;
#pragma unroll
            for (int i = 0; i < N; ++i, base += per * stride) {
                const int r0 = (w * N + i) * per;
                lds_dma(lds + r0 * S::RB, base, in + ((cp ^ swz(r0)) << 4));
            }
        } else {
            const int first = __builtin_ctzll(bits);
#pragma unroll 1
            for (int i = 0; i < N; ++i) {
                const int r0 = (w * N + i) * per, r = r0 + sub;
                const int key = j0 + ((bits >> r) & 1 ? r : first);
                lds_dma(lds + r0 * S::RB, src + (int64_t)key * stride + ((cp ^ swz(r0)) << 4));
            }
        }
    }
};

// The same for fp32 rows in parts: a thread holds its share of the next tile in registers while this one is worked on.
template <int D, int ROWS, int W> struct Parts {
    typedef Shape<bf16_t, D> S;
    static constexpr int N = ROWS * S::CH / (64 * W), per = 64 / S::CH;    // 8 columns of a row each; rows of a wave's instruction
    const char* src;
    int64_t stride;
    f32x4 x[N][2];

    __device__ __forceinline__ void init(const void* p, int64_t bytes) { src = (const char*)p, stride = bytes; }
    __device__ __forceinline__ void load(int j0, uint32_t bits, int wave, int lane) {
        const int first = __builtin_ctz(bits);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = (n * W + wave) * per + lane / S::CH, key = j0 + ((bits >> r) & 1 ? r : first);
            const f32x4* p = reinterpret_cast<const f32x4*>(src + (int64_t)key * stride + lane % S::CH * 32);
            x[n][0] = p[0], x[n][1] = p[1];
        }
    }
    // Returns, if asked to look for them, the keys (bits) whose values were not all finite; those values are zero then (as by take_odd).
    template <bool VALUES> __device__ __forceinline__ uint32_t store(char* lds, int wave, int lane, bool look) {
        uint32_t odd = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = (n * W + wave) * per + lane / S::CH;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[n][e / 4][e % 4];
            if (VALUES && look) {
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool finite = fabsf(v[e]) < INFINITY;
                    bad = bad || !finite;
                    v[e] = finite ? v[e] : 0.f;
                }
                const uint64_t b = __ballot(bad);
#pragma unroll
                for (int i = 0; i < per; ++i)
                    if (b >> (i * S::CH) & ((1ull << S::CH) - 1)) odd |= 1u << ((n * W + wave) * per + i);
            }
            bf16x8 c[3];
            split8(v, c);
            char* at = lds + r * S::RB + (((lane % S::CH) ^ (VALUES ? S::swz_v(r) : S::swz_k(r))) << 4);
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(at + k * ROWS * S::RB) = c[k];
        }
        return odd;
    }
};

// Values that are not finite, in a tile that not every query sees in full (causal): 0 * inf is not 0, so they would reach queries that must not see them.
// Returns the keys (bits) that hold any; take_odd then clears those values in LDS, and a query that does see such a key becomes NaN through its sum.
template <typename T> __device__ __forceinline__ bool odd_chunk(const u32x4& v) {
    constexpr uint32_t exponent = std::is_same<T, float>::value ? 0x7f800000u : std::is_same<T, bf16_t>::value ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t one = std::is_same<T, float>::value ? 0x00800000u : std::is_same<T, bf16_t>::value ? 0x00800080u : 0x04000400u;
    uint32_t t = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) t |= (v[e] & exponent) + one;              // an exponent of ones carries into the sign's place
    return t & (std::is_same<T, float>::value ? 0x80000000u : 0x80008000u);
}
template <typename T, int D, int ROWS> __device__ __forceinline__ uint64_t odd_keys(const char* vt, int lane) {
    typedef Shape<T, D> S;
    constexpr int N = ROWS * S::RB / 1024, per = 64 / S::CH;
    bool any = false;
#pragma unroll 4
    for (int n = 0; n < N; ++n) any |= odd_chunk<T>(*reinterpret_cast<const u32x4*>(vt + (n * 64 + lane) * 16));
    uint64_t keys = 0;
    if (__any(any))
#pragma unroll 1
        for (int n = 0; n < N; ++n) {
            const uint64_t b = __ballot(odd_chunk<T>(*reinterpret_cast<const u32x4*>(vt + (n * 64 + lane) * 16)));
#pragma unroll 1
            for (int r = 0; r < per; ++r)
                if (b >> (r * S::CH) & (S::CH == 64 ? ~0ull : (1ull << (S::CH & 63)) - 1)) keys |= 1ull << (n * per + r);
        }
    return keys;
}
template <typename T, int D, int ROWS> __device__ __forceinline__ void take_odd(char* vt, int lane) {
    constexpr int N = ROWS * Shape<T, D>::RB / (64 * (int)sizeof(T));
#pragma unroll 1
    for (int n = 0; n < N; ++n) {
        T* v = (T*)vt + n * 64 + lane;
        if (!(fabsf(to_f32(*v)) < INFINITY)) *v = (T)0.f;
    }
}

template <typename T, int D> struct Out {
    typedef Shape<T, D> S;
    // writes column blocks cb = first, first + step, ... of a finished row: 4 columns per 4 registers; `ss`: this lane's share of the sum of squares
    template <int STEP, int COUNT>
    static __device__ __forceinline__ void store(const Args& x, const f32x16 (&o)[COUNT], int first, int b, int i, int head, bool live, float factor, int h) {
        if (!live) return;
        T* out = (T*)x.a.out_dev + b * x.a.out_batch_stride + i * x.a.out_token_stride + head * x.a.out_head_stride;
#pragma unroll
        for (int n = 0; n < COUNT; ++n) {
            const int cb = first + n * STEP;
            if (cb >= S::NC) break;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = cb * 32 + 8 * g + 4 * h;
                f32x4 w = {factor, factor, factor, factor};
                if (x.a.norm_weight_dev) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] *= x.a.norm_weight_dev[col + e];
                }
                *reinterpret_cast<typename Traits<T>::vec4*>(out + col) = pack4<T>(o[n][4 * g] * w[0], o[n][4 * g + 1] * w[1], o[n][4 * g + 2] * w[2], o[n][4 * g + 3] * w[3]);
            }
        }
    }
};

// `inverse`: 1 over the first map's sum of weights, 0 where the query sees no key.  Such a row is all zeros, and stays so where an eps of 0 would make its factor infinite.
// (The sum itself in its place: 4 x 5330 tokens, bf16, 535 -> 542 us, other registers.)
__device__ __forceinline__ float norm_factor(const rz_diff_attention_args& a, float sum_of_squares, float inverse) {
    return !a.norm_weight_dev ? a.out_scale : inverse == 0.f ? 0.f : a.out_scale / sqrtf(sum_of_squares / (float)(2 * a.head_dim) + a.norm_eps);
}

template <typename T, int D, bool KEYS, typename F = Form<T, D, KEYS>>
__global__ __launch_bounds__(64 * F::W, F::kWaves) void diff_attention_kernel(const Args x) {
    typedef Shape<typename F::M, D> S;
    constexpr int W = F::W, BN = F::BN, TILE = F::TILE, BUF = F::BUF, NC = F::NC, MAPS = F::MAPS, PLANES = F::PLANES;
    typedef Wave<typename F::M, D, MAPS, PLANES> Rows;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const rz_diff_attention_args& a = x.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work at(x, lane);
    if (!at.any) return;
    for (;;) {
    const int map = MAPS == 1 ? wave & 1 : 0, group = KEYS ? 0 : MAPS == 1 ? wave >> 1 : wave;      // the wave's (first) map, its 32 rows of the unit
    const int row0 = at.rb * F::BR + 32 * group;

    const int n = at.n;
    const int shift = a.causal == RZ_CAUSAL_END ? n - a.n_q : 0;
    auto limit = [&](int query) -> int { return a.causal ? min(n, query + 1 + shift) : n; };       // keys that a query may see at most (may be negative)
    int lim;
    const int last = min((at.rb + 1) * F::BR, x.rows) - 1;
    const int end = max(limit(scalar(last / x.group)), 0);                         // of the workgroup
    const int wave_first = limit(scalar(min(row0, x.rows - 1) / x.group));         // keys that every query of the wave sees, but for hidden ones
    const int unit_first = limit(scalar(at.rb * F::BR / x.group));                 // the same of the workgroup
    const bool whole = at.lo == 0 && at.hi == at.of;
    const int begin = whole ? 0 : at.key(at.lo, end), stop = whole ? end : at.key(at.hi, end);

    Rows wv;
    wv.h = lane >> 5;
    {
        const int rr = min(row0 + (lane & 31), x.rows - 1), i = rr / x.group, head = at.hk * x.group + rr % x.group;
        lim = limit(i);
        wv.init(x, (const T*)a.q_dev + at.b * a.q_batch_stride + i * a.q_token_stride + head * a.q_head_stride + map * D);
    }

    const T *k_src = (const T*)a.k_dev + at.b * a.k_batch_stride + at.hk * a.k_head_stride, *v_src = (const T*)a.v_dev + at.b * a.v_batch_stride + at.hk * a.v_head_stride;
    const int64_t k_step = a.k_token_stride * (int64_t)sizeof(T), v_step = a.v_token_stride * (int64_t)sizeof(T);
    const int64_t* mask = a.mask_dev ? a.mask_dev + at.b * a.mask_batch_stride : nullptr;
    constexpr int STEP = KEYS ? BN * W : BN;
    const int j_first = begin + (KEYS ? wave * BN : 0);
    // Tile k of this workgroup (wave) begins at key j_first + k STEP.  Which of its keys the mask leaves: a bit each; lane n holds those of tile chunk + n, so that
    // a mask is read for 64 tiles at a time and an empty tile costs nothing.
    const int tiles = (max(stop - j_first, 0) + STEP - 1) / STEP;
    int chunk = mask ? -64 : 0;
    uint64_t words = ~0ull;
    auto read_mask = [&](int k) {
        chunk = k;
        const int here = min(tiles - k, 64);
        words = 0;
        constexpr int per = 64 / BN;                                       // tiles of one load
#pragma unroll 4
        for (int n = 0; n < here; n += per) {
            const int key = j_first + (k + n + (per > 1 ? lane / BN : 0)) * STEP + lane % BN;
            const uint64_t b = __ballot(key < stop && mask[key] != 0);
            words = lane == n ? (per > 1 ? b & 0xffffffffu : b) : per > 1 && lane == n + 1 ? b >> 32 : words;
        }
    };
    int k_next = 0;
    uint64_t bits_next = 0;
    auto find = [&] {                                                      // the first tile from k_next on that has a key
        bits_next = 0;
        while (k_next < tiles) {
            if (mask) {
                if (k_next >= chunk + 64) read_mask(k_next);
                const uint64_t some = __ballot(words != 0) >> (k_next - chunk);
                if (!some) {
                    k_next = chunk + 64;
                    continue;
                }
                k_next += __builtin_ctzll(some);
                bits_next = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)words, k_next - chunk) |
                            (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(words >> 32), k_next - chunk) << 32;
            } else {
                bits_next = below(min(stop - (j_first + k_next * STEP), BN));
            }
            return;
        }
    };
    // the queries are there before the first copy leaves: a wait for them inside the loop would be one for the copies too
#pragma unroll
    for (int k = 0; k < PLANES; ++k)
#pragma unroll
        for (int y = 0; y < MAPS; ++y)
#pragma unroll
            for (int t = 0; t < S::NT; ++t) asm volatile("" : "+v"(wv.q[k][y][t]));
    const uint32_t k_at = Rows::k_lane(lane) + map * (S::RB / 2), v_at = TILE + Rows::v_lane(lane);
    find();
    // a wave behind the last row only copies its share of the tiles
    const bool idle = !KEYS && row0 >= x.rows;
    if constexpr (PLANES == 3) {
        Parts<D, BN, W> keys, values;
        keys.init(k_src, k_step);
        values.init(v_src, v_step);
        uint32_t* odd_keys_of = (uint32_t*)(lds + BUF);                   // of each wave's share of a tile
        auto load = [&] {
            const int again = fresh(lane);
            keys.load(j_first + k_next * STEP, (uint32_t)bits_next, wave, again);
            values.load(j_first + k_next * STEP, (uint32_t)bits_next, wave, again);
        };
        auto run = [&](auto live) {
            while (bits_next) {
                const int j = j_first + k_next * STEP, again = fresh(lane);
                const uint32_t bits = (uint32_t)bits_next;
                const bool look = a.causal && j + BN > unit_first;        // the same for all waves that share the tile
                __syncthreads();                                          // the tile before has been read
                keys.template store<false>(lds, wave, again, false);
                const uint32_t here = values.template store<true>(lds + TILE, wave, again, look);
                if (look && lane == 0) odd_keys_of[wave] = here;
                __syncthreads();
                ++k_next;
                find();
                if (bits_next) load();
                uint32_t odd = 0;
                if (look)
#pragma unroll
                    for (int w = 0; w < W; ++w) odd |= (uint32_t)scalar((int)odd_keys_of[w]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (live) {                                     // the queries, operands of products alone, where only those reach: the vector unit works on O
#pragma unroll
                    for (int k = 0; k < PLANES; ++k)
#pragma unroll
                        for (int y = 0; y < MAPS; ++y)
#pragma unroll
                            for (int t = 0; t < S::NT; ++t) asm volatile("" : "+a"(wv.q[k][y][t]));
#pragma unroll
                    for (int y = 0; y < MAPS; ++y)
#pragma unroll
                        for (int cb = 0; cb < NC; ++cb) asm volatile("" : "+v"(wv.o[y][cb]));
                }
                if constexpr (live) wv.block(lds_address(lds) + k_at, lds_address(lds) + v_at, bits, lim - j, bits == ~0u && j + BN <= wave_first, odd);
            }
        };
        if (bits_next) load();
        if (!idle) run(std::true_type{});
        else run(std::false_type{});
    } else {
        Stage<T, D, BN, KEYS ? 1 : W, false> keys;
        Stage<T, D, BN, KEYS ? 1 : W, true> values;
        keys.init(k_src, k_step, KEYS ? 0 : wave, lane);
        values.init(v_src, v_step, KEYS ? 0 : wave, lane);
        auto fill = [&](char* buf, int j, uint64_t bits) {
            keys.fill(buf, j, bits, lane);
            values.fill(buf + TILE, j, bits, lane);
        };
        char* mine = lds + (KEYS ? wave * 2 * BUF : 0);
        if (bits_next) fill(mine, j_first + k_next * STEP, bits_next);
        int turn = 0;
        auto run = [&](auto live) {
            while (bits_next) {
                const int j = j_first + k_next * STEP;
                const uint64_t bits = bits_next;
                // everything asked for so far has landed; the other buffer's readers are done
                landed();
                if constexpr (!KEYS) __syncthreads();
                ++k_next;
                find();
                char* buf = mine + turn * BUF;
                if (bits_next) fill(mine + (turn ^ 1) * BUF, j_first + k_next * STEP, bits_next);
                const bool all = bits == below(BN) && j + BN <= wave_first;
                uint64_t odd = 0;
                if (a.causal && j + BN > unit_first) {                    // the same for all waves that share the tile
                    odd = odd_keys<T, D, BN>(buf + TILE, lane);
                    if (odd) {
                        if constexpr (!KEYS) __syncthreads();
                        take_odd<T, D, BN>(buf + TILE, lane);
                        if constexpr (KEYS) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        else __syncthreads();
                    }
                }
                if constexpr (live) {
                    const uint32_t kt = lds_address(buf) + k_at, vt = lds_address(buf) + v_at;
#pragma unroll
                    for (int kb = 0; kb < BN / 32; ++kb)
                        wv.block(kt + kb * 32 * S::RB, vt + kb * 32 * S::RB, (uint32_t)(bits >> (32 * kb)), lim - j - 32 * kb, all, (uint32_t)(odd >> (32 * kb)));
                }
                turn ^= 1;
            }
        };
        if (!idle) run(std::true_type{});
        else run(std::false_type{});
    }

    // ---- the rows' results ----
    const int again = fresh(lane), h = again >> 5, row = row0 + (again & 31), rr = min(row, x.rows - 1), i = rr / x.group, head = at.hk * x.group + rr % x.group;
    const bool live = row < x.rows;
    float l[MAPS], m[MAPS];
#pragma unroll
    for (int y = 0; y < MAPS; ++y) l[y] = pair_sum(wv.l[y]), m[y] = wv.m[y];
    // keys: block cb of O belongs to wave cb mod W from here on, summed over all waves
    constexpr int OWN = KEYS ? (NC + W - 1) / W : NC, OSTEP = KEYS ? W : 1;
    const int own0 = KEYS ? wave : 0;
    f32x16 o[MAPS][OWN];
    float* f = (float*)lds;
    if constexpr (KEYS) {
        // every wave's share against the rows' common maxima
        float* stat = f + W * 2 * NC * 16 * 64;                            // [wave][map][32] maxima, then sums
        __syncthreads();
        if (h == 0) stat[(wave * 2 + 0) * 32 + lane] = m[0], stat[(wave * 2 + 1) * 32 + lane] = m[1];
        __syncthreads();
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            float mx = -INFINITY;
            for (int w = 0; w < W; ++w) mx = fmaxf(mx, stat[(w * 2 + y) * 32 + (lane & 31)]);
            const float g = m[y] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[y] - mx);
            m[y] = mx;
            l[y] *= g;
#pragma unroll
            for (int cb = 0; cb < NC; ++cb)
#pragma unroll
                for (int e = 0; e < 16; ++e) f[(((wave * 2 + y) * NC + cb) * 16 + e) * 64 + lane] = wv.o[y][cb][e] * g;
        }
        __syncthreads();
        if (h == 0) stat[(wave * 2 + 0) * 32 + lane] = l[0], stat[(wave * 2 + 1) * 32 + lane] = l[1];
        __syncthreads();
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            l[y] = 0.f;
            for (int w = 0; w < W; ++w) l[y] += stat[(w * 2 + y) * 32 + (lane & 31)];
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                const int cb = min(own0 + k * OSTEP, NC - 1);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float t = 0.f;
                    for (int w = 0; w < W; ++w) t += f[(((w * 2 + y) * NC + cb) * 16 + e) * 64 + lane];
                    o[y][k][e] = t;
                }
            }
        }
        __syncthreads();                                                   // stat is used once more below
    } else {
#pragma unroll
        for (int y = 0; y < MAPS; ++y)
#pragma unroll
            for (int k = 0; k < OWN; ++k) o[y][k] = wv.o[y][k];
    }

    if (!whole) {
        const int64_t slot = (int64_t)at.slot * x.part_rows + (row - at.rb * F::BR);
        float* part = x.ws + slot * 4 * D;
        float* stat = x.ws + parts(x) * 4 * D + slot * 4;
        if (live) {
#pragma unroll
            for (int y = 0; y < MAPS; ++y)
#pragma unroll
                for (int k = 0; k < OWN; ++k) {
                    const int cb = own0 + k * OSTEP;
                    if (cb >= NC) break;
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<f32x4*>(part + (map + y) * 2 * D + cb * 32 + 8 * g + 4 * h) = f32x4{o[y][k][4 * g], o[y][k][4 * g + 1], o[y][k][4 * g + 2], o[y][k][4 * g + 3]};
                }
            if (h == 0 && own0 == 0) {
#pragma unroll
                for (int y = 0; y < MAPS; ++y) stat[map + y] = m[y], stat[2 + map + y] = l[y];
            }
        }
        if (KEYS || at.from == at.to) return;
        at.next(x);
        __syncthreads();                                                   // LDS is free for the next piece
        continue;
    }
    float lambda = 0.f;
    if (a.lambda_head_stride == 0) lambda = head_lambda(a, 0, lane);
    else
        for (int g = 0; g < x.group; ++g) {
            const float v = head_lambda(a, at.hk * x.group + g, lane);
            if (rr % x.group == g) lambda = v;
        }
    float r[MAPS];
#pragma unroll
    for (int y = 0; y < MAPS; ++y) r[y] = l[y] == 0.f ? 0.f : (map + y ? lambda : 1.f) / l[y];
    float ss = 0.f;
    if constexpr (MAPS == 1) {
        // the second map's O joins the first's in LDS
        __syncthreads();
        if (map) {
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) f[((group * NC + k) * 16 + e) * 64 + lane] = o[0][k][e] * r[0];
        }
        __syncthreads();
        if (map) return;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[0][k][e] = o[0][k][e] * r[0] - f[((group * NC + k) * 16 + e) * 64 + lane];
                ss = fmaf(o[0][k][e], o[0][k][e], ss);
            }
    } else {
#pragma unroll
        for (int k = 0; k < OWN; ++k)
            if (own0 + k * OSTEP < NC) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    o[0][k][e] = o[0][k][e] * r[0] - o[1][k][e] * r[1];
                    ss = fmaf(o[0][k][e], o[0][k][e], ss);
                }
            }
    }
    ss = pair_sum(ss);
    if constexpr (KEYS) {
        float* stat = f + W * 2 * NC * 16 * 64;
        if (h == 0) stat[wave * 32 + lane] = ss;
        __syncthreads();
        ss = 0.f;
        for (int w = 0; w < W; ++w) ss += stat[w * 32 + (lane & 31)];
    }
    Out<T, D>::template store<OSTEP, OWN>(x, o[0], own0, at.b, i, head, live, norm_factor(a, ss, r[0]), h);
    return;                                                                // a whole unit is a workgroup's only piece
    }
}

// a query row's result from both maps' O (a lane: 2 D / 64 neighbouring columns) and sums, by one wave
template <typename T, int D> __device__ __forceinline__ void finish_row(const Args& x, float (&o)[2][2 * D / 64], float l0, float l1, float lambda, int b, int i, int head, int lane) {
    constexpr int N = 2 * D / 64;
    const rz_diff_attention_args& a = x.a;
    const float r0 = l0 == 0.f ? 0.f : 1.f / l0, r1 = l1 == 0.f ? 0.f : lambda / l1;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        o[0][e] = o[0][e] * r0 - o[1][e] * r1;
        ss = fmaf(o[0][e], o[0][e], ss);
    }
    const float f = norm_factor(a, wave_sum(ss), r0);
    T* out = (T*)a.out_dev + b * a.out_batch_stride + i * a.out_token_stride + head * a.out_head_stride + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = from_f32<T>(o[0][e] * f * (a.norm_weight_dev ? a.norm_weight_dev[lane * N + e] : 1.f));
}

// Few query rows (R at a time) over many keys, bound by HBM: no matrix unit, whose 32 columns would stay empty.  D / 4 lanes take a key, 8 of its columns each: half of
// them the first map's, half the second's; 256 / D keys of a wave at a time, kFly such steps on their way.  Every place of a key keeps its own maxima, sums and O of all rows;
// they meet at the end, in the wave, then in LDS.  Weights stay fp32.
template <typename T, int D, int R> struct Few {
    static constexpr int W = 4, BR = R, LK = D / 4, H = LK / 2, KEYS = 64 / LK, kFly = R >= 4 ? 2 : 4;
    static constexpr int BN = KEYS * kFly;                     // keys of a wave's turn
    static constexpr int kPerCu = R == 1 ? 4 : R == 2 ? 3 : 2;                   // waves of a SIMD, too: registers
    static constexpr int kJoin = W * R * 4 * D * 4, kLds = kJoin + W * R * 4 * 4;
};
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), CTRL, 0xf, 0xf, true)); }
// the sum over the H lanes of a map (H = 4, 8, 16); the value of the other map's lanes, the same in all of them
template <int H> __device__ __forceinline__ float map_sum(float v) {
    v += dpp<0xB1>(v);                                         // lanes 1 apart, 2 apart, then mirrored in 8 and in 16
    v += dpp<0x4E>(v);
    if constexpr (H >= 8) v += dpp<0x141>(v);
    if constexpr (H >= 16) v += dpp<0x140>(v);
    return v;
}
template <int H> __device__ __forceinline__ float other_map(float v) {
    if constexpr (H == 4) return dpp<0x141>(v);
    else if constexpr (H == 8) return dpp<0x140>(v);
    else return __shfl_xor(v, H, 64);
}
template <typename T> struct Eight;                            // 8 columns as they lie in memory
template <> struct Eight<float> {
    f32x4 v[2];
    __device__ __forceinline__ void load(const float* p) { v[0] = reinterpret_cast<const f32x4*>(p)[0], v[1] = reinterpret_cast<const f32x4*>(p)[1]; }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[e / 4][e % 4];
    }
};
template <typename T> struct Eight {
    typename Op<T>::chunk v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const typename Op<T>::chunk*>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_f32((T)v[e]);
    }
};

template <typename T, int D, int R> __global__ __launch_bounds__(256, (Few<T, D, R>::kPerCu)) void diff_attention_few_kernel(const Args x) {
    typedef Few<T, D, R> F;
    constexpr int W = F::W, LK = F::LK, H = F::H, FLY = F::kFly, N = 2 * D / 64;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const rz_diff_attention_args& a = x.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Work at(x, lane);
    if (!at.any) return;
    const int shift = a.causal == RZ_CAUSAL_END ? at.n - a.n_q : 0;
    auto limit = [&](int row) -> int { return a.causal ? min(at.n, scalar(row / x.group) + 1 + shift) : at.n; };
    const int row0 = at.rb * R, rows = min(R, x.rows - row0);
    const int end = max(limit(row0 + rows - 1), 0), first = limit(row0);   // keys of the last row, of all rows
    const bool whole = at.lo == 0 && at.hi == at.of;
    const int begin = whole ? 0 : at.key(at.lo, end), stop = whole ? end : at.key(at.hi, end);

    const int col = lane % LK * 8, place = lane / LK;
    const int64_t* mask = a.mask_dev ? a.mask_dev + at.b * a.mask_batch_stride : nullptr;
    const T* k_src = (const T*)a.k_dev + at.b * a.k_batch_stride + at.hk * a.k_head_stride + col;
    const T* v_src = (const T*)a.v_dev + at.b * a.v_batch_stride + at.hk * a.v_head_stride + col;
    float q[R][8], o[R][2][8], m[R], l[R];
    int lim[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int rr = row0 + min(r, rows - 1), i = scalar(rr / x.group), head = at.hk * x.group + rr - i * x.group;
        Eight<T> e;
        e.load((const T*)a.q_dev + at.b * a.q_batch_stride + i * a.q_token_stride + head * a.q_head_stride + col);
        e.get(q[r]);
        lim[r] = limit(rr);
        m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) o[r][0][c] = o[r][1][c] = 0.f;
    }
    for (int j0 = begin + wave * F::BN; j0 < stop; j0 += W * F::BN) {
        Eight<T> kr[FLY], vr[FLY];
        bool seen[FLY];
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            const int j = j0 + u * F::KEYS + place, key = min(j, stop - 1);
            kr[u].load(k_src + key * a.k_token_stride);
            vr[u].load(v_src + key * a.v_token_stride);
            seen[u] = j < stop && (!mask || mask[key] != 0);
        }
        const bool edge = j0 + F::BN > first;                  // causal: keys that not every row sees
        float s[R][FLY];
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            float k[8];
            kr[u].get(k);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float t = 0.f;
#pragma unroll
                for (int c = 0; c < 8; ++c) t = fmaf(q[r][c], k[c], t);
                t = map_sum<H>(t) * x.c;
                s[r][u] = seen[u] && (!edge || j0 + u * F::KEYS + place < lim[r]) ? t : -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = s[r][0];
#pragma unroll
            for (int u = 1; u < FLY; ++u) top = fmaxf(top, s[r][u]);
            if (__any(top > m[r])) {
                const float mn = fmaxf(m[r], top), f0 = m[r] == mn ? 1.f : __builtin_amdgcn_exp2f(m[r] - mn), f1 = other_map<H>(f0);
                const float own = lane % LK < H ? f0 : f1, other = lane % LK < H ? f1 : f0;
                m[r] = mn;
                l[r] *= f0;
#pragma unroll
                for (int c = 0; c < 8; ++c) o[r][0][c] *= own, o[r][1][c] *= other;
            }
            const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int u = 0; u < FLY; ++u) {
                s[r][u] = __builtin_amdgcn_exp2f(s[r][u] - ref);
                l[r] += s[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            float v[8];
            vr[u].get(v);
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = seen[u] ? v[c] : 0.f;       // 0 * (what a hidden place holds) would not be 0
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float mine = s[r][u], theirs = other_map<H>(mine);
                const float p0 = lane % LK < H ? mine : theirs, p1 = lane % LK < H ? theirs : mine;
                if (edge) {
                    const bool sees = j0 + u * F::KEYS + place < lim[r];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float w = sees ? v[c] : 0.f;
                        o[r][0][c] = fmaf(p0, w, o[r][0][c]);
                        o[r][1][c] = fmaf(p1, w, o[r][1][c]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        o[r][0][c] = fmaf(p0, v[c], o[r][0][c]);
                        o[r][1][c] = fmaf(p1, v[c], o[r][1][c]);
                    }
                }
            }
        }
    }

    // the places of a wave, then the waves: O [wave][row][map][2 D], {m1, m2, l1, l2} [wave][row]
    float* f = (float*)lds;
    f32x4* stat = (f32x4*)(lds + F::kJoin);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float mx = m[r];
#pragma unroll
        for (int d = LK; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        const float g = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - mx), h = other_map<H>(g), g0 = lane % LK < H ? g : h, g1 = lane % LK < H ? h : g;
        float sum = l[r] * g;
#pragma unroll
        for (int d = LK; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
        const float mo = other_map<H>(mx), so = other_map<H>(sum);
        if (lane == 0) stat[wave * R + r] = f32x4{mx, mo, sum, so};
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                float t = o[r][y][c] * (y ? g1 : g0);
#pragma unroll
                for (int d = LK; d < 64; d <<= 1) t += __shfl_xor(t, d, 64);
                if (place == 0) f[((wave * R + r) * 2 + y) * 2 * D + col + c] = t;
            }
    }
    __syncthreads();
    for (int r = wave; r < rows; r += W) {
        f32x4 st[W];
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, t[2][N] = {};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            st[w] = stat[w * R + r];
            m0 = fmaxf(m0, st[w][0]), m1 = fmaxf(m1, st[w][1]);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float g0 = st[w][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[w][0] - m0), g1 = st[w][1] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[w][1] - m1);
            l0 = fmaf(st[w][2], g0, l0), l1 = fmaf(st[w][3], g1, l1);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                t[0][e] = fmaf(f[((w * R + r) * 2 + 0) * 2 * D + lane * N + e], g0, t[0][e]);
                t[1][e] = fmaf(f[((w * R + r) * 2 + 1) * 2 * D + lane * N + e], g1, t[1][e]);
            }
        }
        if (whole) {
            const int i = scalar((row0 + r) / x.group), head = at.hk * x.group + row0 + r - i * x.group;
            finish_row<T, D>(x, t, l0, l1, head_lambda(a, a.lambda_head_stride ? head : 0, lane), at.b, i, head, lane);
        } else {
            const int64_t slot = (int64_t)at.slot * x.part_rows + r;
            float* part = x.ws + slot * 4 * D + lane * N;
#pragma unroll
            for (int e = 0; e < N; ++e) part[e] = t[0][e], part[2 * D + e] = t[1][e];
            if (lane == 0) *reinterpret_cast<f32x4*>(x.ws + parts(x) * 4 * D + slot * 4) = f32x4{m0, m1, l0, l1};
        }
    }
}

// joins the pieces of a query row and head: one wave, a lane owns 2 D / 64 neighbouring columns of both maps
template <typename T, int D> __global__ __launch_bounds__(256) void diff_attention_join_kernel(const Args x, int block_rows) {
    constexpr int N = 2 * D / 64;
    const rz_diff_attention_args& a = x.a;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t tail = id / x.part_rows;
    if (tail >= x.units - x.full) return;
    const int per_batch = a.kv_heads * x.row_blocks, u = x.full + (int)tail, r = (int)(id - tail * x.part_rows), b = u / per_batch, unit = u - b * per_batch;
    const int row = (x.row_blocks - 1 - unit % x.row_blocks) * block_rows + r;
    if (row >= x.rows) return;
    const int i = row / x.group, head = unit / x.row_blocks * x.group + row % x.group;
    int first, step = 1, splits;
    if (x.shared) {
        const Lengths all(x, lane);
        splits = __shfl(all.splits, b, 64);
        first = __shfl(all.first, b, 64) + unit;
        step = per_batch;
    } else {
        const int t = (int)tail, g = range_of(x, t * x.blocks);
        splits = range_of(x, t * x.blocks + x.blocks - 1) - g + 1;
        first = g + t;
    }
    if (splits == 1) return;                                               // it ran whole
    const int64_t slot = (int64_t)first * x.part_rows + r, next = (int64_t)step * x.part_rows;
    const float* part = x.ws + slot * 4 * D + lane * N;
    const float* stat = x.ws + parts(x) * 4 * D + slot * 4;
    const float lambda = head_lambda(a, head, lane);
    f32x4 st = {-INFINITY, -INFINITY, 0.f, 0.f};
    if (lane < splits) st = *reinterpret_cast<const f32x4*>(stat + lane * next * 4);
    const float m0 = wave_max(st[0]), m1 = wave_max(st[1]);
    const float f0 = st[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[0] - m0), f1 = st[1] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[1] - m1);
    const float l0 = wave_sum(st[2] * f0), l1 = wave_sum(st[3] * f1);
    float o[2][N] = {};
    constexpr int kFly = 4;                                                // pieces on their way at a time; those behind the last: the last, of weight 0
    for (int s = 0; s < splits; s += kFly) {
        float p[kFly][2][N];
#pragma unroll
        for (int k = 0; k < kFly; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < N; ++e) p[k][y][e] = part[min(s + k, splits - 1) * next * 4 * D + y * 2 * D + e];
#pragma unroll
        for (int k = 0; k < kFly; ++k) {
            const bool there = s + k < splits;
            const float w0 = there ? __shfl(f0, s + k, 64) : 0.f, w1 = there ? __shfl(f1, s + k, 64) : 0.f;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                o[0][e] = fmaf(p[k][0][e], w0, o[0][e]);
                o[1][e] = fmaf(p[k][1][e], w1, o[1][e]);
            }
        }
    }
    finish_row<T, D>(x, o, l0, l1, lambda, b, i, head, lane);
}

int cu_count() {
    static const int n = [] {
        int dev = 0, v = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) v = 256;
        return v;
    }();
    return n;
}

// Hardly any rows: no matrix unit.  us, with it / without, three caches in turn, head dim 64: bf16, one row, 1 x 6 heads over 257 keys 11.9 / 10.4, 64 x 12 over 300 42 / 27; two
// rows 42 / 30, but 8 x 4 over 300 11.9 / 15.5: only where every CU has a unit; four rows 43 / 60.  fp32, four rows, 8 x 4 over 8192 126 / 63; eight as two blocks of four, each
// key read twice: 64 x 12 over 300, head dims 32, 64, 128 62 / 67, 133 / 93, 198 / 156, head dim 64 over long caches, 8 x 4 x 8192 126 / 82, 1 x 4 x 65536 132 / 96, 1 x 8 238 / 144
// (the pieces of both blocks beside each other, on one XCD, change that by -3 .. +5 %); twelve, 64 x 12 over 300, 62 / 100, 133 / 142, 199 / 237.
template <typename T, int D> bool few_form(const rz_diff_attention_args& a, int64_t rows) {
    return rows <= (sizeof(T) == 4 ? (D == 32 ? 4 : 8) : 1) || (rows == 2 && (int64_t)a.batch * a.kv_heads >= cu_count());
}
// Few rows: the waves of a workgroup share the rows and split the keys (head dims 32 and 64).
template <int D> bool keys_form(int64_t rows) { return D <= 64 && rows <= 32; }

// What the ways to run the last round cost, in microseconds: its longest workgroup, the partial results written and read again (5 TB/s), the join's launch.  A block of
// 64 keys takes a workgroup `alone` on its CU, or beside one or two others, as long as measured here with 256 of them on every CU, 1024 and 2048 keys.
template <typename T, int D> struct Cost {
    static constexpr double alone = sizeof(T) == 4 ? (D == 32 ? 4.75 : D == 64 ? 8.4 : 10.4) : D == 32 ? 1.65 : D == 64 ? 2.24 : 3.07;
    static constexpr double beside = sizeof(T) == 4 ? (D == 32 ? 3.7 : 0.) : D == 32 ? 0.69 : D == 64 ? 0.82 : 0.29;
    static constexpr double join = 5., second = 3.;            // a stretch over two units starts and ends twice
    static double run(int blocks, int64_t groups) { return blocks * (alone + beside * (double)((groups - 1) / cu_count())); }
    static double pieces(int64_t n, int rows) { return n * (rows * (4. * D * sizeof(float)) * 2 / 5e6); }
};

// The units fill the chip's places round by round.  The rest, if any, runs whole, in equal pieces or in stretches that share all places, whichever costs least.  Head dim 64,
// 6 heads, us, whole / equal / stretches: bf16 1370 tokens x 1 59 / 45 / 47, x 3 60 / 69 / 78, 2740 x 1 104 / 74 / 81, 2740 x 2 132 / - / 121, 3800 x 1 142 / 119 / 110;
// fp32 1370 x 1 184 / 87 / 81, x 2 189 / - / 132.
// Keys form: as many equal pieces as there are places, if they would leave more than a quarter of them idle, of at least 4 tiles for every wave.
template <typename T, int D, bool KEYS, typename F> Args make(const rz_diff_attention_args& a, void* ws) {
    Args x;
    x.a = a;
    x.c = a.scale * 1.44269504088896340736f;
    x.up = f16_up(a.n_k);
    x.group = a.heads / a.kv_heads;
    x.rows = a.n_q * x.group;
    x.row_blocks = (x.rows + F::BR - 1) / F::BR;
    x.units = x.row_blocks * a.kv_heads * a.batch;
    const int places = F::kPerCu * cu_count();
    x.cus = cu_count();
    x.full = x.units / places * places;
    const int tail = x.units - x.full;
    x.least = KEYS ? 4 * F::W * F::BN : 4 * F::BN;
    x.splits = 1, x.shared = false;
    x.blocks = (a.n_k + 63) / 64, x.ranges = x.each = x.more = x.slots = 0;
    x.part_rows = min(x.rows, F::BR);
    x.ws = (float*)ws;
    int equal = 1, ranges = 0;
    if (tail && x.blocks && (KEYS || !a.causal || !x.full)) {                          // causal rows: after a full round short units are left, whose places free up one by one
        // a unit has at most 2 + blocks / each pieces
        const int most = min(min(places / tail, x.blocks), kMostSplits);
        if constexpr (KEYS) {
            if ((int64_t)tail * 4 <= (int64_t)places * 3) equal = max(1, min(most, a.n_k / x.least));
        } else {
            typedef Cost<T, D> C;
            double best = C::run(x.blocks, tail);
            for (int k = 2; k <= most; ++k) {
                const double cost = C::run((x.blocks + k - 1) / k, (int64_t)tail * k) + C::pieces((int64_t)tail * k, x.part_rows) + C::join;
                if (cost < best) best = cost, equal = k;
            }
            const int64_t line = (int64_t)tail * x.blocks;
            const int r = (int)min((int64_t)places, line / ((x.blocks + kMostSplits - 3) / (kMostSplits - 2)));
            if (r > tail && line <= INT32_MAX && C::run((int)((line + r - 1) / r), r) + C::pieces(r + tail, x.part_rows) + C::join + C::second < best) ranges = r;
        }
    }
    if (x.full == 0 && a.kv_lens_dev && a.batch <= 64) {
        x.splits = equal, x.shared = equal > 1;
        x.slots = x.shared ? tail * equal : 0;
    } else if (equal > 1 || ranges) {
        if (!ranges) x.blocks = equal, ranges = tail * equal;              // each piece a stretch of its own
        const int64_t line = (int64_t)tail * x.blocks;
        x.ranges = ranges, x.each = (int)(line / ranges), x.more = (int)(line % ranges), x.slots = ranges + tail;
    }
    if (!x.shared && !x.ranges) x.full = x.units;
    return x;
}

int groups(const Args& x) { return x.shared ? x.slots : x.full + x.ranges; }

template <typename T, int D, bool KEYS, typename F> hipError_t launch(void (*k)(Args), const rz_diff_attention_args& a, void* ws, hipStream_t s) {
    const Args x = make<T, D, KEYS, F>(a, ws);
    if (F::kLds > 64 * 1024) {
        static std::atomic<uint64_t> told{0};                              // devices that know
        int dev = 0;
        if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
        if (dev >= 64 || !(told.load(std::memory_order_relaxed) >> dev & 1)) {
            if (hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, F::kLds); e != hipSuccess) return e;
            if (dev < 64) told.fetch_or(1ull << dev, std::memory_order_relaxed);
        }
    }
    const int tail = x.units - x.full;
    hipLaunchKernelGGL(k, dim3((unsigned)groups(x)), dim3(64 * F::W), F::kLds, s, x);
    if (hipError_t err = hipGetLastError(); err != hipSuccess || !tail) return err;
    hipLaunchKernelGGL((diff_attention_join_kernel<T, D>), dim3((unsigned)(((int64_t)tail * x.part_rows + 3) / 4)), dim3(256), 0, s, x, F::BR);
    return hipGetLastError();
}

// One of the forms for these sizes: use(KEYS, form, kernel).
template <typename T, int D, typename Use> auto with_form(const rz_diff_attention_args& a, Use use) {
    const int64_t rows = (int64_t)a.n_q * (a.heads / a.kv_heads);
    if (few_form<T, D>(a, rows)) {
        if (rows == 1) return use(std::true_type{}, Few<T, D, 1>{}, diff_attention_few_kernel<T, D, 1>);
        if (rows == 2) return use(std::true_type{}, Few<T, D, 2>{}, diff_attention_few_kernel<T, D, 2>);
        if constexpr (sizeof(T) == 4) return use(std::true_type{}, Few<T, D, 4>{}, diff_attention_few_kernel<T, D, 4>);
    }
    if constexpr (D <= 64)
        if (keys_form<D>(rows)) return use(std::true_type{}, Form<T, D, true>{}, diff_attention_kernel<T, D, true>);
    return use(std::false_type{}, Form<T, D, false>{}, diff_attention_kernel<T, D, false>);
}
template <typename T, int D> size_t workspace(const rz_diff_attention_args& a) {
    return with_form<T, D>(a, [&](auto keys, auto form, auto) { return (size_t)parts(make<T, D, decltype(keys)::value, decltype(form)>(a, nullptr)) * (4 * D + 4) * sizeof(float); });
}
template <typename T, int D> int workgroups(const rz_diff_attention_args& a) {
    return with_form<T, D>(a, [&](auto keys, auto form, auto) { return groups(make<T, D, decltype(keys)::value, decltype(form)>(a, nullptr)); });
}
template <typename T, int D> hipError_t launch(const rz_diff_attention_args& a, void* ws, hipStream_t s) {
    return with_form<T, D>(a, [&](auto keys, auto form, auto kernel) { return launch<T, D, decltype(keys)::value, decltype(form)>(kernel, a, ws, s); });
}
template <typename T> size_t workspace(const rz_diff_attention_args& a) {
    return a.head_dim == 32 ? workspace<T, 32>(a) : a.head_dim == 64 ? workspace<T, 64>(a) : workspace<T, 128>(a);
}
template <typename T> int workgroups(const rz_diff_attention_args& a) {
    return a.head_dim == 32 ? workgroups<T, 32>(a) : a.head_dim == 64 ? workgroups<T, 64>(a) : workgroups<T, 128>(a);
}
template <typename T> hipError_t launch(const rz_diff_attention_args& a, void* ws, hipStream_t s) {
    return a.head_dim == 32 ? launch<T, 32>(a, ws, s) : a.head_dim == 64 ? launch<T, 64>(a, ws, s) : launch<T, 128>(a, ws, s);
}

}  // namespace

size_t diff_attention_workspace_bytes(const rz_diff_attention_args& a) {
    return a.dtype == DT_F32 ? workspace<float>(a) : a.dtype == DT_BF16 ? workspace<bf16_t>(a) : workspace<f16_t>(a);
}

int diff_attention_workgroups(const rz_diff_attention_args& a) {
    return a.dtype == DT_F32 ? workgroups<float>(a) : a.dtype == DT_BF16 ? workgroups<bf16_t>(a) : workgroups<f16_t>(a);
}

hipError_t launch_diff_attention(const rz_diff_attention_args& a, void* ws, hipStream_t s) {
    return a.dtype == DT_F32 ? launch<float>(a, ws, s) : a.dtype == DT_BF16 ? launch<bf16_t>(a, ws, s) : launch<f16_t>(a, ws, s);
}

}  // namespace rz
