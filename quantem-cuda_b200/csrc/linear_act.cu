// linear_act.cu — matrix product with bias, activation and residual in its
// epilogue, and its backward, on the tcgen05 tensor cores.
//
//   z = (x W^T) [* x_scale * w_scale] + bias,   y = act(z) + residual
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = sum_rows dz
//
// The three products are D[m, n] = sum_k A[m, k] B[n, k] with A and B either
// K-major (the reduction index contiguous) or MN-major (the output index
// contiguous), so one kernel serves them: x, dz and W are K-major in x W^T and as
// dx's A; W as dx's B and both operands of dW are MN-major. All are read as they
// lie, no transposed copy is made.
//
// The backward needs dz = dy act'(z), in 16 bits as the next products' operand
// (at most half a step of its type off: dx and dW, themselves rounded to 16 bits,
// come out 1.4 times as far from their 64-bit values as from an unrounded dz; two
// 16-bit parts of dz would take that away at twice the work of both products), and
// its column sums, taken in fp32 before that rounding. Two ways to it:
// * z is formed again from x and W, and the epilogue multiplies dy by act'(z):
//   nothing is kept, nothing rounded but dz;
// * a large bf16 forward keeps act'(z) itself, which lies within [-0.13, 1.13],
//   in fp16 times 2^12: at most half a step off, 2^-11 of its value (an eighth of
//   dz's own rounding) down to 2^-26, and 2^-37 below; z in 16 bits would add as
//   much as dz's rounding. A pass over dy then gives dz. A training pass of 8192
//   rows of 1024 by 4096 (SiLU) takes 253 us so and 290 us with z formed again,
//   32768 rows of 512 by 512 121 and 134 us, 16384 of 2048 by 2048 413 and 501 us
//   (loops of a second in turn).
//
// fp16 has too few exponents for fp32 upstream gradients (a loss averaged over
// many values, a scaled one): there dz is multiplied by a power of two S that
// brings the largest |dy| to 2^14..2^15 (|act'| <= 1.13, so dz S stays below 2^16),
// and dz W and dz^T x are multiplied by 1/S, which rounds nothing. dz then has
// fp16's 11 bits next to the largest gradient, down to 2^-39 of it. The price
// is a pass over dy for its maximum.
//
// Accumulation is fp32 in tensor memory; bias, activation, residual and scales
// are applied to the fp32 value, which is rounded once.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ml_common.cuh"
#include "tc_common.cuh"

namespace qc {
namespace ml {

__device__ unsigned int g_ml_fault_word = 0;

namespace {

constexpr uint64_t kWaitLimitNs = 2000000000ull;  // 2 s per barrier wait
constexpr int kMaxDevices = 64;
constexpr float kKeptScale = 4096.f;  // of the kept derivative in fp16

// Value i of an array of `total` (debug build; always true otherwise). What TMA
// moves is bounded by its tensor map.
__device__ __forceinline__ bool in_array(long long i, long long total) {
    return QC_IN_BOUNDS(i, total, g_ml_fault_word);
}
// Values of `rows` rows of n values, ld apart.
__device__ __forceinline__ long long extent(long long rows, long long ld, int n) { return (rows - 1) * ld + n; }

// ── activations ──────────────────────────────────────────────────────────

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Phi, the normal distribution function, without erff's branches (its epilogue
// took 116 us on 262144 rows of 256 by 256, bf16).
//
// Forward: Phi(z) = 1/(1 + exp(-g(z))), g the log odds. g(z)/z is an even,
// smooth function: a polynomial of degree 7 in u = z^2 <= 30, fitted by the
// Lawson iteration (least squares, reweighted towards the least largest error)
// so that z Phi(z) is within 7.8e-8, and within 1.4e-3 of its own value as far as
// z = -5.47. Beyond, where it is below 1.3e-7, the absolute bound alone holds (4
// times the value at -6, 125 times at -7). Coefficients are scaled by -1/ln 2. One exponential and one reciprocal per value, no selection by sign.
// KEEP: the derivative Phi(z) + z phi(z) too, to d.
template <bool KEEP = false>
__device__ __forceinline__ void gelu(float &z0, float &z1, float *d = nullptr) {
    const Pair z = pair(z0, z1);
    float u0, u1, e0, e1;
    split(mul2(z, z), u0, u1);
    const Pair u = pair(fminf(u0, 30.f), fminf(u1, 30.f));
    Pair r = fma2(pair(8.26141724e-11f), u, pair(-9.84667015e-09f));
    r = fma2(r, u, pair(4.82880296e-07f));
    r = fma2(r, u, pair(-1.24473117e-05f));
    r = fma2(r, u, pair(0.000164565499f));
    r = fma2(r, u, pair(8.21615176e-05f));
    r = fma2(r, u, pair(-0.104823098f));
    r = fma2(r, u, pair(-2.30221295f));
    split(mul2(r, z), e0, e1);
    split(add2(pair(exp2_approx(e0), exp2_approx(e1)), pair(1.f)), e0, e1);
    const Pair cdf = pair(rcp_approx(e0), rcp_approx(e1));
    split(mul2(z, cdf), z0, z1);
    if constexpr (KEEP) {
        split(mul2(pair(u0, u1), pair(-0.72134752044448170f)), u0, u1);  // -z^2/2 / ln 2
        const Pair e = pair(exp2_approx(u0), exp2_approx(u1));
        split(fma2(mul2(z, pair(0.39894228040143268f)), e, cdf), d[0], d[1]);
    }
}

// Derivative: Phi(z) + z phi(z) needs e = exp(-z^2/2) as well, so Phi comes from
// the same e: Phi(-a) = e t P(t), t = 1/(1 + p a), where exp(a^2/2) Phi(-a) is
// smooth and falls like 1/a. P of degree 7 is within 9.1e-8 of it over
// 0 <= a <= 14 (beyond, e is 0 in fp32), fitted in the same way. Phi is formed as
// 1/2 + copysign(1/2 - Phi(-a), z), within 6e-8.
__device__ __forceinline__ void gelu_grad(float &z0, float &z1) {
    const Pair z = pair(z0, z1);
    float e0, e1, c0, c1;
    split(mul2(mul2(z, z), pair(-0.72134752044448170f)), e0, e1);  // -z^2/2 / ln 2
    const Pair e = pair(exp2_approx(e0), exp2_approx(e1));
    const Pair t = pair(rcp_approx(fmaf(fabsf(z0), 0.30448020f, 1.f)), rcp_approx(fmaf(fabsf(z1), 0.30448020f, 1.f)));
    Pair r = fma2(pair(0.036741964519023895f), t, pair(-0.15402236580848694f));
    r = fma2(r, t, pair(0.18878662586212158f));
    r = fma2(r, t, pair(-0.04037942737340927f));
    r = fma2(r, t, pair(0.12219109386205673f));
    r = fma2(r, t, pair(0.10294676572084427f));
    r = fma2(r, t, pair(0.1223057210445404f));
    r = fma2(r, t, pair(0.12142965942621231f));
    split(fma2(mul2(r, t), mul2(e, pair(-1.f)), pair(0.5f)), c0, c1);
    const Pair phi = add2(pair(copysignf(c0, z0), copysignf(c1, z1)), pair(0.5f));
    split(fma2(mul2(z, pair(0.39894228040143268f)), e, phi), z0, z1);
}

__device__ __forceinline__ float sigmoid(float z) { return rcp_approx(1.f + exp2_approx(z * -1.4426950408889634f)); }

template <int ACT>
__device__ __forceinline__ void act_fwd(float &z0, float &z1) {
    if constexpr (ACT == QC_ACT_RELU) {
        z0 = z0 < 0.f ? 0.f : z0;  // keeps a NaN
        z1 = z1 < 0.f ? 0.f : z1;
    }
    if constexpr (ACT == QC_ACT_SILU) {
        z0 *= sigmoid(z0);
        z1 *= sigmoid(z1);
    }
    if constexpr (ACT == QC_ACT_GELU) {
        gelu(z0, z1);
    }
}

// z to act(z), as act_fwd does, and act'(z) to d
template <int ACT>
__device__ __forceinline__ void act_both(float &z0, float &z1, float &d0, float &d1) {
    const float a = z0, b = z1;
    if constexpr (ACT == QC_ACT_GELU) {
        float d[2];
        gelu<true>(z0, z1, d);
        d0 = d[0], d1 = d[1];
    } else {
        act_fwd<ACT>(z0, z1);
    }
    if constexpr (ACT == QC_ACT_NONE) d0 = d1 = 1.f;
    if constexpr (ACT == QC_ACT_RELU) {
        d0 = a > 0.f ? 1.f : 0.f;
        d1 = b > 0.f ? 1.f : 0.f;
    }
    if constexpr (ACT == QC_ACT_SILU) {
        const float p0 = sigmoid(a), p1 = sigmoid(b);
        d0 = p0 + z0 * (1.f - p0);
        d1 = p1 + z1 * (1.f - p1);
    }
}

// z to act'(z)
template <int ACT>
__device__ __forceinline__ void act_grad(float &z0, float &z1) {
    if constexpr (ACT == QC_ACT_NONE) z0 = z1 = 1.f;
    if constexpr (ACT == QC_ACT_RELU) {
        z0 = z0 > 0.f ? 1.f : 0.f;
        z1 = z1 > 0.f ? 1.f : 0.f;
    }
    if constexpr (ACT == QC_ACT_SILU) {
        const float p0 = sigmoid(z0), p1 = sigmoid(z1);
        z0 = p0 * (1.f + z0 * (1.f - p0));
        z1 = p1 * (1.f + z1 * (1.f - p1));
    }
    if constexpr (ACT == QC_ACT_GELU) {
        gelu_grad(z0, z1);
    }
}

// ── the tiled product ────────────────────────────────────────────────────
//
// Persistent, one CTA per SM, 128 x BN output tiles, 18 warps:
//   warp 0     TMA loads of A (128 x 128 B) and B (BN x 128 B) into a ring;
//   warp 1     tcgen05.mma from the ring into one of two (BN = 256) or four
//              accumulators in tensor memory (the next tile's products run
//              under this tile's epilogue);
//   warps 2-17 epilogue, four groups of four warps (one per quarter of the
//              tensor memory lanes). The groups take the tiles' 128-byte-wide
//              column slabs in turn: accumulator -> registers -> bias,
//              activation, residual -> slab in shared memory -> TMA store. The
//              residual (dy in the backward) is fetched into the slab by TMA as
//              soon as the slab's last store has read it. With two groups of
//              two slabs each the epilogue issued in 45% of the cycles only.
// PAIR: two CTAs (a cluster on one TPC) work on 256 x BN tiles. Each loads its
// 128 rows of A and half of B's rows, and the leading CTA's matrix instructions
// read both halves: a CTA fetches 32 KB instead of 48 KB per 128 x 256 x 64
// products, which is what long reductions are bound by (16384 x 4096 x 4096 in
// bf16: 428 us, single CTAs 488 us, cold; 467 us in a loop of seconds).
// Rows and columns that no 16-byte boundary divides leave by warp-wide plain
// stores from the slab instead (and the residual comes in the same way).

// kActGradScaled is a form of its own for its fp32 dy times S: in kActGrad, the
// scale's branches alone cost 5 of 104 us on 262144 rows of 256 by 256 with GELU.
enum Epilogue { kForward = 0, kActGrad = 1, kPartial = 2, kForwardKeep = 3, kActGradScaled = 4 };
__host__ __device__ constexpr bool is_forward(int epi) { return epi == kForward || epi == kForwardKeep; }
__host__ __device__ constexpr bool is_act_grad(int epi) { return epi == kActGrad || epi == kActGradScaled; }
enum ResidualMode { kResNone = 0, kResTma = 1, kResWarp = 2, kResThread = 3 };

// Division of 0 <= n < 2^31 by a fixed d: with 2^p >= 2^31 d and mul = ceil(2^p/d),
// n mul / 2^p lies less than 1/d above n/d, so its whole part is n/d's.
struct Divisor {
    uint32_t d = 1, mul = 0, shift = 0;
    void set(uint32_t by) {
        d = by;
        int log = 0;
        while ((1ull << log) < by) ++log;
        mul = (uint32_t)(((1ull << (31 + log)) + by - 1) / by);
        shift = log > 0 ? log - 1 : 0;
    }
    __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};

struct Product {
    long long M;  // output rows
    int N, m_tiles, n_tiles, k_blocks, splits;
    Divisor by_split, by_span;  // tiles of one split, of one group of row tiles
    uint32_t idesc;
    const void *bias;
    const float *row_scale, *col_scale;
    const void *res;  // residual (forward) or dy (act grad)
    long long ld_res;
    void *y;  // plain-store outputs: contiguous [M, N]
    uint4 *kept;  // act'(z) kKeptScale in fp16: [row tile][64-column slab][quarter][8 columns][32 rows]
    void *colsum;  // [row tiles][N]: fp32 partial sums, or the sums themselves where there is one row tile
    // The largest finite |dy| as bits, or null: kActGradScaled forms dz S (and
    // divides its column sums by S), the products of dz S are divided by S.
    const unsigned int *dy_max;
    int colsum_type, bias_type, out_type, act, res_mode, tma_store;
};

// 8-column vectors of the kept derivative: 1024 per 128 rows and 64 columns
__host__ __device__ __forceinline__ long long kept_vectors(long long rows, int n) {
    return (rows + 127) / 128 * ((n + 63) / 64) * 1024;
}

// The power of two that takes m (bits of a finite |value|) to [2^14, 2^15), as
// far as it and its reciprocal are normal fp32 numbers; INV: its reciprocal.
template <bool INV>
__device__ __forceinline__ float gradient_scale(unsigned int m) {
    const int e = min(14 + 127 - (int)(m >> 23), 126);
    return __uint_as_float((unsigned int)(127 + (INV ? -e : e)) << 23);
}

constexpr int kGroups = 4;
constexpr int kThreads = 64 + 128 * kGroups;
constexpr int kSlabBytes = 128 * 128;
constexpr int kStageA = 128 * 128;

template <int BN, bool PAIR>
struct Geom {
    static constexpr int kRowsB = PAIR ? BN / 2 : BN;  // B's rows in this CTA
    static constexpr int kStage = kStageA + kRowsB * 128;
    static constexpr int kStages = kStage > 40000 ? 3 : kStage > 30000 ? 4 : 6;
    static constexpr int kAccs = BN == 256 ? 2 : 4;
};

template <int BN, bool PAIR>
struct ProductSmem {
    using G = Geom<BN, PAIR>;
    alignas(1024) unsigned char ring[G::kStages][G::kStage];
    alignas(1024) unsigned char slab[kGroups][kSlabBytes];
    alignas(16) float bias[4 * kGroups][64];
    alignas(16) float col_scale[4 * kGroups][64];
    float colsum[kGroups][2][4][64];  // [group][parity][warp][column]
    uint64_t full[G::kStages], empty[G::kStages];
    uint64_t acc_full[G::kAccs], acc_empty[G::kAccs];
    uint64_t res_full[kGroups];
    uint32_t tmem;
    int gave_up;
};

// Waits for a phase of `bar`, for 2 s at most; a wait that gives up sets the
// fault word and `gave_up`, after which no wait of the CTA lingers. The
// epilogue then runs through its remaining slabs (so that every thread meets
// every barrier), fills them with NaN, and the kernel ends with the fault word set.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *gave_up) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*gave_up) return false;
        if (global_timer_ns() - t0 > kWaitLimitNs) {
            *gave_up = 1;
            atomicOr(&g_ml_fault_word, QC_FAULT_TMA_WAIT);
            return false;
        }
    }
    return true;
}
// Waits for copies or products still in flight before the CTA leaves.
__device__ __forceinline__ bool drain(uint64_t *bar, uint32_t parity) {
    if (mbar_wait_bounded(bar, parity, kWaitLimitNs)) return true;
    atomicOr(&g_ml_fault_word, QC_FAULT_TMA_WAIT);
    return false;
}
constexpr uint32_t kNaNBits = 0xffffffffu;  // two NaN in 16 bits

// Tiles go to the CTAs (pairs) in groups of 2048 rows, rows fastest, so that the
// tiles in flight share rows of A and of B in L2. m counts 128 or 256 rows.
template <bool PAIR>
__device__ __forceinline__ void tile_of(const Product &p, int t, int &m, int &n, int &s) {
    constexpr int kSpan = PAIR ? 8 : 16;
    s = p.by_split.of(t);
    const int u = t - s * (int)p.by_split.d;
    const int g = p.by_span.of(u), r = u - g * (int)p.by_span.d;
    const int first = g * kSpan, rows = min(kSpan, p.m_tiles - first);
    n = rows == kSpan ? r / kSpan : r / rows;
    m = first + r - n * rows;
}
__device__ __forceinline__ void k_range(const Product &p, int s, int &k0, int &k1) {
    k0 = (int)((long long)s * p.k_blocks / p.splits);
    k1 = (int)((long long)(s + 1) * p.k_blocks / p.splits);
}

// byte offset of 16-byte chunk `c` of row `row` in a 128-byte-swizzled slab
__device__ __forceinline__ uint32_t slab_at(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }

__device__ __forceinline__ void unpack8(uint4 q, int type, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == QC_BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
__device__ __forceinline__ uint4 pack8(const float *v, int type) {
    if (type == QC_BF16)
        return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    return make_uint4(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7]));
}

// 32 columns of one row: v holds the accumulators and leaves as what goes into
// the slab. `chunk0`: the slab's first 16-byte chunk of these columns.
// GRAD: a product of dz.
template <int EPI, int ACT, bool GRAD>
__device__ __forceinline__ void epilogue_32(const Product &p, float (&v)[32], unsigned char *slab, int row, int chunk0,
                                            const float *bias, const float *col_scale, float row_scale,
                                            const float *dy_row, int dy_left, uint4 *kept) {
    const bool wide = EPI == kPartial || p.out_type == QC_F32;
    if constexpr (GRAD) {
        if (p.dy_max) {
            const float s = gradient_scale<true>(*p.dy_max);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= s;
        }
    }
    if constexpr (EPI != kPartial) {
        if (p.row_scale) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = v[i] * row_scale * col_scale[i];  // the scales' product may leave fp32
        }
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += bias[i];
        }
    }
    if constexpr (EPI == kForwardKeep) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) act_both<ACT>(v[8 * c + i], v[8 * c + i + 1], d[i], d[i + 1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= kKeptScale;
            if (kept && in_array(kept + 32 * c - p.kept, kept_vectors(p.M, p.N))) kept[32 * c] = pack8(d, QC_F16);
        }
    }
    if constexpr (is_forward(EPI)) {
        if constexpr (EPI == kForward) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) act_fwd<ACT>(v[i], v[i + 1]);
        }
        if (p.res_mode != kResNone) {
            if (wide) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float4 q = *reinterpret_cast<const float4 *>(slab + slab_at(row, chunk0 + c));
                    v[4 * c] += q.x, v[4 * c + 1] += q.y, v[4 * c + 2] += q.z, v[4 * c + 3] += q.w;
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float r[8];
                    unpack8(*reinterpret_cast<const uint4 *>(slab + slab_at(row, chunk0 + c)), p.out_type, r);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[8 * c + i] += r[i];
                }
            }
        }
    }
    if constexpr (is_act_grad(EPI)) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) act_grad<ACT>(v[i], v[i + 1]);
        if (p.res_mode == kResThread) {
            if constexpr (EPI == kActGradScaled) {
                const float s = gradient_scale<false>(*p.dy_max);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= s;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] = i < dy_left && in_array(dy_row + i - static_cast<const float *>(p.res), extent(p.M, p.ld_res, p.N))
                           ? v[i] * dy_row[i]
                           : 0.f;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float r[8];
                unpack8(*reinterpret_cast<const uint4 *>(slab + slab_at(row, chunk0 + c)), p.out_type, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * c + i] *= r[i];
            }
        }
    }
    if (wide) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float4 *>(slab + slab_at(row, chunk0 + c)) =
                make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4 *>(slab + slab_at(row, chunk0 + c)) = pack8(v + 8 * c, p.out_type);
    }
}

// Sums of 32 columns over the warp's 32 rows: lane l leaves with column l's.
__device__ __forceinline__ float column_sums(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    return v[0];
}

// One slab's columns between global memory and this warp's 32 slab rows, lanes
// along the columns, for layouts that TMA cannot tile.
template <bool LOAD>
__device__ __forceinline__ void slab_warp_copy(const Product &p, unsigned char *slab, void *global, long long ld,
                                               long long m0, int row0, int col0, int lane) {
    const bool wide = p.out_type == QC_F32;
    const int rows = (int)min(32ll, p.M - (m0 + row0)), cols = min(wide ? 32 : 64, p.N - col0);
    const long long room = extent(p.M, ld, p.N);
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
        const int row = row0 + r;
        const long long at = (m0 + row) * ld + col0;
        if (wide) {
            if (lane < cols && in_array(at + lane, room)) {
                float *s = reinterpret_cast<float *>(slab + slab_at(row, lane >> 2)) + (lane & 3);
                float *g = static_cast<float *>(global) + at + lane;
                if constexpr (LOAD) *s = *g;
                else *g = *s;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = lane + 32 * h;
                if (c < cols && in_array(at + c, room)) {
                    unsigned short *s = reinterpret_cast<unsigned short *>(slab + slab_at(row, c >> 3)) + (c & 7);
                    unsigned short *g = static_cast<unsigned short *>(global) + at + c;
                    if constexpr (LOAD) *s = *g;
                    else *g = *s;
                }
            }
        }
    }
}

template <bool F8, bool A_MN, bool B_MN, int BN, int EPI, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_r,
                   const __grid_constant__ Product p) {
    using G = Geom<BN, PAIR>;
    using Smem = ProductSmem<BN, PAIR>;
    extern __shared__ unsigned char raw[];
    Smem &sm = *reinterpret_cast<Smem *>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
    constexpr int S = G::kStages;
    constexpr uint32_t kTmemCols = G::kAccs * BN;
    constexpr uint32_t A = G::kAccs;
    constexpr int kStep = F8 ? 128 : 64;  // reduction steps per ring stage
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = p.m_tiles * p.n_tiles * p.splits;
    const int rank = PAIR ? (int)tc::cluster_rank() : 0;
    const int first_tile = PAIR ? blockIdx.x / 2 : blockIdx.x, tile_step = PAIR ? gridDim.x / 2 : gridDim.x;
    const bool wide = EPI == kPartial || p.out_type == QC_F32;
    const int slab_cols = wide ? 32 : 64, slabs = BN / slab_cols;
    constexpr int kLogSlabs16 = BN == 256 ? 2 : BN == 128 ? 1 : 0;
    const int log_slabs = kLogSlabs16 + wide;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int i = 0; i < (int)A; ++i) {
            mbar_init(&sm.acc_full[i], 1);
            mbar_init(&sm.acc_empty[i], (PAIR ? 8 : 4) * slabs);
        }
        for (int i = 0; i < kGroups; ++i) mbar_init(&sm.res_full[i], 1);
        sm.gave_up = 0;
        fence_mbar_init();
        prefetch_tensor_map(&map_a);
        prefetch_tensor_map(&map_b);
    }
    if (warp == 1) tc::tmem_alloc<PAIR>(&sm.tmem, kTmemCols);
    tc::fence_before();
    __syncwarp();
    if constexpr (PAIR) tc::cluster_sync();
    else __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sm.tmem);

    if (warp == 0) {
        if (lane == 0) {
            uint32_t q = 0;
            bool ok = true;
            for (int t = first_tile; t < total && ok; t += tile_step) {
                int m, n, s, k0, k1;
                tile_of<PAIR>(p, t, m, n, s);
                k_range(p, s, k0, k1);
                const int row = (PAIR ? 2 * m + rank : m) * 128, col = n * BN + rank * G::kRowsB;
                for (int k = k0; k < k1; ++k, ++q) {
                    const int st = q % S;
                    if (!(ok = wait(&sm.empty[st], ((q / S) & 1) ^ 1, &sm.gave_up))) break;
                    const uint32_t a = smem_addr(sm.ring[st]), b = a + kStageA;
                    // a pair's loads all complete on the leading CTA's barrier
                    if (rank == 0) mbar_arrive_expect_tx(&sm.full[st], (PAIR ? 2 : 1) * G::kStage);
                    const uint32_t bar = PAIR ? tc::cluster_addr(&sm.full[st], 0) : 0;
                    auto load = [&](uint32_t dst, const CUtensorMap *map, int x, int y) {
                        if constexpr (PAIR) tc::load_2d_pair(dst, map, x, y, bar);
                        else tc::load_2d(dst, map, x, y, &sm.full[st]);
                    };
                    if constexpr (A_MN) {
                        load(a, &map_a, row, k * 64);
                        load(a + 8192, &map_a, row + 64, k * 64);
                    } else {
                        load(a, &map_a, k * kStep, row);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int h = 0; h < G::kRowsB / 64; ++h) load(b + h * 8192, &map_b, col + 64 * h, k * 64);
                    } else {
                        load(b, &map_b, k * kStep, col);
                    }
                }
            }
            // every load has landed, and the products have read it, before
            // this thread leaves (in a pair they signal both CTAs)
            for (uint32_t i = q > S ? q - S : 0; i < q; ++i) drain(&sm.empty[i % S], (i / S) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t q = 0, it = 0;
            bool ok = true;
            for (int t = first_tile; t < total && ok; t += tile_step, ++it) {
                int m, n, s, k0, k1;
                tile_of<PAIR>(p, t, m, n, s);
                k_range(p, s, k0, k1);
                const uint32_t acc = it % A, d = tmem + acc * BN;
                if (!(ok = wait(&sm.acc_empty[acc], ((it / A) & 1) ^ 1, &sm.gave_up))) break;
                tc::fence_after();
                for (int k = k0; k < k1; ++k, ++q) {
                    const int st = q % S;
                    if (!(ok = wait(&sm.full[st], (q / S) & 1, &sm.gave_up))) break;
                    tc::fence_after();
                    const uint32_t a = smem_addr(sm.ring[st]);
                    const uint64_t da = tc::operand_desc(a, A_MN ? 8192 : 16);
                    const uint64_t db = tc::operand_desc(a + kStageA, B_MN ? 8192 : 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        tc::mma<F8, PAIR>(d, da + j * (A_MN ? 128 : 2), db + j * (B_MN ? 128 : 2), p.idesc,
                                          k > k0 || j > 0);
                    tc::mma_commit<PAIR>(&sm.empty[st]);
                }
                if (ok) tc::mma_commit<PAIR>(&sm.acc_full[acc]);  // else the epilogue's wait gives up too
            }
            // the last products have finished reading the ring: the final
            // commits' barriers complete only then
            for (uint32_t i = q > S ? q - S : 0; i < q; ++i) drain(&sm.empty[i % S], (i / S) & 1);
        }
        __syncwarp();
    } else {
        const int ew = warp - 2, group = ew >> 2, quarter = warp & 3;
        const bool leader = (ew & 3) == 0 && lane == 0;
        const int row0 = quarter * 32, row = row0 + lane;
        const int my_tiles = total > first_tile ? (total - 1 - first_tile) / tile_step + 1 : 0;
        // The group's j-th unit (a slab of a tile). In turn over all groups; but
        // with dy to fetch in a memory-bound product, group g takes slabs g%2,
        // g%2 + 2, ... of every second tile: while one pair of groups computes,
        // the other's loads and stores are under way (115 -> 107 us on 262144
        // rows of 256 by 256 with GELU; the forward, 65 us, takes 71 us so).
        const bool in_turn = !is_act_grad(EPI) || PAIR || slabs < 4;
        auto unit = [&](int j, int &it, int &slab) {
            if (!in_turn) {
                it = (j >> (log_slabs - 1)) * 2 + (group >> 1);
                slab = (j & (slabs / 2 - 1)) * 2 + (group & 1);
            } else {
                it = (group + j * kGroups) >> log_slabs;
                slab = (group + j * kGroups) & (slabs - 1);
            }
            return it < my_tiles;
        };
        float *bias_sh = sm.bias[ew], *scale_sh = sm.col_scale[ew];
        unsigned char *buf = sm.slab[group];

        uint32_t fetched = 0;
        auto fetch = [&](int j) {  // leader: residual of the group's j-th unit into the slab
            int it, slab, m, n, s;
            if (!unit(j, it, slab) || *reinterpret_cast<volatile int *>(&sm.gave_up)) return;
            ++fetched;
            tile_of<PAIR>(p, first_tile + it * tile_step, m, n, s);
            if constexpr (PAIR) m = 2 * m + rank;
            mbar_arrive_expect_tx(&sm.res_full[group], kSlabBytes);
            tc::load_3d(smem_addr(buf), &map_r, n * BN + slab * slab_cols, m * 128, 0, &sm.res_full[group]);
        };
        const bool tma_res = EPI != kPartial && p.res_mode == kResTma;
        if (leader && tma_res) fetch(0);

        // the next unit's bias and scales, loaded while this one is computed
        struct {
            float bias[2] = {0.f, 0.f}, scale[2] = {0.f, 0.f}, row_scale = 0.f;
        } ahead;
        auto look_ahead = [&](int j) {
            int it, slab, m, n, s;
            if (!(p.bias || p.row_scale) || !unit(j, it, slab)) return;
            tile_of<PAIR>(p, first_tile + it * tile_step, m, n, s);
            if constexpr (PAIR) m = 2 * m + rank;
            const int c = n * BN + slab * slab_cols + lane;
            const long long r = (long long)m * 128 + row;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool in = c + 32 * h < p.N && in_array(c + 32 * h, p.N);
                if (p.bias) ahead.bias[h] = in ? load_any(p.bias, c + 32 * h, p.bias_type) : 0.f;
                if (p.row_scale) ahead.scale[h] = in ? p.col_scale[c + 32 * h] : 0.f;
            }
            if (p.row_scale) ahead.row_scale = r < p.M && in_array(r, p.M) ? p.row_scale[r] : 0.f;
        };
        if constexpr (EPI != kPartial) look_ahead(0);

        int it, slab;
        bool sound = true;  // no wait of this thread has given up (a later phase of the same parity says nothing)
        for (int j = 0; unit(j, it, slab); ++j) {
            int m, n, s;
            tile_of<PAIR>(p, first_tile + it * tile_step, m, n, s);
            if constexpr (PAIR) m = 2 * m + rank;
            const int col0 = n * BN + slab * slab_cols;
            const long long m0 = (long long)m * 128;
            float row_scale = 1.f;
            if constexpr (EPI != kPartial) {
                if (p.bias) {
                    bias_sh[lane] = ahead.bias[0];
                    bias_sh[lane + 32] = ahead.bias[1];
                }
                if (p.row_scale) {
                    scale_sh[lane] = ahead.scale[0];
                    scale_sh[lane + 32] = ahead.scale[1];
                    row_scale = ahead.row_scale;
                }
                look_ahead(j + 1);
            }
            // the slab may be written: its last store has read it. The leader
            // waited for that before it fetched the residual, else here.
            if (p.tma_store && !tma_res) {
                if (leader) tc::store_wait_read();
                tc::named_barrier(1 + group, 128);
            }
            if (EPI != kPartial && p.res_mode == kResWarp)
                slab_warp_copy<true>(p, buf, const_cast<void *>(p.res), p.ld_res, m0, row0, col0, lane);
            __syncwarp();
            if (tma_res) sound = wait(&sm.res_full[group], j & 1, &sm.gave_up) && sound;
            sound = wait(&sm.acc_full[it % A], (it / A) & 1, &sm.gave_up) && sound;
            __syncwarp();
            tc::fence_after();
            const uint32_t acc = tmem + it % A * BN + slab * slab_cols + ((uint32_t)row0 << 16);
#pragma unroll 1
            for (int h = 0; h < slab_cols / 32; ++h) {
                float v[32];
                tc::tmem_load_32(acc + 32 * h, v);
                const int c0 = col0 + 32 * h;
                const int chunk0 = wide ? 0 : 4 * h;
                const float *dy_row = nullptr;
                int dy_left = 0;
                if (is_act_grad(EPI) && p.res_mode == kResThread && m0 + row < p.M) {
                    dy_row = static_cast<const float *>(p.res) + (m0 + row) * p.ld_res + c0;
                    dy_left = p.N - c0;
                }
                const float *b = bias_sh + 32 * h, *cs = scale_sh + 32 * h;
                uint4 *kept = nullptr;
                if (EPI == kForwardKeep && m0 < p.M && col0 < p.N)
                    kept = p.kept + ((((long long)m * ((p.N + 63) / 64) + col0 / 64) * 4 + quarter) * 8 + 4 * h) * 32 + lane;
                switch (EPI == kPartial ? QC_ACT_NONE : p.act) {
                    case QC_ACT_RELU:
                        epilogue_32<EPI, QC_ACT_RELU, B_MN>(p, v, buf, row, chunk0, b, cs, row_scale, dy_row, dy_left,
                                                      kept);
                        break;
                    case QC_ACT_SILU:
                        epilogue_32<EPI, QC_ACT_SILU, B_MN>(p, v, buf, row, chunk0, b, cs, row_scale, dy_row, dy_left,
                                                      kept);
                        break;
                    case QC_ACT_GELU:
                        epilogue_32<EPI, QC_ACT_GELU, B_MN>(p, v, buf, row, chunk0, b, cs, row_scale, dy_row, dy_left,
                                                      kept);
                        break;
                    default:
                        epilogue_32<EPI, QC_ACT_NONE, B_MN>(p, v, buf, row, chunk0, b, cs, row_scale, dy_row, dy_left,
                                                      kept);
                        break;
                }
                if constexpr (is_act_grad(EPI)) {
                    if (p.colsum) {
                        // rows past the last hold the bias's z times a zero dy
                        if (m0 + row >= p.M) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0.f;
                        }
                        const float sum = column_sums(v, lane);
                        sm.colsum[group][j & 1][ew & 3][32 * h + lane] = sound ? sum : __uint_as_float(kNaNBits);
                    }
                }
            }
            if (!sound) {
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4 *>(buf + row * 128 + 16 * c) = make_uint4(kNaNBits, kNaNBits, kNaNBits, kNaNBits);
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) tc::arrive_cluster(tc::cluster_addr(&sm.acc_empty[it % A], 0));
                else mbar_arrive(&sm.acc_empty[it % A]);
            }
            if (p.tma_store) {
                tc::fence_async_smem();
                tc::named_barrier(1 + group, 128);
                if (leader) {
                    if (col0 < p.N && m0 < p.M) tc::store_3d(&map_y, smem_addr(buf), col0, m * 128, EPI == kPartial ? s : 0);
                    tc::store_commit();
                    if (tma_res) {
                        tc::store_wait_read();
                        fetch(j + 1);
                    }
                }
                if constexpr (is_act_grad(EPI)) {
                    const int c = (ew & 3) * 32 + lane;
                    if (p.colsum && c < 64 && col0 + c < p.N && m0 < p.M &&
                        in_array((long long)m * p.N + col0 + c, (p.M + 127) / 128 * p.N)) {
                        const float *cs = &sm.colsum[group][j & 1][0][c];
                        float sum = (cs[0] + cs[64]) + (cs[128] + cs[192]);
                        if constexpr (EPI == kActGradScaled) sum *= gradient_scale<true>(*p.dy_max);
                        store_any(p.colsum, (long long)m * p.N + col0 + c, p.colsum_type, sum);
                    }
                }
                __syncwarp();
            } else {
                __syncwarp();
                slab_warp_copy<false>(p, buf, p.y, p.N, m0, row0, col0, lane);
                __syncwarp();
            }
        }
        if (leader) {
            // the last residual has landed, also where a wait gave up
            if (fetched) drain(&sm.res_full[group], (fetched - 1) & 1);
            tc::store_wait_all();
        }
        __syncwarp();
    }
    tc::fence_before();
    __syncwarp();
    if constexpr (PAIR) tc::cluster_sync();
    else __syncthreads();
    if (warp == 1) tc::tmem_free<PAIR>(tmem, kTmemCols);
}

// ── few rows: the weights on the rows' side ──────────────────────────────
//
// With few rows (points) the product is bound by reading the weights, so W's
// rows fill the 128 lanes of the matrix instruction and the points its BN
// columns. The reduction is split over the CTAs of a cluster (up to 8), each
// streaming its part of W through a deep ring; the parts are joined over
// distributed shared memory in rank order, so the result does not change from
// run to run, and no workspace is needed.

template <int BN>
struct FewGeom {
    static constexpr int kStage = kStageA + BN * 128;
    static constexpr int kStages = BN <= 16 ? 11 : BN <= 32 ? 10 : BN <= 64 ? 8 : 6;
};
template <int BN>
struct FewSmem {
    alignas(1024) unsigned char ring[FewGeom<BN>::kStages][FewGeom<BN>::kStage];  // then the part [BN][128] fp32
    uint64_t full[FewGeom<BN>::kStages], empty[FewGeom<BN>::kStages], done;
    uint32_t tmem;
    int gave_up;
};

__device__ __forceinline__ void spoil(float (&v)[16], bool sound) {
    if (sound) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(kNaNBits);
}

// One column (feature) per lane, eight rows of x at a time, straight-line code:
// with one warp per scheduler the latencies must overlap within the thread.
template <int ACT, int OT>
struct FewEpilogue {
    const Product &p;
    long long r0;
    int f;
    float bias, col_scale;

    // sums z of rows c..c+8 of this tile, as far as `end`
    __device__ __forceinline__ void finish(float (&z)[8], int c, int end) const {
        if (f >= p.N || !in_array(f, p.N) || !in_array(r0 + min(c + 8, end) - 1, p.M)) return;
        using E = typename ElemOf<OT>::type;
        const long long at = (r0 + c) * p.N + f;
        float res[8] = {};
        if (p.row_scale) {
            float rs[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) rs[i] = c + i < end ? p.row_scale[r0 + c + i] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = z[i] * rs[i] * col_scale;
        }
        if (p.res) {
            const E *from = static_cast<const E *>(p.res) + (r0 + c) * p.ld_res + f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < end) res[i] = load_any(from, i * p.ld_res, OT);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] += bias;
#pragma unroll
        for (int i = 0; i < 8; i += 2) act_fwd<ACT>(z[i], z[i + 1]);
        E *to = static_cast<E *>(p.y) + at;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < end) store_any(to, (long long)i * p.N, OT, z[i] + res[i]);
    }

    // the whole reduction lies in this CTA: from the accumulator
    __device__ __forceinline__ void whole(uint32_t acc, int cols, bool sound) const {
        for (int c = 0; c < cols; c += 16) {
            float v[16], z[8];
            tc::tmem_load_16(acc + c, v);
            spoil(v, sound);
#pragma unroll
            for (int h = 0; h < 16; h += 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = v[h + i];
                if (c + h < cols) finish(z, c + h, cols);
            }
            __syncwarp();
        }
    }

    // from the cluster's parts, added in rank order; `part`: this thread's
    // column in [rows][128]
    __device__ __forceinline__ void joined(const float *part, int parts, int begin, int end) const {
        for (int c = begin; c < end; c += 8) {
            float z[8] = {};
            for (int q = 0; q < parts; ++q) {
                const uint32_t from = tc::cluster_addr(part + c * 128, q);
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = c + i < end ? tc::load_cluster(from + i * 512) : 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] += v[i];
            }
            finish(z, c, end);
        }
    }
};

template <typename F>
__device__ __forceinline__ void with_act_and_type(int act, int out_type, F &&run) {
#define QC_ACT_CASE(ACT)                                                                     \
    case ACT:                                                                                \
        if (out_type == QC_BF16) run(std::integral_constant<int, ACT>(), std::integral_constant<int, QC_BF16>()); \
        else if (out_type == QC_F16) run(std::integral_constant<int, ACT>(), std::integral_constant<int, QC_F16>()); \
        else run(std::integral_constant<int, ACT>(), std::integral_constant<int, QC_F32>()); \
        break;
    switch (act) {
        QC_ACT_CASE(QC_ACT_NONE)
        QC_ACT_CASE(QC_ACT_RELU)
        QC_ACT_CASE(QC_ACT_SILU)
        QC_ACT_CASE(QC_ACT_GELU)
    }
#undef QC_ACT_CASE
}

template <bool F8, int BN>
__global__ void __launch_bounds__(192, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ Product p) {
    using G = FewGeom<BN>;
    constexpr int S = G::kStages;
    constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
    constexpr int kStep = F8 ? 128 : 64;
    extern __shared__ unsigned char raw[];
    FewSmem<BN> &sm = *reinterpret_cast<FewSmem<BN> *>(raw + ((1024 - (smem_addr(raw) & 1023)) & 1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = p.splits;
    const int rank = (int)tc::cluster_rank();
    const int f0 = blockIdx.x / parts * 128;  // first feature (row of W)
    const long long r0 = (long long)blockIdx.y * BN;  // first row of x
    int k0, k1;
    k_range(p, rank, k0, k1);

    auto load = [&](int q) {
        const int st = q % S;
        mbar_arrive_expect_tx(&sm.full[st], G::kStage);
        const uint32_t a = smem_addr(sm.ring[st]);
        tc::load_2d(a, &map_w, (k0 + q) * kStep, f0, &sm.full[st]);
        tc::load_2d(a + kStageA, &map_x, (k0 + q) * kStep, (int)r0, &sm.full[st]);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        mbar_init(&sm.done, 1);
        sm.gave_up = 0;
        fence_mbar_init();
        // the ring is filled before anything else is set up
        for (int q = 0; q < min(S, k1 - k0); ++q) load(q);
    }
    if (warp == 1) tc::tmem_alloc(&sm.tmem, kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sm.tmem);

    if (warp == 0) {
        if (lane == 0) {
            int q = min(S, k1 - k0);
            for (; q < k1 - k0; ++q) {
                if (!wait(&sm.empty[q % S], ((q / S) & 1) ^ 1, &sm.gave_up)) break;
                load(q);
            }
            for (int i = q > S ? q - S : 0; i < q; ++i) drain(&sm.full[i % S], (i / S) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            int q = 0;
            bool ok = true;
            for (int k = k0; k < k1; ++k, ++q) {
                const int st = q % S;
                if (!(ok = wait(&sm.full[st], (q / S) & 1, &sm.gave_up))) break;
                tc::fence_after();
                const uint32_t a = smem_addr(sm.ring[st]);
                const uint64_t da = tc::operand_desc(a, 16), db = tc::operand_desc(a + kStageA, 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) tc::mma<F8>(tmem, da + 2 * j, db + 2 * j, p.idesc, k > k0 || j > 0);
                tc::mma_commit(&sm.empty[st]);
            }
            if (ok) tc::mma_commit(&sm.done);
        }
        __syncwarp();
    }
    // every thread: all products are done, the ring is free (a wait that gave up
    // leaves NaN)
    const bool sound = drain(&sm.done, 0);
    tc::fence_after();
    __syncthreads();
    float *part = reinterpret_cast<float *>(sm.ring);
    const int quarter = warp & 3, f_local = quarter * 32 + lane, f = f0 + f_local;
    const int cols = (int)min((long long)BN, p.M - r0);  // rows of x in this tile
    const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
    float b = 0.f, cs = 1.f;
    if (warp >= 2 && f < p.N) {
        if (p.bias) b = load_any(p.bias, f, p.bias_type);
        if (p.row_scale) cs = p.col_scale[f];
    }
    if (parts == 1) {
        if (warp >= 2) {
            with_act_and_type(p.act, p.out_type, [&](auto act, auto type) {
                FewEpilogue<decltype(act)::value, decltype(type)::value>{p, r0, f, b, cs}.whole(acc, cols, sound);
            });
            tc::fence_before();
        }
        __syncthreads();
        if (warp == 1) tc::tmem_free(tmem, kTmemCols);
        return;
    }
    if (warp >= 2) {
#pragma unroll 1
        for (int c = 0; c < cols; c += 16) {
            float v[16];
            tc::tmem_load_16(acc + c, v);
            spoil(v, sound);
#pragma unroll
            for (int i = 0; i < 16; ++i) part[(c + i) * 128 + f_local] = v[i];
        }
        tc::fence_before();
    }
    __syncwarp();
    tc::cluster_sync();
    if (warp >= 2) {
        const int each = (cols + parts - 1) / parts;  // this CTA's share of the rows
        with_act_and_type(p.act, p.out_type, [&](auto act, auto type) {
            FewEpilogue<decltype(act)::value, decltype(type)::value>{p, r0, f, b, cs}.joined(
                part + f_local, parts, rank * each, min(cols, (rank + 1) * each));
        });
    }
    __syncwarp();
    tc::cluster_sync();  // the parts stay until every CTA has read them
    if (warp == 1) tc::tmem_free(tmem, kTmemCols);
}

// ── small passes ─────────────────────────────────────────────────────────

// Rows copied to a 16-byte-aligned row pitch for TMA (widths and pointers that
// no 16-byte boundary divides). A thread forms one 16-byte vector; 16-bit values
// are read in aligned words, put together again where the row starts between two.
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T *src, long long ld_src, T *dst, long long ld_dst,
                                                        long long rows, int n) {
    constexpr int V = 16 / (int)sizeof(T);
    const int vecs = (int)(ld_dst / V);
    const long long count = rows * vecs, stride = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += stride) {
        const long long r = i / vecs;
        const int c = (int)(i - r * vecs) * V;
        const T *from = src + r * ld_src + c;
        if (!in_array(r * ld_src + min(c + V, n) - 1, extent(rows, ld_src, n)) || !in_array(r * ld_dst + c + V - 1, rows * ld_dst))
            continue;
        uint32_t w[4] = {0, 0, 0, 0};
        if (sizeof(T) == 2 && c + V <= n) {
            if ((reinterpret_cast<uintptr_t>(from) & 3) == 0) {
                const uint32_t *q = reinterpret_cast<const uint32_t *>(from);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = q[k];
            } else {
                const uint32_t *q = reinterpret_cast<const uint32_t *>(from + 1);
                const uint32_t a = q[0], b = q[1], d = q[2], e = (uint32_t)from[V - 1];
                w[0] = (uint32_t)from[0] | (a << 16);
                w[1] = __funnelshift_r(a, b, 16);
                w[2] = __funnelshift_r(b, d, 16);
                w[3] = __funnelshift_r(d, e, 16);
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (c + k < n) w[k * sizeof(T) / 4] |= (uint32_t)from[k] << (8 * (k * sizeof(T) % 4));
        }
        *reinterpret_cast<uint4 *>(dst + r * ld_dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The largest finite |dy| as bits into *out (0 before): bits of non-negative
// floats order like the floats, and a maximum does not depend on its order.
__global__ void __launch_bounds__(256) largest_kernel(const float *dy, long long ld, long long rows, int n,
                                                      unsigned int *out) {
    __shared__ unsigned int sh[8];
    const long long threads = (long long)gridDim.x * 256, id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int lane = threadIdx.x & 31;
    unsigned int m = 0;
    auto take = [&](float v) {
        const unsigned int b = __float_as_uint(v) & 0x7fffffffu;
        if (b < 0x7f800000u) m = max(m, b);
    };
    if (ld == n) {
        const long long count = rows * n;
        long long done = 0;
        if ((reinterpret_cast<uintptr_t>(dy) & 15) == 0) {
            const float4 *q = reinterpret_cast<const float4 *>(dy);
#pragma unroll 4
            for (long long i = id; i < count / 4; i += threads) {
                if (!in_array(4 * i + 3, count)) break;
                const float4 v = q[i];
                take(v.x), take(v.y), take(v.z), take(v.w);
            }
            done = count / 4 * 4;
        }
        for (long long i = done + id; i < count; i += threads) take(dy[i]);
    } else {
        for (long long r = id / 32; r < rows; r += threads / 32)
            for (int c = lane; c < n; c += 32)
                if (in_array(r * ld + c, extent(rows, ld, n))) take(dy[r * ld + c]);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max(m, sh[i]);
        if (m) atomicMax(out, m);
    }
}

// dz = dy where there is no activation: cast to the operands' type (dst may be
// null; times S where the largest |dy| is given), and column sums of blocks of rows. 64 columns x 4 rows of threads.
__global__ void __launch_bounds__(256) cast_colsum_kernel(const void *dy, long long ld, int dy_type, void *dst,
                                                          long long ld_dst, int dst_type, void *colsum, int colsum_type,
                                                          long long rows, int n, long long rows_per_block,
                                                          const unsigned int *dy_max) {
    __shared__ float sh[4][64];
    const float scale = dy_max ? gradient_scale<false>(*dy_max) : 1.f;
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), ry = threadIdx.x >> 6;
    const long long r0 = blockIdx.y * rows_per_block, r1 = min(rows, r0 + rows_per_block);
    float s = 0.f;
    if (c < n)
        for (long long r = r0 + ry; r < r1; r += 4) {
            if (!in_array(r * ld + c, extent(rows, ld, n)) || (dst && !in_array(r * ld_dst + c, rows * ld_dst))) break;
            const float v = load_any(dy, r * ld + c, dy_type);
            if (dst) store_any(dst, r * ld_dst + c, dst_type, v * scale);
            s += v;
        }
    if (!colsum) return;
    sh[ry][threadIdx.x & 63] = s;
    __syncthreads();
    if (ry == 0 && c < n)
        store_any(colsum, (long long)blockIdx.y * n + c, colsum_type,
                  (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]));
}

// dz = dy * act'(z) from what the forward kept (KEPT), and column sums of blocks
// of rows. 8 columns per thread, 32 rows of 64 columns per turn of the block.
template <bool KEPT>
__global__ void __launch_bounds__(256) dz_kernel(const unsigned short *dy, long long ld, const uint4 *kept,
                                                 unsigned short *dz, long long ld_dz, void *colsum, int colsum_type,
                                                 int type, long long rows, int n, long long rows_per_block) {
    __shared__ float sh[8][64];
    const int chunk = threadIdx.x & 7, c = blockIdx.x * 64 + chunk * 8;
    const long long r1 = min(rows, (blockIdx.y + 1) * rows_per_block);
    float sum[8] = {};
    if (c < n) {
#pragma unroll 4
        for (long long r = blockIdx.y * rows_per_block + (threadIdx.x >> 3); r < r1; r += 32) {
            if (!in_array(r * ld + c + 7, extent(rows, ld, n))) break;
            float v[8];
            unpack8(*reinterpret_cast<const uint4 *>(dy + r * ld + c), type, v);
            if constexpr (KEPT) {
                const long long at = ((((r >> 7) * gridDim.x + blockIdx.x) * 4 + ((r >> 5) & 3)) * 8 + chunk) * 32 + (r & 31);
                if (!in_array(at, kept_vectors(rows, n)) || !in_array(r * ld_dz + c + 7, rows * ld_dz)) break;
                float d[8];
                unpack8(kept[at], QC_F16, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= d[i] * (1.f / kKeptScale);
                *reinterpret_cast<uint4 *>(dz + r * ld_dz + c) = pack8(v, type);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[i];
        }
    }
    if (!colsum) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 16);
    }
    if ((threadIdx.x & 31) < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sh[threadIdx.x >> 5][chunk * 8 + i] = sum[i];
    }
    __syncthreads();
    const int at = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && at < n) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += sh[i][threadIdx.x];
        store_any(colsum, (long long)blockIdx.y * n + at, colsum_type, s);
    }
}

// Partial products [splits][rows][ld] added in a fixed order, rounded once. A
// block's 8 warps share the splits of 32 quads of columns.
__global__ void __launch_bounds__(256) join_splits_kernel(const float *part, int splits, long long rows, int n,
                                                          long long ld, void *out, int out_type) {
    __shared__ float4 sh[8][32];
    const int quads = (n + 3) / 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long i = (long long)blockIdx.x * 32 + lane, r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
#pragma unroll 4
        for (int q = warp; q < splits; q += 8) {
            if (!in_array(((long long)q * rows + r) * ld + c + 3, splits * rows * ld)) break;
            const float4 v = *reinterpret_cast<const float4 *>(part + ((long long)q * rows + r) * ld + c);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
    }
    sh[warp][lane] = s;
    __syncthreads();
    if (warp || r >= rows || !in_array(r * n + min(c + 4, n) - 1, rows * n)) return;
#pragma unroll
    for (int q = 1; q < 8; ++q) {
        const float4 v = sh[q][lane];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    if (n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {  // out has 16 bits
        store_vec<4>(out, r * n + c, out_type, v);
    } else {
        for (int k = 0; k < 4 && c + k < n; ++k) store_any(out, r * n + c + k, out_type, v[k]);
    }
}

__global__ void __launch_bounds__(256) zero_kernel(unsigned char *p, long long bytes) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (long long)gridDim.x * 256) p[i] = 0;
}

// ── host side ────────────────────────────────────────────────────────────

CUtensorMapDataType map_type(int t) {
    switch (t) {
        case QC_F32: return CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
        case QC_BF16: return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        case QC_F16: return CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        default: return CU_TENSOR_MAP_DATA_TYPE_UINT8;
    }
}

// [planes][rows][cols] with a row pitch of ld elements, read or written in
// boxes of box_rows rows of 128 bytes, 128-byte swizzle.
int make_map(CUtensorMap *map, const void *base, int type, long long cols, long long rows, long long ld, int box_rows,
             int dims, long long planes = 1) {
    EncodeTiledFn encode = nullptr;
    if (int st = tensor_map_encoder(&encode)) return st;
    const int es = elem_size(type);
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t pitch[2] = {(cuuint64_t)(ld * es), (cuuint64_t)(ld * es * rows)};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = encode(map, map_type(type), dims, const_cast<void *>(base), size, pitch, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(QC_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled failed (CUresult %d) for %lld rows of %lld, pitch %lld",
                         (int)r, rows, cols, ld);
    return 0;
}

// Whether TMA can tile rows of this pitch from this address.
bool tileable(const void *p, long long ld, int type) { return aligned_to(p, 16) && (ld * elem_size(type)) % 16 == 0; }

// Binds the current device's context to this thread (the tensor maps are
// encoded through the driver API; a fresh host thread has none).
int bind_device(int *dev) {
    QC_CUDA_TRY(cudaGetDevice(dev), "cudaGetDevice");
    QC_CUDA_TRY(cudaSetDevice(*dev), "cudaSetDevice");
    return 0;
}

// Opts in to `smem` bytes of dynamic shared memory, once per device and kernel.
template <typename K>
int opt_in(K kernel, size_t smem, std::atomic<unsigned long long> &done, int dev) {
    if (dev < kMaxDevices && (done.load(std::memory_order_relaxed) >> dev) & 1) return 0;
    QC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                "cudaFuncSetAttribute(max dynamic shared memory)");
    if (dev < kMaxDevices) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return 0;
}

struct Operand {
    const void *p;
    long long ld;  // elements
};

template <bool F8, bool A_MN, bool B_MN, int BN, int EPI, bool PAIR>
int launch_product(const Operand &a, const Operand &b, int type, long long K, const CUtensorMap &map_y,
                   const CUtensorMap &map_r, Product p, int sms, int dev, cudaStream_t stream) {
    using G = Geom<BN, PAIR>;
    CUtensorMap map_a, map_b;
    if (int st = A_MN ? make_map(&map_a, a.p, type, p.M, K, a.ld, 64, 2) : make_map(&map_a, a.p, type, K, p.M, a.ld, 128, 2))
        return st;
    if (int st = B_MN ? make_map(&map_b, b.p, type, p.N, K, b.ld, 64, 2)
                      : make_map(&map_b, b.p, type, K, p.N, b.ld, G::kRowsB, 2))
        return st;
    p.m_tiles = (int)((p.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
    p.n_tiles = (p.N + BN - 1) / BN;
    p.by_split.set((uint32_t)std::min<long long>((long long)p.m_tiles * p.n_tiles, 1ll << 30));
    p.by_span.set((uint32_t)std::min<long long>((long long)(PAIR ? 8 : 16) * p.n_tiles, 1ll << 30));
    p.idesc = tc::instr_desc(type == QC_BF16 ? 1 : 0, A_MN, B_MN, BN, PAIR ? 256 : 128);
    auto kernel = product_kernel<F8, A_MN, B_MN, BN, EPI, PAIR>;
    const size_t smem = sizeof(ProductSmem<BN, PAIR>) + 1024;
    static_assert(sizeof(ProductSmem<BN, PAIR>) + 1024 <= 232448, "shared memory");
    static std::atomic<unsigned long long> done{0};
    if (int st = opt_in(kernel, smem, done, dev)) return st;
    const long long total = (long long)p.m_tiles * p.n_tiles * p.splits;
    QC_RETURN_IF(total >= (1ll << 28), QC_ERR_INVALID_ARGUMENT, "linear_act: %lld tiles", total);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(PAIR ? 2 * std::min<long long>(total, sms / 2) : std::min<long long>(total, sms)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 1 : 0;
    QC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_y, map_r, p), "product_kernel launch");
    return 0;
}

// Tile width and whether two CTAs share a tile: the least rounds of tiles over
// the SMs times a round's cost. A round costs little more for a wider tile (a
// reduction of 4096 in bf16, one round: 24.5 us for 64 columns, 24.9 for 128,
// 32 for 256, 29 for 256 in pairs), because the latency of its loads counts
// more than their bytes; 2048 rows of 4096 by 1024 take 45 us in two rounds of
// 64 columns and 27 us in one of 128. Pairs need two row tiles and a reduction
// of at least 16 ring stages (1024 16-bit values): over 4096 they take 195
// against 222 us (8192 rows, 4096 columns), over 1024 57 against 61 us, and
// over 256, where memory and the epilogue bound the product, 71 against 65 us.
// Pairs of 128 columns cost more than single CTAs (26 us) and never less rounds.
constexpr int kPairStages = 16;
struct TileChoice {
    int bn;
    bool pair;
    long long rounds;
};
TileChoice choose_tile(long long M, int n, int k_blocks, int splits, int sms) {
    struct Option {
        int bn, pair, cost;
    };
    constexpr Option options[] = {{256, 1, 120}, {256, 0, 135}, {128, 0, 107}, {64, 0, 100}};
    TileChoice best{64, false, 0};
    long long least = -1;
    for (const Option &o : options) {
        if ((o.bn > 64 && n <= o.bn / 2) || (o.pair && (M <= 128 || k_blocks / splits < kPairStages))) continue;
        const long long rows = o.pair ? 256 : 128, slots = o.pair ? sms / 2 : sms;
        const long long tiles = (M + rows - 1) / rows * ((n + o.bn - 1) / o.bn) * splits;
        const long long rounds = (tiles + slots - 1) / slots, cost = rounds * o.cost;
        if (least < 0 || cost < least) least = cost, best = {o.bn, o.pair != 0, rounds};
    }
    return best;
}

// Ring stages of a reduction over K values.
int stages_of(long long K, int type) { return (int)((K * elem_size(type) + 127) / 128); }

template <bool F8, bool A_MN, bool B_MN, int EPI>
int run_product(const Operand &a, const Operand &b, int type, long long K, const CUtensorMap &map_y,
                const CUtensorMap &map_r, Product p, int sms, int dev, cudaStream_t stream) {
    p.k_blocks = stages_of(K, type);
    const TileChoice c = choose_tile(p.M, p.N, p.k_blocks, p.splits, sms);
#define QC_RUN(BN, PAIR) \
    return launch_product<F8, A_MN, B_MN, BN, EPI, PAIR>(a, b, type, K, map_y, map_r, p, sms, dev, stream)
    if (c.pair) QC_RUN(256, true);
    if (c.bn == 256) QC_RUN(256, false);
    if (c.bn == 128) QC_RUN(128, false);
    QC_RUN(64, false);
#undef QC_RUN
}

// Rows of x in a tile of the few-row form, and the parts of its reduction: as
// many as fill the SMs, two ring stages each at least, from 8 stages on (4
// stages in 2 parts: 10.6 against 6.3 us at 128 rows). Clusters of 8 fill at
// most 3/4 of the SMs: two do not fit into every group of SMs that shares a
// cluster's network, and a cluster left over runs after the others (16 of them
// 19.6 us, 32 of 4 CTAs 13.9 us).
int few_rows_tile(long long rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }
int few_rows_parts(long long rows, int n, int k_blocks, int sms) {
    const long long tiles = (long long)((n + 127) / 128) * ((rows + few_rows_tile(rows) - 1) / few_rows_tile(rows));
    int parts = 1;
    while (parts < 8 && k_blocks >= 8 && 4 * parts <= k_blocks &&
           2 * parts * tiles <= (parts == 4 ? sms * 3 / 4 : sms))
        parts *= 2;
    return parts;
}

template <bool F8, int BN>
int launch_few(const Operand &x, const Operand &w, int type, long long K, Product p, int sms, int dev,
               cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (int st = make_map(&map_w, w.p, type, K, p.N, w.ld, 128, 2)) return st;
    if (int st = make_map(&map_x, x.p, type, K, p.M, x.ld, BN, 2)) return st;
    p.k_blocks = stages_of(K, type);
    p.idesc = tc::instr_desc(type == QC_BF16 ? 1 : 0, false, false, BN);
    const int tiles = (p.N + 127) / 128, parts = few_rows_parts(p.M, p.N, p.k_blocks, sms);
    const long long row_tiles = (p.M + BN - 1) / BN;
    p.splits = parts;
    auto kernel = few_rows_kernel<F8, BN>;
    const size_t smem = sizeof(FewSmem<BN>) + 1024;
    static_assert(sizeof(FewSmem<BN>) + 1024 <= 232448, "shared memory");
    static_assert(sizeof(FewSmem<BN>::ring) >= BN * 512, "the part lies over the ring");
    static std::atomic<unsigned long long> done{0};
    if (int st = opt_in(kernel, smem, done, dev)) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * parts, (unsigned)row_tiles);
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    QC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p), "few_rows_kernel launch");
    return 0;
}

// Whether the weights take the rows' side. Up to 64 rows they always do (64 rows
// of 1024 by 1024: 6.9 against 9.4 us). Beyond, where the tiled product has too
// few tiles to stream a long reduction with all SMs and this form can split it:
// from 32 ring stages (2048 16-bit values) with up to 32 tiles of 128 x 128
// (2048 by 512, 1024 rows: 11.5 against 14.4 us; 4096 by 1024 in 8 bits, 512
// rows: 12.1 against 15.1), from 64 stages with up to 128 (4096 by 1024, 1024
// rows: 20.4 against 24.7 us; 4096 by 4096, 512 rows: equal).
bool few_rows(long long rows, int n, int k, int type) {
    const long long stages = stages_of(k, type);
    const long long tiles = (rows + 127) / 128 * ((n + 127) / 128);
    return rows <= 64 || (stages >= 32 && tiles <= 32) || (stages >= 64 && tiles <= 128);
}

long long round_up(long long v, long long to) { return (v + to - 1) / to * to; }

// Workspace pieces, each 256-byte aligned.
struct Carve {
    size_t used = 0;
    size_t take(size_t bytes) {
        const size_t at = used;
        used += (bytes + 255) / 256 * 256;
        return at;
    }
};

int pack_rows(const void *src, long long ld, void *dst, long long ld_dst, long long rows, int n, int es, int sms,
              cudaStream_t stream) {
    const unsigned grid =
        (unsigned)std::min<long long>((rows * (ld_dst * es / 16) + 255) / 256, (long long)sms * 8);
    if (es == 1)
        pack_rows_kernel<<<grid, 256, 0, stream>>>(static_cast<const unsigned char *>(src), ld,
                                                   static_cast<unsigned char *>(dst), ld_dst, rows, n);
    else
        pack_rows_kernel<<<grid, 256, 0, stream>>>(static_cast<const unsigned short *>(src), ld,
                                                   static_cast<unsigned short *>(dst), ld_dst, rows, n);
    QC_CHECK_LAUNCH("pack_rows_kernel");
    return 0;
}

bool is_16bit(int t) { return t == QC_BF16 || t == QC_F16; }

int check_shape(const char *fn, long M, int N, int K, long ldx, long ldw, int type) {
    QC_RETURN_IF(M < 0 || N < 1 || K < 1, QC_ERR_INVALID_ARGUMENT, "%s: %ld rows, %d outputs, %d inputs", fn, M, N, K);
    QC_RETURN_IF(M >= (1l << 31) - 256, QC_ERR_INVALID_ARGUMENT, "%s: %ld rows (2^31 - 256 at most)", fn, M);
    QC_RETURN_IF(N >= (1 << 30) || K >= (1 << 30), QC_ERR_INVALID_ARGUMENT, "%s: widths %d, %d (below 2^30)", fn, N, K);
    QC_RETURN_IF((M > 1 && ldx < K) || (N > 1 && ldw < K), QC_ERR_INVALID_ARGUMENT,
                 "%s: row strides %ld, %ld below the width %d", fn, ldx, ldw, K);
    QC_RETURN_IF(!is_16bit(type) && type != QC_E4M3, QC_ERR_INVALID_ARGUMENT, "%s: unknown operand type %d", fn, type);
    return 0;
}

struct Packs {
    bool x, w;
    long long ld;
    size_t at_x, at_w;
};
Packs plan_packs(Carve &c, const void *x, const void *w, long M, int N, int K, long ldx, long ldw, int type) {
    Packs k{};
    const int es = elem_size(type);
    k.ld = round_up(K, 16 / es);
    k.x = !tileable(x, M > 1 ? ldx : k.ld, type);
    k.w = !tileable(w, N > 1 ? ldw : k.ld, type);
    if (k.x) k.at_x = c.take((size_t)M * k.ld * es);
    if (k.w) k.at_w = c.take((size_t)N * k.ld * es);
    return k;
}

int apply_packs(const Packs &k, Operand &x, Operand &w, long M, int N, int K, int type, unsigned char *ws, int sms,
                cudaStream_t stream) {
    const int es = elem_size(type);
    if (k.x) {
        if (int st = pack_rows(x.p, x.ld, ws + k.at_x, k.ld, M, K, es, sms, stream)) return st;
        x = {ws + k.at_x, k.ld};
    } else if (M == 1) {
        x.ld = k.ld;  // the stride of a single row is never used
    }
    if (k.w) {
        if (int st = pack_rows(w.p, w.ld, ws + k.at_w, k.ld, N, K, es, sms, stream)) return st;
        w = {ws + k.at_w, k.ld};
    } else if (N == 1) {
        w.ld = k.ld;
    }
    return 0;
}

// Parts of dweight's reduction, which runs over the rows: split until the SMs are
// filled, at least 512 rows (8 ring stages) each, and at most 32768, because the
// tensor cores cut each addition (2^-24 of the sum a step: 2048 steps stay below
// half a step of fp16).
int weight_splits(long long rows, int n, int k, int sms) {
    const long long tiles = (long long)((n + 127) / 128) * ((k + 255) / 256);
    return (int)std::max<long long>({1, std::min<long long>(sms / tiles, rows / 512), (rows + 32767) / 32768});
}

struct GradPlan {
    Packs packs;
    bool make_dz, vectors, scaled;
    long long ld_dz, ld_part, rows_per_block;
    int splits, sum_parts;
    size_t at_dz, at_sum, at_part, at_max, bytes;
};
GradPlan plan_grad(const void *x, const void *w, const void *dy, long M, int N, int K, long ldx, long ldw, long lddy,
                   int type, int dy_type, int act, int want, int sms, bool kept = false) {
    GradPlan g{};
    Carve c;
    g.packs = plan_packs(c, x, w, M, N, K, ldx, ldw, type);
    const bool tiled = dy_type == type && tileable(dy, lddy, type);
    g.make_dz = kept || ((want & 3) && (act != QC_ACT_NONE || !tiled));
    g.ld_dz = round_up(N, 8);
    const bool z_pass = act != QC_ACT_NONE && !kept;
    g.vectors = kept || (act == QC_ACT_NONE && tiled && N % 8 == 0);  // dz_kernel serves
    g.scaled = type == QC_F16 && dy_type == QC_F32 && (want & 3);
    if (g.scaled) g.at_max = c.take(sizeof(unsigned int));
    if (g.make_dz || z_pass) g.at_dz = c.take((size_t)M * g.ld_dz * 2);
    g.make_dz = g.make_dz || z_pass;
    if (want & 4) {
        if (z_pass) {
            g.sum_parts = (int)((M + 127) / 128);
        } else {
            const long long col_blocks = (N + 63) / 64;
            const long long blocks = std::max<long long>(1, std::min<long long>((M + 63) / 64, sms * 8 / col_blocks + 1));
            g.rows_per_block = round_up((M + blocks - 1) / blocks, 32);
            g.sum_parts = (int)((M + g.rows_per_block - 1) / g.rows_per_block);
        }
        if (g.sum_parts > 1) g.at_sum = c.take((size_t)g.sum_parts * N * 4);
    } else if (g.make_dz && !z_pass) {
        g.rows_per_block = std::max<long long>(32, round_up((M + 1023) / 1024, 32));
        g.sum_parts = (int)((M + g.rows_per_block - 1) / g.rows_per_block);
    }
    g.splits = 1;
    if (want & 2) {
        g.splits = weight_splits(M, N, K, sms);
        g.ld_part = round_up(K, 4);
        if (g.splits > 1) g.at_part = c.take((size_t)g.splits * N * g.ld_part * 4);
    }
    g.bytes = c.used;
    return g;
}

}  // namespace

int ml_fault_word(unsigned int *word, int clear) {
    unsigned int w = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&w, g_ml_fault_word, sizeof(w));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_ml_fault_word, &zero, sizeof(zero));
    }
    QC_CUDA_TRY(e, "cudaMemcpyFromSymbol(fault word)");
    unsigned int norm = 0;
    if (int st = norm_fault_word(&norm, clear)) return st;
    *word = w | norm;
    return 0;
}

}  // namespace ml
}  // namespace qc

using namespace qc::ml;

extern "C" {

int linear_act_form(int product, long rows, int n, int k, int type, int sms, int *form) {
    if (int st = check_shape("linear_act_form", rows, n, k, k, k, type)) return st;
    QC_RETURN_IF(product < QC_PRODUCT_FORWARD || product > QC_PRODUCT_DWEIGHT || rows == 0 || !form,
                 QC_ERR_INVALID_ARGUMENT, "linear_act_form: product %d, %ld rows", product, rows);
    if (sms <= 0)
        if (int st = qc::device_sm_count(&sms)) return st;
    const int stages = stages_of(k, type);
    TileChoice c{};
    int parts = 1;
    if (product == QC_PRODUCT_FORWARD && few_rows(rows, n, k, type)) {
        form[0] = 0;
        form[1] = few_rows_tile(rows);
        form[2] = few_rows_parts(rows, n, stages, sms);
        form[3] = 1;
        return 0;
    }
    if (product == QC_PRODUCT_FORWARD || product == QC_PRODUCT_DERIVATIVE) {
        c = choose_tile(rows, n, stages, 1, sms);
    } else if (product == QC_PRODUCT_DX) {
        c = choose_tile(rows, k, stages_of(n, type), 1, sms);
    } else {
        parts = weight_splits(rows, n, k, sms);
        c = choose_tile(n, k, stages_of(rows, type), parts, sms);
    }
    form[0] = c.pair ? 2 : 1;
    form[1] = c.bn;
    form[2] = parts;
    form[3] = (int)c.rounds;
    return 0;
}

size_t linear_act_workspace_bytes(const void *x, const void *weight, long rows, int n, int k, long x_stride,
                                  long weight_stride, int type) {
    if (rows <= 0 || n < 1 || k < 1) return 0;
    Carve c;
    plan_packs(c, x, weight, rows, n, k, x_stride, weight_stride, type);
    return c.used;
}

static int forward(const char *fn, const void *x, const void *weight, const void *bias, const void *residual, void *y,
                   void *kept, const float *x_scale, const float *weight_scale, long rows, int n, int k, long x_stride,
                   long weight_stride, long residual_stride, int type, int out_type, int bias_type, int activation,
                   void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (int st = check_shape(fn, rows, n, k, x_stride, weight_stride, type)) return st;
    QC_RETURN_IF(out_type != QC_F32 && !is_16bit(out_type), QC_ERR_INVALID_ARGUMENT, "%s: unknown output type %d", fn,
                 out_type);
    QC_RETURN_IF(type != QC_E4M3 && is_16bit(out_type) && out_type != type, QC_ERR_INVALID_ARGUMENT,
                 "%s: 16-bit operands give their own type or fp32", fn);
    QC_RETURN_IF(bias && bias_type != QC_F32 && !is_16bit(bias_type), QC_ERR_INVALID_ARGUMENT,
                 "%s: unknown bias type %d", fn, bias_type);
    QC_RETURN_IF(activation < QC_ACT_NONE || activation > QC_ACT_GELU, QC_ERR_INVALID_ARGUMENT,
                 "%s: unknown activation %d", fn, activation);
    QC_RETURN_IF((type == QC_E4M3) != (x_scale != nullptr) || (x_scale != nullptr) != (weight_scale != nullptr),
                 QC_ERR_INVALID_ARGUMENT, "%s: 8-bit operands need both scales, and no others do", fn);
    if (rows == 0) return 0;
    QC_RETURN_IF(!x || !weight || !y, QC_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
    QC_RETURN_IF(residual && rows > 1 && residual_stride < 0, QC_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
    Carve c;
    const Packs packs = plan_packs(c, x, weight, rows, n, k, x_stride, weight_stride, type);
    QC_RETURN_IF(workspace_bytes < c.used, QC_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", fn,
                 workspace_bytes, c.used);
    QC_RETURN_IF(c.used && !aligned_to(workspace, 256), QC_ERR_INVALID_ARGUMENT,
                 "%s: workspace is not 256-byte aligned", fn);
    int sms = 0, dev = 0;
    if (int st = qc::device_sm_count(&sms)) return st;
    if (int st = bind_device(&dev)) return st;
    Operand xo{x, x_stride}, wo{weight, weight_stride};
    if (int st = apply_packs(packs, xo, wo, rows, n, k, type, static_cast<unsigned char *>(workspace), sms, stream))
        return st;

    Product p{};
    p.M = rows;
    p.N = n;
    p.splits = 1;
    p.bias = bias;
    p.bias_type = bias_type;
    p.row_scale = x_scale;
    p.col_scale = weight_scale;
    p.res = residual;
    p.ld_res = residual_stride;
    p.y = y;
    p.out_type = out_type;
    p.act = activation;
    const bool f8 = type == QC_E4M3;
    if (!kept && few_rows(rows, n, k, type)) {
        const int bn = few_rows_tile(rows);
        if (bn == 16)
            return f8 ? launch_few<true, 16>(xo, wo, type, k, p, sms, dev, stream)
                      : launch_few<false, 16>(xo, wo, type, k, p, sms, dev, stream);
        if (bn == 32)
            return f8 ? launch_few<true, 32>(xo, wo, type, k, p, sms, dev, stream)
                      : launch_few<false, 32>(xo, wo, type, k, p, sms, dev, stream);
        if (bn == 64)
            return f8 ? launch_few<true, 64>(xo, wo, type, k, p, sms, dev, stream)
                      : launch_few<false, 64>(xo, wo, type, k, p, sms, dev, stream);
        return f8 ? launch_few<true, 128>(xo, wo, type, k, p, sms, dev, stream)
                  : launch_few<false, 128>(xo, wo, type, k, p, sms, dev, stream);
    }
    CUtensorMap map_y = {}, map_r = {};
    p.tma_store = tileable(y, n, out_type) && (!residual || tileable(residual, residual_stride, out_type)) &&
                  (!residual || residual_stride >= n);
    p.res_mode = !residual ? kResNone : p.tma_store ? kResTma : kResWarp;
    if (p.tma_store) {
        if (int st = make_map(&map_y, y, out_type, n, rows, n, 128, 3)) return st;
        if (residual)
            if (int st = make_map(&map_r, residual, out_type, n, rows, residual_stride, 128, 3)) return st;
    }
    if (kept) {
        p.kept = static_cast<uint4 *>(kept);
        return run_product<false, false, false, kForwardKeep>(xo, wo, type, k, map_y, map_r, p, sms, dev, stream);
    }
    return f8 ? run_product<true, false, false, kForward>(xo, wo, type, k, map_y, map_r, p, sms, dev, stream)
              : run_product<false, false, false, kForward>(xo, wo, type, k, map_y, map_r, p, sms, dev, stream);
}

int linear_act_cuda(const void *x, const void *weight, const void *bias, const void *residual, void *y,
                    const float *x_scale, const float *weight_scale, long rows, int n, int k, long x_stride,
                    long weight_stride, long residual_stride, int type, int out_type, int bias_type, int activation,
                    void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    QC_NVTX("quantem::linear_act");
    return forward("linear_act", x, weight, bias, residual, y, nullptr, x_scale, weight_scale, rows, n, k, x_stride,
                   weight_stride, residual_stride, type, out_type, bias_type, activation, workspace, workspace_bytes,
                   stream);
}

// Where keeping act'(z) pays: large bf16 products with an activation and a reduction
// of 512 or more (the file's head has times; of 256, 262144 rows: 292 against 296
// us, not worth the memory). fp16 dz has too few bits less to hide the rounding, and
// an fp32 bias gradient would show it.
size_t linear_act_kept_bytes(long rows, int n, int k, int type, int out_type, int bias_type, int activation) {
    if (rows <= 512 || n < 8 || n % 8 || k < 512 || type != QC_BF16 || out_type != QC_BF16 || bias_type == QC_F32 ||
        activation <= QC_ACT_NONE || activation > QC_ACT_GELU || few_rows(rows, n, k, type))
        return 0;
    return (size_t)kept_vectors(rows, n) * sizeof(uint4);
}

int linear_act_keep_cuda(const void *x, const void *weight, const void *bias, const void *residual, void *y, void *kept,
                         long rows, int n, int k, long x_stride, long weight_stride, long residual_stride, int type,
                         int bias_type, int activation, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    QC_NVTX("quantem::linear_act_keep");
    QC_RETURN_IF(linear_act_kept_bytes(rows, n, k, type, type, bias ? bias_type : QC_BF16, activation) == 0,
                 QC_ERR_INVALID_ARGUMENT, "linear_act_keep: nothing is kept of such a call (linear_act_kept_bytes is 0)");
    QC_RETURN_IF(!kept || !aligned_to(kept, 16), QC_ERR_INVALID_ARGUMENT,
                 "linear_act_keep: the kept buffer is null or not 16-byte aligned");
    return forward("linear_act_keep", x, weight, bias, residual, y, kept, nullptr, nullptr, rows, n, k, x_stride,
                   weight_stride, residual_stride, type, type, bias_type, activation, workspace, workspace_bytes,
                   stream);
}

static int grad_want(const void *dx, const void *dweight, const void *dbias) {
    return (dx ? 1 : 0) | (dweight ? 2 : 0) | (dbias ? 4 : 0);
}

size_t linear_act_grad_workspace_bytes(const void *x, const void *weight, const void *dy, const void *dx,
                                       const void *dweight, const void *dbias, long rows, int n, int k, long x_stride,
                                       long weight_stride, long dy_stride, int type, int dy_type, int activation,
                                       int device) {
    if (rows <= 0 || n < 1 || k < 1) return 0;
    int sms = 0;
    if (qc::device_sm_count(device, &sms)) return 0;
    if (rows == 1) dy_stride = n;
    return plan_grad(x, weight, dy, rows, n, k, x_stride, weight_stride, dy_stride, type, dy_type, activation,
                     grad_want(dx, dweight, dbias), sms)
        .bytes;
}

static int backward(const char *fn, const void *x, const void *weight, const void *bias, const void *kept,
                    const void *dy, void *dx, void *dweight, void *dbias, long rows, int n, int k, long x_stride,
                    long weight_stride, long dy_stride, int type, int dy_type, int bias_type, int activation,
                    void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (int st = check_shape(fn, rows, n, k, x_stride, weight_stride, type)) return st;
    QC_RETURN_IF(!is_16bit(type), QC_ERR_INVALID_ARGUMENT, "%s: 16-bit operands only", fn);
    QC_RETURN_IF(dy_type != QC_F32 && dy_type != type, QC_ERR_INVALID_ARGUMENT,
                 "%s: the upstream gradient has the operands' type or fp32", fn);
    QC_RETURN_IF((bias || dbias) && bias_type != QC_F32 && !is_16bit(bias_type), QC_ERR_INVALID_ARGUMENT,
                 "%s: unknown bias type %d", fn, bias_type);
    QC_RETURN_IF(activation < QC_ACT_NONE || activation > QC_ACT_GELU, QC_ERR_INVALID_ARGUMENT,
                 "%s: unknown activation %d", fn, activation);
    const int want = grad_want(dx, dweight, dbias);
    if (!want) return 0;
    int sms = 0, dev = 0;
    if (int st = qc::device_sm_count(&sms)) return st;
    if (int st = bind_device(&dev)) return st;
    if (rows == 0) {  // sums over no rows
        for (int i = 0; i < 2; ++i) {
            void *p = i ? dbias : dweight;
            const long long bytes = i ? (long long)n * elem_size(bias_type) : (long long)n * k * 2;
            if (!p) continue;
            zero_kernel<<<(unsigned)std::min<long long>((bytes + 255) / 256, sms * 8), 256, 0, stream>>>(
                static_cast<unsigned char *>(p), bytes);
            QC_CHECK_LAUNCH("zero_kernel");
        }
        return 0;
    }
    QC_RETURN_IF(!x || !weight || !dy, QC_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
    QC_RETURN_IF(rows > 1 && dy_stride < n, QC_ERR_INVALID_ARGUMENT, "%s: gradient row stride %ld below the width %d",
                 fn, dy_stride, n);
    if (rows == 1) dy_stride = n;
    const GradPlan g = plan_grad(x, weight, dy, rows, n, k, x_stride, weight_stride, dy_stride, type, dy_type,
                                 activation, want, sms, kept != nullptr);
    QC_RETURN_IF(workspace_bytes < g.bytes, QC_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", fn,
                 workspace_bytes, g.bytes);
    QC_RETURN_IF(g.bytes && !aligned_to(workspace, 256), QC_ERR_INVALID_ARGUMENT,
                 "%s: workspace is not 256-byte aligned", fn);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    Operand xo{x, x_stride}, wo{weight, weight_stride}, dzo{dy, dy_stride};
    if (int st = apply_packs(g.packs, xo, wo, rows, n, k, type, ws, sms, stream)) return st;
    // one partial sum is the sum
    void *sums = !(want & 4) ? nullptr : g.sum_parts == 1 ? dbias : ws + g.at_sum;
    const int sums_type = g.sum_parts == 1 ? bias_type : QC_F32;
    const CUtensorMap none = {};
    unsigned int *dy_max = g.scaled ? reinterpret_cast<unsigned int *>(ws + g.at_max) : nullptr;
    if (dy_max) {
        QC_CUDA_TRY(cudaMemsetAsync(dy_max, 0, sizeof(*dy_max), stream), "cudaMemsetAsync");
        const long long blocks = ((long long)rows * n + 4095) / 4096;
        largest_kernel<<<(unsigned)std::min<long long>(blocks, (long long)sms * 8), 256, 0, stream>>>(
            static_cast<const float *>(dy), dy_stride, rows, n, dy_max);
        QC_CHECK_LAUNCH("largest_kernel");
    }

    if (activation != QC_ACT_NONE && !kept) {
        Product p{};
        p.M = rows;
        p.N = n;
        p.splits = 1;
        p.bias = bias;
        p.bias_type = bias_type;
        p.res = dy;
        p.ld_res = dy_stride;
        p.out_type = type;
        p.act = activation;
        p.colsum = sums;
        p.colsum_type = sums_type;
        p.dy_max = dy_max;
        p.tma_store = 1;
        p.res_mode = dy_type == QC_F32 ? kResThread : tileable(dy, dy_stride, type) ? kResTma : kResWarp;
        CUtensorMap map_y = {}, map_r = {};
        if (int st = make_map(&map_y, ws + g.at_dz, type, n, rows, g.ld_dz, 128, 3)) return st;
        if (p.res_mode == kResTma)
            if (int st = make_map(&map_r, dy, type, n, rows, dy_stride, 128, 3)) return st;
        if (int st = dy_max ? run_product<false, false, false, kActGradScaled>(xo, wo, type, k, map_y, map_r, p, sms, dev, stream)
                            : run_product<false, false, false, kActGrad>(xo, wo, type, k, map_y, map_r, p, sms, dev, stream))
            return st;
        dzo = {ws + g.at_dz, g.ld_dz};
    } else if (g.vectors && (kept || sums)) {
        const dim3 grid((n + 63) / 64, g.sum_parts);
        const unsigned short *from = static_cast<const unsigned short *>(dy);
        unsigned short *to = reinterpret_cast<unsigned short *>(ws + g.at_dz);
        if (kept) {
            dz_kernel<true><<<grid, 256, 0, stream>>>(from, dy_stride, static_cast<const uint4 *>(kept), to, g.ld_dz,
                                                      sums, sums_type, type, rows, n, g.rows_per_block);
            dzo = {to, g.ld_dz};
        } else {
            dz_kernel<false><<<grid, 256, 0, stream>>>(from, dy_stride, nullptr, nullptr, 0, sums, sums_type, type,
                                                       rows, n, g.rows_per_block);
        }
        QC_CHECK_LAUNCH("dz_kernel");
    } else if (g.make_dz || sums) {
        void *dst = g.make_dz ? ws + g.at_dz : nullptr;
        cast_colsum_kernel<<<dim3((n + 63) / 64, g.sum_parts), 256, 0, stream>>>(
            dy, dy_stride, dy_type, dst, g.ld_dz, type, sums, sums_type, rows, n, g.rows_per_block, dy_max);
        QC_CHECK_LAUNCH("cast_colsum_kernel");
        if (g.make_dz) dzo = {ws + g.at_dz, g.ld_dz};
    }
    if (dbias && g.sum_parts > 1)
        if (int st = launch_colsum_reduce(static_cast<const float *>(sums), g.sum_parts, n, dbias, bias_type, stream)) return st;
    if (dx) {
        Product p{};
        p.M = rows;
        p.N = k;
        p.splits = 1;
        p.y = dx;
        p.out_type = type;
        p.dy_max = dy_max;
        p.tma_store = tileable(dx, k, type);
        CUtensorMap map_y = {};
        if (p.tma_store)
            if (int st = make_map(&map_y, dx, type, k, rows, k, 128, 3)) return st;
        if (int st = run_product<false, false, true, kForward>(dzo, wo, type, n, map_y, none, p, sms, dev, stream))
            return st;
    }
    if (dweight) {
        Product p{};
        p.M = n;
        p.N = k;
        p.splits = g.splits;
        p.dy_max = dy_max;
        CUtensorMap map_y = {};
        if (g.splits > 1) {
            float *part = reinterpret_cast<float *>(ws + g.at_part);
            p.out_type = QC_F32;
            p.tma_store = 1;
            if (int st = make_map(&map_y, part, QC_F32, k, n, g.ld_part, 128, 3, g.splits)) return st;
            if (int st = run_product<false, true, true, kPartial>(dzo, xo, type, rows, map_y, none, p, sms, dev, stream))
                return st;
            const long long quads = (long long)n * ((k + 3) / 4);
            join_splits_kernel<<<(unsigned)((quads + 31) / 32), 256, 0, stream>>>(
                part, g.splits, n, k, g.ld_part, dweight, type);
            QC_CHECK_LAUNCH("join_splits_kernel");
        } else {
            p.y = dweight;
            p.out_type = type;
            p.tma_store = tileable(dweight, k, type);
            if (p.tma_store)
                if (int st = make_map(&map_y, dweight, type, k, n, k, 128, 3)) return st;
            if (int st = run_product<false, true, true, kForward>(dzo, xo, type, rows, map_y, none, p, sms, dev, stream))
                return st;
        }
    }
    return 0;
}

int linear_act_grad_cuda(const void *x, const void *weight, const void *bias, const void *dy, void *dx, void *dweight,
                         void *dbias, long rows, int n, int k, long x_stride, long weight_stride, long dy_stride,
                         int type, int dy_type, int bias_type, int activation, void *workspace, size_t workspace_bytes,
                         cudaStream_t stream) {
    QC_NVTX("quantem::linear_act_grad");
    return backward("linear_act_grad", x, weight, bias, nullptr, dy, dx, dweight, dbias, rows, n, k, x_stride,
                    weight_stride, dy_stride, type, dy_type, bias_type, activation, workspace, workspace_bytes, stream);
}

size_t linear_act_grad_kept_workspace_bytes(const void *x, const void *weight, const void *dy, const void *dx,
                                            const void *dweight, const void *dbias, long rows, int n, int k,
                                            long x_stride, long weight_stride, long dy_stride, int type,
                                            int activation, int device) {
    if (rows <= 0 || n < 1 || k < 1) return 0;
    int sms = 0;
    if (qc::device_sm_count(device, &sms)) return 0;
    return plan_grad(x, weight, dy, rows, n, k, x_stride, weight_stride, dy_stride, type, type, activation,
                     grad_want(dx, dweight, dbias), sms, true)
        .bytes;
}

int linear_act_grad_kept_cuda(const void *x, const void *weight, const void *kept, const void *dy, void *dx,
                              void *dweight, void *dbias, long rows, int n, int k, long x_stride, long weight_stride,
                              long dy_stride, int type, int activation, void *workspace, size_t workspace_bytes,
                              cudaStream_t stream) {
    QC_NVTX("quantem::linear_act_grad_kept");
    const char *fn = "linear_act_grad_kept";
    QC_RETURN_IF(linear_act_kept_bytes(rows, n, k, type, type, QC_BF16, activation) == 0, QC_ERR_INVALID_ARGUMENT,
                 "%s: nothing is kept of such a call", fn);
    QC_RETURN_IF(!kept || !aligned_to(kept, 16) || !dy || !tileable(dy, dy_stride, type), QC_ERR_INVALID_ARGUMENT,
                 "%s: the kept buffer or the gradient is null or not 16-byte aligned", fn);
    return backward(fn, x, weight, nullptr, kept, dy, dx, dweight, dbias, rows, n, k, x_stride, weight_stride,
                    dy_stride, type, type, type, activation, workspace, workspace_bytes, stream);
}

}  // extern "C"
