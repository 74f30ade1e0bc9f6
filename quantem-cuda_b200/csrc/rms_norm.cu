// rms_norm.cu — root-mean-square norm of rows with the residual's addition,
// its backward, and rows in 8 bits with one scale each.
//
//   h = x + residual,  r = 1/sqrt(mean(h^2) + eps),  y = h * r * w
//   q = e4m3(y / s),   s = max(max|y| / 448, 2^-126)        (8-bit output)
//   g = dy * w,  dx = r * (g - h r^2 mean(g h)) + dh,  dw = sum_rows dy * h * r
//
// Bound: HBM. A row is read once, kept in registers while its sums are formed
// and written once. A row belongs to a group of L lanes of a warp (width up to
// 1024 forward, 512 backward) or to one block (wider), so that every thread
// keeps at most 32 (16) values of it; narrow rows go several at a time so
// that enough bytes are in flight, but not so many that registers cost warps
// (262144 rows of 256 in fp32: 65 us for two at a time in 256-bit accesses,
// 75 us in 128-bit ones, 93 us for four at a time). Rows wider than a block keeps in registers
// are read twice (the second time from L2) by the strided kernels at the end.
// All sums are fp32; the weight's gradient is a sum over all rows: each block
// adds its rows in registers and leaves one partial row, and a second kernel
// adds the partial rows in fixed order, so gradients are the same run to run.
//
// y is formed from the unrounded fp32 h. The backward adds x and the residual
// again where they have 16 bits: from the stored h (rounded to 16 bits) the
// weight's gradient came out 1.5 times as far from its 64-bit value (2.5e-3
// against 1.6e-3 of its norm, 65536 rows of 1024 in bf16), for 2 bytes per
// value less traffic. With fp32 rows it reads the stored h.
#include <algorithm>
#include <type_traits>

#include "ml_common.cuh"

namespace qc {
namespace ml {

__device__ unsigned int g_norm_fault_word = 0;

bool aligned_to(const void *p, long long bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

namespace {

// Values first..last of an array of `total` (debug build; always true otherwise).
__device__ __forceinline__ bool in_array(long long first, long long last, long long total) {
    return QC_IN_BOUNDS(first, total, g_norm_fault_word) && QC_IN_BOUNDS(last, total, g_norm_fault_word);
}
// Values of rows of width n, ld apart.
__device__ __forceinline__ long long extent(long long rows, long long ld, int n) { return (rows - 1) * ld + n; }

struct NormArgs {
    const void *x, *res, *weight;
    void *y, *h;
    float *scale;
    long long rows, ldx, ldr;
    int n, out_type, norm;  // norm 0: quantise x as it is
    float eps;
};

constexpr float kE4M3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// Division by a scale of at least 2^-126: the product with its reciprocal and one
// correction by the remainder (Markstein, 1990), which rounds like the quotient itself; the product alone moves
// values across the borders of e4m3's steps twice as often. An infinite scale
// takes finite values to 0 and the infinite one to NaN, as division does.
struct Quotient {
    float inv, minus;
    __device__ __forceinline__ explicit Quotient(float s) : inv(1.f / s), minus(fabsf(s) == INFINITY ? 0.f : -s) {}
    __device__ __forceinline__ float operator()(float y) const {
        const float q = y * inv;
        return fmaf(fmaf(q, minus, y), inv, q);
    }
    __device__ __forceinline__ Pair operator()(Pair y) const {
        const Pair q = mul2(y, pair(inv));
        return fma2(fma2(q, pair(minus), y), pair(inv), q);
    }
};

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Sum (or maximum) over the block. `slot` has one float per warp and is not
// reused before the next barrier: callers alternate between two.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float *slot) {
    v = MAX ? group_max<32>(v) : group_sum<32>(v);
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    float t = slot[0];
    for (int i = 1; i < warps; ++i) t = MAX ? max_nan(t, slot[i]) : t + slot[i];
    return t;
}

// Rows whose width no vector divides (SHIFT): row r begins r*n mod V values past
// a vector boundary, the same in every array when their strides agree mod V. A
// group keeps to rows of one remainder (its rows lie a multiple of V apart), so
// that its vectors lie on the boundaries of every array and its columns, hence
// its weights and its part of dw, stay the same; only the first and the last
// vector of a row are partial. 10007 rows of 999 in fp16: 23 us against 35 us
// forward and 25 against 56 us backward with one value per access.
template <int V, bool SHIFT>
struct Span {
    int n, shift;
    __device__ __forceinline__ int col(int vec) const { return vec * V - (SHIFT ? shift : 0); }
    __device__ __forceinline__ bool any(int c) const { return SHIFT ? c + V > 0 && c < n : c < n; }
    __device__ __forceinline__ bool whole(int c) const { return !SHIFT || (c >= 0 && c + V <= n); }
    __device__ __forceinline__ bool holds(int c) const { return SHIFT ? c >= 0 && c < n : c < n; }

    // Columns c..c+V of a row at `at` in an array of `total` values. A partial
    // vector brings its neighbours' values along; mask() drops them, which
    // waits for the load, so all loads of a row are issued before.
    // whether these columns of the row at `at` lie in an array of `total` values
    __device__ __forceinline__ bool inside(long long at, int c, long long total) const {
        return in_array(at + (SHIFT ? max(c, 0) : c), at + (SHIFT ? min(c + V, n) : c + V) - 1, total);
    }
    template <int T>
    __device__ __forceinline__ void load(Raw<T, V> &r, const void *base, long long at, int c, long long total) const {
        if (!inside(at, c, total)) return;
        if (!SHIFT || (at + c >= 0 && at + c + V <= total)) r.load(base, at + c);
        else r.load_some(base, at + c, -c, n - c);
    }
    template <int T>
    __device__ __forceinline__ void mask(Raw<T, V> &r, int c) const {
        if (!whole(c)) r.keep(-c, n - c);
    }
    __device__ __forceinline__ void store(void *base, long long at, int c, int type, const float (&v)[V],
                                          long long total) const {
        if (!inside(at, c, total)) return;
        if (whole(c)) {
            store_vec<V>(base, at + c, type, v);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (holds(c + i)) store_any(base, at + c + i, type, v[i]);
        }
    }
};

// L lanes per row (L = 0: the block), NV vectors of V values per thread, R
// rows at a time.
template <int XT, int V, int L, int NV, int R, bool SHIFT>
__global__ void __launch_bounds__(L ? 256 : 512) rms_norm_kernel(NormArgs a) {
    __shared__ float slots[2][32];
    constexpr bool kBlock = L == 0;
    constexpr int kL = kBlock ? 32 : L;
    const int lanes = kBlock ? blockDim.x : L;
    const int lane = kBlock ? threadIdx.x : threadIdx.x % kL;
    const long long group = kBlock ? blockIdx.x
                                   : (long long)blockIdx.x * (blockDim.x / kL) + threadIdx.x / kL;
    const long long groups = kBlock ? gridDim.x : (long long)gridDim.x * (blockDim.x / kL);
    // the first row of this warp's groups: loops end for whole warps together
    const long long first = kBlock ? group : group - (threadIdx.x % 32) / kL;
    const Span<V, SHIFT> span{a.n, SHIFT ? (int)(group % V * (a.n % V) % V) : 0};
    const long long total_x = extent(a.rows, a.ldx, a.n), total_r = extent(a.rows, a.ldr, a.n);

    Raw<XT, V> w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = span.col(j * lanes + lane);
        w[j].zero();
        if (a.norm && span.any(c) && span.inside(0, c, a.n)) {
            if constexpr (SHIFT) w[j].load_some(a.weight, c, -c, a.n - c);
            else w[j].load(a.weight, c);
        }
    }
    const float inv_n = 1.f / (float)a.n;

    // Where registers allow it, the next rows are on their way while the present
    // ones are worked on (131072 rows of 1024 in fp16: 90 against 104 us, 300000 of
    // 256: 54 against 63 us). Elsewhere it costs warps or is no faster: fp32 rows
    // of 256 to bf16 66 against 62 us, two vectors per thread (512 wide) 63 against
    // 57 us, odd widths 145 against 88 us.
    constexpr bool kAhead = !SHIFT && XT != QC_F32 && V > 1 && !kBlock && NV != 2;
    Raw<XT, V> xr[R][NV], rr[R][NV];
    auto load_rows = [&](long long it) {
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long row = group + (it * R + q) * groups;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                xr[q][j].zero();
                rr[q][j].zero();
                if (row < a.rows && span.any(c)) {
                    span.load(xr[q][j], a.x, row * a.ldx, c, total_x);
                    if (a.res) span.load(rr[q][j], a.res, row * a.ldr, c, total_r);
                }
            }
        }
    };
    if constexpr (kAhead) load_rows(0);
    for (long long it = 0; first + it * R * groups < a.rows; ++it) {
        float h[R][NV][V];
        if constexpr (!kAhead) load_rows(it);
#pragma unroll
        for (int q = 0; q < R; ++q) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                span.mask(xr[q][j], c);
                span.mask(rr[q][j], c);
#pragma unroll
                for (int i = 0; i < V; ++i) h[q][j][i] = xr[q][j].get(i);
                if (a.res) {
                    if constexpr (V == 1) {
                        h[q][j][0] += rr[q][j].get(0);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i += 2)
                            split(add2(pair(h[q][j][i], h[q][j][i + 1]), pair(rr[q][j].get(i), rr[q][j].get(i + 1))),
                                  h[q][j][i], h[q][j][i + 1]);
                    }
                }
            }
        }
        if constexpr (kAhead) load_rows(it + 1);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long row = group + (it * R + q) * groups;
            float r = 1.f;
            if (a.norm) {
                float ss = 0.f;
                if constexpr (V == 1) {
#pragma unroll
                    for (int j = 0; j < NV; ++j) ss += h[q][j][0] * h[q][j][0];
                } else {
                    Pair ss2 = pair(0.f);
                    float odd;
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int i = 0; i < V; i += 2) {
                            const Pair v = pair(h[q][j][i], h[q][j][i + 1]);
                            ss2 = fma2(v, v, ss2);
                        }
                    split(ss2, ss, odd);
                    ss += odd;
                }
                ss = kBlock ? block_reduce<false>(ss, slots[0]) : group_sum<kL>(ss);
                r = rsqrtf(ss * inv_n + a.eps);
            }
            if (a.h) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = span.col(j * lanes + lane);
                    if (row < a.rows && span.any(c)) span.store(a.h, row * a.n, c, XT, h[q][j], a.rows * a.n);
                }
            }
            if (a.norm) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if constexpr (V == 1) {
                        h[q][j][0] = h[q][j][0] * r * w[j].get(0);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i += 2)
                            split(mul2(mul2(pair(h[q][j][i], h[q][j][i + 1]), pair(r)),
                                       pair(w[j].get(i), w[j].get(i + 1))),
                                  h[q][j][i], h[q][j][i + 1]);
                    }
                }
            }
            if (a.scale) {
                float amax = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) amax = max_nan(amax, fabsf(h[q][j][i]));
                amax = kBlock ? block_reduce<true>(amax, slots[1]) : group_max<kL>(amax);
                const float s = max_nan(amax / kE4M3Max, kMinScale);
                const Quotient by(s);
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if constexpr (V == 1) {
                        h[q][j][0] = by(h[q][j][0]);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i += 2)
                            split(by(pair(h[q][j][i], h[q][j][i + 1])), h[q][j][i], h[q][j][i + 1]);
                    }
                }
                if (lane == 0 && row < a.rows && in_array(row, row, a.rows)) a.scale[row] = s;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                if (row < a.rows && span.any(c)) span.store(a.y, row * a.n, c, a.out_type, h[q][j], a.rows * a.n);
            }
            // two uses of one slot array lie a barrier apart only when both
            // arrays are used (norm and scale); otherwise the block waits here
            if (kBlock && !(a.norm && a.scale)) __syncthreads();
        }
    }
}

// Column c of a row in an array whose rows lie ld apart; in x, the residual and
// the weight.
template <typename Args>
__device__ __forceinline__ bool in_rows(const Args &a, long long row, long long ld, int c) {
    return in_array(row * ld + c, row * ld + c, extent(a.rows, ld, a.n));
}
template <typename Args>
__device__ __forceinline__ bool at_inside(const Args &a, long long row, int c) {
    return in_array(c, c, a.n) && in_rows(a, row, a.ldx, c) && (!a.res || in_rows(a, row, a.ldr, c));
}

// Rows of any width: one block per row, strided, read again for each pass.
template <int XT>
__global__ void __launch_bounds__(1024) rms_norm_wide_kernel(NormArgs a) {
    __shared__ float slots[2][32];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        auto h_at = [&](int c) {
            if (!at_inside(a, row, c)) return 0.f;
            float v = load_any(a.x, row * a.ldx + c, XT);
            if (a.res) v += load_any(a.res, row * a.ldr + c, XT);
            return v;
        };
        float r = 1.f;
        if (a.norm) {
            float ss = 0.f;
            for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
                const float h = h_at(c);
                ss += h * h;
            }
            r = rsqrtf(block_reduce<false>(ss, slots[0]) * (1.f / (float)a.n) + a.eps);
        }
        float s = 1.f;
        if (a.scale) {
            float amax = 0.f;
            for (int c = threadIdx.x; c < a.n; c += blockDim.x)
                amax = max_nan(amax, fabsf(a.norm ? h_at(c) * r * load_any(a.weight, c, XT) : h_at(c)));
            s = max_nan(block_reduce<true>(amax, slots[1]) / kE4M3Max, kMinScale);
            if (threadIdx.x == 0) a.scale[row] = s;
        }
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
            const float h = h_at(c);
            float y = a.norm ? h * r * load_any(a.weight, c, XT) : h;
            if (a.scale) y = Quotient(s)(y);
            if (!in_array(row * a.n + c, row * a.n + c, a.rows * a.n)) continue;
            if (a.h) store_any(a.h, row * a.n + c, XT, h);
            store_any(a.y, row * a.n + c, a.out_type, y);
        }
        __syncthreads();
    }
}

struct NormGradArgs {
    const void *x, *res, *weight, *dy, *dh;  // h = x + res (res may be null)
    void *dx;
    float *dw_part;  // [gridDim.x][n], or null
    void *dw;        // a single block writes the sum itself
    long long rows, ldx, ldr, lddy, lddh;
    int n;
    float eps;
    long long dw_room;  // values that dw_part has room for
};

template <int XT, int YT, int V, int L, int NV, int R, bool SHIFT>
__global__ void __launch_bounds__(L ? 256 : 512) rms_norm_grad_kernel(NormGradArgs a) {
    extern __shared__ float dw_sh[];  // [n], warp groups only
    __shared__ float slots[2][2][32];
    constexpr bool kBlock = L == 0;
    constexpr int kL = kBlock ? 32 : L;
    const int lanes = kBlock ? blockDim.x : L;
    const int lane = kBlock ? threadIdx.x : threadIdx.x % kL;
    const long long group = kBlock ? blockIdx.x
                                   : (long long)blockIdx.x * (blockDim.x / kL) + threadIdx.x / kL;
    const long long groups = kBlock ? gridDim.x : (long long)gridDim.x * (blockDim.x / kL);
    const long long first = kBlock ? group : group - (threadIdx.x % 32) / kL;
    const Span<V, SHIFT> span{a.n, SHIFT ? (int)(group % V * (a.n % V) % V) : 0};

    Raw<XT, V> w[NV];
    float dw[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = span.col(j * lanes + lane);
        w[j].zero();
        if (span.any(c) && span.inside(0, c, a.n)) {
            if constexpr (SHIFT) w[j].load_some(a.weight, c, -c, a.n - c);
            else w[j].load(a.weight, c);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.f;
    }
    const float inv_n = 1.f / (float)a.n;
    int flip = 0;

    for (long long it = 0; first + it * R * groups < a.rows; ++it) {
        Raw<XT, V> x[R][NV], res[R][NV], dh[R][NV];
        Raw<YT, V> dy[R][NV];
#pragma unroll
        for (int q = 0; q < R; ++q)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                const long long row = group + (it * R + q) * groups;
                x[q][j].zero();
                res[q][j].zero();
                dy[q][j].zero();
                dh[q][j].zero();
                if (row < a.rows && span.any(c)) {
                    span.load(x[q][j], a.x, row * a.ldx, c, extent(a.rows, a.ldx, a.n));
                    if (a.res) span.load(res[q][j], a.res, row * a.ldr, c, extent(a.rows, a.ldr, a.n));
                    span.load(dy[q][j], a.dy, row * a.lddy, c, extent(a.rows, a.lddy, a.n));
                    if (a.dh) span.load(dh[q][j], a.dh, row * a.lddh, c, extent(a.rows, a.lddh, a.n));
                }
            }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const long long row = group + (it * R + q) * groups;
            float ss = 0.f, gh = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                span.mask(x[q][j], c);
                span.mask(res[q][j], c);
                span.mask(dy[q][j], c);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float hv = x[q][j].get(i) + res[q][j].get(i);
                    ss += hv * hv;
                    gh += hv * (dy[q][j].get(i) * w[j].get(i));
                }
            }
            if constexpr (kBlock) {
                // both sums behind one barrier; the slots alternate, so a
                // thread still reading the last row's is not overtaken
                ss = group_sum<32>(ss);
                gh = group_sum<32>(gh);
                if ((threadIdx.x & 31) == 0) {
                    slots[flip][0][threadIdx.x >> 5] = ss;
                    slots[flip][1][threadIdx.x >> 5] = gh;
                }
                __syncthreads();
                ss = gh = 0.f;
                for (int k = 0; k < (int)(blockDim.x >> 5); ++k) {
                    ss += slots[flip][0][k];
                    gh += slots[flip][1][k];
                }
                flip ^= 1;
            } else {
                ss = group_sum<kL>(ss);
                gh = group_sum<kL>(gh);
            }
            const float r = rsqrtf(ss * inv_n + a.eps);
            const float k = r * r * (gh * inv_n);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = span.col(j * lanes + lane);
                float dx[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float hv = x[q][j].get(i) + res[q][j].get(i), d = dy[q][j].get(i);
                    dx[i] = r * (d * w[j].get(i) - hv * k);
                    if (a.dh) dx[i] += dh[q][j].get(i);
                    if (row < a.rows) dw[j][i] += d * (hv * r);
                }
                if (a.dx && row < a.rows && span.any(c)) span.store(a.dx, row * a.n, c, XT, dx, a.rows * a.n);
            }
        }
    }
    if (a.dw_part == nullptr) return;
    float *part = a.dw_part + (long long)blockIdx.x * a.n;
    auto dw_inside = [&](int c) {
        const long long at = gridDim.x == 1 ? c : (long long)blockIdx.x * a.n + c;
        return in_array(at, at, gridDim.x == 1 ? a.n : a.dw_room);
    };
    if constexpr (kBlock) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = span.col(j * lanes + lane) + i;
                if (!span.holds(c) || !dw_inside(c)) continue;
                if (gridDim.x == 1) store_any(a.dw, c, XT, dw[j][i]);
                else part[c] = dw[j][i];
            }
    } else {
        // lanes of a warp's groups that hold the same columns (without SHIFT),
        // then the warps (with SHIFT: the groups) in turn
        if constexpr (!SHIFT) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int o = kL; o < 32; o <<= 1) dw[j][i] += __shfl_xor_sync(0xffffffffu, dw[j][i], o);
        }
        constexpr int kTurn = SHIFT ? kL : 32;
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) dw_sh[c] = 0.f;
        __syncthreads();
        for (int k = 0; k < (int)blockDim.x / kTurn; ++k) {
            if ((int)threadIdx.x / kTurn == k && (SHIFT || (threadIdx.x & 31) < kL)) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int c = span.col(j * lanes + lane) + i;
                        if (span.holds(c)) dw_sh[c] += dw[j][i];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
            if (!dw_inside(c)) continue;
            if (gridDim.x == 1) store_any(a.dw, c, XT, dw_sh[c]);
            else part[c] = dw_sh[c];
        }
    }
}

// Any width. The block's partial row lives in the workspace: each thread adds
// to its own columns only.
template <int XT, int YT>
__global__ void __launch_bounds__(1024) rms_norm_grad_wide_kernel(NormGradArgs a) {
    __shared__ float slots[2][32];
    float *part = a.dw_part ? a.dw_part + (long long)blockIdx.x * a.n : nullptr;
    auto h_at = [&](long long row, int c) {
        if (!at_inside(a, row, c) || !in_rows(a, row, a.lddy, c) || (a.dh && !in_rows(a, row, a.lddh, c))) return 0.f;
        float v = load_any(a.x, row * a.ldx + c, XT);
        if (a.res) v += load_any(a.res, row * a.ldr + c, XT);
        return v;
    };
    if (part && !in_array((long long)blockIdx.x * a.n, (long long)(blockIdx.x + 1) * a.n - 1, a.dw_room)) part = nullptr;
    if (part)
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) part[c] = 0.f;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float ss = 0.f, gh = 0.f;
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
            const float h = h_at(row, c);
            ss += h * h;
            gh += h * (load_any(a.dy, row * a.lddy + c, YT) * load_any(a.weight, c, XT));
        }
        ss = block_reduce<false>(ss, slots[0]);
        gh = block_reduce<false>(gh, slots[1]);
        const float r = rsqrtf(ss * (1.f / (float)a.n) + a.eps);
        const float k = r * r * (gh * (1.f / (float)a.n));
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
            const float h = h_at(row, c), d = load_any(a.dy, row * a.lddy + c, YT);
            float dx = r * (d * load_any(a.weight, c, XT) - h * k);
            if (a.dh) dx += load_any(a.dh, row * a.lddh + c, XT);
            if (a.dx && in_array(row * a.n + c, row * a.n + c, a.rows * a.n)) store_any(a.dx, row * a.n + c, XT, dx);
            if (part) part[c] += d * (h * r);
        }
        __syncthreads();
    }
    if (part && gridDim.x == 1)
        for (int c = threadIdx.x; c < a.n; c += blockDim.x) store_any(a.dw, c, XT, part[c]);
}

// 8 columns (one 32-byte sector) per block, 32 threads down the partial rows.
__global__ void __launch_bounds__(256) colsum_reduce_kernel(const float *partial, int parts, int n, void *out,
                                                            int out_type) {
    __shared__ float sh[32][9];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), lane = threadIdx.x >> 3;
    float s = 0.f;
    if (c < n) {
        int p = lane;
        if (!QC_IN_BOUNDS(c, n, g_norm_fault_word)) p = parts;
        for (; p + 224 < parts; p += 256) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = partial[(long long)(p + 32 * i) * n + c];
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; p < parts; p += 32) s += partial[(long long)p * n + c];
    }
    sh[lane][threadIdx.x & 7] = s;
    __syncthreads();
    if (threadIdx.x < 8 && c < n) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sh[i][threadIdx.x];
        store_any(out, c, out_type, s);
    }
}

// ── host side ────────────────────────────────────────────────────────────

constexpr int kLive = 16;  // values per thread of all the rows in flight
constexpr int kFwdPerThread = 32, kBwdPerThread = 16;  // values of a row per thread, at most
constexpr int kMaxParts = 148 * 8;

int pow2_at_least(long long v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// Blocks for `rows`: one group's row each, or as many as the SMs hold. Groups
// number a multiple of 8 unless each has a single row.
long long blocks_for(long long rows, long long rows_per_block, long long most) {
    const long long want = (rows + rows_per_block - 1) / rows_per_block;
    return want <= most ? want : std::max<long long>(8, most / 8 * 8);
}

constexpr int rows_at_a_time(int live, int per_row) {
    return live / per_row < 1 ? 1 : live / per_row > 4 ? 4 : live / per_row;
}

template <int XT, int V, int L, int NV, bool SHIFT>
int launch_fwd(const NormArgs &a, int threads, int sms, cudaStream_t stream) {
    constexpr int R = L ? rows_at_a_time(kLive, NV * V) : 1;
    const long long per_block = L ? (long long)threads / (L ? L : 1) : 1;
    const long long grid = blocks_for(a.rows, per_block, (long long)sms * (2048 / threads));
    rms_norm_kernel<XT, V, L, NV, R, SHIFT><<<(unsigned)grid, threads, 0, stream>>>(a);
    QC_CHECK_LAUNCH("rms_norm_kernel");
    return 0;
}

template <int XT, int V, bool SHIFT>
int dispatch_fwd(const NormArgs &a, int sms, cudaStream_t stream) {
    const long long vecs = SHIFT ? (a.n + 2 * V - 2) / V : (a.n + V - 1) / V;
    if (vecs <= 32 * kFwdPerThread / V) {
        if constexpr (V > 1) {
            if (vecs <= 4) return launch_fwd<XT, V, 4, 1, SHIFT>(a, 256, sms, stream);
            if (vecs <= 8) return launch_fwd<XT, V, 8, 1, SHIFT>(a, 256, sms, stream);
            if (vecs <= 16) return launch_fwd<XT, V, 16, 1, SHIFT>(a, 256, sms, stream);
        }
        switch (pow2_at_least((vecs + 31) / 32)) {
            case 1: return launch_fwd<XT, V, 32, 1, SHIFT>(a, 256, sms, stream);
            case 2: return launch_fwd<XT, V, 32, 2, SHIFT>(a, 256, sms, stream);
            case 4: return launch_fwd<XT, V, 32, 4, SHIFT>(a, 256, sms, stream);
            case 8:
                if constexpr (V <= 4) return launch_fwd<XT, V, 32, 8, SHIFT>(a, 256, sms, stream);
                break;
            default:
                if constexpr (V == 1) return launch_fwd<XT, V, 32, 32, SHIFT>(a, 256, sms, stream);
                break;
        }
    }
    for (int threads = 256; threads <= 512; threads *= 2) {
        const long long nv = (vecs + threads - 1) / threads;
        if (nv * V > kFwdPerThread) continue;
        if (nv <= 1) return launch_fwd<XT, V, 0, 1, SHIFT>(a, threads, sms, stream);
        if (nv <= 2) return launch_fwd<XT, V, 0, 2, SHIFT>(a, threads, sms, stream);
        if (nv <= 4) return launch_fwd<XT, V, 0, 4, SHIFT>(a, threads, sms, stream);
        if constexpr (V <= 4)
            if (nv <= 8) return launch_fwd<XT, V, 0, 8, SHIFT>(a, threads, sms, stream);
        if constexpr (V == 1) return launch_fwd<XT, V, 0, 32, SHIFT>(a, threads, sms, stream);
    }
    rms_norm_wide_kernel<XT><<<(unsigned)blocks_for(a.rows, 1, sms * 2), 1024, 0, stream>>>(a);
    QC_CHECK_LAUNCH("rms_norm_wide_kernel");
    return 0;
}

// Whether vectors of V values lie alike in an array (a null one does): rows of
// stride ld from an address aligned to `bytes`.
template <int V>
bool alike(const void *p, long long ld, const NormArgs &a, int bytes) {
    return !p || (aligned_to(p, bytes) && (a.rows <= 1 || (ld - a.n) % V == 0));
}

template <int XT>
int run_fwd(const NormArgs &a, int sms, cudaStream_t stream) {
    constexpr int V = 8, kX = V * (XT == QC_F32 ? 4 : 2);
    if (alike<V>(a.x, a.ldx, a, kX) && alike<V>(a.res, a.ldr, a, kX) && alike<V>(a.weight, a.n, a, kX) &&
        alike<V>(a.h, a.n, a, kX) && alike<V>(a.y, a.n, a, V * elem_size(a.out_type)))
        return a.n % V == 0 ? dispatch_fwd<XT, V, false>(a, sms, stream) : dispatch_fwd<XT, V, true>(a, sms, stream);
    return dispatch_fwd<XT, 1, false>(a, sms, stream);
}

template <int XT, int YT, int V, int L, int NV, bool SHIFT>
int launch_bwd(const NormGradArgs &a, int threads, long long grid, cudaStream_t stream) {
    constexpr int R = L ? rows_at_a_time(kLive, NV * V) : 1;
    const size_t smem = L && a.dw_part ? (size_t)a.n * 4 : 0;
    rms_norm_grad_kernel<XT, YT, V, L, NV, R, SHIFT><<<(unsigned)grid, threads, smem, stream>>>(a);
    QC_CHECK_LAUNCH("rms_norm_grad_kernel");
    return 0;
}

// Blocks of a backward: each leaves a partial row in the workspace. A small one
// takes one block, which needs no second kernel (3 us of a call's host time); its
// groups then take rows 8 or more apart, as odd widths need.
long long grad_blocks(long long rows, int n, long long rows_per_block, long long most) {
    if (rows_per_block > 1 && rows * n <= 16384) return 1;
    return blocks_for(rows, rows_per_block, std::min<long long>(most, kMaxParts));
}

template <int XT, int YT, int V, bool SHIFT>
int dispatch_bwd(const NormGradArgs &a, int sms, int *parts, cudaStream_t stream) {
    const long long vecs = SHIFT ? (a.n + 2 * V - 2) / V : (a.n + V - 1) / V;
    if (vecs <= 32 * kBwdPerThread / V) {
        const int L = V == 1 ? 32 : vecs <= 4 ? 4 : vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32;
        const long long grid = grad_blocks(a.rows, a.n, 256 / L, sms * 4);
        *parts = (int)grid;
        if constexpr (V > 1) {
            if (L == 4) return launch_bwd<XT, YT, V, 4, 1, SHIFT>(a, 256, grid, stream);
            if (L == 8) return launch_bwd<XT, YT, V, 8, 1, SHIFT>(a, 256, grid, stream);
            if (L == 16) return launch_bwd<XT, YT, V, 16, 1, SHIFT>(a, 256, grid, stream);
        }
        switch (pow2_at_least((vecs + 31) / 32)) {
            case 1: return launch_bwd<XT, YT, V, 32, 1, SHIFT>(a, 256, grid, stream);
            case 2: return launch_bwd<XT, YT, V, 32, 2, SHIFT>(a, 256, grid, stream);
            case 4:
                if constexpr (V <= 4) return launch_bwd<XT, YT, V, 32, 4, SHIFT>(a, 256, grid, stream);
                break;
            default:
                if constexpr (V == 1) return launch_bwd<XT, YT, V, 32, 16, SHIFT>(a, 256, grid, stream);
                break;
        }
    }
    for (int threads = 128; threads <= 512; threads *= 2) {
        const long long nv = (vecs + threads - 1) / threads;
        if (nv * V > kBwdPerThread) continue;
        const long long grid = grad_blocks(a.rows, a.n, 1, (long long)sms * (1024 / threads));
        *parts = (int)grid;
        if (nv <= 1) return launch_bwd<XT, YT, V, 0, 1, SHIFT>(a, threads, grid, stream);
        if (nv <= 2) return launch_bwd<XT, YT, V, 0, 2, SHIFT>(a, threads, grid, stream);
        if constexpr (V <= 4)
            if (nv <= 4) return launch_bwd<XT, YT, V, 0, 4, SHIFT>(a, threads, grid, stream);
        if constexpr (V == 1) return launch_bwd<XT, YT, V, 0, 16, SHIFT>(a, threads, grid, stream);
    }
    const long long grid = grad_blocks(a.rows, a.n, 1, sms * 2);
    *parts = (int)grid;
    rms_norm_grad_wide_kernel<XT, YT><<<(unsigned)grid, 1024, 0, stream>>>(a);
    QC_CHECK_LAUNCH("rms_norm_grad_wide_kernel");
    return 0;
}

template <int V>
bool alike(const void *p, long long ld, const NormGradArgs &a, int bytes) {
    return !p || (aligned_to(p, bytes) && (a.rows <= 1 || (ld - a.n) % V == 0));
}

template <int XT, int YT>
int run_bwd(const NormGradArgs &a, int sms, int *parts, cudaStream_t stream) {
    constexpr int V = XT == QC_F32 ? 4 : 8, kX = 16;
    if (alike<V>(a.x, a.ldx, a, kX) && alike<V>(a.res, a.ldr, a, kX) && alike<V>(a.weight, a.n, a, kX) &&
        alike<V>(a.dy, a.lddy, a, V * elem_size(YT)) && alike<V>(a.dh, a.lddh, a, kX) && alike<V>(a.dx, a.n, a, kX))
        return a.n % V == 0 ? dispatch_bwd<XT, YT, V, false>(a, sms, parts, stream)
                            : dispatch_bwd<XT, YT, V, true>(a, sms, parts, stream);
    return dispatch_bwd<XT, YT, 1, false>(a, sms, parts, stream);
}

int check_rows(const char *fn, const void *x, const void *weight, long rows, int n, long ldx, long ldr,
               const void *res, int x_type) {
    QC_RETURN_IF(rows < 0 || n < 1, QC_ERR_INVALID_ARGUMENT, "%s: rows %ld, width %d", fn, rows, n);
    QC_RETURN_IF(x_type != QC_F32 && x_type != QC_BF16 && x_type != QC_F16, QC_ERR_INVALID_ARGUMENT,
                 "%s: unknown element type %d", fn, x_type);
    QC_RETURN_IF(rows > 0 && (x == nullptr || weight == nullptr), QC_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
    QC_RETURN_IF(ldx < 0 || (res != nullptr && ldr < 0), QC_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
    return 0;
}

int norm_forward(const char *fn, const NormArgs &a, int x_type, cudaStream_t stream) {
    if (a.rows == 0) return 0;
    int sms = 0;
    if (int st = device_sm_count(&sms)) return st;
    switch (x_type) {
        case QC_F32: return run_fwd<QC_F32>(a, sms, stream);
        case QC_BF16: return run_fwd<QC_BF16>(a, sms, stream);
        default: return run_fwd<QC_F16>(a, sms, stream);
    }
}

}  // namespace

int launch_colsum_reduce(const float *partial, int parts, int n, void *out, int out_type, cudaStream_t stream) {
    colsum_reduce_kernel<<<(n + 7) / 8, 256, 0, stream>>>(partial, parts, n, out, out_type);
    QC_CHECK_LAUNCH("colsum_reduce_kernel");
    return 0;
}

int norm_fault_word(unsigned int *word, int clear) {
    unsigned int w = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&w, g_norm_fault_word, sizeof(w));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_norm_fault_word, &zero, sizeof(zero));
    }
    QC_CUDA_TRY(e, "cudaMemcpyFromSymbol(fault word)");
    *word = w;
    return 0;
}

}  // namespace ml
}  // namespace qc

using namespace qc::ml;

extern "C" {

int rms_norm_cuda(const void *x, const void *residual, const void *weight, void *y, void *h, float *scale, long rows,
                  int n, long x_stride, long residual_stride, int x_type, int out_type, float eps,
                  cudaStream_t stream) {
    QC_NVTX("quantem::rms_norm");
    if (int st = check_rows("rms_norm", x, weight, rows, n, x_stride, residual_stride, residual, x_type)) return st;
    QC_RETURN_IF(out_type < QC_F32 || out_type > QC_E4M3, QC_ERR_INVALID_ARGUMENT, "rms_norm: unknown output type %d",
                 out_type);
    QC_RETURN_IF((out_type == QC_E4M3) != (scale != nullptr) && rows > 0, QC_ERR_INVALID_ARGUMENT,
                 "rms_norm: 8-bit output needs scales, and no other does");
    QC_RETURN_IF(rows > 0 && y == nullptr, QC_ERR_INVALID_ARGUMENT, "rms_norm: null output");
    QC_RETURN_IF((residual != nullptr) != (h != nullptr) && rows > 0, QC_ERR_INVALID_ARGUMENT,
                 "rms_norm: the sum h is written exactly when a residual is added");
    NormArgs a{x, residual, weight, y, h, scale, rows, x_stride, residual_stride, n, out_type, 1, eps};
    return norm_forward("rms_norm", a, x_type, stream);
}

int quantize_rows_cuda(const void *x, void *q, float *scale, long rows, int n, long x_stride, int x_type,
                       cudaStream_t stream) {
    QC_NVTX("quantem::quantize_rows");
    if (int st = check_rows("quantize_rows", x, x, rows, n, x_stride, 0, nullptr, x_type)) return st;
    QC_RETURN_IF(rows > 0 && (q == nullptr || scale == nullptr), QC_ERR_INVALID_ARGUMENT,
                 "quantize_rows: null output");
    NormArgs a{x, nullptr, nullptr, q, nullptr, scale, rows, x_stride, 0, n, QC_E4M3, 0, 0.f};
    return norm_forward("quantize_rows", a, x_type, stream);
}

size_t rms_norm_grad_workspace_bytes(long rows, int n) {
    if (rows <= 0 || n <= 0) return 0;
    const long parts = rows < kMaxParts ? rows : kMaxParts;
    return (size_t)parts * n * sizeof(float);
}

int rms_norm_grad_cuda(const void *x, const void *residual, const void *weight, const void *dy, const void *dh,
                       void *dx, void *dweight, long rows, int n, long x_stride, long residual_stride, long dy_stride,
                       long dh_stride, int x_type, int dy_type, float eps, void *workspace, size_t workspace_bytes,
                       cudaStream_t stream) {
    QC_NVTX("quantem::rms_norm_grad");
    if (int st = check_rows("rms_norm_grad", x, weight, rows, n, x_stride, residual_stride, residual, x_type)) return st;
    QC_RETURN_IF(dy_type != QC_F32 && dy_type != QC_BF16 && dy_type != QC_F16, QC_ERR_INVALID_ARGUMENT,
                 "rms_norm_grad: unknown gradient type %d", dy_type);
    QC_RETURN_IF(rows > 0 && dy == nullptr, QC_ERR_INVALID_ARGUMENT, "rms_norm_grad: null upstream gradient");
    QC_RETURN_IF(dy_stride < 0 || dh_stride < 0, QC_ERR_INVALID_ARGUMENT, "rms_norm_grad: negative row stride");
    QC_RETURN_IF(dweight && workspace_bytes < rms_norm_grad_workspace_bytes(rows, n), QC_ERR_WORKSPACE_TOO_SMALL,
                 "rms_norm_grad: workspace of %zu bytes, %zu needed", workspace_bytes,
                 rms_norm_grad_workspace_bytes(rows, n));
    QC_RETURN_IF(dweight && rows > 0 && !aligned_to(workspace, 4), QC_ERR_INVALID_ARGUMENT,
                 "rms_norm_grad: workspace is not 4-byte aligned");
    int sms = 0;
    if (int st = qc::device_sm_count(&sms)) return st;
    int parts = 0;
    if (rows > 0) {
        NormGradArgs a{x, residual, weight, dy, dh, dx, dweight ? static_cast<float *>(workspace) : nullptr, dweight,
                       rows, x_stride, residual_stride, dy_stride, dh_stride, n, eps,
                       (long long)(workspace_bytes / sizeof(float))};
        int st = 0;
        const int key = x_type * 4 + dy_type;
        switch (key) {
#define QC_CASE(X, Y) \
    case X * 4 + Y: st = run_bwd<X, Y>(a, sms, &parts, stream); break;
            QC_CASE(QC_F32, QC_F32)
            QC_CASE(QC_F32, QC_BF16)
            QC_CASE(QC_F32, QC_F16)
            QC_CASE(QC_BF16, QC_BF16)
            QC_CASE(QC_BF16, QC_F32)
            QC_CASE(QC_F16, QC_F16)
            QC_CASE(QC_F16, QC_F32)
#undef QC_CASE
            default:
                return qc::set_error(QC_ERR_INVALID_ARGUMENT, "rms_norm_grad: a gradient of type %d for rows of type %d",
                                     dy_type, x_type);
        }
        if (st) return st;
    }
    // no rows: the gradient of the weight is zero; one block has written it
    if (dweight && parts != 1) return launch_colsum_reduce(static_cast<const float *>(workspace), parts, n, dweight, x_type, stream);
    return 0;
}

}  // extern "C"
