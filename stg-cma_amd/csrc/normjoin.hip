// Norm after a block, gate, scaled residual sum, norm before the next block -- one row pass forward, one row pass backward:
//     n = Norm(h) w1 (+ b1),   x' = alpha x + gate o n,   y = Norm(x') w2 (+ b2)          Norm: LayerNorm or RMS norm over the last dim
// As separate passes the chain moves the branch h, the stream x and their images six to eight times; here every tensor crosses HBM once
// (forward: h, x in, x', y out; backward: dy, dx', x', h in, dx, dh out), which is the floor: the arithmetic (~15 / ~30 operations per element)
// stays under it.  The gradients of the weights and the gate are column sums over all rows: every block keeps its columns' sums in registers
// over its share of the rows and leaves ONE partial row, added up in a fixed order by a second kernel -- no atomics, repeatable bit for bit.
// x' is rounded to the stream's type before the second norm reads it, so that the backward, which reads the stored x', sees the same values.
// 62720 x 512, fp32 stream: 75 us forward (5.1 TB/s), 122 us backward (4.7 TB/s), plain copies of 256 MiB .. 8 GiB on such a card 5.4 .. 4.7; 16384 x 4096, bf16 stream: 100 us forward
// (5.4 TB/s).
#include <math.h>
#include "common.h"
#include "../../include/stgcma.h"

namespace {

struct JP {
    const void* x; int64_t ldx;
    const bf16_t* h; int64_t ldh;
    const float* gate; int gate_kind; int64_t rpg;        // 0 none, 1 scalar, 2 [C], 3 [groups, C] with rpg rows to a group
    const float* w1; const float* b1; const float* w2; const float* b2;
    float alpha, eps;
    void* xo; int64_t ldxo;
    bf16_t* y; int64_t ldy;
    float* stats;                                         // [rows, 4]: mean1, rstd1, mean2, rstd2 (means 0 for RMS)
    int64_t rows; int C; int rms;
    const bf16_t* dy; int64_t lddy;
    const void* dxo; int64_t lddxo;
    void* dx; int64_t lddx;
    bf16_t* dh; int64_t lddh;
    float* part; int64_t pcols;                           // [blocks, pcols]: dw1, db1 (if b1), dw2, db2 (if b2), dgate ([C] or one value)
    float* gpart;                                         // gate_kind 3: [groups * W, C]
    int64_t G; int W; int64_t gpw, piece;                 // row groups, splits of a group, groups of a block, rows of a split
};

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void unpack8(const u4_t& u, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const bf16_t* p, float* v) { unpack8(*reinterpret_cast<const u4_t*>(p), v); }
__device__ __forceinline__ void load8(const float* p, float* v) {
    const f4_t a = *reinterpret_cast<const f4_t*>(p), b = *reinterpret_cast<const f4_t*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ u4_t packed8(const float* v) { return (u4_t){pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])}; }
__device__ __forceinline__ void store8(bf16_t* p, const float* v) { *reinterpret_cast<u4_t*>(p) = packed8(v); }
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<f4_t*>(p) = (f4_t){v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f4_t*>(p + 4) = (f4_t){v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void round_as(float*, const float*) {}                     // fp32 stream: stored as computed
__device__ __forceinline__ void round_as(bf16_t*, float* v) { const u4_t u = packed8(v); unpack8(u, v); }

// sum over the TPR threads that share a row (every wave of the block calls it the same number of times)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum<(TPR < 64 ? TPR : 64)>(v);
    if (TPR <= 64) return v;
    const int wave = threadIdx.x >> 6, w0 = wave / (TPR / 64) * (TPR / 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) t += red[w0 + w];
    return t;
}
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
    a = wave_sum<(TPR < 64 ? TPR : 64)>(a);
    b = wave_sum<(TPR < 64 ? TPR : 64)>(b);
    if (TPR <= 64) return;
    const int wave = threadIdx.x >> 6, w0 = wave / (TPR / 64) * (TPR / 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { red[wave] = a; red[8 + wave] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) { a += red[w0 + w]; b += red[8 + w0 + w]; }
}

// Eight elements as they lie in memory: a row's loads are asked for one row ahead, so they stay raw until their turn.
template <typename T> struct Raw8 { u4_t a, b; };
template <> struct Raw8<bf16_t> { u4_t a; };
__device__ __forceinline__ void ask(Raw8<bf16_t>& r, const bf16_t* p) { r.a = *reinterpret_cast<const u4_t*>(p); }
__device__ __forceinline__ void ask(Raw8<float>& r, const float* p) { r.a = *reinterpret_cast<const u4_t*>(p); r.b = *reinterpret_cast<const u4_t*>(p + 4); }
__device__ __forceinline__ void none(Raw8<bf16_t>& r) { r.a = (u4_t){0u, 0u, 0u, 0u}; }
__device__ __forceinline__ void none(Raw8<float>& r) { r.a = r.b = (u4_t){0u, 0u, 0u, 0u}; }
__device__ __forceinline__ void open8(const Raw8<bf16_t>& r, float* v) { unpack8(r.a, v); }
__device__ __forceinline__ void open8(const Raw8<float>& r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(r.a[i]); v[4 + i] = __uint_as_float(r.b[i]); }
}

// TPR threads own a row, 8 NCH columns each (16 .. 512 threads: rows of up to 128 columns go four to a wave), and keep the columns' weights in registers over
// their rows; a block of NT threads has RG rows in flight.
template <int TPR> struct Blk { static constexpr int NT = TPR <= 256 ? 256 : TPR, RG = NT / TPR; };

template <typename XT, int TPR, int NCH>
__global__ void __launch_bounds__(Blk<TPR>::NT) norm_join_fwd_kernel(JP a) {
    constexpr int RG = Blk<TPR>::RG;
    __shared__ float red[16];
    const int rg = threadIdx.x / TPR, col0 = 8 * (threadIdx.x % TPR);
    const float invC = 1.0f / (float)a.C;
    float w1[NCH][8], b1[NCH][8], w2[NCH][8], b2[NCH][8], g[NCH][8];
    bool on[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int col = col0 + 8 * TPR * c;
        on[c] = col < a.C;
        const float s = a.gate_kind == 1 ? a.gate[0] : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { w1[c][i] = b1[c][i] = w2[c][i] = b2[c][i] = 0.f; g[c][i] = s; }
        if (on[c]) {
            load8(a.w1 + col, w1[c]);
            load8(a.w2 + col, w2[c]);
            if (a.b1) load8(a.b1 + col, b1[c]);
            if (a.b2) load8(a.b2 + col, b2[c]);
            if (a.gate_kind == 2) load8(a.gate + col, g[c]);
        }
    }
    Raw8<bf16_t> rh[NCH];
    Raw8<XT> rx[NCH];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = col0 + 8 * TPR * c;
            none(rh[c]);
            none(rx[c]);
            if (on[c] && row < a.rows) {
                ask(rh[c], a.h + row * a.ldh + col);
                ask(rx[c], (const XT*)a.x + row * a.ldx + col);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * RG;
    fetch((int64_t)blockIdx.x * RG + rg);
    for (int64_t base = (int64_t)blockIdx.x * RG; base < a.rows; base += step) {
        const int64_t row = base + rg;
        float h[NCH][8], x[NCH][8];
        float m1 = 0.f, m2 = 0.f, s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            open8(rh[c], h[c]);
            open8(rx[c], x[c]);
            if (a.gate_kind == 3 && on[c] && row < a.rows) load8(a.gate + (row / a.rpg) * a.C + col0 + 8 * TPR * c, g[c]);
        }
        fetch(row + step);
        if (!a.rms) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) s += h[c][i];
            m1 = row_sum<TPR>(s, red) * invC;
        }
        s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) { h[c][i] = on[c] ? h[c][i] - m1 : 0.f; s = fmaf(h[c][i], h[c][i], s); }
        const float r1 = rsqrtf(row_sum<TPR>(s, red) * invC + a.eps);
        s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = fmaf(h[c][i] * r1, w1[c][i], b1[c][i]);
                x[c][i] = fmaf(g[c][i], n, a.alpha * x[c][i]);
            }
            round_as((XT*)nullptr, x[c]);
            if (on[c] && row < a.rows) store8((XT*)a.xo + row * a.ldxo + col0 + 8 * TPR * c, x[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += on[c] ? x[c][i] : 0.f;
        }
        if (!a.rms) m2 = row_sum<TPR>(s, red) * invC;
        s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[c][i] = on[c] ? x[c][i] - m2 : 0.f; s = fmaf(x[c][i], x[c][i], s); }
        const float r2 = rsqrtf(row_sum<TPR>(s, red) * invC + a.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[c][i] = fmaf(x[c][i] * r2, w2[c][i], b2[c][i]);
            if (on[c] && row < a.rows) store8(a.y + row * a.ldy + col0 + 8 * TPR * c, x[c]);
        }
        if (a.stats && row < a.rows && col0 == 0) *reinterpret_cast<f4_t*>(a.stats + 4 * row) = (f4_t){m1, r1, m2, r2};
    }
}

// partial row of one parameter: the RG row groups of the block are summed in LDS, in order
template <int TPR, int NCH>
__device__ __forceinline__ void flush8(const float (&v)[NCH][8], float* s, float* out, int C, const bool (&on)[NCH]) {
    constexpr int RG = Blk<TPR>::RG;
    const int rg = threadIdx.x / TPR, col0 = 8 * (threadIdx.x % TPR);
    if (RG > 1) {
        __syncthreads();
        if (on[0]) store8(s + rg * C + col0, v[0]);
        __syncthreads();
        if (on[0] && rg == 0) {
            float t[8], u[8];
            load8(s + col0, t);
#pragma unroll
            for (int k = 1; k < RG; ++k) {
                load8(s + k * C + col0, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] += u[i];
            }
            store8(out + col0, t);
        }
    } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (on[c]) store8(out + col0 + 8 * TPR * c, v[c]);
    }
}

// The rows of a block: `gpw` row groups (gate_kind 3; otherwise all rows are one group), or the piece `blockIdx % W` of one.  SOLO (at least RG groups to a
// block): each of the RG row groups of threads takes whole gate groups and writes their gate gradients itself; otherwise the RG work on one
// group together and meet in LDS at its end.
template <typename XT, int TPR, int NCH, bool SOLO>
__global__ void __launch_bounds__(Blk<TPR>::NT) norm_join_bwd_kernel(JP a) {
    constexpr int RG = Blk<TPR>::RG, NW = Blk<TPR>::NT / 64;
    static_assert(NCH == 1 || RG == 1, "flush8");
    // 16 columns a thread leave no room for their weights and a row ahead beside the five sums: the weights come from L2 each time
    constexpr bool HOLD = NCH == 1;
    __shared__ float red[16];
    __shared__ __attribute__((aligned(16))) float sum[RG > 1 ? 2048 : 4];     // RG * C <= 2048
    const int rg = threadIdx.x / TPR, col0 = 8 * (threadIdx.x % TPR);
    const float invC = 1.0f / (float)a.C;
    float w1[HOLD ? NCH : 1][8], b1[HOLD ? NCH : 1][8], w2[HOLD ? NCH : 1][8], g[HOLD ? NCH : 1][8];
    float aw1[NCH][8], ab1[NCH][8], aw2[NCH][8], ab2[NCH][8], ag[NCH][8];
    bool on[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int col = col0 + 8 * TPR * c;
        on[c] = col < a.C;
#pragma unroll
        for (int i = 0; i < 8; ++i) aw1[c][i] = ab1[c][i] = aw2[c][i] = ab2[c][i] = ag[c][i] = 0.f;
    }
    const bool one = a.gate_kind == 1;                                  // ag[0]: its gradient's sum and compensation
    const float gate0 = one ? a.gate[0] : 1.f;
    auto set = [&](int c, int k, int64_t gr, bool fresh) {              // weights and gate of chunk c into slot k; fresh: the group's gate alone
        const int col = col0 + 8 * TPR * c;
        if (!fresh) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { w1[k][i] = b1[k][i] = w2[k][i] = 0.f; g[k][i] = gate0; }
            if (on[c]) {
                load8(a.w1 + col, w1[k]);
                load8(a.w2 + col, w2[k]);
                if (a.b1) load8(a.b1 + col, b1[k]);
                if (a.gate_kind == 2) load8(a.gate + col, g[k]);
            }
        }
        if (a.gate_kind == 3 && on[c] && gr < a.G) load8(a.gate + gr * a.C + col, g[k]);
    };
    if (HOLD) set(0, 0, a.G, false);
    const int64_t part = blockIdx.x % a.W, g0 = blockIdx.x / a.W * a.gpw;
    const int64_t g1 = g0 + a.gpw < a.G ? g0 + a.gpw : a.G;
    const int64_t turns = SOLO ? (g1 - g0 + RG - 1) / RG : g1 - g0;     // groups (of RG) in turn, `count` rows each: the same for every wave
    const int64_t count = SOLO ? a.rpg : (a.piece + RG - 1) / RG;
    auto row_of = [&](int64_t turn, int64_t i) -> int64_t {             // the row, or -1
        const int64_t gr = SOLO ? g0 + turn * RG + rg : g0 + turn;
        const int64_t in = SOLO ? i : part * a.piece + i * RG + rg;     // inside the group
        const int64_t row = gr * a.rpg + in;
        const bool ok = gr < g1 && in < a.rpg && (SOLO || i * RG + rg < a.piece) && row < a.rows;
        return ok ? row : -1;
    };
    Raw8<bf16_t> rdy[NCH], rh[NCH];
    Raw8<XT> rz[NCH], rt[NCH];
    f4_t rs;
    auto fetch = [&](int64_t row) {
        rs = (f4_t){0.f, 0.f, 0.f, 0.f};
        if (row >= 0) rs = *reinterpret_cast<const f4_t*>(a.stats + 4 * row);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = col0 + 8 * TPR * c;
            none(rdy[c]);
            none(rh[c]);
            none(rz[c]);
            none(rt[c]);
            if (on[c] && row >= 0) {
                ask(rdy[c], a.dy + row * a.lddy + col);
                ask(rz[c], (const XT*)a.xo + row * a.ldxo + col);
                ask(rh[c], a.h + row * a.ldh + col);
                if (a.dxo) ask(rt[c], (const XT*)a.dxo + row * a.lddxo + col);
            }
        }
    };
    if (HOLD && turns > 0 && count > 0) fetch(row_of(0, 0));
    for (int64_t turn = 0; turn < turns; ++turn) {
        const int64_t gr = SOLO ? g0 + turn * RG + rg : g0 + turn;
        if (HOLD && gr < g1) set(0, 0, gr, true);
        for (int64_t i = 0; i < count; ++i) {
            const int64_t row = row_of(turn, i);
            float dy[NCH][8], t[NCH][8], z[NCH][8], h[NCH][8];
            if (!HOLD) fetch(row);
            const f4_t st = rs;
#pragma unroll
            for (int c = 0; c < NCH; ++c) { open8(rdy[c], dy[c]); open8(rt[c], t[c]); open8(rz[c], z[c]); open8(rh[c], h[c]); }
            if (HOLD) fetch(i + 1 < count ? row_of(turn, i + 1) : (turn + 1 < turns ? row_of(turn + 1, 0) : -1));
            float c1 = 0.f, c2 = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const bool ok = on[c] && row >= 0;
                const int u = HOLD ? c : 0;
                if (!HOLD) set(c, 0, gr, false);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    z[c][k] = ok ? (z[c][k] - st[2]) * st[3] : 0.f;     // second norm's normalised row
                    aw2[c][k] = fmaf(dy[c][k], z[c][k], aw2[c][k]);
                    ab2[c][k] += dy[c][k];
                    dy[c][k] *= w2[u][k];
                    c1 += dy[c][k];
                    c2 = fmaf(dy[c][k], z[c][k], c2);
                }
            }
            row_sum2<TPR>(c1, c2, red);
            c1 = a.rms ? 0.f : c1 * invC;
            c2 *= invC;
            float e1 = 0.f, e2 = 0.f, gsum = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const bool ok = on[c] && row >= 0;
                const int u = HOLD ? c : 0;
                if (!HOLD) set(c, 0, gr, false);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    t[c][k] = fmaf(st[3], dy[c][k] - fmaf(z[c][k], c2, c1), t[c][k]);     // gradient of x'
                    h[c][k] = ok ? (h[c][k] - st[0]) * st[1] : 0.f;
                    t[c][k] = ok ? t[c][k] : 0.f;
                    const float n = fmaf(h[c][k], w1[u][k], b1[u][k]);
                    if (one) gsum = fmaf(t[c][k], n, gsum);
                    else ag[c][k] = fmaf(t[c][k], n, ag[c][k]);
                    const float dn = t[c][k] * g[u][k];
                    aw1[c][k] = fmaf(dn, h[c][k], aw1[c][k]);
                    ab1[c][k] += dn;
                    dy[c][k] = dn * w1[u][k];
                    e1 += dy[c][k];
                    e2 = fmaf(dy[c][k], h[c][k], e2);
                    t[c][k] *= a.alpha;
                }
                if (ok) store8((XT*)a.dx + row * a.lddx + col0 + 8 * TPR * c, t[c]);
            }
            if (one) {                                                  // one sum of every element: compensated, or it loses what cancels in it
                const float v = gsum - ag[0][1], q = ag[0][0] + v;
                ag[0][1] = (q - ag[0][0]) - v;
                ag[0][0] = q;
            }
            row_sum2<TPR>(e1, e2, red);
            e1 = a.rms ? 0.f : e1 * invC;
            e2 *= invC;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
#pragma unroll
                for (int k = 0; k < 8; ++k) h[c][k] = st[1] * (dy[c][k] - fmaf(h[c][k], e2, e1));
                if (on[c] && row >= 0) store8(a.dh + row * a.lddh + col0 + 8 * TPR * c, h[c]);
            }
        }
        if (a.gate_kind == 3 && a.gpart) {
            if (SOLO) {
                if (gr < g1) {
#pragma unroll
                    for (int c = 0; c < NCH; ++c)
                        if (on[c]) store8(a.gpart + gr * a.C + col0 + 8 * TPR * c, ag[c]);
                }
            } else flush8<TPR, NCH>(ag, sum, a.gpart + (gr * a.W + part) * a.C, a.C, on);
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) ag[c][k] = 0.f;
        }
    }
    if (a.part) {
        float* out = a.part + (int64_t)blockIdx.x * a.pcols;
        flush8<TPR, NCH>(aw1, sum, out, a.C, on); out += a.C;
        if (a.b1) { flush8<TPR, NCH>(ab1, sum, out, a.C, on); out += a.C; }
        flush8<TPR, NCH>(aw2, sum, out, a.C, on); out += a.C;
        if (a.b2) { flush8<TPR, NCH>(ab2, sum, out, a.C, on); out += a.C; }
        if (a.gate_kind == 2) flush8<TPR, NCH>(ag, sum, out, a.C, on);
        if (one) {
            __shared__ double wsum[NW];
            double v = (double)ag[0][0] - (double)ag[0][1];
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
            if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = v;
            __syncthreads();
            if (threadIdx.x == 0) {
                double t = 0.0;
                for (int w = 0; w < NW; ++w) t += wsum[w];
                out[0] = (float)t;
            }
        }
    }
}

// out[b][c] = sum_i in[b][i][c]: 16 columns x 64 row strides to a block (many blocks with few serial loads each), in a fixed order
__global__ void __launch_bounds__(1024) norm_join_sum_kernel(const float* in, float* out, int n, int64_t cols) {
    __shared__ double s[64][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c;
    const float* p = in + (int64_t)blockIdx.y * n * cols;
    double t = 0.0;
    if (col < cols) {
#pragma unroll 4
        for (int i = k; i < n; i += 64) t += p[(int64_t)i * cols + col];
    }
    s[k][c] = t;
    __syncthreads();
    for (int w = 32; w > 0; w >>= 1) {
        if (k < w) s[k][c] += s[k + w][c];
        __syncthreads();
    }
    if (k == 0 && col < cols) out[(int64_t)blockIdx.y * cols + col] = (float)s[0][c];
}

// the same for a handful of rows: a thread per column
__global__ void __launch_bounds__(256) norm_join_few_kernel(const float* in, float* out, int n, int64_t cols) {
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col >= cols) return;
    const float* p = in + (int64_t)blockIdx.y * n * cols + col;
    double t = 0.0;
    for (int i = 0; i < n; ++i) t += p[(int64_t)i * cols];
    out[(int64_t)blockIdx.y * cols + col] = (float)t;
}

bool bad16(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check(const char* who, const stg_norm_join_args* a) {
    STG_CHECK(a != nullptr, -1, "%s: null arguments", who);
    STG_CHECK(a->x_dtype == STG_F32 || a->x_dtype == STG_BF16, -2, "%s: the stream is fp32 or bf16", who);
    STG_CHECK(a->rows >= 0 && a->C > 0 && a->C % 8 == 0 && a->C <= 8192, -2, "%s: rows=%lld, width %d (a multiple of 8 up to 8192)", who, (long long)a->rows, a->C);
    STG_CHECK(a->gate_kind >= 0 && a->gate_kind <= 3 && ((a->gate_kind == 0) == (a->gate == nullptr) || (a->gate_kind == 3 && a->rows == 0)), -2, "%s: gate kind %d (0..3, 0 without a gate)", who, a->gate_kind);
    STG_CHECK(a->gate_kind != 3 || a->rows_per_group > 0, -2, "%s: a gate by group needs rows_per_group > 0", who);
    STG_CHECK(a->w1 && a->w2 && (a->rows == 0 || (a->h && a->xo)), -1, "%s: null tensor", who);
    STG_CHECK(a->ldh >= a->C && a->ldxo >= a->C && a->ldh % 8 == 0 && a->ldxo % 8 == 0, -3, "%s: leading dimensions must be multiples of 8 and >= the width", who);
    STG_CHECK(!bad16(a->h) && !bad16(a->xo) && !bad16(a->w1) && !bad16(a->w2) && !bad16(a->b1) && !bad16(a->b2) && (a->gate_kind < 2 || !bad16(a->gate)) && !bad16(a->stats),
              -3, "%s: tensors must be 16-byte aligned", who);
    STG_CHECK(a->eps >= 0.f, -2, "%s: eps %g", who, a->eps);
    return 0;
}

JP make(const stg_norm_join_args* a) {
    JP p{};
    p.x = a->x; p.ldx = a->ldx; p.h = (const bf16_t*)a->h; p.ldh = a->ldh;
    p.gate = a->gate; p.gate_kind = a->gate_kind; p.rpg = a->rows > 0 ? a->rows : 1;
    if (a->gate_kind == 3 && a->rows_per_group < p.rpg) p.rpg = a->rows_per_group;
    p.w1 = a->w1; p.b1 = a->b1; p.w2 = a->w2; p.b2 = a->b2; p.alpha = a->alpha; p.eps = a->eps;
    p.xo = a->xo; p.ldxo = a->ldxo; p.y = (bf16_t*)a->y; p.ldy = a->ldy; p.stats = a->stats;
    p.rows = a->rows; p.C = a->C; p.rms = a->rms != 0;
    return p;
}

// threads of a row: 8 columns each up to 4096, 16 beyond (with 1024 threads a row the backward's 170 registers spilled: 600 us instead of 225 us
// at 8192 x 5120)
int threads_per_row(int C) { return C <= 128 ? 16 : C <= 256 ? 32 : C <= 512 ? 64 : C <= 1024 ? 128 : C <= 2048 ? 256 : 512; }
int rows_in_flight(int C) { const int t = threads_per_row(C); return t <= 256 ? 256 / t : 1; }

// How the backward's blocks share the rows: as many blocks as stay resident together (two of 256 threads or one of 512 per compute unit at 200
// registers; a few more would cost a second round), since every further block leaves another partial row of up to 5 C floats (8192 x 4096, bf16 stream:
// 130 us with 1024 blocks, 115 us with 256); fewer when a block's row groups would be left without a row.  More gate groups than blocks: several
// groups to a block; fewer: a group is split W ways.
void plan_bwd(JP& p) {
    const int64_t rgn = rows_in_flight(p.C), target = threads_per_row(p.C) <= 256 ? 512 : 256;
    p.G = (p.rows + p.rpg - 1) / p.rpg;
    p.W = 1;
    p.gpw = 1;
    p.piece = p.rpg;
    if (p.G >= target) p.gpw = (p.G + target - 1) / target;
    else if (p.G > 0) {
        const int64_t most = (p.rpg + rgn - 1) / rgn, w = target / p.G;
        p.W = (int)(w < most ? w : most);
        p.piece = ((p.rpg + p.W - 1) / p.W + rgn - 1) / rgn * rgn;
        p.W = (int)((p.rpg + p.piece - 1) / p.piece);
    }
}
int64_t blocks_of(const JP& p) { return (p.G + p.gpw - 1) / p.gpw * p.W; }
int64_t part_cols(const JP& p) {
    return (int64_t)p.C * (2 + (p.b1 ? 1 : 0) + (p.b2 ? 1 : 0) + (p.gate_kind == 2 ? 1 : 0)) + (p.gate_kind == 1 ? 1 : 0);
}
// the partial rows start 16-byte aligned
int64_t part_pitch(const JP& p) { return (part_cols(p) + 3) / 4 * 4; }

bool solo(const JP& p) { return p.W == 1 && p.gate_kind == 3 && p.gpw >= rows_in_flight(p.C); }

#define BY_WIDTH(CALL)                                                          \
    switch (threads_per_row(p.C)) {                                             \
        case 16: { constexpr int T = 16, N = 1; CALL; break; }                  \
        case 32: { constexpr int T = 32, N = 1; CALL; break; }                  \
        case 64: { constexpr int T = 64, N = 1; CALL; break; }                  \
        case 128: { constexpr int T = 128, N = 1; CALL; break; }                \
        case 256: { constexpr int T = 256, N = 1; CALL; break; }                \
        default:                                                                \
            if (p.C <= 4096) { constexpr int T = 512, N = 1; CALL; }            \
            else { constexpr int T = 512, N = 2; CALL; }                        \
    }

template <typename XT>
int launch_fwd(const JP& p, hipStream_t st) {
    int64_t n = (p.rows + rows_in_flight(p.C) - 1) / rows_in_flight(p.C);
    n = n < 2048 ? n : 2048;
    BY_WIDTH((norm_join_fwd_kernel<XT, T, N><<<dim3((unsigned)n), Blk<T>::NT, 0, st>>>(p)));
    STG_LAUNCH_CHECK();
    return 0;
}
template <typename XT>
int launch_bwd(const JP& p, hipStream_t st) {
    const dim3 g((unsigned)blocks_of(p));
    if (solo(p)) { BY_WIDTH((norm_join_bwd_kernel<XT, T, N, true><<<g, Blk<T>::NT, 0, st>>>(p))); }
    else { BY_WIDTH((norm_join_bwd_kernel<XT, T, N, false><<<g, Blk<T>::NT, 0, st>>>(p))); }
    STG_LAUNCH_CHECK();
    return 0;
}

}  // namespace

// out[b] = column sums of in[b] ([n, cols]) for `batch` of them.  Up to 16 rows: a thread per column (2 rows of 768 columns, 80 batches: 4.1 us against 9.9 us
// for blocks of 64 row strides); more: 64 row strides per column (980 rows of 2 052 columns: 5.4 us against 24 us for 16 strides).
static int launch_sum(const float* in, float* out, int64_t n, int64_t cols, int64_t batch, hipStream_t st) {
    for (int64_t b0 = 0; b0 < batch; b0 += 65535) {                     // the grid's y limit
        const unsigned nb = (unsigned)(batch - b0 < 65535 ? batch - b0 : 65535);
        const float* i = in + b0 * n * cols;
        float* o = out + b0 * cols;
        if (n <= 16) norm_join_few_kernel<<<dim3((unsigned)((cols + 255) / 256), nb), 256, 0, st>>>(i, o, (int)n, cols);
        else norm_join_sum_kernel<<<dim3((unsigned)((cols + 15) / 16), nb), 1024, 0, st>>>(i, o, (int)n, cols);
        STG_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int stg_norm_join_fwd(const stg_norm_join_args* a, void* stream) {
    const int rc = check("stg_norm_join_fwd", a);
    if (rc) return rc;
    STG_CHECK(a->rows == 0 || (a->x && a->y), -1, "stg_norm_join_fwd: null tensor");
    STG_CHECK(a->ldx >= a->C && a->ldy >= a->C && a->ldx % 8 == 0 && a->ldy % 8 == 0, -3, "stg_norm_join_fwd: leading dimensions must be multiples of 8 and >= the width");
    STG_CHECK(!bad16(a->x) && !bad16(a->y), -3, "stg_norm_join_fwd: tensors must be 16-byte aligned");
    if (a->rows == 0) return 0;
    const JP p = make(a);
    return a->x_dtype == STG_F32 ? launch_fwd<float>(p, (hipStream_t)stream) : launch_fwd<bf16_t>(p, (hipStream_t)stream);
}

extern "C" int64_t stg_norm_join_param_floats(const stg_norm_join_args* a) { return a == nullptr ? -1 : part_pitch(make(a)); }

extern "C" int64_t stg_norm_join_bwd_ws_floats(const stg_norm_join_args* a) {
    if (a == nullptr || a->rows < 0 || a->C <= 0 || (a->gate_kind == 3 && a->rows_per_group <= 0)) return -1;
    JP p = make(a);
    plan_bwd(p);
    return blocks_of(p) * part_pitch(p) + (p.gate_kind == 3 && p.W > 1 ? p.G * p.W * p.C : 0) + 4;
}

extern "C" int stg_norm_join_bwd(const stg_norm_join_args* a, const void* dy, int64_t lddy, const void* dxo, int64_t lddxo, void* dx, int64_t lddx,
                                 void* dh, int64_t lddh, float* dparams, float* dgate_groups, float* ws, int64_t ws_floats, void* stream) {
    const int rc = check("stg_norm_join_bwd", a);
    if (rc) return rc;
    STG_CHECK(a->rows == 0 || (dy && dx && dh && a->stats), -1, "stg_norm_join_bwd: null tensor");
    STG_CHECK(lddy >= a->C && lddx >= a->C && lddh >= a->C && (!dxo || lddxo >= a->C) && lddy % 8 == 0 && lddx % 8 == 0 && lddh % 8 == 0 && (!dxo || lddxo % 8 == 0), -3,
              "stg_norm_join_bwd: leading dimensions must be multiples of 8 and >= the width");
    STG_CHECK(!bad16(dy) && !bad16(dx) && !bad16(dh) && !bad16(dxo) && !bad16(dgate_groups) && !bad16(ws), -3, "stg_norm_join_bwd: tensors must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    JP p = make(a);
    plan_bwd(p);
    p.dy = (const bf16_t*)dy; p.lddy = lddy; p.dxo = dxo; p.lddxo = lddxo; p.dx = dx; p.lddx = lddx; p.dh = (bf16_t*)dh; p.lddh = lddh;
    const int64_t nb = blocks_of(p), pitch = part_pitch(p);
    STG_CHECK(nb <= INT32_MAX, -2, "stg_norm_join_bwd: too many row groups");
    const bool groups = p.gate_kind == 3 && dgate_groups != nullptr;
    if (dparams || (groups && p.W > 1))
        STG_CHECK(ws != nullptr && ws_floats >= stg_norm_join_bwd_ws_floats(a), -4, "stg_norm_join_bwd: workspace of %lld floats is too small", (long long)ws_floats);
    p.pcols = pitch;
    if (dparams) p.part = ws;
    if (groups) p.gpart = p.W > 1 ? ws + nb * pitch : dgate_groups;
    if (a->rows > 0) {
        const int e = a->x_dtype == STG_F32 ? launch_bwd<float>(p, st) : launch_bwd<bf16_t>(p, st);
        if (e) return e;
    }
    if (dparams) { const int e = launch_sum(p.part, dparams, a->rows > 0 ? nb : 0, pitch, 1, st); if (e) return e; }
    if (groups && p.W > 1) { const int e = launch_sum(p.gpart, dgate_groups, p.W, p.C, p.G, st); if (e) return e; }
    return 0;
}
