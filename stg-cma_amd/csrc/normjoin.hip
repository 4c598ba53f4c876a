// Norm after a block, gate, scaled residual sum, norm before the next block -- one row pass forward, one row pass backward:
//     n = Norm(h) w1 (+ b1),   x' = alpha x + gate o n,   y = Norm(x') w2 (+ b2)          Norm: LayerNorm or RMS norm over the last dim
// As separate passes the chain moves the branch h, the stream x and their images six to eight times; here every tensor crosses HBM once
// (forward: h, x in, x', y out; backward: dy, dx', x', h in, dx, dh out), which is the floor: the arithmetic (~15 / ~30 operations per element)
// stays under it.  The gradients of the weights and the gate are column sums over all rows: every block keeps its columns' sums in registers
// over its share of the rows and leaves ONE partial row, added up in a fixed order by a second kernel -- no atomics, repeatable bit for bit.
// x' is rounded to the stream's type before the second norm reads it, so that the backward, which reads the stored x', sees the same values.
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

// sums over the W waves that share a row (WPR waves; every wave of the block calls it the same number of times)
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* red, int wave) {
    v = wave_sum<64>(v);
    if (WPR == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    const int w0 = wave / WPR * WPR;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) t += red[w0 + w];
    return t;
}
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int wave) {
    a = wave_sum<64>(a);
    b = wave_sum<64>(b);
    if (WPR == 1) return;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { red[wave] = a; red[16 + wave] = b; }
    __syncthreads();
    const int w0 = wave / WPR * WPR;
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) { a += red[w0 + w]; b += red[16 + w0 + w]; }
}

// A lane owns 8 columns of the row (WPR waves of 64 lanes cover 512 WPR columns) and keeps their weights in registers over its rows.
template <typename XT, int WPR>
__global__ void __launch_bounds__(WPR <= 4 ? 256 : 64 * WPR) norm_join_fwd_kernel(JP a) {
    constexpr int NW = WPR <= 4 ? 4 : WPR, RG = NW / WPR;               // waves of the block, rows in flight
    __shared__ float red[32];
    const int wave = threadIdx.x >> 6;
    const int col = 8 * ((wave % WPR) * 64 + (threadIdx.x & 63));
    const bool on = col < a.C;
    const float invC = 1.0f / (float)a.C;
    float w1[8] = {}, b1[8] = {}, w2[8] = {}, b2[8] = {}, g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = 1.f;
    if (on) {
        load8(a.w1 + col, w1);
        load8(a.w2 + col, w2);
        if (a.b1) load8(a.b1 + col, b1);
        if (a.b2) load8(a.b2 + col, b2);
        if (a.gate_kind == 2) load8(a.gate + col, g);
    }
    if (a.gate_kind == 1) {
        const float s = a.gate[0];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = s;
    }
    const int64_t step = (int64_t)gridDim.x * RG;
    for (int64_t base = (int64_t)blockIdx.x * RG; base < a.rows; base += step) {
        const int64_t row = base + wave / WPR;
        const bool ok = on && row < a.rows;
        float h[8] = {}, x[8] = {};
        if (ok) {
            load8(a.h + row * a.ldh + col, h);
            load8((const XT*)a.x + row * a.ldx + col, x);
            if (a.gate_kind == 3) load8(a.gate + (row / a.rpg) * a.C + col, g);
        }
        float m1 = 0.f, m2 = 0.f, s = 0.f;
        if (!a.rms) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s += h[i];
            m1 = row_sum<WPR>(s, red, wave) * invC;
        }
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { h[i] = on ? h[i] - m1 : 0.f; s = fmaf(h[i], h[i], s); }
        const float r1 = rsqrtf(row_sum<WPR>(s, red, wave) * invC + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float n = fmaf(h[i] * r1, w1[i], b1[i]);
            x[i] = fmaf(g[i], n, a.alpha * x[i]);
        }
        round_as((XT*)nullptr, x);
        if (ok) store8((XT*)a.xo + row * a.ldxo + col, x);
        s = 0.f;
        if (!a.rms) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s += on ? x[i] : 0.f;
            m2 = row_sum<WPR>(s, red, wave) * invC;
        }
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { x[i] = on ? x[i] - m2 : 0.f; s = fmaf(x[i], x[i], s); }
        const float r2 = rsqrtf(row_sum<WPR>(s, red, wave) * invC + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i] * r2, w2[i], b2[i]);
        if (ok) store8(a.y + row * a.ldy + col, x);
        if (a.stats && row < a.rows && col == 0) *reinterpret_cast<f4_t*>(a.stats + 4 * row) = (f4_t){m1, r1, m2, r2};
    }
}

// partial row of one parameter: the RG row groups of the block are summed in LDS, in order
template <int RG>
__device__ __forceinline__ void flush8(const float* v, float* s, float* out, int C, int rg, int col, bool on) {
    if (RG > 1) {
        __syncthreads();
        if (on) store8(s + rg * C + col, v);
        __syncthreads();
        if (on && rg == 0) {
            float t[8], u[8];
            load8(s + col, t);
#pragma unroll
            for (int k = 1; k < RG; ++k) {
                load8(s + k * C + col, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] += u[i];
            }
            store8(out + col, t);
        }
    } else if (on) store8(out + col, v);
}

template <typename XT, int WPR>
__global__ void __launch_bounds__(WPR <= 4 ? 256 : 64 * WPR) norm_join_bwd_kernel(JP a) {
    constexpr int NW = WPR <= 4 ? 4 : WPR, RG = NW / WPR;
    __shared__ float red[32];
    __shared__ __attribute__((aligned(16))) float sum[RG > 1 ? 2048 : 4];     // RG * C <= 2048
    const int wave = threadIdx.x >> 6, rg = wave / WPR;
    const int col = 8 * ((wave % WPR) * 64 + (threadIdx.x & 63));
    const bool on = col < a.C;
    const float invC = 1.0f / (float)a.C;
    float w1[8] = {}, b1[8] = {}, w2[8] = {}, g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = 1.f;
    if (on) {
        load8(a.w1 + col, w1);
        load8(a.w2 + col, w2);
        if (a.b1) load8(a.b1 + col, b1);
        if (a.gate_kind == 2) load8(a.gate + col, g);
    }
    if (a.gate_kind == 1) {
        const float s = a.gate[0];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = s;
    }
    float aw1[8] = {}, ab1[8] = {}, aw2[8] = {}, ab2[8] = {}, ag[8] = {};
    const int64_t part = blockIdx.x % a.W, g0 = blockIdx.x / a.W * a.gpw;
    const int64_t g1 = g0 + a.gpw < a.G ? g0 + a.gpw : a.G;
    for (int64_t gr = g0; gr < g1; ++gr) {
        const int64_t first = gr * a.rpg + part * a.piece;
        int64_t last = first + a.piece, gend = (gr + 1) * a.rpg;
        gend = gend < a.rows ? gend : a.rows;
        last = last < gend ? last : gend;
        if (a.gate_kind == 3 && on) load8(a.gate + gr * a.C + col, g);
        for (int64_t base = first; base < last; base += RG) {
            const int64_t row = base + rg;
            const bool in = row < last, ok = on && in;
            float dy[8] = {}, t[8] = {}, z[8] = {}, h[8] = {};
            f4_t st = {0.f, 0.f, 0.f, 0.f};
            if (in) st = *reinterpret_cast<const f4_t*>(a.stats + 4 * row);
            if (ok) {
                load8(a.dy + row * a.lddy + col, dy);
                load8((const XT*)a.xo + row * a.ldxo + col, z);
                load8(a.h + row * a.ldh + col, h);
                if (a.dxo) load8((const XT*)a.dxo + row * a.lddxo + col, t);
            }
            float c1 = 0.f, c2 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] = ok ? (z[i] - st[2]) * st[3] : 0.f;               // second norm's normalised row
                aw2[i] = fmaf(dy[i], z[i], aw2[i]);
                ab2[i] += dy[i];
                dy[i] *= w2[i];
                c1 += dy[i];
                c2 = fmaf(dy[i], z[i], c2);
            }
            row_sum2<WPR>(c1, c2, red, wave);
            c1 = a.rms ? 0.f : c1 * invC;
            c2 *= invC;
            float e1 = 0.f, e2 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[i] = fmaf(st[3], dy[i] - fmaf(z[i], c2, c1), t[i]);   // gradient of x'
                h[i] = ok ? (h[i] - st[0]) * st[1] : 0.f;
                t[i] = ok ? t[i] : 0.f;
                ag[i] = fmaf(t[i], fmaf(h[i], w1[i], b1[i]), ag[i]);
                const float dn = t[i] * g[i];
                aw1[i] = fmaf(dn, h[i], aw1[i]);
                ab1[i] += dn;
                dy[i] = dn * w1[i];
                e1 += dy[i];
                e2 = fmaf(dy[i], h[i], e2);
                t[i] *= a.alpha;
            }
            if (ok) store8((XT*)a.dx + row * a.lddx + col, t);
            row_sum2<WPR>(e1, e2, red, wave);
            e1 = a.rms ? 0.f : e1 * invC;
            e2 *= invC;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = st[1] * (dy[i] - fmaf(h[i], e2, e1));
            if (ok) store8(a.dh + row * a.lddh + col, h);
        }
        if (a.gate_kind == 3 && a.gpart) {
            flush8<RG>(ag, sum, a.gpart + (gr * a.W + part) * a.C, a.C, rg, col, on);
#pragma unroll
            for (int i = 0; i < 8; ++i) ag[i] = 0.f;
        }
    }
    if (a.part) {
        float* out = a.part + (int64_t)blockIdx.x * a.pcols;
        flush8<RG>(aw1, sum, out, a.C, rg, col, on); out += a.C;
        if (a.b1) { flush8<RG>(ab1, sum, out, a.C, rg, col, on); out += a.C; }
        flush8<RG>(aw2, sum, out, a.C, rg, col, on); out += a.C;
        if (a.b2) { flush8<RG>(ab2, sum, out, a.C, rg, col, on); out += a.C; }
        if (a.gate_kind == 2) flush8<RG>(ag, sum, out, a.C, rg, col, on);
        if (a.gate_kind == 1) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) v += ag[i];
            v = wave_sum<64>(v);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) red[wave] = v;
            __syncthreads();
            if (threadIdx.x == 0) {
                float s = 0.f;
                for (int w = 0; w < NW; ++w) s += red[w];
                out[0] = s;
            }
        }
    }
}

// out[b][c] = sum_i in[b][i][c]: 16 columns x 64 row strides to a block (many blocks with few serial loads each), in a fixed order
__global__ void __launch_bounds__(1024) norm_join_sum_kernel(const float* in, float* out, int n, int64_t cols) {
    __shared__ float s[64][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c;
    const float* p = in + (int64_t)blockIdx.y * n * cols;
    float t = 0.f;
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
    if (k == 0 && col < cols) out[(int64_t)blockIdx.y * cols + col] = s[0][c];
}

// the same for a handful of rows: a thread per column
__global__ void __launch_bounds__(256) norm_join_few_kernel(const float* in, float* out, int n, int64_t cols) {
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col >= cols) return;
    const float* p = in + (int64_t)blockIdx.y * n * cols + col;
    float t = 0.f;
    for (int i = 0; i < n; ++i) t += p[(int64_t)i * cols];
    out[(int64_t)blockIdx.y * cols + col] = t;
}

bool bad16(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check(const char* who, const stg_norm_join_args* a) {
    STG_CHECK(a != nullptr, -1, "%s: null arguments", who);
    STG_CHECK(a->x_dtype == STG_F32 || a->x_dtype == STG_BF16, -2, "%s: the stream is fp32 or bf16", who);
    STG_CHECK(a->rows >= 0 && a->C > 0 && a->C % 8 == 0 && a->C <= 8192, -2, "%s: rows=%lld, width %d (a multiple of 8 up to 8192)", who, (long long)a->rows, a->C);
    STG_CHECK(a->gate_kind >= 0 && a->gate_kind <= 3 && (a->gate_kind == 0) == (a->gate == nullptr), -2, "%s: gate kind %d (0..3, 0 without a gate)", who, a->gate_kind);
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
    p.gate = a->gate; p.gate_kind = a->gate_kind; p.rpg = a->gate_kind == 3 ? a->rows_per_group : (a->rows > 0 ? a->rows : 1);
    p.w1 = a->w1; p.b1 = a->b1; p.w2 = a->w2; p.b2 = a->b2; p.alpha = a->alpha; p.eps = a->eps;
    p.xo = a->xo; p.ldxo = a->ldxo; p.y = (bf16_t*)a->y; p.ldy = a->ldy; p.stats = a->stats;
    p.rows = a->rows; p.C = a->C; p.rms = a->rms != 0;
    return p;
}

int waves_per_row(int C) { return C <= 512 ? 1 : C <= 1024 ? 2 : C <= 2048 ? 4 : C <= 4096 ? 8 : 16; }

// How the backward's blocks share the rows.  Few rows: one block per compute unit, down to one row for each of its wave groups (latency).  Many: at
// least 8 rows for each (a block's partial row costs as much traffic as a few rows) and at most 1024 blocks.  Groups (gate_kind 3) longer than
// a block's share are split W ways, shorter ones go several to a block.
void plan_bwd(JP& p) {
    const int wpr = waves_per_row(p.C), rgn = wpr <= 4 ? 4 / wpr : 1;
    int64_t share = (p.rows + 255) / 256;
    share = share < 8 * rgn ? share : 8 * rgn;
    const int64_t most = (p.rows + 1023) / 1024;
    share = share > most ? share : most;
    share = share > rgn ? share : rgn;
    share = (share + rgn - 1) / rgn * rgn;
    p.G = (p.rows + p.rpg - 1) / p.rpg;
    if (p.rpg > share) {
        p.W = (int)((p.rpg + share - 1) / share);
        p.piece = ((p.rpg + p.W - 1) / p.W + rgn - 1) / rgn * rgn;
        p.gpw = 1;
    } else {
        p.W = 1;
        p.piece = p.rpg;
        p.gpw = share / p.rpg;
    }
}
int64_t blocks_of(const JP& p) { return (p.G + p.gpw - 1) / p.gpw * p.W; }
int64_t part_cols(const JP& p) {
    return (int64_t)p.C * (2 + (p.b1 ? 1 : 0) + (p.b2 ? 1 : 0) + (p.gate_kind == 2 ? 1 : 0)) + (p.gate_kind == 1 ? 1 : 0);
}
// the partial rows start 16-byte aligned
int64_t part_pitch(const JP& p) { return (part_cols(p) + 3) / 4 * 4; }

template <typename XT>
int launch_fwd(const JP& p, hipStream_t st) {
    const int wpr = waves_per_row(p.C), rgn = wpr <= 4 ? 4 / wpr : 1;
    int64_t n = (p.rows + rgn - 1) / rgn;
    n = n < 2048 ? n : 2048;
    const dim3 g((unsigned)n);
    switch (wpr) {
        case 1: norm_join_fwd_kernel<XT, 1><<<g, 256, 0, st>>>(p); break;
        case 2: norm_join_fwd_kernel<XT, 2><<<g, 256, 0, st>>>(p); break;
        case 4: norm_join_fwd_kernel<XT, 4><<<g, 256, 0, st>>>(p); break;
        case 8: norm_join_fwd_kernel<XT, 8><<<g, 512, 0, st>>>(p); break;
        default: norm_join_fwd_kernel<XT, 16><<<g, 1024, 0, st>>>(p); break;
    }
    STG_LAUNCH_CHECK();
    return 0;
}
template <typename XT>
int launch_bwd(const JP& p, hipStream_t st) {
    const dim3 g((unsigned)blocks_of(p));
    switch (waves_per_row(p.C)) {
        case 1: norm_join_bwd_kernel<XT, 1><<<g, 256, 0, st>>>(p); break;
        case 2: norm_join_bwd_kernel<XT, 2><<<g, 256, 0, st>>>(p); break;
        case 4: norm_join_bwd_kernel<XT, 4><<<g, 256, 0, st>>>(p); break;
        case 8: norm_join_bwd_kernel<XT, 8><<<g, 512, 0, st>>>(p); break;
        default: norm_join_bwd_kernel<XT, 16><<<g, 1024, 0, st>>>(p); break;
    }
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

extern "C" int64_t stg_norm_join_param_floats(const stg_norm_join_args* a) { return a == nullptr ? -1 : part_cols(make(a)); }

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
