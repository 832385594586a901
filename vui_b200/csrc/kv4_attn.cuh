// Attention over the paged 4-bit cache (layout: kv4_kernels.cuh).  With V and K the values that the codes stand for, row r of a
// sequence at position p and query head j:  out = sum_{i <= p} softmax_i(scale q . K_i) V_i,  K and V of kv head j / group.
#pragma once
#include "kv4_kernels.cuh"

namespace vuik {

constexpr int KA_THREADS = 128, KA_WARPS = 4;
constexpr int KA_STEP = 64;                    // positions that a warp takes at once

struct Kv4AttnArgs {
    Kv4Cache c;
    const int4* entries; const int32_t* cu_rows; const int32_t* cu_units;
    int n, n_rows, group, split;
    const __nv_bfloat16* q; long long q_stride;
    __nv_bfloat16* out; long long out_stride;
    float scale_log2;                          // scale * log2(e)
    float* acc;                                // partial sums: (unit, column, dim), where a sequence has more than one split
    float2* ml;                                // maximum (of log2 scores) and sum: (unit, column)
};

// m16n8k16, f16 in, fp32 out: D += A B.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The eight codes of a word as four pairs of the values that they stand for.  A nibble under the exponent of 1024 is 1024 + c, one
// that sits four bits higher 1024 + 16 c: both are exact in f16, and so is what is left when 1024 is taken off again.
__device__ __forceinline__ void kv4_values(uint32_t w, uint32_t s, uint32_t z, uint32_t (&r)[4]) {
    const uint32_t v = w >> 8;
    uint32_t x[4];
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[0]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[1]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[2]) : "r"(v));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[3]) : "r"(v));
    const __half2 hs = *reinterpret_cast<const __half2*>(&s), hz = *reinterpret_cast<const __half2*>(&z);
    const __half2 low = __half2half2(__ushort_as_half(0xE400)), sixteenth = __half2half2(__ushort_as_half(0x2C00)),
                  less = __half2half2(__ushort_as_half(0xD400));   // -1024, 1 / 16, -64
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = *reinterpret_cast<const __half2*>(&x[j]);
        const __half2 code = j & 1 ? __hfma2(h, sixteenth, less) : __hadd2(h, low);
        const __half2 value = __hfma2(hs, code, hz);
        r[j] = *reinterpret_cast<const uint32_t*>(&value);
    }
}

// A unit: a tile of columns of one sequence (its rows times the query heads of a kv head, COLS at a time), a kv head, a split of the
// positions.  Units lie in the order sequence, column tile, kv head, split.
struct Kv4Unit {
    int entry, ctile, head, split, splits;      // splits: of the sequence
    int slot, start, rows, row0;
};

template <int COLS>
__device__ __forceinline__ void unit_enter(const Kv4AttnArgs& a, Kv4Unit& u) {
    const int4 e = __ldcg(a.entries + u.entry);
    u.slot = e.x; u.start = e.y; u.rows = e.z; u.row0 = e.w;
    u.splits = (e.y + e.z + a.split - 1) / a.split;
}

// The place of work item w (< cu_units[n] * n_kv) by a search over the sequences' first units.
template <int COLS>
__device__ __forceinline__ Kv4Unit unit_at(const Kv4AttnArgs& a, long long w) {
    Kv4Unit u;
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)__ldcg(a.cu_units + mid) * a.c.n_kv <= w) lo = mid; else hi = mid;
    }
    u.entry = lo;
    unit_enter<COLS>(a, u);
    const long long off = w - (long long)__ldcg(a.cu_units + lo) * a.c.n_kv;
    u.split = (int)(off % u.splits);
    const long long rest = off / u.splits;
    u.head = (int)(rest % a.c.n_kv);
    u.ctile = (int)(rest / a.c.n_kv);
    return u;
}

template <int COLS>
__device__ __forceinline__ void unit_next(const Kv4AttnArgs& a, Kv4Unit& u) {
    if (++u.split < u.splits) return;
    u.split = 0;
    if (++u.head < a.c.n_kv) return;
    u.head = 0;
    if (++u.ctile < (u.rows * a.group + COLS - 1) / COLS) return;
    u.ctile = 0;
    do {
        if (++u.entry >= a.n) return;
        unit_enter<COLS>(a, u);
    } while (u.rows == 0);
}

// mma.sync form: 4 warps share a unit's positions 64 at a time.  Keys are the A operand (16 positions of a tile), queries the B
// operand (8 columns), so that one or a few query heads waste nothing but columns; the scores' transpose for the second product is
// one movmatrix a fragment.  Softmax statistics and sums are fp32; the weights enter the second product as f16 (2^-12 relative,
// where bf16's 2^-9 would be as much as the output's own rounding).
template <int NG, int NT>
__global__ void __launch_bounds__(KA_THREADS) k_kv4_attn(const Kv4AttnArgs a) {
    constexpr int HD = NG * KV4_GROUP, COLS = NT * 8;
    __shared__ float sm_acc[KA_WARPS][COLS][HD + 4];
    __shared__ float2 sm_ml[KA_WARPS][COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch();
    const long long total = (long long)__ldcg(a.cu_units + a.n) * a.c.n_kv;
    const long long first = total * blockIdx.x / gridDim.x, last = total * (blockIdx.x + 1) / gridDim.x;
    if (first >= last) return;
    Kv4Unit u = unit_at<COLS>(a, first);
    const int tiles = 1 << (a.c.block_shift - 4);
    uint32_t qf[NT][NG][4];
    float factor[NT][2];
    int limit[NT][2];       // last position that the column sees

    for (long long w = first; w < last; ++w) {
        const int cols = u.rows * a.group - u.ctile * COLS;                 // valid ones of this tile, if fewer than COLS
        if (w == first || u.split == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int col = u.ctile * COLS + nt * 8 + g;
                const bool there = nt * 8 + g < cols;
                const int row = there ? col / a.group : 0, head = u.head * a.group + (there ? col % a.group : 0);
                uint4 raw[NG];
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    raw[i] = make_uint4(0, 0, 0, 0);
                    if (there)
                        raw[i] = __ldcg(reinterpret_cast<const uint4*>(a.q + (long long)(u.row0 + row) * a.q_stride + head * HD + i * KV4_GROUP + t * 8));
                    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) big = max(big, max(x[j] & 0x7fffu, x[j] >> 16 & 0x7fffu));
                }
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // the column times a power of two, so that its largest element lies in [1, 2): exact in f16 but for elements 2^14 times smaller
                const int e = min(max((int)(big >> 7), 1), 253);
                const float down = __int_as_float((254 - e) << 23), up = __int_as_float(e << 23);
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        qf[nt][i][j] = pack_h2(__uint_as_float(x[j] << 16) * down, __uint_as_float(x[j] & 0xffff0000u) * down);
                }
                const float f = a.scale_log2 * up;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c2 = nt * 8 + 2 * t + j;
                    factor[nt][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
                    limit[nt][j] = c2 < cols ? u.start + (u.ctile * COLS + c2) / a.group : -1;
                }
            }
        }
        const int top_row = (u.ctile * COLS) / a.group, end_row = (u.ctile * COLS + min(cols, COLS) - 1) / a.group;
        const int lo = u.split * a.split;
        const int hi = (int)min((long long)lo + a.split, (long long)u.start + end_row + 1);
        float acc[NT][2 * NG][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }
        const int32_t* row_table = a.c.table + (size_t)u.slot * a.c.max_blocks;
        for (int base = lo + warp * KA_STEP; base < hi; base += KA_WARPS * KA_STEP) {
            const int nk = min(4, (hi - base + 15) >> 4);
            const bool whole = base + KA_STEP - 1 <= u.start + top_row;   // every column sees all 64
            float s[4][NT][4];
            const unsigned char* at[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < nk) {
                    const int pos = base + k * 16;
                    int b = __ldcg(row_table + (pos >> a.c.block_shift));
                    if ((unsigned)b >= (unsigned)a.c.n_blocks) {
                        if (lane == 0) atomicOr(a.c.flag, KV4_BAD_BLOCK);
                        b = 0;
                    }
                    at[k] = a.c.pool + ((size_t)((long long)b * a.c.n_kv + u.head) * tiles + ((pos & ((1 << a.c.block_shift) - 1)) >> 4)) * (NG * KV4_GT);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[k][nt][0] = s[k][nt][1] = s[k][nt][2] = s[k][nt][3] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < nk) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const unsigned char* p = at[k] + i * KV4_GT;
                        const uint2 code = __ldcg(reinterpret_cast<const uint2*>(p + lane * 8));
                        const uint2 par = __ldcg(reinterpret_cast<const uint2*>(p + KV4_KPAR + g * 8));
                        uint32_t x[4], y[4];
                        kv4_values(code.x, __byte_perm(par.x, 0, 0x1010), __byte_perm(par.x, 0, 0x3232), x);
                        kv4_values(code.y, __byte_perm(par.y, 0, 0x1010), __byte_perm(par.y, 0, 0x3232), y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(s[k][nt], x[0], y[0], x[1], y[1], qf[nt][i][0], qf[nt][i][1]);
                            mma16816(s[k][nt], x[2], y[2], x[3], y[3], qf[nt][i][2], qf[nt][i][3]);
                        }
                    }
                }
            }
            uint32_t p[4][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[k][nt][j] *= factor[nt][j & 1];
                        if (!whole && base + k * 16 + g + (j >> 1) * 8 > limit[nt][j & 1]) s[k][nt][j] = -INFINITY;
                        top[j & 1] = fmaxf(top[j & 1], s[k][nt][j]);
                    }
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
                }
                float old[2], now[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float best = fmaxf(m[nt][j], top[j]);
                    now[j] = best == -INFINITY ? 0.f : best;    // nothing seen yet: weights of exp(-inf) = 0
                    old[j] = ex2(m[nt][j] - now[j]);
                    m[nt][j] = best;
                    l[nt][j] *= old[j];
                }
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) {
                    acc[nt][i][0] *= old[0]; acc[nt][i][1] *= old[1];
                    acc[nt][i][2] *= old[0]; acc[nt][i][3] *= old[1];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[j] = ex2(s[k][nt][j] - now[j & 1]);
                        l[nt][j & 1] += e[j];
                    }
                    p[k][nt][0] = movmatrix(pack_h2(e[0], e[1]));
                    p[k][nt][1] = movmatrix(pack_h2(e[2], e[3]));
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < nk) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const unsigned char* q = at[k] + i * KV4_GT;
                        const uint2 code = __ldcg(reinterpret_cast<const uint2*>(q + KV4_VCODE + lane * 8));
                        const uint4 par = __ldcg(reinterpret_cast<const uint4*>(q + KV4_VPAR + t * 16));
                        uint32_t x[4], y[4];
                        kv4_values(code.x, par.x, par.y, x);
                        kv4_values(code.y, par.z, par.w, y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(acc[nt][2 * i], x[0], x[1], y[0], y[1], p[k][nt][0], p[k][nt][1]);
                            mma16816(acc[nt][2 * i + 1], x[2], x[3], y[2], y[3], p[k][nt][0], p[k][nt][1]);
                        }
                    }
                }
            }
        }
        // the warps' states, added in the order of the warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], o);
                l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], o);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = nt * 8 + 2 * t + j;
                if (col < cols) {
                    if (g == 0) sm_ml[warp][col] = make_float2(m[nt][j], l[nt][j]);
#pragma unroll
                    for (int i = 0; i < NG; ++i)
                        *reinterpret_cast<float4*>(&sm_acc[warp][col][i * KV4_GROUP + 4 * g]) =
                            make_float4(acc[nt][2 * i][j], acc[nt][2 * i][2 + j], acc[nt][2 * i + 1][j], acc[nt][2 * i + 1][2 + j]);
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < min(cols, COLS) * (HD / 4); i += KA_THREADS) {
            const int col = i / (HD / 4), d = i % (HD / 4) * 4;
            float best = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < KA_WARPS; ++k) best = fmaxf(best, sm_ml[k][col].x);
            const float now = best == -INFINITY ? 0.f : best;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < KA_WARPS; ++k) {
                const float2 part = sm_ml[k][col];
                const float f = ex2(part.x - now);
                const float4 v = *reinterpret_cast<const float4*>(&sm_acc[k][col][d]);
                sum += f * part.y;
                o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
            }
            if (u.splits == 1) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const int c = u.ctile * COLS + col;
                __nv_bfloat162 lo2 = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi2 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
                uint2 v = make_uint2(*reinterpret_cast<uint32_t*>(&lo2), *reinterpret_cast<uint32_t*>(&hi2));
                *reinterpret_cast<uint2*>(a.out + (long long)(u.row0 + c / a.group) * a.out_stride + (u.head * a.group + c % a.group) * HD + d) = v;
            } else {
                *reinterpret_cast<float4*>(a.acc + (size_t)(w * COLS + col) * HD + d) = o;
                if (d == 0) a.ml[w * COLS + col] = make_float2(best, sum);
            }
        }
        __syncthreads();
        unit_next<COLS>(a, u);
    }
}

// Adds up the splits of every row that has more than one, in the order of the positions: a warp a (row, query head).
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_merge(const Kv4AttnArgs a, const int cols) {
    constexpr int HD = NG * KV4_GROUP;
    const int lane = threadIdx.x & 31, heads = a.c.n_kv * a.group;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch();
    const int row = (int)(id / heads), head = (int)(id % heads), kv = head / a.group;
    if (row >= a.n_rows || row >= __ldcg(a.cu_rows + a.n)) return;
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(a.cu_rows + mid) <= row) lo = mid; else hi = mid;
    }
    const int4 e = __ldcg(a.entries + lo);
    const int all = (e.y + e.z + a.split - 1) / a.split;
    if (all == 1) return;
    const int own = (e.y + row - e.w) / a.split + 1;        // splits that the row sees
    const int c = (row - e.w) * a.group + head % a.group;
    const long long w = (long long)__ldcg(a.cu_units + lo) * a.c.n_kv + ((long long)(c / cols) * a.c.n_kv + kv) * all;
    const float2* ml = a.ml + w * cols + c % cols;
    const float* acc = a.acc + (size_t)(w * cols + c % cols) * HD + lane * NG;
    float best = -INFINITY;
    for (int i = lane; i < own; i += 32) best = fmaxf(best, __ldcg(&ml[(size_t)i * cols].x));
#pragma unroll
    for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    const float now = best == -INFINITY ? 0.f : best;
    float sum = 0.f, out[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) out[j] = 0.f;
#pragma unroll 4
    for (int i = 0; i < own; ++i) {
        const float2 part = __ldcg(ml + (size_t)i * cols);
        const float f = ex2(part.x - now);
        sum += f * part.y;
#pragma unroll
        for (int j = 0; j < NG; ++j) out[j] += f * __ldcg(acc + (size_t)i * cols * HD + j);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NG; ++j) a.out[(long long)row * a.out_stride + head * HD + lane * NG + j] = __float2bfloat16_rn(out[j] * inv);
}

}  // namespace vuik
