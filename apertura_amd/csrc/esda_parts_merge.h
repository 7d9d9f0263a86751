// esda_parts_merge.h -- the merge of the partials (m, l, O) that the runs and tiles of a decode step
// leave (gfx950): esda_prefix.hip and esda_tree.hip.
//
//   out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the n partials of a row
//
// Row, made from the parameters and a row's number, says where they are: n of them, ml(j) and acc(j) +
// at(j) * D; most(): the plan's for any row; write(): the row is written (else its sequence was skipped);
// EMPTY: a row may have no key, and is 0 then.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "esda_device.h"

namespace {

// A thread per row and 4 dims: plans of at most NS partials a row.  Every partial is loaded at once,
// beside the position that says how many of the own ones count (the others are dropped by a select).
template <int D, int NS, class Row>
__global__ __launch_bounds__(256) void merge_few_kernel(typename Row::Params p) {
    const long long t = (long long) blockIdx.x * 256 + threadIdx.x;
    const int row = (int) (t / (D / 4)), d = (int) (t % (D / 4)) * 4;
    if (row >= Row::rows(p)) return;
    const Row r(p, row);
    f32x2 ml[NS];
    f32x4 a[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        ml[j] = f32x2{-INFINITY, 0.0f};
        a[j] = 0.0f;
        if (j < r.most()) {
            ml[j] = r.ml(j);
            a[j] = *reinterpret_cast<const f32x4 *>(r.acc(j) + r.at(j) * D + d);
        }
    }
    if (!r.write()) return;
    float M = -INFINITY;
#pragma unroll
    for (int j = 0; j < NS; ++j) M = j < r.n ? fmaxf(M, ml[j][0]) : M;
    if (Row::EMPTY && M == -INFINITY) M = 0.0f;
    float den = 0.0f;
    f32x4 num = 0.0f;
#pragma unroll
    for (int j = 0; j < NS; ++j)
        if (j < r.n) {
            const float w = __builtin_amdgcn_exp2f(ml[j][0] - M);
            den = __builtin_fmaf(ml[j][1], w, den);
            num += a[j] * w;
        }
    if (Row::EMPTY && den == 0.0f) den = 1.0f;
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (__bf16) (num[e] / den);
    *reinterpret_cast<bf16x4 *>(p.out + (size_t) row * D + d) = o;
}

// A workgroup per row and 64 dims: 16 groups of 16 lanes x 4 dims take the partials in turn, U of
// them in flight, each against its own maximum; the groups meet in LDS.
template <int D, class Row>
__global__ __launch_bounds__(256) void merge_many_kernel(typename Row::Params p) {
    constexpr int U = 4;
    __shared__ f32x4 part[16][16];
    __shared__ f32x2 gml[16];
    const int row = blockIdx.x / (D / 64), lane = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int d = (int) (blockIdx.x % (D / 64)) * 64 + lane * 4;
    const Row r(p, row);
    if (!r.write()) return;
    float M = -INFINITY, den = 0.0f;
    f32x4 num = 0.0f;
    for (int j0 = g; j0 < r.n; j0 += 16 * U) {
        f32x2 ml[U];
        f32x4 a[U];
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 16 * u;
            ml[u] = f32x2{-INFINITY, 0.0f};
            a[u] = 0.0f;
            if (j < r.n) {
                ml[u] = r.ml(j);
                a[u] = *reinterpret_cast<const f32x4 *>(r.acc(j) + r.at(j) * D + d);
            }
            top = fmaxf(top, ml[u][0]);
        }
        const float c = __builtin_amdgcn_exp2f(M - (top == -INFINITY ? 0.0f : top));
        num *= c;
        den *= c;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = __builtin_amdgcn_exp2f(ml[u][0] - (top == -INFINITY ? 0.0f : top));
            den = __builtin_fmaf(ml[u][1], w, den);
            num += a[u] * w;
        }
        M = top;
    }
    part[g][lane] = num;
    if (lane == 0) gml[g] = f32x2{M, den};
    __syncthreads();
    if (g == 0) {
        float top = gml[0][0], l = 0.0f;
#pragma unroll
        for (int u = 1; u < 16; ++u) top = fmaxf(top, gml[u][0]);
        f32x4 o = 0.0f;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float w = gml[u][0] == -INFINITY && gml[u][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(gml[u][0] - top);
            l = __builtin_fmaf(gml[u][1], w, l);
            o += part[u][lane] * w;
        }
        if (Row::EMPTY && l == 0.0f) l = 1.0f;
        bf16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (__bf16) (o[e] / l);
        *reinterpret_cast<bf16x4 *>(p.out + (size_t) row * D + d) = b;
    }
}

// The threads of the first form hold a row's partials side by side: up to 8 of them always, up to 40
// where there are threads to cover the loads.  64 rows (2,048 .. 8,192 threads) in 21 partials, first
// form / second: 10.5 / 8.9, 19.0 / 17.5, 15.4 / 14.1 us a step (D = 128, 256, 512); 32,768 threads, 11
// 15.3 / 16.3 and 20.9 / 21.8, 21 20.7 / 20.5 and 22.2 / 22.3; 65,536 20.1 / 23.7 and 24.7 / 28.4, 31
// 33.6 / 35.5 and 41.3 / 43.6; 262,144 in 11 37.6 / 48.5, in 31 77.4 / 79.6.  n: most partials of a row.
template <int D, class Row>
void launch_parts_merge(const typename Row::Params &m, int n, hipStream_t st) {
    const int rows = Row::rows(m);
    const long long threads = (long long) rows * (D / 4);
    const unsigned few = (unsigned) ((threads + 255) / 256);
    if (n <= 4) hipLaunchKernelGGL((merge_few_kernel<D, 4, Row>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 8) hipLaunchKernelGGL((merge_few_kernel<D, 8, Row>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 16 && threads >= 1 << 15) hipLaunchKernelGGL((merge_few_kernel<D, 16, Row>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 24 && threads >= 1 << 15) hipLaunchKernelGGL((merge_few_kernel<D, 24, Row>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 40 && threads >= 1 << 16) hipLaunchKernelGGL((merge_few_kernel<D, 40, Row>), dim3(few), dim3(256), 0, st, m);
    else hipLaunchKernelGGL((merge_many_kernel<D, Row>), dim3(rows * (D / 64)), dim3(256), 0, st, m);
}

}  // namespace
