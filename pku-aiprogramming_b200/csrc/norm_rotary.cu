// Norms of query and key heads with rotary positions in the same pass, forward and backward, and the same on the way into a paged cache.
//
//   forward   r = (mean_c x_c^2 + eps)^-1/2 over a head's D channels, y_c = w_c r x_c, z = y with its first R channels turned by the token's position
//   backward  g = dz turned back, dw_c = sum over rows of g_c r x_c, and with h_c = w_c g_c, m = r mean_c(h_c x_c): dx_c = r (h_c - r x_c m)
//
// HBM-bound: a row is read once, its sum of squares is met by the lanes that hold it, and it is written once.  A row of D channels is
// units of two accesses of kV values, the two halves of kV pairs (or kV pairs of neighbours, or channels that only are normed); 2^n lanes
// have a row, so the sums are n shuffles, and the rows of a warp lie next to each other.
#include "rotary_parts.cuh"

namespace ttk {

constexpr int kHeadThreads = 256;

// A token's rows of one of the tensors, of head 0: where they come from, where they go, and for keys on their way into a cache a second place.
template <typename Tin, typename Tout>
struct alignas(16) HdRows {
    const Tin* x;
    Tout* y;
};
template <typename Tin, typename Tout>
struct alignas(16) HdRows3 {
    const Tin* x;
    Tout *y, *also;
};

// A lane's units of a row: unit u turns for u < turned, channels c0 .. and c1 .., each there or not.
template <int kV, int kUnits, bool kNeighbours>
struct HdUnits {
    int c0[kUnits], c1[kUnits], at[kUnits];
    unsigned has0, has1, turns;   // a bit per unit
    __device__ __forceinline__ HdUnits(int lane, int lanes, int D, int R) : has0(0), has1(0), turns(0) {
        const int turned = (R / 2 + kV - 1) / kV;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int u = lane + k * lanes;
            at[k] = u;
            if (u < turned) {
                turns |= 1u << k;
                has0 |= 1u << k;
                c0[k] = kNeighbours ? 2 * u * kV : u * kV;
                c1[k] = kNeighbours ? c0[k] + kV : c0[k] + R / 2;
                if (c1[k] < R) has1 |= 1u << k;
            } else {
                c0[k] = R + 2 * (u - turned) * kV;
                c1[k] = c0[k] + kV;
                if (c0[k] < D) has0 |= 1u << k;
                if (c1[k] < D) has1 |= 1u << k;
            }
        }
    }
};

// The table of sines: kV pairs of a unit, two beside each other and then the same two of the next unit, so that what the lanes of a row read at a time is
// whole banks.
template <int kV>
__device__ __forceinline__ int hd_place(int pair, int turned) {
    const int u = pair / kV, e = pair % kV;
    return kV == 1 ? u : 2 * ((e >> 1) * turned + u) + (e & 1);
}
template <int kV>
__device__ __forceinline__ void hd_sines(float2* cs, const RotaryArgs& a, const RtPlaces& places, int here, int tid, float per_half) {
    const int half = a.R / 2, turned = (half + kV - 1) / kV;
    for (int i = tid; i < here * half; i += kHeadThreads) {
        const int t = (int)(((float)i + 0.5f) * per_half), pair = i - t * half;   // i < 2^13: exact
        int b, s;
        places.at(t, &b, &s);
        const int axis = a.axes ? min(max(a.axes[pair], 0), a.n_axes - 1) : 0;
        const int p = a.pos[axis * a.pos_axis + b * a.pos_batch + s];
        cs[t * (turned * kV) + hd_place<kV>(pair, turned)] = rt_turn(p, a.inv_freq[pair], a.scale, a.back);
    }
}
// kV pairs of floats turned: (x[0][e], x[1][e]), or neighbours among x[0] and then among x[1]
template <int kV, bool kNeighbours>
__device__ __forceinline__ void hd_turn(float (&x)[2][kV], const float2* cs, int u, int turned) {
    float2 f[kV];
    if (kV == 1) {
        f[0] = cs[u];
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2) {
            const float4 z = *reinterpret_cast<const float4*>(cs + 2 * ((e >> 1) * turned + u));
            f[e] = make_float2(z.x, z.y);
            f[(e + 1) % kV] = make_float2(z.z, z.w);
        }
    }
#pragma unroll
    for (int e = 0; e < kV; ++e) {
        float &p = kNeighbours && kV > 1 ? x[2 * e / kV][2 * e % kV] : x[0][e], &q = kNeighbours && kV > 1 ? x[2 * e / kV][(2 * e + 1) % kV] : x[1][e];
        const float x1 = p, x2 = q;
        p = x1 * f[e].x - x2 * f[e].y;
        q = x2 * f[e].x + x1 * f[e].y;
    }
}
__device__ __forceinline__ float hd_weight(const void* w, int bf16, int c) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[c]) : static_cast<const float*>(w)[c];
}

// blockDim = kHeadThreads; 2^log_lanes lanes to a row.  kAppend: keys and values go into the pools' rows (a third tensor, which is copied).
template <typename Tin, typename Tout, int kV, int kUnits, bool kNeighbours, bool kNorm, bool kAppend>
__global__ void __launch_bounds__(kHeadThreads) heads_kernel(const NormRotaryArgs a, int tokens_per_cta, int log_lanes, float per_half) {
    using In = RtVec<Tin, kV>;
    using Out = RtVec<Tout, kV>;
    using Rows = typename std::conditional<kAppend, HdRows3<Tin, Tout>, HdRows<Tin, Tout>>::type;
    constexpr int kTensors = kAppend ? 3 : 2, kAhead = 2;
    extern __shared__ float4 sm[];
    Rows* rows = reinterpret_cast<Rows*>(sm);   // [tokens_per_cta][kTensors]
    float2* cs = reinterpret_cast<float2*>(rows + kTensors * tokens_per_cta);
    const RotaryArgs& r = a.r;
    const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes, groups = kHeadThreads >> log_lanes;
    const unsigned t0 = blockIdx.x * (unsigned)tokens_per_cta, n_tok = (unsigned)r.B * (unsigned)r.S;
    const int here = (int)min((unsigned)tokens_per_cta, n_tok - t0), turned = (r.R / 2 + kV - 1) / kV;
    const RtPlaces places(t0, r.B, r.S);
    const HdUnits<kV, kUnits, kNeighbours> units(lane, lanes, r.D, r.R);
    grid_let_next_start();
    grid_wait_for_previous();
    hd_sines<kV>(cs, r, places, here, tid, per_half);
    for (int i = kHeadThreads - 1 - tid; i < kTensors * here; i += kHeadThreads) {
        const int t = i / kTensors, w = i - t * kTensors;
        int b, s;
        places.at(t, &b, &s);
        if constexpr (kAppend) {
            Rows z{};
            if (w == 0) {
                z.x = (const Tin*)r.x[0] + s * r.xs[0][2];
                z.y = (Tout*)r.y[0] + s * r.ys[0][2];
            } else {
                z.x = w == 1 ? (const Tin*)r.x[1] + s * r.xs[1][2] : (const Tin*)a.v + s * a.v_stride[0];
                if (w == 1 && r.y[1]) z.also = (Tout*)r.y[1] + s * r.ys[1][2];
                const int slot = a.slots[s];
                if (slot >= 0 && slot < a.n_slots) {
                    const int page = slot / a.page;
                    z.y = (Tout*)a.pool[w - 1] + ((long long)page * r.heads[1] * a.page + (slot - page * a.page)) * r.D;
                }
            }
            rows[i] = z;
        } else {
            rows[i] = Rows{(const Tin*)r.x[w] + b * r.xs[w][0] + s * r.xs[w][2], (Tout*)r.y[w] + b * r.ys[w][0] + s * r.ys[w][2]};
        }
    }
    __syncthreads();
    const float inv_D = 1.f / (float)r.D;
#pragma unroll 1
    for (int w = 0; w < kTensors; ++w) {
        const int heads = w < 2 ? r.heads[w] : r.heads[1];
        if (heads == 0) continue;
        const bool moved = kAppend && w == 2;   // as it is
        const long long x_head = moved ? a.v_stride[1] : r.xs[w][1], y_head = kAppend && w > 0 ? (long long)a.page * r.D : r.ys[w][1], also_head = r.ys[1][1];
        float weight[kUnits][2][kV];
        if (kNorm && !moved) {
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    weight[k][0][e] = units.has0 >> k & 1 ? hd_weight(a.w[w], a.w_bf16, units.c0[k] + e) : 0.f;
                    weight[k][1][e] = units.has1 >> k & 1 ? hd_weight(a.w[w], a.w_bf16, units.c1[k] + e) : 0.f;
                }
        }
        const int total = here * heads, dt = groups / heads, dh = groups - dt * heads;
        int t = group / heads, h = group - t * heads;
        for (int base = 0; base < total; base += kAhead * groups) {
            In v[kAhead][kUnits][2];
            int at_t[kAhead], at_h[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                at_t[j] = base + j * groups + group < total ? t : -1;
                at_h[j] = h;
                if (at_t[j] >= 0) {
                    const Tin* x = rows[kTensors * t + w].x + h * x_head;
#pragma unroll
                    for (int k = 0; k < kUnits; ++k) {
                        if (units.has0 >> k & 1) v[j][k][0] = *reinterpret_cast<const In*>(x + units.c0[k]);
                        if (units.has1 >> k & 1) v[j][k][1] = *reinterpret_cast<const In*>(x + units.c1[k]);
                    }
                }
                t += dt;
                h += dh;
                if (h >= heads) {
                    h -= heads;
                    ++t;
                }
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                float x[kUnits][2][kV], sum = 0.f;
#pragma unroll
                for (int k = 0; k < kUnits; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < kV; ++e) {
                            x[k][i][e] = at_t[j] >= 0 && ((i ? units.has1 : units.has0) >> k & 1) ? rt_get(v[j][k][i].v[e]) : 0.f;
                            if (kNorm) sum = fmaf(x[k][i][e], x[k][i][e], sum);
                        }
                if (kNorm && !moved) {
                    for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    const float by = rsqrtf(sum * inv_D + a.eps);
#pragma unroll
                    for (int k = 0; k < kUnits; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < kV; ++e) x[k][i][e] = x[k][i][e] * by * weight[k][i][e];
                }
                if (at_t[j] < 0) continue;
                const Rows& row = rows[kTensors * at_t[j] + w];
                Tout* y = row.y ? row.y + at_h[j] * y_head : nullptr;
                Tout* also = nullptr;
                if constexpr (kAppend) {
                    if (row.also) also = row.also + at_h[j] * also_head;
                }
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    if (!moved && (units.turns >> k & 1)) hd_turn<kV, kNeighbours>(x[k], cs + at_t[j] * (turned * kV), units.at[k], turned);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!((i ? units.has1 : units.has0) >> k & 1)) continue;
                        Out z;
#pragma unroll
                        for (int e = 0; e < kV; ++e) z.v[e] = rt_put<Tout>(x[k][i][e]);
                        const int c = i ? units.c1[k] : units.c0[k];
                        if (!kAppend || y) *reinterpret_cast<Out*>(y + c) = z;
                        if (kAppend && also) *reinterpret_cast<Out*>(also + c) = z;
                    }
                }
            }
        }
    }
}

// The gradient: CTAs below ctas[0] have rows of query heads, the others of key heads, so that the weight's sums of one tensor stay in registers; tiles of tokens go
// round them.  Each leaves its sums [D] in `partial`, which the next kernel adds up in their order: results repeat to the bit.
template <typename T>
struct alignas(16) HdRowsBack {
    const T *g, *x;
    T* y;
};
template <typename T, int kV, int kUnits, bool kNeighbours>
__global__ void __launch_bounds__(kHeadThreads) heads_backward_kernel(const NormRotaryArgs a, int tokens_per_tile, int log_lanes, float per_half, int ctas_q, float* partial) {
    using Vec = RtVec<T, kV>;
    using Rows = HdRowsBack<T>;
    constexpr int kAhead = 2, kWarps = kHeadThreads / 32;
    extern __shared__ float4 sm[];
    Rows* rows = reinterpret_cast<Rows*>(sm);   // [tokens_per_tile]
    float2* cs = reinterpret_cast<float2*>(rows + tokens_per_tile);
    const RotaryArgs& r = a.r;
    const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes, groups = kHeadThreads >> log_lanes;
    const int w = (int)blockIdx.x >= ctas_q, cta = (int)blockIdx.x - (w ? ctas_q : 0), n_cta = w ? (int)gridDim.x - ctas_q : ctas_q;
    const int heads = r.heads[w], turned = (r.R / 2 + kV - 1) / kV;
    const unsigned n_tok = (unsigned)r.B * (unsigned)r.S, tiles = (n_tok + tokens_per_tile - 1) / tokens_per_tile;
    const HdUnits<kV, kUnits, kNeighbours> units(lane, lanes, r.D, r.R);
    grid_let_next_start();
    grid_wait_for_previous();
    float weight[kUnits][2][kV], dw[kUnits][2][kV];
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            weight[k][0][e] = units.has0 >> k & 1 ? hd_weight(a.w[w], a.w_bf16, units.c0[k] + e) : 0.f;
            weight[k][1][e] = units.has1 >> k & 1 ? hd_weight(a.w[w], a.w_bf16, units.c1[k] + e) : 0.f;
            dw[k][0][e] = dw[k][1][e] = 0.f;
        }
    const float inv_D = 1.f / (float)r.D;
    const int dt = groups / heads, dh = groups - dt * heads;
    for (unsigned tile = cta; tile < tiles; tile += n_cta) {
        const unsigned t0 = tile * tokens_per_tile;
        const int here = (int)min((unsigned)tokens_per_tile, n_tok - t0), total = here * heads;
        const RtPlaces places(t0, r.B, r.S);
        __syncthreads();   // the tile before has been read
        hd_sines<kV>(cs, r, places, here, tid, per_half);
        for (int t = kHeadThreads - 1 - tid; t < here; t += kHeadThreads) {
            int b, s;
            places.at(t, &b, &s);
            rows[t] = Rows{(const T*)r.x[w] + b * r.xs[w][0] + s * r.xs[w][2], (const T*)a.in[w] + b * a.in_stride[w][0] + s * a.in_stride[w][2],
                           (T*)r.y[w] + b * r.ys[w][0] + s * r.ys[w][2]};
        }
        __syncthreads();
        int t = group / heads, h = group - t * heads;
        for (int base = 0; base < total; base += kAhead * groups) {
            Vec vg[kAhead][kUnits][2], vx[kAhead][kUnits][2];
            int at_t[kAhead], at_h[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                at_t[j] = base + j * groups + group < total ? t : -1;
                at_h[j] = h;
                if (at_t[j] >= 0) {
                    const T *g = rows[t].g + h * r.xs[w][1], *x = rows[t].x + h * a.in_stride[w][1];
#pragma unroll
                    for (int k = 0; k < kUnits; ++k) {
                        if (units.has0 >> k & 1) {
                            vg[j][k][0] = *reinterpret_cast<const Vec*>(g + units.c0[k]);
                            vx[j][k][0] = *reinterpret_cast<const Vec*>(x + units.c0[k]);
                        }
                        if (units.has1 >> k & 1) {
                            vg[j][k][1] = *reinterpret_cast<const Vec*>(g + units.c1[k]);
                            vx[j][k][1] = *reinterpret_cast<const Vec*>(x + units.c1[k]);
                        }
                    }
                }
                t += dt;
                h += dh;
                if (h >= heads) {
                    h -= heads;
                    ++t;
                }
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                float g[kUnits][2][kV], x[kUnits][2][kV], squares = 0.f, along = 0.f;
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < kV; ++e) {
                            const bool there = at_t[j] >= 0 && ((i ? units.has1 : units.has0) >> k & 1);
                            g[k][i][e] = there ? rt_get(vg[j][k][i].v[e]) : 0.f;
                            x[k][i][e] = there ? rt_get(vx[j][k][i].v[e]) : 0.f;
                        }
                    if (at_t[j] >= 0 && (units.turns >> k & 1)) hd_turn<kV, kNeighbours>(g[k], cs + at_t[j] * (turned * kV), units.at[k], turned);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < kV; ++e) {
                            if (!((i ? units.has1 : units.has0) >> k & 1)) g[k][i][e] = 0.f;   // (turned by what no pair has)
                            squares = fmaf(x[k][i][e], x[k][i][e], squares);
                            along = fmaf(g[k][i][e] * weight[k][i][e], x[k][i][e], along);
                        }
                }
                for (int d = 1; d < lanes; d <<= 1) {
                    squares += __shfl_xor_sync(0xffffffffu, squares, d);
                    along += __shfl_xor_sync(0xffffffffu, along, d);
                }
                const float by = rsqrtf(squares * inv_D + a.eps), less = along * inv_D * by * by;
                if (at_t[j] < 0) continue;
                T* y = rows[at_t[j]].y + at_h[j] * r.ys[w][1];
#pragma unroll
                for (int k = 0; k < kUnits; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!((i ? units.has1 : units.has0) >> k & 1)) continue;
                        Vec z;
#pragma unroll
                        for (int e = 0; e < kV; ++e) {
                            dw[k][i][e] = fmaf(g[k][i][e], x[k][i][e] * by, dw[k][i][e]);
                            z.v[e] = rt_put<T>(by * (g[k][i][e] * weight[k][i][e] - x[k][i][e] * less));
                        }
                        *reinterpret_cast<Vec*>(y + (i ? units.c1[k] : units.c0[k])) = z;
                    }
            }
        }
    }
    // the rows of a warp, then the warps
    float* sums = reinterpret_cast<float*>(sm);   // [kWarps][D]
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                float y = dw[k][i][e];
                for (int d = lanes; d < 32; d <<= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
                if ((tid & 31) < lanes && ((i ? units.has1 : units.has0) >> k & 1)) sums[(tid >> 5) * r.D + (i ? units.c1[k] : units.c0[k]) + e] = y;
            }
    __syncthreads();
    for (int c = tid; c < r.D; c += kHeadThreads) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) y += sums[i * r.D + c];
        partial[(long long)blockIdx.x * r.D + c] = y;
    }
}
// One tensor's sums, 32 channels to a CTA.
__global__ void __launch_bounds__(1024) heads_weight_kernel(const float* partial, int ctas_q, int ctas_k, int D, void* dw_q, void* dw_k, int bf16) {
    __shared__ float sums[32][33];
    const int w = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x, n = w ? ctas_k : ctas_q;
    const float* from = partial + (w ? (long long)ctas_q * D : 0) + c;
    grid_let_next_start();
    grid_wait_for_previous();
    float y = 0.f;
    if (c < D)
        for (int i = threadIdx.y; i < n; i += 32) y += from[(long long)i * D];
    sums[threadIdx.y][threadIdx.x] = y;
    __syncthreads();
    y = sums[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
    const int out = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && out < D) {
        void* dw = w ? dw_k : dw_q;
        if (bf16) static_cast<__nv_bfloat16*>(dw)[out] = __float2bfloat16_rn(y);
        else static_cast<float*>(dw)[out] = y;
    }
}

// Lanes of a row, and whether they are enough for kUnits units each.
static bool hd_lanes(int units, int per_lane, int* log_lanes) {
    *log_lanes = 0;
    while ((per_lane << *log_lanes) < units) ++*log_lanes;
    return *log_lanes <= 5;
}
constexpr int hd_units(int kV) { return kV >= 4 ? 1 : kV == 2 ? 3 : 5; }   // of a lane, at most: 256 channels to 32 lanes
static int hd_units_of_row(int D, int R, int kV) { return (R / 2 + kV - 1) / kV + (D - R + 2 * kV - 1) / (2 * kV); }
// The widest accesses that fit: rows at multiples of `aligned` bytes, channels in whole accesses
static bool hd_fits(int D, int R, int interleaved, int kV, int size, int aligned) {
    int log_lanes;
    return kV * size <= aligned && (kV == 1 || ((interleaved ? R : R / 2) % kV == 0 && D % kV == 0)) && hd_lanes(hd_units_of_row(D, R, kV), hd_units(kV), &log_lanes);
}
// Bytes that all of some rows lie at multiples of, or-ed together: the lowest bit set.
struct HdPlaces {
    unsigned long long bits = 0;
    void add(const void* p, const long long* stride, const int* n, int dims, int size) {
        bits |= (uintptr_t)p;
        for (int d = 0; d < dims; ++d)
            if (n[d] > 1) bits |= (unsigned long long)stride[d] * size;
    }
    int aligned(int most) const { return (int)((bits | most) & (0 - (bits | most))); }
};

// Tokens per CTA: four rows to each group of lanes, fewer where all CTAs are resident at once then.
static int hd_tokens(long long n_tok, int heads, int groups, size_t token, long long resident) {
    const long long one_wave = (n_tok + resident - 1) / resident;
    long long per = 4LL * groups / heads;
    if (per > one_wave || 3 * per >= 2 * one_wave) per = one_wave;
    const long long fits = 27 * 1024 / (long long)token;
    if (per > fits) per = fits;
    return per < 1 ? 1 : (int)per;
}

template <typename Tin, typename Tout, int kV, bool kNorm, bool kAppend>
static cudaError_t launch_heads(const NormRotaryArgs& a, int interleaved, cudaStream_t st) {
    constexpr int kUnits = hd_units(kV);
    int log_lanes;
    hd_lanes(hd_units_of_row(a.r.D, a.r.R, kV), kUnits, &log_lanes);
    const int turned = (a.r.R / 2 + kV - 1) / kV, heads = a.r.heads[0] + a.r.heads[1] * (kAppend ? 2 : 1);
    const size_t token = (size_t)turned * kV * sizeof(float2) + (kAppend ? 3 * 32 : 2 * 16);
    const long long n_tok = (long long)a.r.B * a.r.S;
    const int per = hd_tokens(n_tok, heads, kHeadThreads >> log_lanes, token, 3LL * sm_count());
    LaunchScope ls(kAppend ? K_CACHE_APPEND_ROTARY : K_NORM_ROTARY, st);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, (unsigned)((n_tok + per - 1) / per), kHeadThreads, per * token, st, a, per, log_lanes, 2.f / (float)a.r.R);
    };
    return interleaved ? go(heads_kernel<Tin, Tout, kV, kUnits, true, kNorm, kAppend>) : go(heads_kernel<Tin, Tout, kV, kUnits, false, kNorm, kAppend>);
}
template <typename Tin, typename Tout, bool kNorm, bool kAppend, int kV = 16 / sizeof(Tin)>
static cudaError_t launch_heads_width(const NormRotaryArgs& a, int interleaved, int aligned, cudaStream_t st) {
    if constexpr (kV > 1) {
        if (!hd_fits(a.r.D, a.r.R, interleaved, kV, sizeof(Tin), aligned)) return launch_heads_width<Tin, Tout, kNorm, kAppend, kV / 2>(a, interleaved, aligned, st);
    }
    return launch_heads<Tin, Tout, kV, kNorm, kAppend>(a, interleaved, st);
}
static void hd_add_rows(HdPlaces* p, const RotaryArgs& a, int i, int in_size, int out_size) {
    const int n[3] = {a.B, a.heads[i], a.S};
    if (!a.heads[i]) return;
    p->add(a.x[i], a.xs[i], n, 3, in_size);
    if (a.y[i]) p->add(a.y[i], a.ys[i], n, 3, out_size);
}
cudaError_t norm_rotary(const NormRotaryArgs& a, int bf16, int interleaved, cudaStream_t st) {
    HdPlaces places;
    for (int i = 0; i < 2; ++i) hd_add_rows(&places, a.r, i, bf16 ? 2 : 4, bf16 ? 2 : 4);
    const int aligned = places.aligned(16);
    return bf16 ? launch_heads_width<__nv_bfloat16, __nv_bfloat16, true, false>(a, interleaved, aligned, st) : launch_heads_width<float, float, true, false>(a, interleaved, aligned, st);
}
cudaError_t cache_append_rotary(const NormRotaryArgs& a, int bf16, int interleaved, cudaStream_t st) {
    // places in units of the input's type: the outputs are bf16
    const int size = bf16 ? 2 : 4;
    HdPlaces in, out;
    const int n[2] = {a.r.S, a.r.heads[1]};
    for (int i = 0; i < 2; ++i) {
        const int m[3] = {1, a.r.heads[i], a.r.S};
        if (!a.r.heads[i]) continue;
        in.add(a.r.x[i], a.r.xs[i], m, 3, size);
        if (a.r.y[i]) out.add(a.r.y[i], a.r.ys[i], m, 3, 2);
        out.add(a.pool[i], nullptr, nullptr, 0, 2);
    }
    in.add(a.v, a.v_stride, n, 2, size);
    const int from = in.aligned(16), to = out.aligned(16) * (size / 2), aligned = from < to ? from : to;
    auto go = [&](auto type) {
        using T = decltype(type);
        return a.w[0] || a.w[1] ? launch_heads_width<T, __nv_bfloat16, true, true>(a, interleaved, aligned, st) : launch_heads_width<T, __nv_bfloat16, false, true>(a, interleaved, aligned, st);
    };
    return bf16 ? go(__nv_bfloat16{}) : go(float{});
}

// CTAs of the gradient: what the SMs hold at once, shared out by the heads; fewer where there are not rows for them.
constexpr int kBackCtas = 2;   // per SM
static void hd_ctas(const NormRotaryArgs& a, int (&ctas)[2]) {
    const long long n_tok = (long long)a.r.B * a.r.S, all = (long long)sm_count() * kBackCtas, heads = a.r.heads[0] + a.r.heads[1];
    for (int i = 0; i < 2; ++i) {
        long long n = (all * a.r.heads[i] + heads / 2) / heads;
        if (i == 0 && n >= all && a.r.heads[1]) n = all - 1;
        if (i == 1) n = all - ctas[0];
        if (n > n_tok) n = n_tok;
        ctas[i] = !a.r.heads[i] || !n_tok ? 0 : n < 1 ? 1 : (int)n;
    }
}
size_t norm_rotary_backward_workspace(int D) { return align256((size_t)sm_count() * kBackCtas * D * sizeof(float)); }

template <typename T, int kV>
static cudaError_t launch_heads_back(const NormRotaryArgs& a, int interleaved, float* partial, const int (&ctas)[2], cudaStream_t st) {
    constexpr int kUnits = hd_units(kV);
    int log_lanes;
    hd_lanes(hd_units_of_row(a.r.D, a.r.R, kV), kUnits, &log_lanes);
    const int turned = (a.r.R / 2 + kV - 1) / kV, groups = kHeadThreads >> log_lanes;
    const size_t token = (size_t)turned * kV * sizeof(float2) + sizeof(HdRowsBack<T>), sums = (size_t)kHeadThreads / 32 * a.r.D * sizeof(float);
    const int most = a.r.heads[0] > a.r.heads[1] ? a.r.heads[0] : a.r.heads[1];
    int per = 4 * groups / most;
    const int fits = (int)(27 * 1024 / token);
    per = per > fits ? fits : per < 1 ? 1 : per;
    const size_t smem = per * token > sums ? per * token : sums;
    LaunchScope ls(K_NORM_ROTARY_BWD, st);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, (unsigned)(ctas[0] + ctas[1]), kHeadThreads, smem, st, a, per, log_lanes, 2.f / (float)a.r.R, ctas[0], partial);
    };
    return interleaved ? go(heads_backward_kernel<T, kV, kUnits, true>) : go(heads_backward_kernel<T, kV, kUnits, false>);
}
template <typename T, int kV = 16 / sizeof(T)>
static cudaError_t launch_heads_back_width(const NormRotaryArgs& a, int interleaved, int aligned, float* partial, const int (&ctas)[2], cudaStream_t st) {
    if constexpr (kV > 1) {
        if (!hd_fits(a.r.D, a.r.R, interleaved, kV, sizeof(T), aligned)) return launch_heads_back_width<T, kV / 2>(a, interleaved, aligned, partial, ctas, st);
    }
    return launch_heads_back<T, kV>(a, interleaved, partial, ctas, st);
}
cudaError_t norm_rotary_backward(const NormRotaryArgs& a, int bf16, int interleaved, void* workspace, cudaStream_t st) {
    HdPlaces places;
    for (int i = 0; i < 2; ++i) {
        hd_add_rows(&places, a.r, i, bf16 ? 2 : 4, bf16 ? 2 : 4);
        const int n[3] = {a.r.B, a.r.heads[i], a.r.S};
        if (a.r.heads[i]) places.add(a.in[i], a.in_stride[i], n, 3, bf16 ? 2 : 4);
    }
    int ctas[2];
    hd_ctas(a, ctas);
    float* partial = static_cast<float*>(workspace);
    if (ctas[0] + ctas[1]) {
        const int aligned = places.aligned(16);
        const cudaError_t e = bf16 ? launch_heads_back_width<__nv_bfloat16>(a, interleaved, aligned, partial, ctas, st)
                                   : launch_heads_back_width<float>(a, interleaved, aligned, partial, ctas, st);
        if (e != cudaSuccess) return e;
    }
    LaunchScope ls(K_NORM_ROTARY_DW, st);
    return launch_overlapped(heads_weight_kernel, dim3((unsigned)(a.r.D + 31) / 32, a.r.heads[1] ? 2 : 1), dim3(32, 32), 0, st, (const float*)partial, ctas[0], ctas[1], a.r.D, a.dw[0],
                             a.dw[1], a.w_bf16);
}

}  // namespace ttk
