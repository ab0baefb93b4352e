// Norms of query and key heads with rotary positions in the same pass, forward and backward, and the same on the way into a paged cache.
//
//   forward   r = (mean_c x_c^2 + eps)^-1/2 over a head's D channels, y_c = w_c r x_c, z = y with its first R channels turned by the token's position
//   backward  g = dz turned back, dw_c = sum over rows of g_c r x_c, and with h_c = w_c g_c, m = r mean_c(h_c x_c): dx_c = r (h_c - r x_c m)
//
// HBM-bound: a row is read once, its sum of squares is met by the lanes that hold it, and it is written once.  A row of D channels is
// units of two accesses of kV values, the two halves of kV pairs (or kV pairs of neighbours, or channels that only are normed); 2^n lanes
// have a row, so the sums are n shuffles, and the rows of a warp lie next to each other.
//
// Beside the bytes stand sixteen conversions, products and roundings for 32 bytes of bf16, and a token's sines, exact for any position, which are worth five
// of its rows; fewer of them were faster, though issue slots are half busy (45 %, the gradient 51 %): what is left waits within a row, on its loads, on shared memory
// and the lanes' sums, on its own arithmetic (1.6, 3.0 and 1.1 cycles an issue, in the gradient 1.8, 1.3 and 1.4), with the 16 or 24 warps per SM that the registers
// leave.  So sines, weights and places lie in shared memory, made a tile of tokens ahead, each CTA that is resident has an equal share of the tokens, and two rows
// of a lane are on their way at once.  Replayed from a graph: 16384 tokens of 32 + 8 heads of 128 in bf16, all
// channels turned, 62.2 us, 5.4 TB/s (a copy runs at 6.6); the gradient of 8192 of them 56.5 us, 4.5 TB/s; of 4094 tokens of 8 + 8 heads of 64 floats 15.0 us, 3.4 TB/s; 13,000
// tokens turned and written into a cache of pages of 16 58.2 us, 5.5 TB/s; 64 single tokens 4 us, a launch.
#include "rotary_parts.cuh"
#include "sm100_ptx.cuh"

namespace ttk {
using namespace sm100;

constexpr int kHeadThreads = 256;
// CTAs per SM, as many as hold two rows of a lane in registers.  16384 tokens of 40 heads of 128, all channels turned: with one unit a lane 3, 63.6 us (4, which
// spill, 69.4), with two 2, 62.2 us (3, which spill, 82.7).
constexpr int hd_ctas_per_sm(int units) { return units == 1 ? 3 : 2; }
constexpr int kBackCtas = 2;   // of the gradient: 8192 of those tokens 56.5 us; 3, which spill, 77.7

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

// A lane's units of a row: unit u turns for u < turned, channels c0 .. and c1 .., each there or not.  kWhole: all are there.
template <int kV, int kUnits, bool kNeighbours, bool kWhole>
struct HdUnits {
    int c0[kUnits], c1[kUnits], at[kUnits];
    unsigned there[2], turning;   // a bit per unit
    __device__ __forceinline__ HdUnits(int lane, int lanes, int D, int R) : there{0, 0}, turning(0) {
        const int turned = (R / 2 + kV - 1) / kV;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int u = lane + k * lanes;
            const bool turn = u < turned;
            at[k] = u;
            c0[k] = !turn ? R + 2 * (u - turned) * kV : kNeighbours ? 2 * u * kV : u * kV;
            c1[k] = turn && !kNeighbours ? c0[k] + R / 2 : c0[k] + kV;
            if (turn) turning |= 1u << k;
            if (c0[k] < D) there[0] |= 1u << k;
            if (c1[k] < (turn ? R : D)) there[1] |= 1u << k;
        }
    }
    __device__ __forceinline__ int channel(int k, int chunk) const { return chunk ? c1[k] : c0[k]; }
    __device__ __forceinline__ bool has(int k, int chunk) const { return kWhole || (there[chunk] >> k & 1); }
    __device__ __forceinline__ bool turns(int k) const { return turning >> k & 1; }
    // The flags differ among the lanes of a row, which meet in every turn of a loop: they are made unknown to the compiler in each, so that it cannot make
    // loops of their own for lanes with one and with another.
    __device__ __forceinline__ void forget() { asm volatile("" : "+r"(there[0]), "+r"(there[1]), "+r"(turning)); }
};

// Tables in shared memory lie as the lanes of a row read them, 16 bytes of one unit beside the same of the next, so that a read is whole banks.
// The sines: (cos, sin) of two pairs of a unit, in halves cosines first; kV = 1: of the unit's pair.
template <int kV, bool kNeighbours>
__device__ __forceinline__ void hd_put_turn(float* cs, int pair, int turned, float2 f) {
    const int u = pair / kV, e = pair % kV;
    if (kV == 1) {
        cs[2 * u] = f.x;
        cs[2 * u + 1] = f.y;
    } else {
        float* at = cs + 4 * ((e >> 1) * turned + u);
        at[kNeighbours ? 2 * (e & 1) : e & 1] = f.x;
        at[kNeighbours ? 2 * (e & 1) + 1 : 2 + (e & 1)] = f.y;
    }
}
// of a tile's tokens: a thread keeps its pair
template <int kV, bool kNeighbours>
__device__ __forceinline__ void hd_sines(float* cs, const RotaryArgs& a, const RtPlaces& places, int here, int tid) {
    const int half = a.R / 2, turned = (half + kV - 1) / kV, at_once = kHeadThreads / half;   // half is at most 128
    const int first = tid / half, pair = tid - first * half;
    if (first >= at_once) return;
    const int axis = a.axes ? min(max(a.axes[pair], 0), a.n_axes - 1) : 0;
    const double freq = a.inv_freq[pair];
    const int* pos = a.pos + axis * a.pos_axis;
    for (int t = first; t < here; t += at_once) {
        int b, s;
        places.at(t, &b, &s);
        hd_put_turn<kV, kNeighbours>(cs + t * (2 * turned * kV), pair, turned, rt_turn(pos[b * a.pos_batch + s], freq, a.scale, a.back));
    }
}
// kV pairs of floats turned: (x[0][e], x[1][e]), or neighbours among x[0] and then among x[1]
template <int kV, bool kNeighbours>
__device__ __forceinline__ void hd_turn(float (&x)[2][kV], const float* cs, int u, int turned) {
    auto turn = [](float& p, float& q, float c, float s) {
        const float x1 = p, x2 = q;
        p = x1 * c - x2 * s;
        q = x2 * c + x1 * s;
    };
    if constexpr (kV == 1) {
        const float2 f = reinterpret_cast<const float2*>(cs)[u];
        turn(x[0][0], x[1][0], f.x, f.y);
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2) {
            const float4 z = reinterpret_cast<const float4*>(cs)[(e >> 1) * turned + u];
            if (kNeighbours) {
                turn(x[2 * e / kV][2 * e % kV], x[2 * e / kV][2 * e % kV + 1], z.x, z.y);
                turn(x[(2 * e + 2) / kV][(2 * e + 2) % kV], x[(2 * e + 2) / kV][(2 * e + 2) % kV + 1], z.z, z.w);
            } else {
                const uint64_t c = pack_f32x2(z.x, z.y), s = pack_f32x2(z.z, z.w);
                const uint64_t x1 = pack_f32x2(x[0][e], x[0][e + 1]), x2 = pack_f32x2(x[1][e], x[1][e + 1]);
                float less[2];   // (there is no packed subtraction, and changing signs is two operations)
                unpack_f32x2(mul_f32x2(x2, s), less[0], less[1]);
                unpack_f32x2(fma_f32x2(x2, c, mul_f32x2(x1, s)), x[1][e], x[1][e + 1]);
                x[0][e] = fmaf(x[0][e], z.x, -less[0]);
                x[0][e + 1] = fmaf(x[0][e + 1], z.y, -less[1]);
            }
        }
    }
}
// The weights of a tensor, up to 4 channels of a chunk of a unit at a time.  What no channel has stays as it is.
template <int kV, bool kNeighbours>
__device__ __forceinline__ void hd_weights(float* ws, const void* w, int bf16, int n_units, int D, int R, int tid) {
    constexpr int kQuad = kV < 4 ? kV : 4;
    const int turned = (R / 2 + kV - 1) / kV;
    for (int c = tid; c < D; c += kHeadThreads) {
        const bool paired = !kNeighbours && c < R;   // in halves
        const int in = paired ? (c < R / 2 ? c : c - R / 2) : c < R ? c : c - R;   // (of the chunks, or of those behind R)
        const int chunk = paired ? c >= R / 2 : in / kV & 1, u = (paired ? in / kV : in / (2 * kV)) + (c < R ? 0 : turned), e = in % kV;
        ws[((chunk * (kV / kQuad) + e / kQuad) * n_units + u) * kQuad + e % kQuad] =
            bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[c]) : static_cast<const float*>(w)[c];
    }
}
template <int kV>
__device__ __forceinline__ void hd_weight(float (&w)[2][kV], const float* ws, int u, int n_units) {
    constexpr int kQuad = kV < 4 ? kV : 4;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < kV; e += kQuad) {
            const RtVec<float, kQuad> z = reinterpret_cast<const RtVec<float, kQuad>*>(ws)[(i * (kV / kQuad) + e / kQuad) * n_units + u];
#pragma unroll
            for (int j = 0; j < kQuad; ++j) w[i][e + j] = z.v[j];
        }
}
// Values of a chunk in floats, and of two of them at a time f(a, b) = a * b, or + c
template <typename T, int kV>
__device__ __forceinline__ void hd_floats(float (&x)[kV], const RtVec<T, kV>& v) {
    if constexpr (sizeof(T) == 2 && kV > 1) {
        RtVec<uint32_t, kV / 2> w;
        memcpy(&w, &v, sizeof w);
#pragma unroll
        for (int e = 0; e < kV / 2; ++e) {
            x[2 * e] = __uint_as_float(w.v[e] << 16);
            x[2 * e + 1] = __uint_as_float(w.v[e] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) x[e] = rt_get(v.v[e]);
    }
}
template <typename T, int kV>
__device__ __forceinline__ RtVec<T, kV> hd_rounded(const float (&x)[kV]) {
    RtVec<T, kV> z;
    if constexpr (sizeof(T) == 2 && kV > 1) {
#pragma unroll
        for (int e = 0; e < kV; e += 2) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(x[e], x[e + 1]);
            z.v[e] = two.x;
            z.v[e + 1] = two.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) z.v[e] = rt_put<T>(x[e]);
    }
    return z;
}
template <int kV>
__device__ __forceinline__ void hd_mul(float (&y)[kV], const float (&a)[kV], const float (&b)[kV]) {
    if constexpr (kV == 1) {
        y[0] = a[0] * b[0];
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2) unpack_f32x2(mul_f32x2(pack_f32x2(a[e], a[e + 1]), pack_f32x2(b[e], b[e + 1])), y[e], y[e + 1]);
    }
}
template <int kV>
__device__ __forceinline__ void hd_mul(float (&y)[kV], const float (&a)[kV], float b) {
    if constexpr (kV == 1) {
        y[0] = a[0] * b;
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2) unpack_f32x2(mul_f32x2(pack_f32x2(a[e], a[e + 1]), pack_f32x2(b, b)), y[e], y[e + 1]);
    }
}
// y += a b, over the channels into two sums or into one for each
template <int kV>
__device__ __forceinline__ void hd_add_products(float (&sum)[2], const float (&a)[kV], const float (&b)[kV]) {
    if constexpr (kV == 1) {
        sum[0] = fmaf(a[0], b[0], sum[0]);
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2)
            unpack_f32x2(fma_f32x2(pack_f32x2(a[e], a[e + 1]), pack_f32x2(b[e], b[e + 1]), pack_f32x2(sum[0], sum[1])), sum[0], sum[1]);
    }
}
template <int kV>
__device__ __forceinline__ void hd_fma(float (&y)[kV], const float (&a)[kV], const float (&b)[kV], const float (&c)[kV]) {
    if constexpr (kV == 1) {
        y[0] = fmaf(a[0], b[0], c[0]);
    } else {
#pragma unroll
        for (int e = 0; e < kV; e += 2)
            unpack_f32x2(fma_f32x2(pack_f32x2(a[e], a[e + 1]), pack_f32x2(b[e], b[e + 1]), pack_f32x2(c[e], c[e + 1])), y[e], y[e + 1]);
    }
}
template <int kV>
__device__ __forceinline__ void hd_fma(float (&y)[kV], const float (&a)[kV], float b, const float (&c)[kV]) {
    float bs[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) bs[e] = b;
    hd_fma<kV>(y, a, bs, c);
}
// What a lane has of a row, as it comes; 0 for channels that are not there
template <typename T, int kV, int kUnits>
struct HdRaw {
    RtVec<T, kV> v[kUnits][2];
    template <typename Units>
    __device__ __forceinline__ void load(const T* x, const Units& units) {
#pragma unroll
        for (int k = 0; k < kUnits; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (units.has(k, i)) {
                    v[k][i] = *reinterpret_cast<const RtVec<T, kV>*>(x + units.channel(k, i));
                } else {
#pragma unroll
                    for (int e = 0; e < kV; ++e) v[k][i].v[e] = rt_put<T>(0.f);
                }
            }
    }
};
// The sum over a row's lanes, 2^n of them.
__device__ __forceinline__ float hd_sum(float x, int lanes) {
#pragma unroll
    for (int d = 16; d; d >>= 1)
        if (d < lanes) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
// A walk of a group of lanes over the rows (token, head) of a tile, as many apart as there are groups.  Every group takes as many turns; where there is no row
// left it takes the tile's first one, for nothing.
struct HdWalk {
    int t, h, dt, dh, heads, row, total, apart;
    __device__ __forceinline__ HdWalk(int group, int groups, int n_heads, int tokens) : heads(n_heads), row(group), total(tokens * n_heads), apart(groups) {
        t = group / n_heads;
        h = group - t * n_heads;
        dt = groups / n_heads;
        dh = groups - dt * n_heads;
        stay();
    }
    __device__ __forceinline__ int turns() const { return (total + apart - 1) / apart; }
    __device__ __forceinline__ bool there() const { return row < total; }
    __device__ __forceinline__ void stay() {
        if (!there()) t = h = 0;
    }
    __device__ __forceinline__ void next() {
        row += apart;
        t += dt;
        h += dh;
        if (h >= heads) {
            h -= heads;
            ++t;
        }
        stay();
    }
};
// A CTA's tokens of n: equal shares.
__device__ __forceinline__ unsigned hd_share(unsigned n, unsigned cta, unsigned ctas) { return (unsigned)((unsigned long long)n * cta / ctas); }

// blockDim = kHeadThreads; 2^log_lanes lanes to a row.  A CTA goes through its tokens tile by tile; the next tile's sines are made before the rows of the one at
// hand.  kAppend: keys and values go into the pools' rows (a third tensor, which is copied).
template <typename Tin, typename Tout, int kV, int kUnits, bool kNeighbours, bool kNorm, bool kAppend, bool kWhole>
__global__ void __launch_bounds__(kHeadThreads, hd_ctas_per_sm(kUnits)) heads_kernel(const NormRotaryArgs a, int tile_tokens, int log_lanes) {
    using Out = RtVec<Tout, kV>;
    using Raw = HdRaw<Tin, kV, kUnits>;
    using Rows = typename std::conditional<kAppend, HdRows3<Tin, Tout>, HdRows<Tin, Tout>>::type;
    constexpr int kTensors = kAppend ? 3 : 2;
    extern __shared__ float4 sm[];
    const RotaryArgs& r = a.r;
    const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes, groups = kHeadThreads >> log_lanes;
    const int turned = (r.R / 2 + kV - 1) / kV, n_units = lanes * kUnits, tile_sines = tile_tokens * (2 * turned * kV);
    Rows* all_rows = reinterpret_cast<Rows*>(sm);                                     // [2][tile_tokens][kTensors]
    float* ws = reinterpret_cast<float*>(all_rows + 2 * kTensors * tile_tokens);      // [2][n_units * 2 * kV]
    float* all_cs = ws + (kNorm ? 4 * n_units * kV : 0);                              // [2][tile_tokens][2 * turned * kV]
    const unsigned n_tok = (unsigned)r.B * (unsigned)r.S, first = hd_share(n_tok, blockIdx.x, gridDim.x), last = hd_share(n_tok, blockIdx.x + 1, gridDim.x);
    const HdUnits<kV, kUnits, kNeighbours, kWhole> all_units(lane, lanes, r.D, r.R);
    grid_let_next_start();
    grid_wait_for_previous();
    auto tile_of = [&](unsigned t0) { return (int)min((unsigned)tile_tokens, last - t0); };
    auto prepare = [&](unsigned t0, int which) {
        const int here = tile_of(t0);
        const RtPlaces places(t0, r.B, r.S);
        hd_sines<kV, kNeighbours>(all_cs + which * tile_sines, r, places, here, tid);
        Rows* rows = all_rows + which * (kTensors * tile_tokens);
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
    };
    prepare(first, 0);
    if (kNorm) {
        if (!kWhole) {
            for (int i = tid; i < 4 * n_units * kV; i += kHeadThreads) ws[i] = 0.f;
            __syncthreads();
        }
        for (int w = 0; w < 2; ++w)
            if (r.heads[w]) hd_weights<kV, kNeighbours>(ws + w * (2 * n_units * kV), a.w[w], a.w_bf16, n_units, r.D, r.R, tid);
    }
    __syncthreads();
    const float inv_D = 1.f / (float)r.D;
    const int up_to_k = r.heads[0], up_to_v = r.heads[0] + r.heads[1], heads = up_to_v + (kAppend ? r.heads[1] : 0);
    int which = 0;
    for (unsigned t0 = first; t0 < last; t0 += tile_tokens, which ^= 1) {
        if (last - t0 > (unsigned)tile_tokens) prepare(t0 + tile_tokens, which ^ 1);
        const Rows* rows = all_rows + which * (kTensors * tile_tokens);
        const float* cs = all_cs + which * tile_sines;
        HdWalk at(group, groups, heads, tile_of(t0));
        // what is to be done with a row that is on its way
        struct Job {
            Raw raw;
            Tout *y, *also;   // null: nowhere
            int sines, w;
        };
        auto fetch = [&](Job& to, const HdWalk& x) {
            const int w = x.h < up_to_k ? 0 : !kAppend || x.h < up_to_v ? 1 : 2, h = x.h - (w == 0 ? 0 : w == 1 ? up_to_k : up_to_v);
            const Rows row = rows[kTensors * x.t + w];
            to.raw.load(row.x + h * (kAppend && w == 2 ? a.v_stride[1] : w ? r.xs[1][1] : r.xs[0][1]), all_units);
            to.y = x.there() && (!kAppend || row.y) ? row.y + h * (w == 0 ? r.ys[0][1] : kAppend ? (long long)a.page * r.D : r.ys[1][1]) : nullptr;
            if constexpr (kAppend) to.also = x.there() && row.also ? row.also + h * r.ys[1][1] : nullptr;
            to.sines = x.t * (2 * turned * kV);
            to.w = w;
        };
        auto work = [&](const Job& job) {
            HdUnits<kV, kUnits, kNeighbours, kWhole> units = all_units;
            units.forget();
            const bool moved = kAppend && job.w == 2;   // as it is
            float x[kUnits][2][kV];
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) hd_floats<Tin, kV>(x[k][i], job.raw.v[k][i]);
            if (kNorm) {
                // unit by unit, and the lanes the farthest first: in one order whether a lane has one unit of a whole row or two
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    float sums[2] = {0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 2; ++i) hd_add_products<kV>(sums, x[k][i], x[k][i]);
                    sum += sums[0] + sums[1];
                }
                // the row times its weights while the lanes meet
                const float* weights = ws + (moved ? 0 : job.w) * (2 * n_units * kV);
                float y[kUnits][2][kV];
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    float wt[2][kV];
                    hd_weight<kV>(wt, weights, units.at[k], n_units);
#pragma unroll
                    for (int i = 0; i < 2; ++i) hd_mul<kV>(y[k][i], x[k][i], wt[i]);
                }
                __syncwarp();
                sum = hd_sum(sum, lanes);
                if (!moved) {
                    const float by = rsqrtf(sum * inv_D + a.eps);
#pragma unroll
                    for (int k = 0; k < kUnits; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) hd_mul<kV>(x[k][i], y[k][i], by);
                }
            }
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                if (!moved && units.turns(k)) hd_turn<kV, kNeighbours>(x[k], cs + job.sines, units.at[k], turned);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!units.has(k, i)) continue;
                    const Out z = hd_rounded<Tout, kV>(x[k][i]);
                    if (job.y) *reinterpret_cast<Out*>(job.y + units.channel(k, i)) = z;
                    if (kAppend && job.also) *reinterpret_cast<Out*>(job.also + units.channel(k, i)) = z;
                }
            }
        };
        // a row is loaded ahead of the one at hand
        const int turns = at.turns();
        Job one, two;
        fetch(one, at);
        for (int turn = 0; turn < turns; turn += 2) {
            at.next();
            fetch(two, at);
            work(one);
            at.next();
            fetch(one, at);
            work(two);
        }
        __syncthreads();   // the tables of the next tile are there, those of this one read
    }
}

// The gradient: CTAs below ctas[0] have rows of query heads, the others of key heads, so that the weight's sums of one tensor stay in registers; tiles of tokens go
// round them.  Each leaves its sums [D] in `partial`, which the next kernel adds up in their order: results repeat to the bit.
template <typename T>
struct alignas(16) HdRowsBack {
    const T *g, *x;
    T* y;
};
template <typename T, int kV, int kUnits, bool kNeighbours, bool kWhole>
__global__ void __launch_bounds__(kHeadThreads, kBackCtas) heads_backward_kernel(const NormRotaryArgs a, int tile_tokens, int log_lanes, int ctas_q, float* partial) {
    using Rows = HdRowsBack<T>;
    using Raw = HdRaw<T, kV, kUnits>;
    constexpr int kWarps = kHeadThreads / 32;
    extern __shared__ float4 sm[];
    const RotaryArgs& r = a.r;
    const int tid = threadIdx.x, lanes = 1 << log_lanes, lane = tid & (lanes - 1), group = tid >> log_lanes, groups = kHeadThreads >> log_lanes;
    const int turned = (r.R / 2 + kV - 1) / kV, n_units = lanes * kUnits, tile_sines = tile_tokens * (2 * turned * kV);
    Rows* all_rows = reinterpret_cast<Rows*>(sm);                          // [2][tile_tokens]
    float* ws = reinterpret_cast<float*>(all_rows + 2 * tile_tokens);      // [n_units * 2 * kV]
    float* all_cs = ws + 2 * n_units * kV;                                 // [2][tile_tokens][2 * turned * kV]
    const int w = (int)blockIdx.x >= ctas_q, cta = (int)blockIdx.x - (w ? ctas_q : 0), n_cta = w ? (int)gridDim.x - ctas_q : ctas_q;
    const int heads = r.heads[w];
    const unsigned n_tok = (unsigned)r.B * (unsigned)r.S, first = hd_share(n_tok, cta, n_cta), last = hd_share(n_tok, cta + 1, n_cta);
    const HdUnits<kV, kUnits, kNeighbours, kWhole> all_units(lane, lanes, r.D, r.R);
    const float inv_D = 1.f / (float)r.D;
    const long long g_head = r.xs[w][1], x_head = a.in_stride[w][1], y_head = r.ys[w][1];
    float dw[kUnits][2][kV];
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
        for (int e = 0; e < kV; ++e) dw[k][0][e] = dw[k][1][e] = 0.f;
    grid_let_next_start();
    grid_wait_for_previous();
    auto tile_of = [&](unsigned t0) { return (int)min((unsigned)tile_tokens, last - t0); };
    auto prepare = [&](unsigned t0, int which) {
        const int here = tile_of(t0);
        const RtPlaces places(t0, r.B, r.S);
        hd_sines<kV, kNeighbours>(all_cs + which * tile_sines, r, places, here, tid);
        for (int t = kHeadThreads - 1 - tid; t < here; t += kHeadThreads) {
            int b, s;
            places.at(t, &b, &s);
            all_rows[which * tile_tokens + t] = Rows{(const T*)r.x[w] + b * r.xs[w][0] + s * r.xs[w][2], (const T*)a.in[w] + b * a.in_stride[w][0] + s * a.in_stride[w][2],
                                                     (T*)r.y[w] + b * r.ys[w][0] + s * r.ys[w][2]};
        }
    };
    prepare(first, 0);
    if (!kWhole) {
        for (int i = tid; i < 2 * n_units * kV; i += kHeadThreads) ws[i] = 0.f;
        __syncthreads();
    }
    hd_weights<kV, kNeighbours>(ws, a.w[w], a.w_bf16, n_units, r.D, r.R, tid);
    __syncthreads();
    int which = 0;
    for (unsigned t0 = first; t0 < last; t0 += tile_tokens, which ^= 1) {
        if (last - t0 > (unsigned)tile_tokens) prepare(t0 + tile_tokens, which ^ 1);
        const Rows* rows = all_rows + which * tile_tokens;
        const float* cs = all_cs + which * tile_sines;
        HdWalk at(group, groups, heads, tile_of(t0));
        struct Job {
            Raw g, x;
            T* y;   // null: nowhere
            int sines;
        };
        auto fetch = [&](Job& to, const HdWalk& from) {
            const Rows row = rows[from.t];
            to.g.load(row.g + from.h * g_head, all_units);
            to.x.load(row.x + from.h * x_head, all_units);
            to.y = from.there() ? row.y + from.h * y_head : nullptr;
            to.sines = from.t * (2 * turned * kV);
        };
        auto work = [&](const Job& job) {
            HdUnits<kV, kUnits, kNeighbours, kWhole> units = all_units;
            units.forget();
            float g[kUnits][2][kV], x[kUnits][2][kV], squares[2] = {0.f, 0.f}, alongs[2] = {0.f, 0.f};
            const float* sines = cs + job.sines;
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                float wt[2][kV];
                hd_weight<kV>(wt, ws, units.at[k], n_units);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    hd_floats<T, kV>(g[k][i], job.g.v[k][i]);
                    hd_floats<T, kV>(x[k][i], job.x.v[k][i]);
                }
                if (units.turns(k)) hd_turn<kV, kNeighbours>(g[k], sines, units.at[k], turned);
                if (!units.has(k, 1))
#pragma unroll
                    for (int e = 0; e < kV; ++e) g[k][1][e] = 0.f;   // (turned by what no pair has)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float h[kV];
                    hd_mul<kV>(h, g[k][i], wt[i]);
                    hd_add_products<kV>(squares, x[k][i], x[k][i]);
                    hd_add_products<kV>(alongs, h, x[k][i]);
                }
            }
            __syncwarp();
            const float square = hd_sum(squares[0] + squares[1], lanes), along = hd_sum(alongs[0] + alongs[1], lanes);
            const float by = rsqrtf(square * inv_D + a.eps), less = -along * inv_D * by * by;
            if (job.y) {
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    float wt[2][kV];
                    hd_weight<kV>(wt, ws, units.at[k], n_units);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!units.has(k, i)) continue;
                        float unit[kV], h[kV];
                        hd_mul<kV>(unit, x[k][i], by);
                        hd_fma<kV>(dw[k][i], g[k][i], unit, dw[k][i]);
                        hd_mul<kV>(h, g[k][i], wt[i]);
                        hd_fma<kV>(h, x[k][i], less, h);
                        hd_mul<kV>(h, h, by);
                        *reinterpret_cast<RtVec<T, kV>*>(job.y + units.channel(k, i)) = hd_rounded<T, kV>(h);
                    }
                }
            }
        };
        const int turns = at.turns();
        Job one, two;
        fetch(one, at);
        for (int turn = 0; turn < turns; turn += 2) {
            at.next();
            fetch(two, at);
            work(one);
            at.next();
            fetch(one, at);
            work(two);
        }
        __syncthreads();   // the tables of the next tile are there, those of this one read
    }
    // the rows of a warp, then the warps
    float* sums = reinterpret_cast<float*>(sm);   // [kWarps][D]; (the barrier at a tile's end: the tables have been read)
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                float y = dw[k][i][e];
                for (int d = lanes; d < 32; d <<= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
                if ((tid & 31) < lanes && all_units.has(k, i)) sums[(tid >> 5) * r.D + all_units.channel(k, i) + e] = y;
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

// Whether all of a row's lanes have two whole chunks of it.
static bool hd_whole(int D, int R, int interleaved, int kV, int n_units) { return n_units * 2 * kV == D && R % (2 * kV) == 0 && (interleaved || R / 2 % kV == 0); }
// Tokens per tile: rows for so many turns of every group of lanes, as the tables of two have room for.  A tile's first rows are loaded behind a barrier: 16384 tokens of 40
// heads of 128 71.2 / 67.7 / 65.1 / 63.6 us with 4 / 8 / 14 / 28 turns of one unit, the gradient of 8192 88.0 / 61.1 / 59.3 / 56.5.  Of two units, whose turns have twice
// the rows, 67.6 / 67.5 / 62.0 / 62.0 with 4 / 7 / 14 / 28, and into a cache, half of the channels turned, 60.4 / 58.8 / 58.2 / 59.6: 14.
static int hd_tile(long long n_tok, long long ctas, int turns, int heads, int groups, size_t token) {
    long long per = (long long)turns * groups / heads;
    const long long fits = 12 * 1024 / (long long)token, share = (n_tok + ctas - 1) / ctas;
    per = per > fits ? fits : per;
    per = per > share ? share : per;
    return per < 1 ? 1 : (int)per;
}

template <typename Tin, typename Tout, int kV, int kUnits, bool kNorm, bool kAppend, bool kWhole>
static cudaError_t launch_heads_units(const NormRotaryArgs& a, int interleaved, int log_lanes, cudaStream_t st) {
    const int turned = (a.r.R / 2 + kV - 1) / kV, heads = a.r.heads[0] + a.r.heads[1] * (kAppend ? 2 : 1), n_units = kUnits << log_lanes;
    const size_t token = (size_t)turned * kV * sizeof(float2) + (kAppend ? 3 * 32 : 2 * 16), weights = kNorm ? (size_t)n_units * kV * 16 : 0;
    const long long n_tok = (long long)a.r.B * a.r.S, resident = (long long)hd_ctas_per_sm(kUnits) * sm_count(), ctas = n_tok < resident ? n_tok : resident;
    const int per = hd_tile(n_tok, ctas, kUnits == 1 ? 28 : 14, heads, kHeadThreads >> log_lanes, token);
    LaunchScope ls(kAppend ? K_CACHE_APPEND_ROTARY : K_NORM_ROTARY, st);
    auto go = [&](auto kernel) { return launch_overlapped(kernel, (unsigned)ctas, kHeadThreads, weights + 2 * per * token, st, a, per, log_lanes); };
    return interleaved ? go(heads_kernel<Tin, Tout, kV, kUnits, true, kNorm, kAppend, kWhole>) : go(heads_kernel<Tin, Tout, kV, kUnits, false, kNorm, kAppend, kWhole>);
}
template <typename Tin, typename Tout, int kV, bool kNorm, bool kAppend>
static cudaError_t launch_heads(const NormRotaryArgs& a, int interleaved, cudaStream_t st) {
    constexpr int kUnits = hd_units(kV);
    int log_lanes;
    const int units = hd_units_of_row(a.r.D, a.r.R, kV);
    // Whole rows: two units to a lane, so that what a row costs beside its values is shared by more of them (TB/s with one unit and two, 20 heads: floats of 128, 64
    // channels turned, 5.58 and 5.66, of 64 and 64, where it is otherwise, 5.45 and 5.32; bf16 of 256 and 128 5.24 and 5.40).  But bf16 norms of rows of four units, where
    // a warp then has 16 rows, and of few heads that turn all channels, where the CTAs make sines for longer, have three CTAs per SM, and one unit (64 and 64 4.59 and 4.06,
    // 64 and 16 5.03 and 4.92, 128 and 128 4.91 and 4.59, 256 and 256 5.01 and 4.82).  Around the border of 32 heads, all of 128 channels turned, the two are within 2 %:
    // with one unit and two 24 heads 67.3 and 70.9 us, 28 66.0 and 65.2, 32 65.0 and 65.2, 36 64.3 and 65.5, 40 63.6 and 62.2, 56 62.8 and 60.5.
    if constexpr (kUnits == 1) {
        if constexpr (sizeof(Tin) == 2 && kNorm && !kAppend) {
            hd_lanes(units, 1, &log_lanes);
            if ((units <= 4 || (a.r.heads[0] + a.r.heads[1]) * a.r.D < 32LL * a.r.R) && hd_whole(a.r.D, a.r.R, interleaved, kV, 1 << log_lanes))
                return launch_heads_units<Tin, Tout, kV, 1, kNorm, kAppend, true>(a, interleaved, log_lanes, st);
        }
        hd_lanes(units, 2, &log_lanes);
        if (hd_whole(a.r.D, a.r.R, interleaved, kV, 2 << log_lanes)) return launch_heads_units<Tin, Tout, kV, 2, kNorm, kAppend, true>(a, interleaved, log_lanes, st);
    }
    hd_lanes(units, kUnits, &log_lanes);
    return launch_heads_units<Tin, Tout, kV, kUnits, kNorm, kAppend, false>(a, interleaved, log_lanes, st);
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
        out.add(a.pool[i], nullptr, nullptr, 0, 2);   // keys' and values', with and without queries
        if (!a.r.heads[i]) continue;
        in.add(a.r.x[i], a.r.xs[i], m, 3, size);
        if (a.r.y[i]) out.add(a.r.y[i], a.r.ys[i], m, 3, 2);
    }
    in.add(a.v, a.v_stride, n, 2, size);
    const int from = in.aligned(16), to = out.aligned(16) * (size / 2), aligned = from < to ? from : to;
    auto go = [&](auto type) {
        using T = decltype(type);
        return a.w[0] || a.w[1] ? launch_heads_width<T, __nv_bfloat16, true, true>(a, interleaved, aligned, st) : launch_heads_width<T, __nv_bfloat16, false, true>(a, interleaved, aligned, st);
    };
    return bf16 ? go(__nv_bfloat16{}) : go(float{});
}

// CTAs of the gradient: what the SMs hold at once, shared out by what the rows of the two tensors cost; fewer where there are not tokens for them.  A token's sines, where
// all channels turn, take as long as five rows: 8192 tokens of 32 and 8 heads 67.2 / 63.7 / 59.0 / 56.5 / 58.2 us if that is taken for 0 / 1 / 3 / 5 / 7 rows.
static void hd_ctas(const NormRotaryArgs& a, int (&ctas)[2]) {
    const long long n_tok = (long long)a.r.B * a.r.S, all = (long long)sm_count() * kBackCtas, sines = 5LL * a.r.R;
    const long long cost[2] = {(long long)a.r.heads[0] * a.r.D + sines, a.r.heads[1] ? (long long)a.r.heads[1] * a.r.D + sines : 0};
    long long q = (all * cost[0] + (cost[0] + cost[1]) / 2) / (cost[0] + cost[1]);
    if (q >= all && cost[1]) q = all - 1;
    if (q < 1) q = 1;
    const long long n[2] = {q, cost[1] ? all - q : 0};
    for (int i = 0; i < 2; ++i) ctas[i] = (int)(n[i] < n_tok ? n[i] : n_tok);
}
size_t norm_rotary_backward_workspace(int D) { return align256((size_t)sm_count() * kBackCtas * D * sizeof(float)); }

template <typename T, int kV>
static cudaError_t launch_heads_back(const NormRotaryArgs& a, int interleaved, float* partial, const int (&ctas)[2], cudaStream_t st) {
    constexpr int kUnits = hd_units(kV);
    int log_lanes;
    hd_lanes(hd_units_of_row(a.r.D, a.r.R, kV), kUnits, &log_lanes);
    const int turned = (a.r.R / 2 + kV - 1) / kV, n_units = kUnits << log_lanes, most = a.r.heads[0] > a.r.heads[1] ? a.r.heads[0] : a.r.heads[1];
    const size_t token = (size_t)turned * kV * sizeof(float2) + sizeof(HdRowsBack<T>), sums = (size_t)kHeadThreads / 32 * a.r.D * sizeof(float);
    const int per = hd_tile((long long)a.r.B * a.r.S, ctas[0], 28, most, kHeadThreads >> log_lanes, token);
    const size_t tables = 2 * per * token + (size_t)n_units * kV * 8, smem = tables > sums ? tables : sums;
    LaunchScope ls(K_NORM_ROTARY_BWD, st);
    auto go = [&](auto kernel) { return launch_overlapped(kernel, (unsigned)(ctas[0] + ctas[1]), kHeadThreads, smem, st, a, per, log_lanes, ctas[0], partial); };
    if constexpr (kUnits == 1) {
        if (hd_whole(a.r.D, a.r.R, interleaved, kV, n_units)) return interleaved ? go(heads_backward_kernel<T, kV, 1, true, true>) : go(heads_backward_kernel<T, kV, 1, false, true>);
    }
    return interleaved ? go(heads_backward_kernel<T, kV, kUnits, true, false>) : go(heads_backward_kernel<T, kV, kUnits, false, false>);
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
