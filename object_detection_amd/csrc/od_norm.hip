// Group norm with an activation on channels-last maps, forward and backward: the [GroupNorm, ReLU] pair between the
// convolutions of the head towers (reference object_detection/retinanet/retinanet_model.py:47-52 passes
// partial(nn.GroupNorm, 32); torchvision's FCOS head has the same pair).
//
//   x, y: [batch, pixels, channels], channels contiguous;  a group is channels/groups neighbouring channels
//   mean, rstd over the pixels * channels/groups values of one (image, group);  xhat = (x - mean) * rstd
//   u = xhat * gamma + beta;  y = act(u), act = identity, max(u, 0) or u * sigmoid(u)
//   backward, du = dy * act'(u):  dbeta_c = sum du,  dgamma_c = sum du * xhat  (over images and pixels),
//   dx = rstd * (gamma du - mean_g(gamma du) - xhat * mean_g(gamma du * xhat))
//
// Both directions are HBM streams; the arithmetic is fp32 for every element type and a 16-bit result is rounded once.
// A thread owns one 16-byte column vector (8 or 4 channels) and walks down the pixels, so a row of the map is read in
// whole cache lines and the per-channel coefficients stay in registers.
//
// Statistics: a thread sums x - k and (x - k)^2 with k its own first value of the channel, which bounds what the
// subtraction of the two sums can lose by the number of its pixels whatever the mean of the map is: four pixels in 32 bits,
// the fours in 64.  Everything above a thread is merged in 64 bits as (count, mean, M2) in two passes, M2 = sum M2_i + n_i
// (mean_i - mean)^2.  Fixed order, no atomics.  Mean and 1/std stay 64-bit: a rectifier's gradient is all or nothing, and
// since a 16-bit map holds few different values, hundreds of pixels of a channel lie on its corner together; where fp32
// cannot tell the side, 64 bits decide.  The sums in 64 bits cost the statistics of 16 x 64 x 64 x 256 bf16 12.0 us instead of
// 11.2 and those of 16 x 256 x 256 x 256 nothing; with sums in 32 bits one in twenty of the large maps had a channel whose
// corner fell to the other side than by 64 bits throughout, with them one in five hundred.
#include "od_common.h"
#include "../../include/od_boxes.h"
#include "od_elem.h"

#pragma clang fp contract(fast)

namespace {

using namespace od;

constexpr int NT = 256;                 // threads per workgroup
constexpr int MAX_CHUNKS = 256;         // pixel chunks per image of the two-pass form

struct NormShape {
    long long batch, pixels;            // images, pixels per image
    int channels, groups, per_group;    // per_group = channels / groups
    int chunks;                         // workgroups per image (two-pass form)
    long long chunk_pixels;
    float eps;
};

// weight or bias of channel c in the parameters' own type; a missing table is the constant `none`
__device__ __forceinline__ float param(const void* p, int dtype, int c, float none) {
    if (!p) return none;
    if (dtype == OD_DTYPE_F32) return ((const float*)p)[c];
    if (dtype == OD_DTYPE_F16) return (float)((const _Float16*)p)[c];
    return Elem<bf16_t>::to_float(((const bf16_t*)p)[c]);
}
// the same of channels c .. c + VEC, with all loads in flight together
template <int VEC>
__device__ __forceinline__ void params(const void* p, int dtype, int c, float none, float (&out)[VEC]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = none;
    } else if (dtype == OD_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = ((const float*)p)[c + i];
    } else if (dtype == OD_DTYPE_F16) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = (float)((const _Float16*)p)[c + i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = Elem<bf16_t>::to_float(((const bf16_t*)p)[c + i]);
    }
}
// (mean, 1/std) of the groups of channels c .. c + VEC
template <int VEC>
__device__ __forceinline__ void group_stats(const double2* stats, int per_group, int c, double2 (&out)[VEC]) {
    if (per_group % VEC == 0 && c % VEC == 0) {                     // one group
        const double2 v = stats[c / per_group];
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = v;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = stats[(c + i) / per_group];
    }
}
__device__ __forceinline__ void store_param(void* p, int dtype, int c, float v) {
    if (dtype == OD_DTYPE_F32) ((float*)p)[c] = v;
    else if (dtype == OD_DTYPE_F16) ((_Float16*)p)[c] = (_Float16)v;
    else ((bf16_t*)p)[c] = Elem<bf16_t>::from_float(v);
}

// 1 / (1 + exp(-u)) with the hardware exponential and reciprocal: relative error below 1e-6 for |u| < 16
template <int ACT>
__device__ __forceinline__ float act_value(float u) {
    if (ACT == OD_ACT_RELU) return u < 0.0f ? 0.0f : u;              // NaN stays NaN
    if (ACT == OD_ACT_SILU) return u * __builtin_amdgcn_rcpf(1.0f + __expf(-u));
    return u;
}
// dy * act'(u)
template <int ACT>
__device__ __forceinline__ float act_grad(float u, float dy) {
    if (ACT == OD_ACT_RELU) return u <= 0.0f ? 0.0f : dy;
    if (ACT == OD_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-u));
        return dy * s * (1.0f + u * (1.0f - s));
    }
    return dy;
}

// Threads of a workgroup laid over a window of `cols` column vectors: `width` of them side by side (all of them, or NT
// at a time), NT / width pixel rows below each other; threads left over idle.
struct Lay {
    int width, rows, tx, ty;
    bool active;
    __device__ __forceinline__ explicit Lay(int cols) {
        width = cols < NT ? cols : NT;
        rows = NT / width;
        tx = threadIdx.x % width;
        ty = threadIdx.x / width;
        active = ty < rows;
    }
};

// pixels that row ty of `rows` takes out of n < 2^31: ty, ty + rows, ...
__device__ __forceinline__ int taken(long long n, int ty, int rows) {
    const uint32_t m = (uint32_t)n, r = (uint32_t)rows;
    return (int)(m / r + ((uint32_t)ty < m % r ? 1 : 0));
}

// A value per channel out of the workgroup's rows: sum over r of f(r, c) for the `here` channels c of a window, spread over
// all threads; every thread of a channel gets the sum.  scratch: NT doubles.
struct Gather {
    int here, rows, slices, c, slice;
    __device__ __forceinline__ Gather(int channels, int nrows) {
        here = channels;
        rows = nrows;
        slices = here < NT ? NT / here : 1;
        slices = slices < rows ? slices : rows;
        c = here < NT ? threadIdx.x % here : threadIdx.x;
        slice = here < NT ? threadIdx.x / here : 0;
    }
    template <typename F>
    __device__ __forceinline__ double sum(double* scratch, F f) const {
        double v = 0.0;
        if (slice < slices)
            for (int r = slice; r < rows; r += slices) v += f(r);
        __syncthreads();
        scratch[threadIdx.x] = v;
        __syncthreads();
        v = 0.0;
        if (slice < slices)
            for (int k = 0; k < slices; ++k) v += scratch[k * here + c];
        return v;
    }
};

// Statistics of channels [c0, c0 + nc) over `n` pixels at src (row stride `channels`), by the whole workgroup.
// Leaves (mean, M2) of each channel in ch[0 .. nc).  red: 3 * NT * VEC floats, scratch: NT doubles.
template <typename T, int VEC>
__device__ __forceinline__ void channel_stats(const T* src, int channels, int c0, int nc, long long n, double2* ch,
                                              double* scratch, float* red) {
    const int cols = nc / VEC;
    const Lay lay(cols);
    for (int base = 0; base < cols; base += lay.width) {
        const int col = base + lay.tx;
        const bool on = lay.active && col < cols;
        float k[VEC];
        double s1[VEC], s2[VEC];                        // sums of x - k and its square
#pragma unroll
        for (int i = 0; i < VEC; ++i) k[i] = 0.0f, s1[i] = s2[i] = 0.0;
        const int mine = on ? taken(n, lay.ty, lay.rows) : 0;
        if (mine > 0) {
            const T* p = src + (long long)lay.ty * channels + c0 + col * VEC;
            const long long step = (long long)lay.rows * channels;
            load_vec<T, VEC>(p, k);
            p += step;
            int j = 1;
            for (; j + 4 <= mine; j += 4) {             // four loads in flight
                float v[4][VEC];
#pragma unroll
                for (int q = 0; q < 4; ++q) load_vec<T, VEC>(p + q * step, v[q]);
                p += 4 * step;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float d = v[0][i] - k[i], a = d, b = d * d;
#pragma unroll
                    for (int q = 1; q < 4; ++q) {
                        d = v[q][i] - k[i];
                        a += d;
                        b = fmaf(d, d, b);
                    }
                    s1[i] += (double)a;
                    s2[i] += (double)b;
                }
            }
            for (; j < mine; ++j, p += step) {
                float v[VEC];
                load_vec<T, VEC>(p, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = v[i] - k[i];
                    s1[i] += (double)d;
                    s2[i] += (double)(d * d);
                }
            }
        }
        __syncthreads();                                // red may still be read for the previous columns
        if (on) {
            const double inv = mine > 0 ? 1.0 / (double)mine : 0.0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {             // the thread's mean in two parts, and its M2
                const int at = (lay.ty * lay.width + lay.tx) * VEC + i;
                const double mean = (double)k[i] + s1[i] * inv;
                red[at] = (float)mean;
                red[NT * VEC + at] = (float)(mean - (double)(float)mean);
                red[2 * NT * VEC + at] = (float)(s2[i] - s1[i] * s1[i] * inv);
            }
        }
        __syncthreads();
        const int here = min(lay.width, cols - base) * VEC;              // channels of this window
        for (int first = 0; first < here; first += NT) {
            const Gather all(min(NT, here - first), lay.rows);
            const int c = first + all.c;
            const uint32_t each = (uint32_t)n / lay.rows, more = (uint32_t)n % lay.rows;
            auto count = [&](int r) { return (double)(each + ((uint32_t)r < more ? 1 : 0)); };
            auto at = [&](int r, int what) { return (double)red[what * NT * VEC + r * lay.width * VEC + c]; };
            const double mean = all.sum(scratch, [&](int r) { return count(r) * (at(r, 0) + at(r, 1)); }) / (double)n;
            double m2 = all.sum(scratch, [&](int r) {
                const double d = at(r, 0) + at(r, 1) - mean;
                return count(r) > 0.0 ? at(r, 2) + count(r) * d * d : 0.0;
            });
            m2 = m2 < 0.0 ? 0.0 : m2;                                   // NaN stays NaN
            if (all.slice == 0 && all.c < all.here) ch[base * VEC + c] = make_double2(mean, m2);
        }
    }
    __syncthreads();
}

// lanes that share one group of `per` values: the power of two not below it, at most a wave
__device__ __forceinline__ int lanes_of(int per) {
    int l = 1;
    while (l < per && l < 64) l <<= 1;
    return l;
}
template <typename F>
__device__ __forceinline__ F lane_sum(F v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// (mean, M2) of group g over n pixels out of its channels' values ch[g * per ..); f(g, mean, M2) once per group
template <typename F>
__device__ __forceinline__ void merge_groups(const double2* ch, int groups, int per, long long n, F f) {
    const int lanes = lanes_of(per);
    const int at = threadIdx.x % lanes;
    for (int g0 = 0; g0 < groups; g0 += NT / lanes) {
        const int g = g0 + threadIdx.x / lanes;
        double mean = 0.0, m2 = 0.0;
        if (g < groups)
            for (int c = at; c < per; c += lanes) mean += ch[g * per + c].x;
        mean = lane_sum(mean, lanes) / (double)per;
        if (g < groups)
            for (int c = at; c < per; c += lanes) {
                const double d = ch[g * per + c].x - mean;
                m2 += ch[g * per + c].y + (double)n * d * d;
            }
        m2 = lane_sum(m2, lanes);
        if (g < groups && at == 0) f(g, mean, m2);
    }
}

// ---- two-pass form ------------------------------------------------------------------------------------------
// part[(image * chunks + chunk) * groups + g] = (mean, M2) of the chunk
template <typename T, int VEC>
__global__ __launch_bounds__(NT) void norm_stats_kernel(NormShape s, const T* __restrict__ x, double2* __restrict__ part) {
    extern __shared__ double smem[];
    double2* ch = reinterpret_cast<double2*>(smem);
    double* scratch = reinterpret_cast<double*>(ch + s.channels);
    float* red = reinterpret_cast<float*>(scratch + NT);
    const long long b = blockIdx.x / s.chunks;
    const int chunk = blockIdx.x % s.chunks;
    const long long p0 = chunk * s.chunk_pixels;
    const long long n = min(s.chunk_pixels, s.pixels - p0);
    channel_stats<T, VEC>(x + (b * s.pixels + p0) * s.channels, s.channels, 0, s.channels, n, ch, scratch, red);
    double2* out = part + (long long)blockIdx.x * s.groups;
    merge_groups(ch, s.groups, s.per_group, n, [&](int g, double mean, double m2) { out[g] = make_double2(mean, m2); });
}

// y of one window of channels and pixels; stats: (mean, 1/std) per group, counted from the window's first channel
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void apply_window(const NormShape& s, const T* src, T* dst, int c0, int nc, long long n,
                                             const double2* stats, const void* weight, const void* bias, int pdtype) {
    const int cols = nc / VEC;
    const Lay lay(cols);
    for (int base = 0; base < cols; base += lay.width) {
        const int col = base + lay.tx;
        if (!lay.active || col >= cols) continue;
        float mean[VEC], a[VEC], beta[VEC];
        double2 st[VEC];
        group_stats<VEC>(stats, s.per_group, col * VEC, st);
        params<VEC>(weight, pdtype, c0 + col * VEC, 1.0f, a);
        params<VEC>(bias, pdtype, c0 + col * VEC, 0.0f, beta);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            mean[i] = (float)st[i].x;
            a[i] = (float)(st[i].y * (double)a[i]);
        }
        const int mine = taken(n, lay.ty, lay.rows);
        const long long off = (long long)lay.ty * s.channels + c0 + col * VEC;
        const long long step = (long long)lay.rows * s.channels;
        const T* p = src + off;
        T* q = dst + off;
        int j = 0;
        for (; j + 4 <= mine; j += 4) {
            float v[4][VEC];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_vec<T, VEC>(p + u * step, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = act_value<ACT>(fmaf(v[u][i] - mean[i], a[i], beta[i]));
                store_vec<T, VEC>(q + u * step, v[u]);
            }
            p += 4 * step;
            q += 4 * step;
        }
        for (; j < mine; ++j, p += step, q += step) {
            float v[VEC];
            load_vec<T, VEC>(p, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = act_value<ACT>(fmaf(v[i] - mean[i], a[i], beta[i]));
            store_vec<T, VEC>(q, v);
        }
    }
}

// The chunks of one image joined: a workgroup takes 8 groups, 32 slices of the chunks each.
__global__ __launch_bounds__(NT) void norm_join_kernel(NormShape s, const double2* __restrict__ part,
                                                       double2* __restrict__ stats) {
    __shared__ double red[NT];
    const int blocks = (s.groups + 7) / 8;
    const long long b = blockIdx.x / blocks;
    const int g = (int)(blockIdx.x % blocks) * 8 + (threadIdx.x & 7);
    const bool on = g < s.groups;
    const double2* mine = part + b * s.chunks * s.groups;
    auto count = [&](int k) { return (double)min(s.chunk_pixels, s.pixels - k * s.chunk_pixels); };
    auto joined = [&](double v) {
        __syncthreads();
        red[threadIdx.x] = v;
        __syncthreads();
        v = 0.0;
        for (int r = 0; r < NT / 8; ++r) v += red[r * 8 + (threadIdx.x & 7)];
        return v;
    };
    double mean = 0.0;
    if (on)
        for (int k = threadIdx.x >> 3; k < s.chunks; k += NT / 8) mean += count(k) * mine[(long long)k * s.groups + g].x;
    mean = joined(mean) / (double)s.pixels;
    double m2 = 0.0;
    if (on)
        for (int k = threadIdx.x >> 3; k < s.chunks; k += NT / 8) {
            const double2 v = mine[(long long)k * s.groups + g];
            const double d = v.x - mean;
            m2 += v.y + count(k) * s.per_group * d * d;
        }
    m2 = joined(m2);
    if (on && threadIdx.x < 8)
        stats[b * s.groups + g] = make_double2(mean, 1.0 / sqrt(m2 / ((double)s.pixels * s.per_group) + (double)s.eps));
}

// part: chunks to be joined here (by every workgroup of the image for itself), or null: stats are there
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(NT) void norm_apply_kernel(NormShape s, const T* __restrict__ x, T* __restrict__ y,
                                                        const void* __restrict__ weight, const void* __restrict__ bias,
                                                        int pdtype, const double2* __restrict__ part, double2* stats) {
    extern __shared__ double smem[];
    const long long b = blockIdx.x / s.chunks;
    const int chunk = blockIdx.x % s.chunks;
    const long long p0 = chunk * s.chunk_pixels;
    const long long first = (b * s.pixels + p0) * s.channels;
    stats += b * s.groups;
    const double2* mine = stats;
    if (part) {
        double2* joined = reinterpret_cast<double2*>(smem + NT);
        part += b * s.chunks * s.groups;
        auto count = [&](int k) { return (double)min(s.chunk_pixels, s.pixels - k * s.chunk_pixels); };
        for (int g0 = 0; g0 < s.groups; g0 += NT) {
            const Gather all(min(NT, s.groups - g0), s.chunks);
            const int g = g0 + all.c;
            const double mean = all.sum(smem, [&](int k) { return count(k) * part[(long long)k * s.groups + g].x; }) /
                                (double)s.pixels;
            const double m2 = all.sum(smem, [&](int k) {
                const double2 v = part[(long long)k * s.groups + g];
                return v.y + count(k) * s.per_group * (v.x - mean) * (v.x - mean);
            });
            if (all.slice == 0 && all.c < all.here) {
                const double2 v = make_double2(mean, 1.0 / sqrt(m2 / ((double)s.pixels * s.per_group) + (double)s.eps));
                joined[g] = v;
                if (chunk == 0) stats[g] = v;
            }
        }
        __syncthreads();
        mine = joined;
    }
    apply_window<T, VEC, ACT>(s, x + first, y + first, 0, s.channels, min(s.chunk_pixels, s.pixels - p0), mine, weight, bias,
                              pdtype);
}

// ---- one-launch form: a workgroup takes `slab` channels (whole groups) of one image over all its pixels -----------
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(NT) void norm_small_kernel(NormShape s, int slab, const T* __restrict__ x, T* __restrict__ y,
                                                        const void* __restrict__ weight, const void* __restrict__ bias,
                                                        int pdtype, double2* __restrict__ stats_out) {
    extern __shared__ double smem[];
    double2* ch = reinterpret_cast<double2*>(smem);
    double2* stats = ch + slab;
    double* scratch = reinterpret_cast<double*>(stats + slab / s.per_group);
    float* red = reinterpret_cast<float*>(scratch + NT);
    const int slabs = (s.channels + slab - 1) / slab;
    const long long b = blockIdx.x / slabs;
    const int c0 = (int)(blockIdx.x % slabs) * slab;
    const int nc = min(slab, s.channels - c0);
    const long long first = b * s.pixels * s.channels;
    channel_stats<T, VEC>(x + first, s.channels, c0, nc, s.pixels, ch, scratch, red);
    const long long g0 = b * s.groups + c0 / s.per_group;
    merge_groups(ch, nc / s.per_group, s.per_group, s.pixels, [&](int g, double mean, double m2) {
        const double2 v = make_double2(mean, 1.0 / sqrt(m2 / ((double)s.pixels * s.per_group) + (double)s.eps));
        stats[g] = v;
        stats_out[g0 + g] = v;
    });
    __syncthreads();
    apply_window<T, VEC, ACT>(s, x + first, y + first, c0, nc, s.pixels, stats, weight, bias, pdtype);
}

// ---- backward ---------------------------------------------------------------------------------------------------
// What a thread holds of its VEC channels, and du = dy act'(u) of a vector of them.
template <int VEC, int ACT>
struct Channels {
    float mean[VEC], rstd[VEC], a[VEC], beta[VEC], corner[VEC];     // a = gamma / std
    const double2* stats;
    const void *weight, *bias;
    int pdtype, per_group, c0;
    __device__ __forceinline__ void init(const double2* st, const void* w, const void* b, int dtype, int per, int first) {
        stats = st; weight = w; bias = b; pdtype = dtype; per_group = per; c0 = first;
        double2 v[VEC];
        group_stats<VEC>(stats, per_group, c0, v);
        params<VEC>(weight, pdtype, c0, 1.0f, a);
        params<VEC>(bias, pdtype, c0, 0.0f, beta);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            mean[i] = (float)v[i].x;
            rstd[i] = (float)v[i].y;
            a[i] = (float)(v[i].y * (double)a[i]);
            // u is off by a few half steps of its terms, |x - mean| |a| = |beta| where it is zero, and by what the mean lost.
            // Zero: fp32 has the side exactly, and nothing is near.  Else a fresh norm (gamma and beta zero) or a map of one
            // value would ask at every pixel: 16 x 128 x 128 x 256 bf16 634 us backward instead of 139.
            corner[i] = 5.0e-7f * fabsf(beta[i]) + 2.0f * fabsf((float)(v[i].x - (double)mean[i]) * a[i]);
        }
    }
    // d = x - mean and du, from x and dy; whether some du has to be decided again, see decide()
    __device__ __forceinline__ bool run(const float* x, const float* dy, float* d, float* du) const {
        bool near = false;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            d[i] = x[i] - mean[i];
            const float u = fmaf(d[i], a[i], beta[i]);
            du[i] = act_grad<ACT>(u, dy[i]);
            if (ACT == OD_ACT_RELU) near = near || fabsf(u) < corner[i];
        }
        return near;
    }
    // du of the elements on which fp32 cannot decide, in 64 bits.  Rare (a channel in thousands has a value there): the
    // loops run without it and go over their pixels once more where run() asked for it.
    __device__ __forceinline__ void decide(const float* x, const float* dy, const float* d, float* du) const {
        int c = c0;
        asm volatile("" : "+v"(c));                                 // keeps what is loaded here out of the loops around
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (fabsf(fmaf(d[i], a[i], beta[i])) < corner[i]) {
                const double2 v = stats[(c + i) / per_group];
                const double u = ((double)x[i] - v.x) * v.y * (double)param(weight, pdtype, c + i, 1.0f)
                                 + (double)param(bias, pdtype, c + i, 0.0f);
                du[i] = u <= 0.0 ? 0.0f : dy[i];
            }
        }
    }
};

// Per-channel sums (du, du * xhat) of `n` pixels of channels [c0, c0 + nc); into out[0 .. nc).  red: 2 * NT * VEC floats,
// scratch: NT doubles.  A thread's own sums are fp32: off by 1e-6 of a gradient that is the same everywhere for 16 x 256 x 256
// x 256, where a thread adds 64 pixels, by 6e-6 at 1024 pixels (one map of 2048 x 2048 x 64), 5e-5 at 8192.  64 bits every 64
// pixels leave 9e-7 throughout and cost 6 % (a step of 16 x 256 x 256 x 256 bf16 871 us instead of 820).
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void channel_sums(const NormShape& s, const T* x, const T* dy, int c0, int nc, long long n,
                                             const double2* stats_b, const void* weight, const void* bias, int pdtype,
                                             float2* out, double* scratch, float* red) {
    const int cols = nc / VEC;
    const Lay lay(cols);
    for (int base = 0; base < cols; base += lay.width) {
        const int col = base + lay.tx;
        const bool on = lay.active && col < cols;
        float s1[VEC], s2[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = 0.0f;
        if (on) {
            Channels<VEC, ACT> ch;
            ch.init(stats_b, weight, bias, pdtype, s.per_group, c0 + col * VEC);
            const int mine = taken(n, lay.ty, lay.rows);
            const long long step = (long long)lay.rows * s.channels;
            long long off = (long long)lay.ty * s.channels + c0 + col * VEC;
            bool again = false;
            auto add = [&](const float* v, const float* g) {
                float d[VEC], du[VEC];
                again = ch.run(v, g, d, du) || again;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    s1[i] += du[i];
                    s2[i] = fmaf(du[i], d[i], s2[i]);               // times 1/std at the end
                }
            };
            int j = 0;
            for (; j + 2 <= mine; j += 2, off += 2 * step) {
                float v0[VEC], v1[VEC], g0[VEC], g1[VEC];
                load_vec<T, VEC>(x + off, v0);
                load_vec<T, VEC>(dy + off, g0);
                load_vec<T, VEC>(x + off + step, v1);
                load_vec<T, VEC>(dy + off + step, g1);
                add(v0, g0);
                add(v1, g1);
            }
            if (j < mine) {
                float v0[VEC], g0[VEC];
                load_vec<T, VEC>(x + off, v0);
                load_vec<T, VEC>(dy + off, g0);
                add(v0, g0);
            }
            if (ACT == OD_ACT_RELU && again) {
                off = (long long)lay.ty * s.channels + c0 + col * VEC;
#pragma unroll 1
                for (j = 0; j < mine; ++j, off += step) {
                    float v[VEC], g[VEC], d[VEC], du[VEC], right[VEC];
                    load_vec<T, VEC>(x + off, v);
                    load_vec<T, VEC>(dy + off, g);
                    if (!ch.run(v, g, d, du)) continue;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) right[i] = du[i];
                    ch.decide(v, g, d, right);
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (right[i] != du[i]) {
                            s1[i] += right[i] - du[i];
                            s2[i] = fmaf(right[i] - du[i], d[i], s2[i]);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) s2[i] *= ch.rstd[i];
        }
        __syncthreads();
        if (on)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                red[(lay.ty * lay.width + lay.tx) * VEC + i] = s1[i];
                red[NT * VEC + (lay.ty * lay.width + lay.tx) * VEC + i] = s2[i];
            }
        __syncthreads();
        const int here = min(lay.width, cols - base) * VEC;
        for (int first = 0; first < here; first += NT) {
            const Gather all(min(NT, here - first), lay.rows);
            const int c = first + all.c;
            const double a = all.sum(scratch, [&](int r) { return (double)red[r * lay.width * VEC + c]; });
            const double q = all.sum(scratch, [&](int r) { return (double)red[NT * VEC + r * lay.width * VEC + c]; });
            if (all.slice == 0 && all.c < all.here) out[base * VEC + c] = make_float2((float)a, (float)q);
        }
    }
}

template <typename T, int VEC, int ACT>
__device__ __forceinline__ void grad_window(const NormShape& s, const T* x, const T* dy, T* dx, int c0, int nc, long long n,
                                            const double2* stats_b, const float2* s_avg, int g_first, const void* weight,
                                            const void* bias, int pdtype) {
    const int cols = nc / VEC;
    const Lay lay(cols);
    for (int base = 0; base < cols; base += lay.width) {
        const int col = base + lay.tx;
        if (!lay.active || col >= cols) continue;
        Channels<VEC, ACT> ch;
        ch.init(stats_b, weight, bias, pdtype, s.per_group, c0 + col * VEC);
        float shift[VEC], slope[VEC];                   // dx = a du - shift - d slope
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float2 avg = s_avg[(c0 + col * VEC + i) / s.per_group - g_first];
            shift[i] = ch.rstd[i] * avg.x;
            slope[i] = ch.rstd[i] * ch.rstd[i] * avg.y;
        }
        const int mine = taken(n, lay.ty, lay.rows);
        const long long step = (long long)lay.rows * s.channels;
        long long off = (long long)lay.ty * s.channels + c0 + col * VEC;
        bool again = false;
        auto grad = [&](float* v, const float* g) {
            float d[VEC], du[VEC];
            again = ch.run(v, g, d, du) || again;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = fmaf(ch.a[i], du[i], -shift[i]) - d[i] * slope[i];
        };
        int j = 0;
        for (; j + 2 <= mine; j += 2, off += 2 * step) {
            float v0[VEC], v1[VEC], g0[VEC], g1[VEC];
            load_vec<T, VEC>(x + off, v0);
            load_vec<T, VEC>(dy + off, g0);
            load_vec<T, VEC>(x + off + step, v1);
            load_vec<T, VEC>(dy + off + step, g1);
            grad(v0, g0);
            store_vec<T, VEC>(dx + off, v0);
            grad(v1, g1);
            store_vec<T, VEC>(dx + off + step, v1);
        }
        if (j < mine) {
            float v0[VEC], g0[VEC];
            load_vec<T, VEC>(x + off, v0);
            load_vec<T, VEC>(dy + off, g0);
            grad(v0, g0);
            store_vec<T, VEC>(dx + off, v0);
        }
        if (ACT == OD_ACT_RELU && again) {
            off = (long long)lay.ty * s.channels + c0 + col * VEC;
#pragma unroll 1
            for (j = 0; j < mine; ++j, off += step) {
                float v[VEC], g[VEC], d[VEC], du[VEC];
                load_vec<T, VEC>(x + off, v);
                load_vec<T, VEC>(dy + off, g);
                if (!ch.run(v, g, d, du)) continue;
                ch.decide(v, g, d, du);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = fmaf(ch.a[i], du[i], -shift[i]) - d[i] * slope[i];
                store_vec<T, VEC>(dx + off, v);
            }
        }
    }
}

// group means of (gamma du, gamma du xhat) from the channel sums ch[0 .. groups * per)
template <typename F>
__device__ __forceinline__ void group_averages(const float2* ch, int groups, int per, int c0, double count,
                                               const void* weight, int pdtype, F f) {
    const int lanes = lanes_of(per);
    const int at = threadIdx.x % lanes;
    const float inv = (float)(1.0 / count);
    for (int g0 = 0; g0 < groups; g0 += NT / lanes) {
        const int g = g0 + threadIdx.x / lanes;
        float a = 0.0f, q = 0.0f;
        if (g < groups)
            for (int c = at; c < per; c += lanes) {
                const float w = param(weight, pdtype, c0 + g * per + c, 1.0f);
                a += w * ch[g * per + c].x;
                q += w * ch[g * per + c].y;
            }
        a = lane_sum(a, lanes);
        q = lane_sum(q, lanes);
        if (g < groups && at == 0) f(g, a * inv, q * inv);
    }
}

// part[(image * chunks + chunk) * channels + c] = channel sums of the chunk
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(NT) void norm_bwd_sums_kernel(NormShape s, const T* __restrict__ x, const T* __restrict__ dy,
                                                           const double2* __restrict__ stats,
                                                           const void* __restrict__ weight, const void* __restrict__ bias,
                                                           int pdtype, float2* __restrict__ part) {
    extern __shared__ double smem[];
    const long long b = blockIdx.x / s.chunks;
    const int chunk = blockIdx.x % s.chunks;
    const long long p0 = chunk * s.chunk_pixels;
    const long long first = (b * s.pixels + p0) * s.channels;
    channel_sums<T, VEC, ACT>(s, x + first, dy + first, 0, s.channels, min(s.chunk_pixels, s.pixels - p0),
                              stats + b * s.groups, weight, bias, pdtype, part + (long long)blockIdx.x * s.channels, smem,
                              reinterpret_cast<float*>(smem + NT));
}

// Rows of `channels` float2 joined: one workgroup takes 16 channels, 16 slices of the rows each, 8 rows in flight.
__device__ __forceinline__ float2 join_rows(const float2* part, long long rows, int channels, int c, float2* red) {
    const int slice = threadIdx.x >> 4;
    double a = 0.0, q = 0.0;
    if (c < channels) {
        long long k = slice;
        for (; k + 7 * 16 < rows; k += 8 * 16) {
            float2 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = part[(k + i * 16) * channels + c];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a += v[i].x;
                q += v[i].y;
            }
        }
        for (; k < rows; k += 16) {
            const float2 v = part[k * channels + c];
            a += v.x;
            q += v.y;
        }
    }
    red[threadIdx.x] = make_float2((float)a, (float)q);
    __syncthreads();
    a = q = 0.0;
    for (int k = 0; k < 16; ++k) {
        a += red[k * 16 + (threadIdx.x & 15)].x;
        q += red[k * 16 + (threadIdx.x & 15)].y;
    }
    return make_float2((float)a, (float)q);
}

// sums[image * channels + c] = the chunks of one image joined
__global__ __launch_bounds__(NT) void norm_bwd_join_kernel(NormShape s, const float2* __restrict__ part,
                                                           float2* __restrict__ sums) {
    __shared__ float2 red[NT];
    const int blocks = (s.channels + 15) / 16;
    const long long b = blockIdx.x / blocks;
    const int c = (int)(blockIdx.x % blocks) * 16 + (threadIdx.x & 15);
    const float2 v = join_rows(part + b * s.chunks * s.channels, s.chunks, s.channels, c, red);
    if (threadIdx.x < 16 && c < s.channels) sums[b * s.channels + c] = v;
}

// dgamma, dbeta: the images' channel sums joined, 16 channels per workgroup
struct ParamGrads {
    void *dweight, *dbias;
    int dtype;
    __device__ __forceinline__ void run(int block, long long batch, int channels, const float2* sums, float2* red) const {
        const int c = block * 16 + (threadIdx.x & 15);
        const float2 v = join_rows(sums, batch, channels, c, red);
        if (threadIdx.x < 16 && c < channels) {
            if (dbias) store_param(dbias, dtype, c, v.x);
            if (dweight) store_param(dweight, dtype, c, v.y);
        }
    }
};

// The first `grad_blocks` workgroups form the parameters' gradients, which need the same sums.
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(NT) void norm_bwd_apply_kernel(NormShape s, const T* __restrict__ x, const T* __restrict__ dy,
                                                            T* __restrict__ dx, const double2* __restrict__ stats,
                                                            const void* __restrict__ weight,
                                                            const void* __restrict__ bias, int pdtype,
                                                            const float2* __restrict__ sums, ParamGrads grads,
                                                            unsigned grad_blocks) {
    extern __shared__ double smem[];
    float2* avg = reinterpret_cast<float2*>(smem);
    if (blockIdx.x < grad_blocks) {
        grads.run(blockIdx.x, s.batch, s.channels, sums, avg);
        return;
    }
    const unsigned block = blockIdx.x - grad_blocks;
    const long long b = block / s.chunks;
    const int chunk = block % s.chunks;
    group_averages(sums + b * s.channels, s.groups, s.per_group, 0, (double)s.pixels * s.per_group, weight, pdtype,
                   [&](int g, float a, float q) { avg[g] = make_float2(a, q); });
    __syncthreads();
    const long long p0 = chunk * s.chunk_pixels;
    const long long first = (b * s.pixels + p0) * s.channels;
    grad_window<T, VEC, ACT>(s, x + first, dy + first, dx + first, 0, s.channels, min(s.chunk_pixels, s.pixels - p0),
                             stats + b * s.groups, avg, 0, weight, bias, pdtype);
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(NT) void norm_bwd_small_kernel(NormShape s, int slab, const T* __restrict__ x,
                                                            const T* __restrict__ dy, T* __restrict__ dx,
                                                            const double2* __restrict__ stats,
                                                            const void* __restrict__ weight, const void* __restrict__ bias,
                                                            int pdtype, float2* __restrict__ sums) {
    extern __shared__ double smem[];
    float* red = reinterpret_cast<float*>(smem + NT);
    float2* ch = reinterpret_cast<float2*>(red + 2 * NT * VEC);
    float2* avg = ch + slab;
    const int slabs = (s.channels + slab - 1) / slab;
    const long long b = blockIdx.x / slabs;
    const int c0 = (int)(blockIdx.x % slabs) * slab;
    const int nc = min(slab, s.channels - c0);
    const long long first = b * s.pixels * s.channels;
    channel_sums<T, VEC, ACT>(s, x + first, dy + first, c0, nc, s.pixels, stats + b * s.groups, weight, bias, pdtype, ch, smem,
                              red);
    __syncthreads();
    for (int c = threadIdx.x; c < nc; c += NT) sums[b * s.channels + c0 + c] = ch[c];
    if (dx) {
        group_averages(ch, nc / s.per_group, s.per_group, c0, (double)s.pixels * s.per_group, weight, pdtype,
                       [&](int g, float a, float q) { avg[g] = make_float2(a, q); });
        __syncthreads();
        grad_window<T, VEC, ACT>(s, x + first, dy + first, dx + first, c0, nc, s.pixels, stats + b * s.groups, avg,
                                 c0 / s.per_group, weight, bias, pdtype);
    }
}

__global__ __launch_bounds__(NT) void norm_param_grads_kernel(long long batch, int channels, const float2* __restrict__ sums,
                                                              ParamGrads grads) {
    __shared__ float2 red[NT];
    grads.run(blockIdx.x, batch, channels, sums, red);
}

// ---- host ---------------------------------------------------------------------------------------------------
int elem_size(int dtype) { return dtype == OD_DTYPE_F32 ? 4 : 2; }

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// channels per workgroup of the one-launch form: whole groups, whole vectors, at least 64 bytes of a row
int slab_channels(int channels, int per_group, int vec, int size) {
    const int unit = per_group / gcd(per_group, vec) * vec;
    const int want = (64 / size + unit - 1) / unit * unit;
    return want < channels ? want : channels;
}

// The one-launch form reads its slab twice, the second time out of the caches, with one workgroup per slab of an image.
// Forward it is ahead up to 64 KiB a slab (16 x 32 x 32 x 256 bf16: 11.8 us against 17.4), backward, with two maps to read,
// up to 32 (22 us against 25 at 64).
bool small_form(const NormShape& s, int slab, int size, int limit) { return s.pixels * slab * size <= limit; }

// Statistics of an image's chunks, 16 bytes each, up to which the workgroups that normalise join them themselves: a launch
// less for the host, which bounds a training step on such maps (77 -> 72 us with the parameters' gradients in the launch of
// dx).  Forward over maps of 64 x 64 in 1, 2, 4 or 8 images, joined here against by a launch of its own: 1024 statistics 13.4
// us against 14.1, 2048 13.8 against 14.4 (eight images 18.0 against 17.6), 2304 15.3 against 15.2, 2560 15.3 against 15.0
// (eight images 22.8 against 21.0), 3328 16.6 against 15.3, 4096 16.7 against 14.8.
constexpr int APPLY_JOINS = 2304;

NormShape shape_of(long long batch, long long pixels, int channels, int groups, float eps, int size) {
    NormShape s;
    s.batch = batch;
    s.pixels = pixels;
    s.channels = channels;
    s.groups = groups;
    s.per_group = channels / groups;
    s.eps = eps;
    // workgroups of at least 64 KiB (a smaller one is mostly its own start: 39 us instead of 15 to normalise
    // 16 x 64 x 64 x 256 bf16 by 2048 of 16 KiB), two to eight per compute unit, at most MAX_CHUNKS per image, at least 16 pixels each
    long long blocks = (long long)((double)batch * pixels * channels * size / 65536.0);
    blocks = blocks < 512 ? 512 : blocks > 2048 ? 2048 : blocks;
    long long chunks = batch > 0 ? (blocks + batch - 1) / batch : 1;
    if (chunks > MAX_CHUNKS) chunks = MAX_CHUNKS;
    if (chunks > (pixels + 15) / 16) chunks = (pixels + 15) / 16;
    if (chunks < 1) chunks = 1;
    s.chunk_pixels = (pixels + chunks - 1) / chunks;
    if (s.chunk_pixels < 1) s.chunk_pixels = 1;
    s.chunks = (int)((pixels + s.chunk_pixels - 1) / s.chunk_pixels);
    if (s.chunks < 1) s.chunks = 1;
    return s;
}

int check_shape(int32_t dtype, int64_t batch, int64_t pixels, int32_t channels, int32_t groups, int32_t param_dtype,
                int32_t activation) {
    if (dtype < OD_DTYPE_F32 || dtype > OD_DTYPE_BF16 || param_dtype < OD_DTYPE_F32 || param_dtype > OD_DTYPE_BF16)
        return OD_ERR_ARG;
    if (activation < OD_ACT_NONE || activation > OD_ACT_SILU) return OD_ERR_ARG;
    if (batch < 0 || pixels < 0 || channels <= 0 || groups <= 0 || channels % groups) return OD_ERR_ARG;
    if (channels > OD_MAX_NORM_CHANNELS || pixels > OD_MAX_NORM_PIXELS || batch > OD_MAX_NORM_BATCH) return OD_ERR_LIMIT;
    return OD_OK;
}

struct FwdCall {
    NormShape s;
    const void *x, *weight, *bias;
    void* y;
    int pdtype;
    double2* stats;
    void* ws;
    hipStream_t stream;
};

template <typename T, int VEC, int ACT>
int forward_typed(const FwdCall& c) {
    const int slab = slab_channels(c.s.channels, c.s.per_group, VEC, sizeof(T));
    const T* x = (const T*)c.x;
    T* y = (T*)c.y;
    if (small_form(c.s, slab, sizeof(T), 64 << 10)) {
        const long long grid = c.s.batch * ((c.s.channels + slab - 1) / slab);
        const size_t lds = (size_t)(slab + slab / c.s.per_group) * sizeof(double2) + NT * sizeof(double) +
                           3 * NT * VEC * sizeof(float);
        OD_LAUNCH_KERNEL(OD_KERNEL_NORM_APPLY, (norm_small_kernel<T, VEC, ACT>), dim3((unsigned)grid), dim3(NT), lds, c.stream,
                         c.s, slab, x, y, c.weight, c.bias, c.pdtype, c.stats);
        return OD_OK;
    }
    double2* part = (double2*)c.ws;
    const long long grid = c.s.batch * c.s.chunks;
    OD_LAUNCH_KERNEL(OD_KERNEL_NORM_STATS, (norm_stats_kernel<T, VEC>), dim3((unsigned)grid), dim3(NT),
                     c.s.channels * sizeof(double2) + NT * sizeof(double) + 3 * NT * VEC * sizeof(float), c.stream, c.s, x, part);
    const bool joined = c.s.chunks * c.s.groups > APPLY_JOINS;
    if (joined) {
        hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(c.s.batch * ((c.s.groups + 7) / 8))), dim3(NT), 0, c.stream, c.s,
                           (const double2*)part, c.stats);
        OD_LAUNCH_CHECK();
    }
    OD_LAUNCH_KERNEL(OD_KERNEL_NORM_APPLY, (norm_apply_kernel<T, VEC, ACT>), dim3((unsigned)grid), dim3(NT),
                     joined ? 0 : NT * sizeof(double) + c.s.groups * sizeof(double2), c.stream, c.s, x, y, c.weight, c.bias,
                     c.pdtype, joined ? (const double2*)nullptr : (const double2*)part, c.stats);
    return OD_OK;
}

struct BwdCall {
    NormShape s;
    const void *x, *dy, *weight, *bias;
    void *dx, *dweight, *dbias;
    int pdtype;
    const double2* stats;
    void* ws;
    hipStream_t stream;
};

template <typename T, int VEC, int ACT>
int backward_typed(const BwdCall& c) {
    const int slab = slab_channels(c.s.channels, c.s.per_group, VEC, sizeof(T));
    const T *x = (const T*)c.x, *dy = (const T*)c.dy;
    T* dx = (T*)c.dx;
    float2* sums = (float2*)c.ws;
    const ParamGrads grads = {c.dweight, c.dbias, c.pdtype};
    const unsigned grad_blocks = c.dweight || c.dbias ? (c.s.channels + 15) / 16 : 0;
    if (small_form(c.s, slab, sizeof(T), 32 << 10)) {
        const long long grid = c.s.batch * ((c.s.channels + slab - 1) / slab);
        const size_t lds = NT * sizeof(double) + (2 * NT * VEC + 4 * (size_t)slab) * sizeof(float);
        OD_LAUNCH_KERNEL(OD_KERNEL_NORM_BWD_APPLY, (norm_bwd_small_kernel<T, VEC, ACT>), dim3((unsigned)grid), dim3(NT), lds,
                         c.stream, c.s, slab, x, dy, dx, c.stats, c.weight, c.bias, c.pdtype, sums);
    } else {
        float2* part = sums + c.s.batch * c.s.channels;
        const long long grid = c.s.batch * c.s.chunks;
        OD_LAUNCH_KERNEL(OD_KERNEL_NORM_BWD_SUMS, (norm_bwd_sums_kernel<T, VEC, ACT>), dim3((unsigned)grid), dim3(NT),
                         NT * sizeof(double) + 2 * NT * VEC * sizeof(float), c.stream, c.s, x, dy, c.stats, c.weight, c.bias,
                         c.pdtype, part);
        hipLaunchKernelGGL(norm_bwd_join_kernel, dim3((unsigned)(c.s.batch * ((c.s.channels + 15) / 16))), dim3(NT), 0, c.stream,
                           c.s, (const float2*)part, sums);
        OD_LAUNCH_CHECK();
        if (dx) {
            const size_t lds = 2 * sizeof(float) * (size_t)(c.s.groups > NT ? c.s.groups : NT);
            OD_LAUNCH_KERNEL(OD_KERNEL_NORM_BWD_APPLY, (norm_bwd_apply_kernel<T, VEC, ACT>), dim3((unsigned)grid + grad_blocks),
                             dim3(NT), lds, c.stream, c.s, x, dy, dx, c.stats, c.weight, c.bias, c.pdtype, (const float2*)sums,
                             grads, grad_blocks);
            return OD_OK;
        }
    }
    if (grad_blocks > 0) {
        hipLaunchKernelGGL(norm_param_grads_kernel, dim3(grad_blocks), dim3(NT), 0, c.stream, c.s.batch, c.s.channels,
                           (const float2*)sums, grads);
        OD_LAUNCH_CHECK();
    }
    return OD_OK;
}

// The vector width follows from the channel count and the addresses; the activation and the type are compiled in.
#define OD_NORM_DISPATCH(fn, call, aligned)                                                              \
    do {                                                                                                 \
        auto by_act = [&](auto vec, auto elem) -> int {                                                  \
            using T = decltype(elem);                                                                    \
            constexpr int V = decltype(vec)::value;                                                      \
            if (activation == OD_ACT_RELU) return fn<T, V, OD_ACT_RELU>(call);                           \
            if (activation == OD_ACT_SILU) return fn<T, V, OD_ACT_SILU>(call);                           \
            return fn<T, V, OD_ACT_NONE>(call);                                                          \
        };                                                                                               \
        const int width_ = (aligned);                                                                    \
        using V1 = std::integral_constant<int, 1>;                                                       \
        using V4 = std::integral_constant<int, 4>;                                                       \
        using V8 = std::integral_constant<int, 8>;                                                       \
        if (dtype == OD_DTYPE_F32) return width_ >= 4 ? by_act(V4{}, float{}) : by_act(V1{}, float{});   \
        if (dtype == OD_DTYPE_F16)                                                                       \
            return width_ >= 8 ? by_act(V8{}, _Float16{}) : width_ >= 4 ? by_act(V4{}, _Float16{})       \
                                                                        : by_act(V1{}, _Float16{});      \
        return width_ >= 8 ? by_act(V8{}, bf16_t{}) : width_ >= 4 ? by_act(V4{}, bf16_t{})               \
                                                                  : by_act(V1{}, bf16_t{});              \
    } while (0)

// elements per access: what divides the channel count and keeps every pointer aligned
int vector_width(int dtype, int channels, uintptr_t addresses) {
    const int size = elem_size(dtype);
    for (int v = 16 / size; v >= 4; v /= 2)
        if (channels % v == 0 && addresses % (uintptr_t)(v * size) == 0) return v;
    return 1;
}

}  // namespace

extern "C" size_t od_group_norm_act_workspace_bytes(int64_t batch, int64_t pixels, int32_t channels, int32_t groups) {
    if (check_shape(OD_DTYPE_F32, batch, pixels, channels, groups, OD_DTYPE_F32, OD_ACT_NONE) != OD_OK) return 0;
    // part: at most 2048 + batch chunks in a launch, of a float2 per channel or a double2 per group; sums: one per image
    const long long chunks = 2048 + batch, each = (long long)channels * sizeof(float2) > groups * (long long)sizeof(double2)
                                                      ? (long long)channels * sizeof(float2) : groups * (long long)sizeof(double2);
    return (size_t)(chunks * each + batch * channels * (long long)sizeof(float2)) + 256;
}

extern "C" int od_group_norm_act_forward(const void* x, int32_t dtype, int64_t batch, int64_t pixels, int32_t channels,
                                         int32_t groups, const void* weight, const void* bias, int32_t param_dtype,
                                         float eps, int32_t activation, void* y, double* stats, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    const int rc = check_shape(dtype, batch, pixels, channels, groups, param_dtype, activation);
    if (rc != OD_OK) return rc;
    if (batch == 0 || pixels == 0) return OD_OK;
    if (!x || !y || !stats || ((uintptr_t)stats & 15) || !workspace || ((uintptr_t)workspace & 255)) return OD_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)y) % elem_size(dtype)) return OD_ERR_ARG;
    if (workspace_bytes < od_group_norm_act_workspace_bytes(batch, pixels, channels, groups)) return OD_ERR_WORKSPACE;
    const FwdCall call = {shape_of(batch, pixels, channels, groups, eps, elem_size(dtype)), x, weight, bias, y, param_dtype,
                          (double2*)stats, workspace, (hipStream_t)stream};
    OD_NORM_DISPATCH(forward_typed, call, vector_width(dtype, channels, (uintptr_t)x | (uintptr_t)y));
}

extern "C" int od_group_norm_act_backward(const void* x, const void* dy, int32_t dtype, int64_t batch, int64_t pixels,
                                          int32_t channels, int32_t groups, const void* weight, const void* bias,
                                          int32_t param_dtype, int32_t activation, const double* stats, void* dx,
                                          void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_shape(dtype, batch, pixels, channels, groups, param_dtype, activation);
    if (rc != OD_OK) return rc;
    if (batch == 0 || pixels == 0) return OD_OK;
    if (!x || !dy || !stats || ((uintptr_t)stats & 15) || !workspace || ((uintptr_t)workspace & 255)) return OD_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx) % elem_size(dtype)) return OD_ERR_ARG;
    if (workspace_bytes < od_group_norm_act_workspace_bytes(batch, pixels, channels, groups)) return OD_ERR_WORKSPACE;
    const BwdCall call = {shape_of(batch, pixels, channels, groups, 0.0f, elem_size(dtype)), x, dy, weight, bias, dx, dweight,
                          dbias, param_dtype, (const double2*)stats, workspace, (hipStream_t)stream};
    OD_NORM_DISPATCH(backward_typed, call, vector_width(dtype, channels, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx));
}
