// Losses of a classification head whose classes are a large vocabulary of embeddings: softmax cross entropy and
// distillation from a teacher's top logits, with their gradients, without the [rows, classes] logits ever being kept.
//
//   z = (F W^T + b) / T            F [rows, dim], W [classes, dim], b [classes]
//   q = softmax(z) over the classes, lse = log sum exp z
//   target distribution p of a row: one class (cross entropy, T = 1), or softmax(t / T) over the classes a teacher names
//   loss_n = T^2 (sum p log p - sum p z_class + lse)
//   dz = g T (q - p), g the gradient of the row's loss;   dF = dz W,  dW = dz^T F,  db = sum_n dz
//
// Forward: one product over tiles of 128 rows x 128 classes whose epilogue folds a tile into a running maximum and sum
// per row (in the lane that owns the row: no traffic between lanes before the end); the classes are split over
// workgroups and joined by a second kernel, which also forms the few logits of the targets by dot products.
// Backward: the classes are taken in pieces; a piece's dz is recomputed from the saved lse into a buffer of bounded size
// (in the type of the inputs: it is an operand of the two products that follow), the target entries are corrected, and
// dF and dW accumulate in fp32.  16-bit dz: bf16 keeps the exponents of fp32; fp16 rows are scaled by one power of two,
// taken from the largest row gradient, so that small probabilities do not underflow; the scale leaves in the fp32 results.
//
// Rows without a target (negative class; no finite teacher entry) are left out at the start: the valid rows are listed in
// order and their features packed densely, so that masked rows cost nothing and whatever they hold (infinities, NaN)
// reaches no product.  All sums run in a fixed order; there are no atomics.
#include "od_common.h"
#include "../../include/od_boxes.h"
#include "od_elem.h"

#pragma clang fp contract(fast)

namespace {

using namespace od;

constexpr int VT = 256;                 // threads per workgroup: four waves in a 2 x 2 arrangement
constexpr int TILE = 128;               // rows and columns of a workgroup's tile (64 x 64 per wave)
constexpr int STAGE = TILE * 128;       // bytes of one operand's stage in LDS
constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.69314718055994531f;
constexpr float LOWEST = -3.402823466e38f;      // start of a running maximum: finite, so that -inf - LOWEST stays -inf

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// A fragment is 16 bytes per lane: 32 rows (lane % 32) x one 32-byte slab of K (halves lane / 32).  Any assignment of K
// to the slots of a slab gives the same product as long as both operands use it.
template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
    static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {
    static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
        const vec4f x = __builtin_bit_cast(vec4f, a), y = __builtin_bit_cast(vec4f, b);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, c, 0, 0, 0);
    }
};

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) uint32_t* global_words;

// 16 bytes per lane from global memory straight into LDS: lane l lands at base + 16 l
__device__ __forceinline__ void stage16(const char* src, char* base) {
    __builtin_amdgcn_global_load_lds((global_words)src, (__attribute__((address_space(3))) uint32_t*)base, 16, 0, 0);
}

// ---- operand with K contiguous: 128 rows x 128 bytes of K.  The 16-byte chunks of a row are permuted by row % 8, which
// spreads the eight rows that a quarter wave reads at once over all banks.
struct ChunkedOperand {
    const char* row[4];                 // this lane's source rows (four rows of eight per wave and instruction)
    int chunk;
    __device__ __forceinline__ void init(const char* base, long long pitch, long long first, long long last) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            long long r = first + (wave * 4 + i) * 8 + (lane >> 3);
            row[i] = base + (r < last ? r : last) * pitch;          // rows past the end repeat the last one
        }
        chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    }
    __device__ __forceinline__ void stage(char* lds, long long kbytes) const {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < 4; ++i) stage16(row[i] + kbytes + chunk, lds + (wave * 4 + i) * 1024);
    }
    // fragment of rows [r0, r0 + 32), slab j of four
    static __device__ __forceinline__ u32x4 frag(const char* lds, int r0, int j) {
        const int lane = threadIdx.x & 63;
        const int r = r0 + (lane & 31);
        return *reinterpret_cast<const u32x4*>(lds + r * 128 + (((2 * j + (lane >> 5)) ^ (r & 7)) << 4));
    }
};

// ---- operand with K strided: KE rows of K x 128 contiguous elements; read transposed.
template <typename T>
struct StridedOperand {
    static constexpr int KE = 128 / sizeof(T);                      // K per stage
    static constexpr int ROWB = TILE * sizeof(T);                   // bytes per K row
    static constexpr int CHUNKS = ROWB / 16;
    static constexpr int RPI = 1024 / ROWB;                         // K rows per wave and instruction
    const char* base;
    long long pitch;
    int lane_row, first_byte, last_byte;
    // chunk permutation of K row k: the rows that one transposing read touches at once go to different banks
    static __device__ __forceinline__ int swizzle(int k) {
        return sizeof(T) == 2 ? (((k & 3) | (((k >> 3) & 1) << 2)) << 1) : (((k >> 2) & 1) << 3);
    }
    __device__ __forceinline__ void init(const char* b, long long p, long long first_col, long long cols) {
        base = b;
        pitch = p;
        lane_row = (threadIdx.x & 63) / CHUNKS;
        first_byte = (int)(first_col * sizeof(T));
        last_byte = (int)(cols * sizeof(T)) - 16;                   // columns past the end repeat the last chunk
    }
    // K rows [k0, k0 + KE); rows past `last` repeat it
    __device__ __forceinline__ void stage(char* lds, long long k0, long long last) const {
        const int wave = threadIdx.x >> 6, pos = (threadIdx.x & 63) % CHUNKS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = (wave * 4 + i) * RPI + lane_row;
            const long long r = k0 + k;
            const int byte = first_byte + ((pos ^ swizzle(k)) << 4);
            stage16(base + (r < last ? r : last) * pitch + (byte < last_byte ? byte : last_byte), lds + (wave * 4 + i) * 1024);
        }
    }
    static __device__ __forceinline__ u32x4 frag(const char* lds, int m0, int j) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // a transposing read hands lane i of 16 the i-th element of the four rows that lanes 4r .. 4r+3 point at
            const int r = (lane & 15) >> 2;
            const int chunk = (m0 >> 3) + (((lane >> 4) & 1) << 1) + ((lane & 3) >> 1);
            const char* p = lds + (16 * j + 8 * h + r) * ROWB + ((chunk ^ ((r | (h << 2)) << 1)) << 4) + ((lane & 1) << 3);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * ROWB));
            const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
            u32x4 v; v.x = a.x; v.y = a.y; v.z = b.x; v.w = b.y;
            return v;
        } else {
            const char* p = lds + (8 * j + 4 * h) * ROWB + (((m0 + (lane & 31)) << 2) ^ (h << 7));
            u32x4 v;
            v.x = *reinterpret_cast<const uint32_t*>(p);
            v.y = *reinterpret_cast<const uint32_t*>(p + ROWB);
            v.z = *reinterpret_cast<const uint32_t*>(p + 2 * ROWB);
            v.w = *reinterpret_cast<const uint32_t*>(p + 3 * ROWB);
            return v;
        }
    }
};

// Every load into LDS of this wave has landed, and every wave has got here.
__device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
}

// Workgroup number -> work number such that each of the eight XCDs (hardware hands workgroups to them in turn) gets one
// contiguous range: neighbours share their operands in one L2.
__device__ __forceinline__ int xcd_range(int id, int total) {
    const int per = total / 8;
    return id < per * 8 ? (id % 8) * per + id / 8 : id;
}

// ---- preparation --------------------------------------------------------------------------------------------------
// Number of valid rows, their list and each row's place in it, in row order, by one workgroup; clears row_loss.
// A row is valid if valid_of(targets, flags) says so.
struct RowLists {
    int* count;
    int* row_of;                        // [rows] valid rows in order
    int* place;                         // [rows] index into row_of, or -1
};

__global__ __launch_bounds__(1024) void list_rows_kernel(const long long* __restrict__ targets,
                                                         const unsigned char* __restrict__ flags, int rows, RowLists lists,
                                                         float* __restrict__ row_loss) {
    __shared__ int sums[1024];
    const int per = (rows + 1023) / 1024;
    const int a = min(rows, (int)threadIdx.x * per), b = min(rows, a + per);
    int n = 0;
    for (int r = a; r < b; ++r) n += flags ? flags[r] : (targets[r] >= 0);
    sums[threadIdx.x] = n;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {                            // inclusive scan
        const int v = (int)threadIdx.x >= o ? sums[threadIdx.x - o] : 0;
        __syncthreads();
        sums[threadIdx.x] += v;
        __syncthreads();
    }
    int at = sums[threadIdx.x] - n;
    for (int r = a; r < b; ++r) {
        const bool on = flags ? flags[r] != 0 : targets[r] >= 0;
        lists.place[r] = on ? at : -1;
        if (on) lists.row_of[at++] = r;
        row_loss[r] = 0.0f;
    }
    if (threadIdx.x == 1023) *lists.count = sums[1023];
}

// Teacher's distribution of a row over its listed classes, one wave per row: p = softmax(t / T) over the entries with a
// class >= 0 and a logit above -inf.  Entries that name the same class are one class: the first of them gets the sum, the
// others 0, and the entropy term sum p log p is the merged distribution's.
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <typename T>
__global__ __launch_bounds__(VT) void teacher_kernel(const long long* __restrict__ classes, const T* __restrict__ logits,
                                                     int rows, int top, float inv_temp, float* __restrict__ prob,
                                                     float* __restrict__ entropy, unsigned char* __restrict__ flags) {
    __shared__ long long s_class[VT / 64][OD_MAX_TEACHER_TOP];
    __shared__ float s_prob[VT / 64][OD_MAX_TEACHER_TOP];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row = blockIdx.x * (VT / 64) + wave;
    constexpr int PER = OD_MAX_TEACHER_TOP / 64;
    float t[PER];
    float top_value = LOWEST;
    bool any = false;
    if (row < rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int k = i * 64 + lane;
            t[i] = -__builtin_inff();
            if (k < top) {
                const long long c = classes[(long long)row * top + k];
                const float v = Elem<T>::to_float(logits[(long long)row * top + k]);
                s_class[wave][k] = c;
                if (c >= 0) t[i] = v;
            }
            any = any || !(t[i] == -__builtin_inff());               // NaN counts: it has to reach the loss
            top_value = fmaxf(top_value, t[i]);
        }
    }
    top_value = wave_max(top_value);
    const bool on = __any(any);
    float total = 0.0f;
    if (row < rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            t[i] = (t[i] - top_value) * inv_temp;                   // -inf stays -inf: exp gives 0
            total += expf(t[i]);
        }
    }
    total = wave_sum(total);
    const float log_total = logf(total);
    if (row < rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int k = i * 64 + lane;
            if (k < top) s_prob[wave][k] = (t[i] == -__builtin_inff()) ? 0.0f : expf(t[i] - log_total);
        }
    }
    __syncthreads();
    float h = 0.0f;
    if (row < rows) {
        for (int k = lane; k < top; k += 64) {
            const long long c = s_class[wave][k];
            float p = 0.0f;
            bool first = true;
            for (int o = 0; o < top; ++o)
                if (s_class[wave][o] == c) {
                    if (o < k) first = false;
                    p += s_prob[wave][o];
                }
            p = (c >= 0 && first) ? p : 0.0f;
            prob[(long long)row * top + k] = p;
            if (!(p == 0.0f)) h += p * logf(p);
        }
    }
    h = wave_sum(h);
    if (row < rows && lane == 0) {
        flags[row] = on ? 1 : 0;
        entropy[row] = h;
    }
}

// Features of the valid rows, dense: [rows rounded up to TILE][dim_pad], zero behind the last valid row and the last
// column.  A thread copies one 16-byte chunk; sources that are not aligned for it are read element by element.
template <typename T>
__global__ __launch_bounds__(VT) void pack_rows_kernel(const T* __restrict__ src, long long pitch, int dim, int dim_pad,
                                                       const int* __restrict__ row_of, const int* __restrict__ count,
                                                       long long rows_out, T* __restrict__ dst) {
    constexpr int E = 16 / sizeof(T);
    const int chunks = dim_pad / E;
    const long long at = (long long)blockIdx.x * VT + threadIdx.x;
    const long long r = at / chunks;
    if (r >= rows_out) return;
    const int c = (int)(at % chunks) * E;
    const long long limit = count ? *count : rows_out;
    alignas(16) T v[E];
    if (r < limit) {
        const T* p = src + (row_of ? (long long)row_of[r] : r) * pitch + c;
        if (c + E <= dim && ((uintptr_t)p & 15) == 0) {
            *reinterpret_cast<u32x4*>(v) = *reinterpret_cast<const u32x4*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = c + i < dim ? p[i] : Elem<T>::from_float(0.0f);
        }
    } else {
        if (count && r >= (limit + TILE - 1) / TILE * TILE) return;            // no tile reads behind the last one's end
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = Elem<T>::from_float(0.0f);
    }
    *reinterpret_cast<u32x4*>(dst + r * dim_pad + c) = *reinterpret_cast<const u32x4*>(v);
}

// bias in units of log2, -inf behind the last class: the tiles' tail then drops out of maxima and sums by itself
template <typename T>
__global__ __launch_bounds__(VT) void bias_kernel(const T* __restrict__ bias, int classes, int classes_pad, float scale,
                                                  float* __restrict__ out) {
    const int v = blockIdx.x * VT + threadIdx.x;
    if (v < classes_pad) out[v] = v >= classes ? -__builtin_inff() : bias ? Elem<T>::to_float(bias[v]) * scale : 0.0f;
}

// ---- the product ----------------------------------------------------------------------------------------------------
struct ProductArgs {
    const char* weight;                 // [classes][weight_pitch bytes], K contiguous, dim_pad elements readable
    long long weight_pitch;
    const char* features;               // packed rows, dim_pad elements each
    int dim_pad;
    long long first_class, last_class;  // of the piece; last class of all
    const float* bias2;                 // at the piece's first class
    const int* count;
    int tiles, splits;                  // class tiles of the piece, workgroups per row tile
    float scale;                        // log2(e) / temperature
    long long rows_pad;
    // forward
    float2* part;                       // [splits][rows_pad] (maximum, sum), log2 units
    // backward
    const float* lse2;                  // [rows_pad] in log2 units
    const float* row_grad;              // [rows_pad]
    void* dz;                           // [rows_pad][piece]
    long long piece;
};

// Accumulators: acc[f][g] holds classes f*32 + 8*(i/4) + 4*(lane/32) + i%4 (i = 0 .. 15) of row g*32 + lane%32.
template <typename T, bool GRAD>
__global__ __launch_bounds__(VT, 2) void product_kernel(ProductArgs p) {
    __shared__ __align__(1024) char lds[4 * STAGE];                 // two stages of (classes, rows)
    __shared__ float2 joined[2][TILE];
    const int id = xcd_range(blockIdx.x, gridDim.x);
    const int split = id % p.splits;
    const long long r0 = (long long)(id / p.splits) * TILE;
    if (r0 >= *p.count) return;
    const int t0 = (int)((long long)p.tiles * split / p.splits), t1 = (int)((long long)p.tiles * (split + 1) / p.splits);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
    const int wc = (wave & 1) * 64, wr = (wave >> 1) * 64;          // this wave's classes and rows within the tile
    constexpr int KE = 128 / sizeof(T);
    const int ksteps = p.dim_pad / KE;

    ChunkedOperand rows, cls;
    rows.init(p.features, (long long)p.dim_pad * sizeof(T), r0, r0 + TILE);

    float m[2], s[2], lse2[2], grad[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        m[g] = LOWEST;
        s[g] = 0.0f;
        if (GRAD) {
            lse2[g] = p.lse2[r0 + wr + g * 32 + (lane & 31)];
            grad[g] = p.row_grad[r0 + wr + g * 32 + (lane & 31)];
        }
    }

    f32x16 acc[2][2];
    int buf = 0;
    if (t0 < t1) {
        cls.init(p.weight, p.weight_pitch, p.first_class + (long long)t0 * TILE, p.last_class);
        cls.stage(lds, 0);
        rows.stage(lds + STAGE, 0);
    }
    for (int t = t0; t < t1; ++t) {
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[f][g][i] = 0.0f;
        for (int k = 0; k < ksteps; ++k) {
            stage_barrier();
            const char* now = lds + buf * 2 * STAGE;
            char* next = lds + (buf ^ 1) * 2 * STAGE;
            if (k + 1 < ksteps) {
                cls.stage(next, (long long)(k + 1) * 128);
                rows.stage(next + STAGE, (long long)(k + 1) * 128);
            } else if (t + 1 < t1) {
                cls.init(p.weight, p.weight_pitch, p.first_class + (long long)(t + 1) * TILE, p.last_class);
                cls.stage(next, 0);
                rows.stage(next + STAGE, 0);
            }
            buf ^= 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 a[2], b[2];
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    a[f] = ChunkedOperand::frag(now, wc + f * 32, j);
                    b[f] = ChunkedOperand::frag(now + STAGE, wr + f * 32, j);
                }
#pragma unroll
                for (int f = 0; f < 2; ++f)
#pragma unroll
                    for (int g = 0; g < 2; ++g) acc[f][g] = Mma<T>::run(a[f], b[g], acc[f][g]);
            }
        }
        const float* bias = p.bias2 + (long long)t * TILE + wc + 4 * h;
        if (!GRAD) {
            float top[2] = {m[0], m[1]};
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const vec4f bq = *reinterpret_cast<const vec4f*>(bias + f * 32 + 8 * q);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float z = fmaf(acc[f][g][4 * q + e], p.scale, bq[e]);
                            acc[f][g][4 * q + e] = z;
                            top[g] = fmaxf(top[g], z);
                        }
                }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float sum = s[g] * __builtin_amdgcn_exp2f(m[g] - top[g]);
#pragma unroll
                for (int f = 0; f < 2; ++f)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(acc[f][g][i] - top[g]);
                m[g] = top[g];
                s[g] = sum;
            }
        } else {
            T* out = (T*)p.dz + (long long)t * TILE + wc + 4 * h;
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const vec4f bq = *reinterpret_cast<const vec4f*>(bias + f * 32 + 8 * q);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float z = fmaf(acc[f][g][4 * q + e], p.scale, bq[e] - lse2[g]);
                            v[e] = grad[g] == 0.0f ? 0.0f : grad[g] * __builtin_amdgcn_exp2f(z);
                        }
                        store_vec<T, 4>(out + (r0 + wr + g * 32 + (lane & 31)) * p.piece + f * 32 + 8 * q, v);
                    }
                }
        }
    }
    if (!GRAD) {
        // a row's classes lie in two lanes and two waves
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const float om = __shfl_xor(m[g], 32, 64), os = __shfl_xor(s[g], 32, 64);
            const float top = fmaxf(m[g], om);
            s[g] = s[g] * __builtin_amdgcn_exp2f(m[g] - top) + os * __builtin_amdgcn_exp2f(om - top);
            m[g] = top;
            if (h == 0) joined[wave & 1][wr + g * 32 + lane] = make_float2(m[g], s[g]);
        }
        __syncthreads();
        if (threadIdx.x < TILE) {
            const float2 a = joined[0][threadIdx.x], b = joined[1][threadIdx.x];
            const float top = fmaxf(a.x, b.x);
            p.part[(long long)split * p.rows_pad + r0 + threadIdx.x] =
                make_float2(top, a.y * __builtin_amdgcn_exp2f(a.x - top) + b.y * __builtin_amdgcn_exp2f(b.x - top));
        }
    }
}

// ---- forward's end -----------------------------------------------------------------------------------------------------
struct TargetArgs {
    const char* features;               // packed
    int dim, dim_pad;
    const void* weight;                 // the caller's rows
    long long weight_pitch;             // elements
    const void* bias;
    long long classes;
    const long long* targets;           // [rows] or [rows, top]
    int top;                            // 0: cross entropy
    const float* prob;                  // [rows, top]
    const float* entropy;               // [rows]
    RowLists lists;
    const float2* part;
    int splits;
    long long rows_pad;
    float temperature;
    float* lse2;                        // [rows_pad]
    float* target_logit;                // [rows, max(top, 1)] by place, natural units, divided by the temperature
    float* row_loss;                    // [rows]
};

// One wave per valid row: joins the splits, forms the targets' logits (16 lanes a dot product), writes the row's loss.
// A class past the vocabulary makes the row's lse, and with it loss and gradient, NaN; it is not followed.
template <typename T>
__global__ __launch_bounds__(VT) void targets_kernel(TargetArgs p) {
    const int lane = threadIdx.x & 63;
    const long long place = (long long)blockIdx.x * (VT / 64) + (threadIdx.x >> 6);
    const int count = *p.lists.count;
    if (place >= count) {
        if (place < p.rows_pad && lane == 0) p.lse2[place] = 0.0f;
        return;
    }
    const long long row = p.lists.row_of[place];
    float m = LOWEST, s = 0.0f;
    for (int k = lane; k < p.splits; k += 64) {
        const float2 v = p.part[(long long)k * p.rows_pad + place];
        const float top = fmaxf(m, v.x);
        s = s * __builtin_amdgcn_exp2f(m - top) + v.y * __builtin_amdgcn_exp2f(v.x - top);
        m = top;
    }
    const float top = wave_max(m);
    s = wave_sum(s * __builtin_amdgcn_exp2f(m - top));
    float lse = (top + log2f(s)) * LN2;

    const int n = p.top > 0 ? p.top : 1;
    const float inv_temp = 1.0f / p.temperature;
    const T* f = (const T*)p.features + place * p.dim_pad;
    float dot_sum = 0.0f;                                           // sum p z over this group of 16 lanes' entries
    bool outside = false;
    for (int k0 = 0; k0 < n; k0 += 4) {
        const int k = k0 + (lane >> 4);
        const long long c = k < n ? p.targets[row * n + k] : -1;
        float z = 0.0f;
        if (c >= p.classes) outside = true;
        if (c >= 0 && c < p.classes) {
            const T* w = (const T*)p.weight + c * p.weight_pitch;
            for (int d = lane & 15; d < p.dim; d += 16) z = fmaf(Elem<T>::to_float(f[d]), Elem<T>::to_float(w[d]), z);
        }
        for (int o = 8; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
        if (c >= 0 && c < p.classes) {
            if (p.bias) z += Elem<T>::to_float(((const T*)p.bias)[c]);
            z *= inv_temp;
            const float prob = p.top > 0 ? p.prob[row * n + k] : 1.0f;
            if ((lane & 15) == 0) {
                p.target_logit[place * n + k] = z;
                if (!(prob == 0.0f)) dot_sum += prob * z;           // an entry without weight takes no part: 0 * inf
            }
        }
    }
    dot_sum = wave_sum(dot_sum);
    if (__any(outside)) lse = __builtin_nanf("");
    if (lane == 0) {
        p.lse2[place] = lse * LOG2E;
        const float t2 = p.temperature * p.temperature;
        p.row_loss[row] = ((p.top > 0 ? p.entropy[row] : 0.0f) + lse - dot_sum) * t2;
    }
}

// loss[0] = sum of the row losses, over the number of valid rows where the mean is asked for
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* __restrict__ row_loss, int rows,
                                                        const int* __restrict__ count, int reduction,
                                                        float* __restrict__ loss) {
    __shared__ double red[1024];
    double v = 0.0;
    for (int r = threadIdx.x; r < rows; r += 1024) v += (double)row_loss[r];
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)(reduction == OD_REDUCE_MEAN ? red[0] / (double)max(1, *count) : red[0]);
}

// ---- backward ------------------------------------------------------------------------------------------------------
// row_grad[place] = gradient of the row's loss times the temperature, times `scale[0]`; scale[1] = 1 / scale[0].
// fp16: scale is the power of two that brings the largest |row_grad| into [2^13, 2^14): |dz| <= |row_grad| stays finite
// and a probability of 2^-28 is still a normal number.  The other types take 1.
__global__ __launch_bounds__(1024) void row_grads_kernel(const float* __restrict__ upstream, int reduction, RowLists lists,
                                                         long long rows_pad, float temperature, int scaled,
                                                         float* __restrict__ row_grad, float* __restrict__ scale) {
    __shared__ float red[1024];
    const int count = *lists.count;
    const float share = temperature / (reduction == OD_REDUCE_MEAN ? (float)max(1, count) : 1.0f);
    float top = 0.0f;
    if (scaled)
        for (int i = threadIdx.x; i < count; i += 1024) {
            const float g = fabsf(upstream[reduction == OD_REDUCE_NONE ? lists.row_of[i] : 0] * share);
            if (g < 3.0e38f) top = fmaxf(top, g);                  // infinities and NaN go through as they are
        }
    red[threadIdx.x] = top;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + o]);
        __syncthreads();
    }
    float s = 1.0f;
    if (scaled && red[0] > 0.0f) {
        int e = 0;
        (void)frexpf(red[0], &e);                                   // red[0] = f * 2^e, f in [0.5, 1)
        e = min(max(14 - e, -100), 100);
        s = ldexpf(1.0f, e);
    }
    for (long long i = threadIdx.x; i < rows_pad; i += 1024)
        row_grad[i] = i < count ? upstream[reduction == OD_REDUCE_NONE ? lists.row_of[i] : 0] * share * s : 0.0f;
    if (threadIdx.x == 0) {
        scale[0] = s;
        scale[1] = 1.0f / s;
    }
}

// The target entries of a piece of dz: g (q - p).  Next to p = 1 it is expm1(log q) + (1 - p), which keeps the digits of
// 1 - q of a confident row; for small p that sum would lose those of q and p.  Each (row, class) is written once: repeated classes carry their whole p in the first entry.
template <typename T>
__global__ __launch_bounds__(VT) void correct_targets_kernel(const long long* __restrict__ targets, int top,
                                                             const float* __restrict__ prob, RowLists lists,
                                                             const float* __restrict__ lse2,
                                                             const float* __restrict__ target_logit,
                                                             const float* __restrict__ row_grad, long long first_class,
                                                             long long piece, long long classes, T* __restrict__ dz) {
    const int n = top > 0 ? top : 1;
    const long long at = (long long)blockIdx.x * VT + threadIdx.x;
    const long long place = at / n;
    if (place >= *lists.count) return;
    const long long row = lists.row_of[place];
    const long long src = row * n + at % n;
    const long long c = targets[src];
    if (c < first_class || c >= first_class + piece || c >= classes) return;
    const float p = top > 0 ? prob[src] : 1.0f;
    if (p == 0.0f) return;                                          // what the product wrote is q already
    const float log_q = target_logit[at] - lse2[place] * LN2;
    const float g = row_grad[place];
    const float v = g == 0.0f ? 0.0f : g * (p > 0.5f ? expm1f(log_q) + (1.0f - p) : expf(log_q) - p);
    dz[place * piece + (c - first_class)] = Elem<T>::from_float(v);
}

struct GradArgs {
    const char* a;                      // [K][a_pitch bytes], dim_pad columns: weight rows of the piece, or packed features
    long long a_pitch, a_last;          // last readable K row
    const char* dz;                     // [rows_pad][piece]
    long long piece;
    int dim_pad;
    const int* count;
    long long cols;                     // columns of the result: rows_pad, or piece
    long long ksteps;                   // K steps of all splits (of rows: at most, see count)
    int splits;
    float* out;                         // [splits][cols][dim_pad]
    int accumulate;
    float* bias_out;                    // [splits][cols] sums of dz over K, or null
};

// out[col][d] = sum_k dz(k, col) * a[k][d].  ROWS: columns are rows of dz and K runs over the classes of the piece (dF);
// otherwise columns are classes and K runs over the valid rows (dW).
template <typename T, bool ROWS>
__global__ __launch_bounds__(VT, 2) void grad_kernel(GradArgs p) {
    __shared__ __align__(1024) char lds[4 * STAGE];
    constexpr int KE = 128 / sizeof(T);
    const int dtiles = (p.dim_pad + TILE - 1) / TILE;
    const int id = xcd_range(blockIdx.x, gridDim.x);
    const int d0 = (id % dtiles) * TILE;
    const long long ctiles = p.cols / TILE;
    const long long c0 = (id / dtiles) % ctiles * TILE;
    const int split = (int)(id / dtiles / ctiles);
    const int count = *p.count;
    if (ROWS && c0 >= count) return;
    long long ksteps = p.ksteps;
    if (!ROWS) ksteps = min(ksteps, (long long)(count + KE - 1) / KE);
    const long long k_first = ksteps * split / p.splits, k_end = ksteps * (split + 1) / p.splits;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
    const int wd = (wave & 1) * 64, wcol = (wave >> 1) * 64;

    StridedOperand<T> a, bs;
    ChunkedOperand bc;
    a.init(p.a, p.a_pitch, d0, p.dim_pad);
    if (ROWS) bc.init(p.dz, p.piece * (long long)sizeof(T), c0, p.cols - 1);
    else bs.init(p.dz, p.piece * (long long)sizeof(T), c0, p.piece);

    f32x16 acc[2][2];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[f][g][i] = 0.0f;
    float bias[2] = {0.0f, 0.0f};
    const bool want_bias = !ROWS && p.bias_out && d0 == 0 && wd == 0;

    auto stage = [&](char* to, long long k) {
        a.stage(to, k * KE, p.a_last);
        if (ROWS) bc.stage(to + STAGE, k * 128);
        else bs.stage(to + STAGE, k * KE, k * KE + KE);
    };
    int buf = 0;
    if (k_first < k_end) stage(lds, k_first);
    for (long long k = k_first; k < k_end; ++k) {
        stage_barrier();
        const char* now = lds + buf * 2 * STAGE;
        if (k + 1 < k_end) stage(lds + (buf ^ 1) * 2 * STAGE, k + 1);
        buf ^= 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 x[2], y[2];
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                x[f] = StridedOperand<T>::frag(now, wd + f * 32, j);
                y[f] = ROWS ? ChunkedOperand::frag(now + STAGE, wcol + f * 32, j)
                            : StridedOperand<T>::frag(now + STAGE, wcol + f * 32, j);
            }
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int g = 0; g < 2; ++g) acc[f][g] = Mma<T>::run(x[f], y[g], acc[f][g]);
            if (want_bias) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (sizeof(T) == 2) {
                            float lo, hi;
                            unpack2(y[g][w], lo, hi, (const T*)nullptr);
                            bias[g] += lo + hi;
                        } else {
                            bias[g] += u2f(y[g][w]);
                        }
                    }
            }
        }
    }
    float* out = p.out + ((long long)split * p.cols + c0) * p.dim_pad + d0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        float* line = out + (long long)(wcol + g * 32 + (lane & 31)) * p.dim_pad;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = wd + f * 32 + 8 * q + 4 * h;
                if (d0 + d >= p.dim_pad) continue;                  // dim_pad is a multiple of four
                vec4f v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[f][g][4 * q + e];
                vec4f* at = reinterpret_cast<vec4f*>(line + d);
                if (p.accumulate) v += *at;
                *at = v;
            }
        if (want_bias) {
            const float sum = bias[g] + __shfl_xor(bias[g], 32, 64);
            if (h == 0) p.bias_out[(long long)split * p.cols + c0 + wcol + g * 32 + lane] = sum;
        }
    }
}

// out[row][0 .. dim) = the splits' sum over line place[row] (or row itself), times scale[1]; zero where place < 0
template <typename T>
__global__ __launch_bounds__(VT) void finish_kernel(const float* __restrict__ part, long long cols, int splits, int dim,
                                                    int dim_pad, const int* __restrict__ place,
                                                    const float* __restrict__ scale, long long rows, T* __restrict__ out) {
    const int groups = (dim + 3) / 4;
    const long long at = (long long)blockIdx.x * VT + threadIdx.x;
    const long long row = at / groups;
    if (row >= rows) return;
    const int d = (int)(at % groups) * 4;
    const long long line = place ? place[row] : row;
    vec4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (line >= 0) {
        for (int s = 0; s < splits; ++s)
            v += *reinterpret_cast<const vec4f*>(part + ((long long)s * cols + line) * dim_pad + d);
        v *= scale[1];
    }
    T* to = out + row * dim + d;
    if (dim % 4 == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0) {
        const float f[4] = {v.x, v.y, v.z, v.w};
        store_vec<T, 4>(to, f);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < dim) to[i] = Elem<T>::from_float(v[i]);
    }
}

template <typename T>
__global__ __launch_bounds__(VT) void finish_bias_kernel(const float* __restrict__ part, long long cols, int splits,
                                                         const float* __restrict__ scale, long long classes,
                                                         T* __restrict__ out) {
    const long long v = (long long)blockIdx.x * VT + threadIdx.x;
    if (v >= classes) return;
    float sum = 0.0f;
    for (int s = 0; s < splits; ++s) sum += part[(long long)s * cols + v];
    out[v] = Elem<T>::from_float(sum * scale[1]);
}

// ---- host ---------------------------------------------------------------------------------------------------------
constexpr long long DZ_BYTES = 256ll << 20;     // size aimed at for a piece of dz
constexpr int FILL = 512;                       // workgroups that fill the chip: two per compute unit

long long up(long long v, long long to) { return (v + to - 1) / to * to; }
long long least(long long a, long long b) { return a < b ? a : b; }
long long most(long long a, long long b) { return a > b ? a : b; }
int elem_size(int dtype) { return dtype == OD_DTYPE_F32 ? 4 : 2; }

// Everything that follows from the sizes.
struct Plan {
    long long rows, rows_pad, classes, classes_pad;
    int dim, dim_pad, size, n;                  // n: targets per row
    int tiles, splits;                          // forward
    long long piece;                            // classes per piece
    int pieces, splits_f, splits_w;             // backward
    // saved buffer
    size_t o_count, o_row_of, o_place, o_lse, o_logit, o_prob, o_packed, saved;
    // forward's scratch
    size_t f_weight, f_bias, f_part, f_entropy, f_flags, forward;
    // backward's scratch
    size_t b_weight, b_bias, b_grad, b_scale, b_dz, b_part_f, b_part_w, b_part_b, backward;
};

size_t take(size_t& at, long long bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
}

bool plan_of(long long rows, long long classes, int dim, int top, int dtype, Plan& p) {
    p.size = elem_size(dtype);
    p.rows = rows;
    p.rows_pad = up(most(rows, 1), TILE);
    p.classes = classes;
    p.classes_pad = up(classes, TILE);
    p.dim = dim;
    p.dim_pad = (int)up(dim, 128 / p.size);
    // one thread per 16 bytes of the packed operands, fewer than 2^32 threads in a launch
    if (most(p.rows_pad, p.classes_pad) * p.dim_pad * p.size / 16 > (1ll << 31)) return false;
    p.n = top > 0 ? top : 1;
    p.tiles = (int)(p.classes_pad / TILE);
    const long long row_tiles = p.rows_pad / TILE;
    // splits of the classes: enough workgroups to fill the chip twice, in eights (one range per XCD) where there are tiles
    long long s = (2 * FILL + row_tiles - 1) / row_tiles;
    if (s > 1) s = up(s, 8);
    p.splits = (int)least(s, p.tiles);
    long long piece = most(TILE, DZ_BYTES / (p.rows_pad * p.size) / TILE * TILE);
    p.pieces = (int)((p.classes_pad + piece - 1) / piece);
    p.piece = up((p.classes_pad + p.pieces - 1) / p.pieces, TILE);
    p.pieces = (int)((p.classes_pad + p.piece - 1) / p.piece);
    const long long dtiles = (p.dim_pad + TILE - 1) / TILE;
    const long long ke = 128 / p.size;
    // splits of K where the result has too few tiles; at least eight steps each
    p.splits_f = (int)most(1, least((FILL + row_tiles * dtiles - 1) / (row_tiles * dtiles), p.piece / ke / 8));
    p.splits_w = (int)most(1, least((FILL + p.piece / TILE * dtiles - 1) / (p.piece / TILE * dtiles), p.rows_pad / ke / 8));

    size_t at = 0;
    p.o_count = take(at, 4);
    p.o_row_of = take(at, 4 * p.rows_pad);
    p.o_place = take(at, 4 * p.rows_pad);
    p.o_lse = take(at, 4 * p.rows_pad);
    p.o_logit = take(at, 4 * p.rows_pad * p.n);
    p.o_prob = take(at, top > 0 ? 4 * p.rows_pad * p.n : 0);
    p.o_packed = take(at, p.rows_pad * p.dim_pad * p.size);
    p.saved = at;

    at = 0;
    p.f_weight = take(at, p.classes * p.dim_pad * p.size);
    p.f_bias = take(at, 4 * p.classes_pad);
    p.f_part = take(at, 8 * p.rows_pad * p.splits);
    p.f_entropy = take(at, 4 * p.rows_pad);
    p.f_flags = take(at, p.rows_pad);
    p.forward = at;

    at = 0;
    p.b_weight = take(at, p.classes * p.dim_pad * p.size);
    p.b_bias = take(at, 4 * p.classes_pad + 4 * p.piece);
    p.b_grad = take(at, 4 * p.rows_pad);
    p.b_scale = take(at, 8);
    p.b_dz = take(at, p.rows_pad * p.piece * p.size);
    p.b_part_f = take(at, 4 * p.rows_pad * p.dim_pad * p.splits_f);
    p.b_part_w = take(at, 4 * p.piece * p.dim_pad * p.splits_w);
    p.b_part_b = take(at, 4 * p.piece * p.splits_w);
    p.backward = at;
    return true;
}

int check_call(int64_t rows, int64_t classes, int32_t dim, int32_t top, int32_t dtype, int32_t teacher_dtype,
               float temperature, int32_t reduction) {
    if (dtype < OD_DTYPE_F32 || dtype > OD_DTYPE_BF16 || teacher_dtype < OD_DTYPE_F32 || teacher_dtype > OD_DTYPE_BF16)
        return OD_ERR_ARG;
    if (rows < 0 || classes <= 0 || dim <= 0 || top < 0) return OD_ERR_ARG;
    if (!(temperature > 0.0f) || temperature > 3.0e38f || (top == 0 && temperature != 1.0f)) return OD_ERR_ARG;
    if (reduction < OD_REDUCE_NONE || reduction > OD_REDUCE_SUM) return OD_ERR_ARG;
    if (rows > OD_MAX_VOCAB_ROWS || classes > OD_MAX_VOCAB_CLASSES || dim > OD_MAX_VOCAB_DIM || top > OD_MAX_TEACHER_TOP)
        return OD_ERR_LIMIT;
    return OD_OK;
}

unsigned blocks_of(long long n, int per) { return (unsigned)((n + per - 1) / per); }

// Whether tiles can be read from the caller's weight rows: whole stages of K and 16-byte chunks.
bool weight_in_place(const Plan& p, const void* weight, long long pitch) {
    return p.dim == p.dim_pad && (pitch * p.size) % 16 == 0 && ((uintptr_t)weight & 15) == 0;
}

struct Call {
    Plan p;
    const void *features, *weight, *bias, *teacher_logits;
    long long feature_pitch, weight_pitch;
    const long long* targets;
    int top, teacher_dtype, reduction;
    float temperature;
    float *row_loss, *loss;
    const float* upstream;
    void *dfeatures, *dweight, *dbias;
    char *saved, *ws;
    hipStream_t stream;
};

// weight rows as the product reads them: in place, or packed into the scratch
template <typename T>
int weight_rows(const Call& c, size_t scratch, const char** rows, long long* pitch) {
    const Plan& p = c.p;
    if (weight_in_place(p, c.weight, c.weight_pitch)) {
        *rows = (const char*)c.weight;
        *pitch = c.weight_pitch * p.size;
        return OD_OK;
    }
    const long long chunks = p.classes * (p.dim_pad * p.size / 16);
    hipLaunchKernelGGL(pack_rows_kernel<T>, dim3(blocks_of(chunks, VT)), dim3(VT), 0, c.stream, (const T*)c.weight,
                       c.weight_pitch, p.dim, p.dim_pad, (const int*)nullptr, (const int*)nullptr, p.classes,
                       (T*)(c.ws + scratch));
    OD_LAUNCH_CHECK();
    *rows = c.ws + scratch;
    *pitch = (long long)p.dim_pad * p.size;
    return OD_OK;
}

RowLists lists_of(const Call& c) {
    return {(int*)(c.saved + c.p.o_count), (int*)(c.saved + c.p.o_row_of), (int*)(c.saved + c.p.o_place)};
}

template <typename T>
int forward_typed(const Call& c) {
    const Plan& p = c.p;
    const RowLists lists = lists_of(c);
    unsigned char* flags = nullptr;
    float* prob = (float*)(c.saved + p.o_prob);
    float* entropy = (float*)(c.ws + p.f_entropy);
    if (c.top > 0) {
        flags = (unsigned char*)(c.ws + p.f_flags);
        const dim3 grid(blocks_of(p.rows, VT / 64));
        const float inv = 1.0f / c.temperature;
        if (c.teacher_dtype == OD_DTYPE_F32)
            hipLaunchKernelGGL(teacher_kernel<float>, grid, dim3(VT), 0, c.stream, c.targets, (const float*)c.teacher_logits,
                               (int)p.rows, c.top, inv, prob, entropy, flags);
        else if (c.teacher_dtype == OD_DTYPE_F16)
            hipLaunchKernelGGL(teacher_kernel<_Float16>, grid, dim3(VT), 0, c.stream, c.targets,
                               (const _Float16*)c.teacher_logits, (int)p.rows, c.top, inv, prob, entropy, flags);
        else
            hipLaunchKernelGGL(teacher_kernel<bf16_t>, grid, dim3(VT), 0, c.stream, c.targets,
                               (const bf16_t*)c.teacher_logits, (int)p.rows, c.top, inv, prob, entropy, flags);
        OD_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(list_rows_kernel, dim3(1), dim3(1024), 0, c.stream, c.targets, (const unsigned char*)flags, (int)p.rows,
                       lists, c.row_loss);
    OD_LAUNCH_CHECK();
    const long long chunks = p.rows_pad * (p.dim_pad * p.size / 16);
    hipLaunchKernelGGL(pack_rows_kernel<T>, dim3(blocks_of(chunks, VT)), dim3(VT), 0, c.stream, (const T*)c.features,
                       c.feature_pitch, p.dim, p.dim_pad, (const int*)lists.row_of, (const int*)lists.count, p.rows_pad,
                       (T*)(c.saved + p.o_packed));
    OD_LAUNCH_CHECK();
    const float scale = LOG2E / c.temperature;
    hipLaunchKernelGGL(bias_kernel<T>, dim3(blocks_of(p.classes_pad, VT)), dim3(VT), 0, c.stream, (const T*)c.bias,
                       (int)p.classes, (int)p.classes_pad, scale, (float*)(c.ws + p.f_bias));
    OD_LAUNCH_CHECK();
    ProductArgs a = {};
    const int rc = weight_rows<T>(c, p.f_weight, &a.weight, &a.weight_pitch);
    if (rc != OD_OK) return rc;
    a.features = c.saved + p.o_packed;
    a.dim_pad = p.dim_pad;
    a.first_class = 0;
    a.last_class = p.classes - 1;
    a.bias2 = (const float*)(c.ws + p.f_bias);
    a.count = lists.count;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.scale = scale;
    a.rows_pad = p.rows_pad;
    a.part = (float2*)(c.ws + p.f_part);
    OD_LAUNCH_KERNEL(OD_KERNEL_VOCAB_LSE, (product_kernel<T, false>), dim3((unsigned)(p.rows_pad / TILE * p.splits)), dim3(VT),
                     0, c.stream, a);
    TargetArgs t = {};
    t.features = a.features;
    t.dim = p.dim;
    t.dim_pad = p.dim_pad;
    t.weight = c.weight;
    t.weight_pitch = c.weight_pitch;
    t.bias = c.bias;
    t.classes = p.classes;
    t.targets = c.targets;
    t.top = c.top;
    t.prob = prob;
    t.entropy = entropy;
    t.lists = lists;
    t.part = a.part;
    t.splits = p.splits;
    t.rows_pad = p.rows_pad;
    t.temperature = c.temperature;
    t.lse2 = (float*)(c.saved + p.o_lse);
    t.target_logit = (float*)(c.saved + p.o_logit);
    t.row_loss = c.row_loss;
    hipLaunchKernelGGL(targets_kernel<T>, dim3(blocks_of(p.rows_pad, VT / 64)), dim3(VT), 0, c.stream, t);
    OD_LAUNCH_CHECK();
    if (c.reduction != OD_REDUCE_NONE) {
        hipLaunchKernelGGL(sum_rows_kernel, dim3(1), dim3(1024), 0, c.stream, (const float*)c.row_loss, (int)p.rows,
                           (const int*)lists.count, c.reduction, c.loss);
        OD_LAUNCH_CHECK();
    }
    return OD_OK;
}

template <typename T>
int backward_typed(const Call& c) {
    const Plan& p = c.p;
    const RowLists lists = lists_of(c);
    float* row_grad = (float*)(c.ws + p.b_grad);
    float* scale = (float*)(c.ws + p.b_scale);
    hipLaunchKernelGGL(row_grads_kernel, dim3(1), dim3(1024), 0, c.stream, c.upstream, c.reduction, lists, p.rows_pad,
                       c.temperature, (int)std::is_same<T, _Float16>::value, row_grad, scale);
    OD_LAUNCH_CHECK();
    const float log2_scale = LOG2E / c.temperature;
    const long long bias_len = p.classes_pad + p.piece;             // the last piece may reach past the last tile
    hipLaunchKernelGGL(bias_kernel<T>, dim3(blocks_of(bias_len, VT)), dim3(VT), 0, c.stream, (const T*)c.bias,
                       (int)p.classes, (int)bias_len, log2_scale, (float*)(c.ws + p.b_bias));
    OD_LAUNCH_CHECK();
    ProductArgs a = {};
    const int rc = weight_rows<T>(c, p.b_weight, &a.weight, &a.weight_pitch);
    if (rc != OD_OK) return rc;
    a.features = c.saved + p.o_packed;
    a.dim_pad = p.dim_pad;
    a.last_class = p.classes - 1;
    a.count = lists.count;
    a.tiles = (int)(p.piece / TILE);
    const long long row_tiles = p.rows_pad / TILE;
    long long s = (4 * FILL + row_tiles - 1) / row_tiles;
    a.splits = (int)most(1, least(s, a.tiles));
    a.scale = log2_scale;
    a.rows_pad = p.rows_pad;
    a.lse2 = (const float*)(c.saved + p.o_lse);
    a.row_grad = row_grad;
    a.dz = c.ws + p.b_dz;
    a.piece = p.piece;
    const int dtiles = (p.dim_pad + TILE - 1) / TILE;
    const int ke = 128 / p.size;
    for (int k = 0; k < p.pieces; ++k) {
        const long long first = k * p.piece;
        a.first_class = first;
        a.bias2 = (const float*)(c.ws + p.b_bias) + first;
        OD_LAUNCH_KERNEL(OD_KERNEL_VOCAB_DZ, (product_kernel<T, true>), dim3((unsigned)(row_tiles * a.splits)), dim3(VT), 0,
                         c.stream, a);
        hipLaunchKernelGGL(correct_targets_kernel<T>, dim3(blocks_of(p.rows * p.n, VT)), dim3(VT), 0, c.stream, c.targets,
                           c.top, (const float*)(c.saved + p.o_prob), lists, a.lse2,
                           (const float*)(c.saved + p.o_logit), (const float*)row_grad, first, p.piece, p.classes,
                           (T*)(c.ws + p.b_dz));
        OD_LAUNCH_CHECK();
        GradArgs g = {};
        g.dz = c.ws + p.b_dz;
        g.piece = p.piece;
        g.dim_pad = p.dim_pad;
        g.count = lists.count;
        if (c.dfeatures) {
            g.a = a.weight + first * a.weight_pitch;
            g.a_pitch = a.weight_pitch;
            g.a_last = p.classes - 1 - first;
            g.cols = p.rows_pad;
            g.ksteps = p.piece / ke;
            g.splits = p.splits_f;
            g.out = (float*)(c.ws + p.b_part_f);
            g.accumulate = k > 0;
            OD_LAUNCH_KERNEL(OD_KERNEL_VOCAB_GRAD_ROWS, (grad_kernel<T, true>),
                             dim3((unsigned)(dtiles * row_tiles * g.splits)), dim3(VT), 0, c.stream, g);
        }
        if (c.dweight || c.dbias) {
            g.a = a.features;
            g.a_pitch = (long long)p.dim_pad * p.size;
            g.a_last = p.rows_pad - 1;
            g.cols = p.piece;
            g.ksteps = p.rows_pad / ke;
            g.splits = p.splits_w;
            g.out = (float*)(c.ws + p.b_part_w);
            g.accumulate = 0;
            g.bias_out = c.dbias ? (float*)(c.ws + p.b_part_b) : nullptr;
            OD_LAUNCH_KERNEL(OD_KERNEL_VOCAB_GRAD_CLASSES, (grad_kernel<T, false>),
                             dim3((unsigned)(dtiles * (p.piece / TILE) * g.splits)), dim3(VT), 0, c.stream, g);
            const long long here = least(p.piece, p.classes - first);
            if (c.dweight) {
                hipLaunchKernelGGL(finish_kernel<T>, dim3(blocks_of(here * ((p.dim + 3) / 4), VT)), dim3(VT), 0, c.stream,
                                   (const float*)g.out, p.piece, p.splits_w, p.dim, p.dim_pad, (const int*)nullptr,
                                   (const float*)scale, here, (T*)c.dweight + first * p.dim);
                OD_LAUNCH_CHECK();
            }
            if (c.dbias) {
                hipLaunchKernelGGL(finish_bias_kernel<T>, dim3(blocks_of(here, VT)), dim3(VT), 0, c.stream,
                                   (const float*)g.bias_out, p.piece, p.splits_w, (const float*)scale, here,
                                   (T*)c.dbias + first);
                OD_LAUNCH_CHECK();
            }
        }
    }
    if (c.dfeatures) {
        hipLaunchKernelGGL(finish_kernel<T>, dim3(blocks_of(p.rows * ((p.dim + 3) / 4), VT)), dim3(VT), 0, c.stream,
                           (const float*)(c.ws + p.b_part_f), p.rows_pad, p.splits_f, p.dim, p.dim_pad,
                           (const int*)lists.place, (const float*)scale, p.rows, (T*)c.dfeatures);
        OD_LAUNCH_CHECK();
    }
    return OD_OK;
}

}  // namespace

extern "C" size_t od_vocab_loss_saved_bytes(int64_t rows, int64_t classes, int32_t dim, int32_t top, int32_t dtype) {
    if (check_call(rows, classes, dim, top, dtype, dtype, 1.0f, 0) != OD_OK) return 0;
    Plan p;
    return plan_of(rows, classes, dim, top, dtype, p) ? p.saved : 0;
}

extern "C" size_t od_vocab_loss_workspace_bytes(int64_t rows, int64_t classes, int32_t dim, int32_t top, int32_t dtype,
                                                int32_t backward) {
    if (check_call(rows, classes, dim, top, dtype, dtype, 1.0f, 0) != OD_OK) return 0;
    Plan p;
    if (!plan_of(rows, classes, dim, top, dtype, p)) return 0;
    return backward ? p.backward : p.forward;
}

extern "C" int od_vocab_loss_forward(const void* features, int64_t feature_pitch, const void* weight, int64_t weight_pitch,
                                     const void* bias, int32_t dtype, int64_t rows, int64_t classes, int32_t dim,
                                     const int64_t* targets, int32_t top, const void* teacher_logits, int32_t teacher_dtype,
                                     float temperature, int32_t reduction, float* row_loss, float* loss, void* saved,
                                     size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_call(rows, classes, dim, top, dtype, teacher_dtype, temperature, reduction);
    if (rc != OD_OK) return rc;
    Call c = {};
    if (!plan_of(rows, classes, dim, top, dtype, c.p)) return OD_ERR_LIMIT;
    if (!weight || (rows > 0 && !row_loss) || !saved || !workspace || ((uintptr_t)saved & 255) || ((uintptr_t)workspace & 255) ||
        (reduction != OD_REDUCE_NONE && !loss))
        return OD_ERR_ARG;
    if (rows > 0 && (!features || !targets || (top > 0 && !teacher_logits))) return OD_ERR_ARG;
    if (feature_pitch < dim || weight_pitch < dim) return OD_ERR_ARG;
    if (((uintptr_t)features | (uintptr_t)weight | (uintptr_t)bias) % c.p.size) return OD_ERR_ARG;
    if (saved_bytes < c.p.saved || workspace_bytes < c.p.forward) return OD_ERR_WORKSPACE;
    if (rows == 0 && reduction == OD_REDUCE_NONE) return OD_OK;
    c.features = features;
    c.feature_pitch = feature_pitch;
    c.weight = weight;
    c.weight_pitch = weight_pitch;
    c.bias = bias;
    c.targets = (const long long*)targets;
    c.top = rows > 0 ? top : 0;
    c.teacher_logits = teacher_logits;
    c.teacher_dtype = teacher_dtype;
    c.temperature = temperature;
    c.reduction = reduction;
    c.row_loss = row_loss;
    c.loss = loss;
    c.saved = (char*)saved;
    c.ws = (char*)workspace;
    c.stream = (hipStream_t)stream;
    if (dtype == OD_DTYPE_F32) return forward_typed<float>(c);
    if (dtype == OD_DTYPE_F16) return forward_typed<_Float16>(c);
    return forward_typed<bf16_t>(c);
}

extern "C" int od_vocab_loss_backward(const void* weight, int64_t weight_pitch, const void* bias, int32_t dtype, int64_t rows,
                                      int64_t classes, int32_t dim, const int64_t* targets, int32_t top, float temperature,
                                      int32_t reduction, const float* upstream, const void* saved, size_t saved_bytes,
                                      void* dfeatures, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    const int rc = check_call(rows, classes, dim, top, dtype, dtype, temperature, reduction);
    if (rc != OD_OK) return rc;
    Call c = {};
    if (!plan_of(rows, classes, dim, top, dtype, c.p)) return OD_ERR_LIMIT;
    if (rows == 0) return OD_OK;
    if (!weight || !targets || !upstream || !saved || !workspace || ((uintptr_t)saved & 255) || ((uintptr_t)workspace & 255))
        return OD_ERR_ARG;
    if (weight_pitch < dim) return OD_ERR_ARG;
    if (((uintptr_t)weight | (uintptr_t)bias | (uintptr_t)dfeatures | (uintptr_t)dweight | (uintptr_t)dbias) % c.p.size)
        return OD_ERR_ARG;
    if (saved_bytes < c.p.saved || workspace_bytes < c.p.backward) return OD_ERR_WORKSPACE;
    c.weight = weight;
    c.weight_pitch = weight_pitch;
    c.bias = bias;
    c.targets = (const long long*)targets;
    c.top = top;
    c.temperature = temperature;
    c.reduction = reduction;
    c.upstream = upstream;
    c.saved = (char*)saved;
    c.dfeatures = dfeatures;
    c.dweight = dweight;
    c.dbias = dbias;
    c.ws = (char*)workspace;
    c.stream = (hipStream_t)stream;
    if (dtype == OD_DTYPE_F32) return backward_typed<float>(c);
    if (dtype == OD_DTYPE_F16) return backward_typed<_Float16>(c);
    return backward_typed<bf16_t>(c);
}
