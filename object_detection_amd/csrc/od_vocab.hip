// Losses of a classification head whose classes are a large vocabulary of embeddings: softmax cross entropy and
// distillation from a teacher's top logits, with their gradients, without the [rows, classes] logits ever being kept.
//
//   z = (F W^T + b) / T            F [rows, dim], W [classes, dim], b [classes]
//   q = softmax(z) over the classes, lse = log sum exp z
//   target distribution p of a row: one class (cross entropy, T = 1), or softmax(t / T) over the classes a teacher names
//   loss_n = T^2 (sum p log p - sum p z_class + lse)
//   dz = g T (q - p), g the gradient of the row's loss;   dF = dz W,  dW = dz^T F,  db = sum_n dz
//
// Forward: one product whose epilogue folds each tile of logits into a running maximum and sum per row, in the lane that
// owns the row: nothing passes between lanes before the end.  The classes are split over workgroups; a second kernel joins
// the splits and forms the few logits of the targets by dot products.
// Backward: the classes are taken in pieces.  A piece's dz is recomputed from the saved lse into a buffer of 256 MB, or of 256
// classes for every row where that is more (from 524288 rows on in 16 bits, half of that in 32; 4 and 8 GiB at the limit of
// rows); its target entries are corrected, and the two products that read it, dF and dW, accumulate in fp32.
// Operands of those two products, for 16-bit inputs: dz, features and weight in fp16, dz times 2^14 and the others (bf16, or
// weighted by a gradient per row) under one power of two each, which brings the largest value to [2^13, 2^14).  dz has 11
// bits down to 2^-28 of a row's gradient and none below 2^-39.  Its rounding and the final one are independent: bf16 gradients
// lie 1.00 final roundings off the exact ones (dz in bf16 would make it 1.4), fp16 gradients 1.2 to 1.4 (dz in fp32 would
// make it 1.0, for twice the traffic of the buffer and a sixth of the matrix rate).  bf16 values no more than 2^27 times smaller
// than the largest come through unchanged; the powers of two leave in the fp32 results.
//
// Rows without a target (negative class; no finite teacher entry) are left out at the start: the valid rows are listed in
// order and their features packed densely, so that whatever masked rows hold (infinities, NaN) reaches no product.  The
// products cost what the valid rows cost; buffers and the width of a piece are sized for all rows, since the host does not
// know how many are valid: where nearly all are masked, taking the valid rows out beforehand makes for fewer pieces (786240 x
// 32000 x 256 bf16 with 0.2 % valid: 7.4 ms a step in 125 pieces, 0.4 with the rows taken out).  All sums run in a fixed
// order; the only atomics are maxima and sums of integers, whose order changes nothing.
//
// A product of n rows, V classes and dim D costs 2 n V D operations, four times a training step (forward, dz again, dF, dW).
#include "od_common.h"
#include "../../include/od_boxes.h"
#include "od_elem.h"

#pragma clang fp contract(fast)

namespace {

using namespace od;

constexpr int VT = 256;                 // threads per workgroup (twice that in the gradient products)
constexpr int TILE = 128;               // rows and classes of a workgroup's tile where both operands stream
constexpr int ROW_TILE = 256;           // rows and classes are padded to this: tiles of every kernel divide it
constexpr int STAGE = TILE * 128;       // bytes of one operand's stage in LDS
constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.69314718055994531f;
constexpr float LOWEST = -3.402823466e38f;      // start of a running maximum: finite, so that -inf - LOWEST stays -inf

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// An operand of the matrix units: 32 rows (lane % 32) x 16 of K, eight per lane (halves lane / 32).  It is read as slabs of
// 32 bytes of K, 16 bytes per lane: one slab in 16 bits, two in fp32.  Any assignment of K to the slots of a fragment gives
// the same product as long as both operands use it.
//
// fp32 products by bf16 matrix instructions: x = h + m + l, each the nearest bf16 to what is left, h within 2^-9 of x, m
// within 2^-9 of the rest, l 2^-9 again, so that 24 bits are there exactly.  Of the nine products the three smallest, below
// 2^-25 of the whole together, are left out, half of what rounding each product to fp32 would cost; sums are fp32 as ever.
// Six instructions of 32 cycles do 16 of K, for which the fp32 instruction takes 512 cycles; taking the operands apart, 11
// vector instructions for two elements, runs beside them and bounds the product.  A training step of 4096 x 8000 x 512, a
// tenth of the rows left out, 802 us instead of 1115, of 21577 x 4938 x 128 806 instead of 1372.  What rounds to an infinite
// h (from 3.39e38 on) gives NaN.
template <typename T> struct Fragment {
    static constexpr int SLABS = 1, PRODUCTS = 1;                   // of K; matrix instructions per product of fragments
    u32x4 v;
    __device__ __forceinline__ void set(const u32x4 (&slab)[1]) { v = slab[0]; }
};
template <> struct Fragment<float> {
    static constexpr int SLABS = 2, PRODUCTS = 6;
    u32x4 h, m, l;
    __device__ __forceinline__ void set(const u32x4 (&slab)[2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = u2f(slab[i >> 1][2 * (i & 1)]), y = u2f(slab[i >> 1][2 * (i & 1) + 1]), a, b;
            h[i] = pack2(x, y, (const bf16_t*)nullptr);
            unpack2(h[i], a, b, (const bf16_t*)nullptr);
            x -= a;
            y -= b;
            m[i] = pack2(x, y, (const bf16_t*)nullptr);
            unpack2(m[i], a, b, (const bf16_t*)nullptr);
            l[i] = pack2(x - a, y - b, (const bf16_t*)nullptr);
        }
    }
};

__device__ __forceinline__ f32x16 mma_bf16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Fragment<bf16_t>& a, const Fragment<bf16_t>& b, f32x16 c) {
    return mma_bf16(a.v, b.v, c);
}
__device__ __forceinline__ f32x16 mma(const Fragment<_Float16>& a, const Fragment<_Float16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a.v), __builtin_bit_cast(h16x8, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Fragment<float>& a, const Fragment<float>& b, f32x16 c) {
    c = mma_bf16(a.l, b.h, c);                                      // the small ones first
    c = mma_bf16(a.h, b.l, c);
    c = mma_bf16(a.m, b.m, c);
    c = mma_bf16(a.m, b.h, c);
    c = mma_bf16(a.h, b.m, c);
    return mma_bf16(a.h, b.h, c);
}

typedef __attribute__((address_space(3))) char lds_char;
typedef const __attribute__((address_space(1))) uint32_t* global_words;

__device__ __forceinline__ long long up_to(long long v, int to) { return (v + to - 1) / to * to; }

// 16 bytes per lane from global memory straight into LDS: lane l lands at base + 16 l
__device__ __forceinline__ void stage16(const char* src, char* base) {
    __builtin_amdgcn_global_load_lds((global_words)src, (__attribute__((address_space(3))) uint32_t*)base, 16, 0, 0);
}

// A tile of classes is the A operand, whose 32 rows reach a lane's accumulators in four groups of four; reading tile row
// class_row(r) as row r of the operand makes them 16 neighbouring classes: acc[i] is class 16 (lane / 32) + i of the 32.
__device__ __forceinline__ int class_row(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

// LDS serves 16 lanes of a 16-byte read at a time, from 64 banks.  The 16-byte chunks of a tile row are permuted by an
// exclusive-or with a function of the row under which those 16 lanes' chunks lie in 16 different bank groups: for the row
// order of class_row (rows 0-3, 16-19, 4-7, 20-23, ...), and for rows in order.
// ROW bytes a row: a multiple of 256 needs four bits; an odd multiple of 128 has one from the row's own parity.
template <int ROW>
__device__ __forceinline__ int class_swizzle(int r) {
    return ROW % 256 == 0 ? ((r & 7) | (((r >> 4) & 1) << 3)) : (((r >> 1) & 3) | (((r >> 4) & 1) << 2));
}
__device__ __forceinline__ int line_swizzle(int r) { return (r >> 1) & 7; }     // rows of 128 bytes, in order

// ---- operand with K contiguous, streamed: R rows x 128 bytes of K per stage, by THREADS threads
template <int R, int THREADS, bool CLASSES>
struct ChunkedOperand {
    static constexpr int PASSES = R * 8 / THREADS;
    const char* base;                   // the tile's first row
    uint32_t offset[PASSES];            // this lane's rows and chunks, within 31 bits
    __device__ __forceinline__ void init(const char* from, long long pitch, long long first, long long last) {
        first = min(first, last);                                   // a tile wholly behind the last row
        base = from + first * pitch;
        const int most = (int)min(last - first, (long long)R);      // rows past the last one repeat it
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = (i * THREADS + threadIdx.x) >> 3;
            const int swz = CLASSES ? class_swizzle<128>(r) : line_swizzle(r);
            offset[i] = (uint32_t)min(r, most) * (uint32_t)pitch + (((threadIdx.x & 7) ^ swz) << 4);
        }
    }
    __device__ __forceinline__ void stage(char* lds, long long kbytes) const {
        const char* from = base + kbytes;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) stage16(from + offset[i], lds + i * THREADS * 16 + (threadIdx.x >> 6) * 1024);
    }
    // fragment of rows [r0, r0 + 32), slab j of four
    static __device__ __forceinline__ u32x4 frag(const char* lds, int r0, int j, int lane) {
        const int r = r0 + (CLASSES ? class_row(lane & 31) : (lane & 31));
        const int swz = CLASSES ? class_swizzle<128>(r) : line_swizzle(r);
        return *reinterpret_cast<const u32x4*>(lds + r * 128 + (((2 * j + (lane >> 5)) ^ swz) << 4));
    }
};

// ---- operand with K strided, streamed: KE rows of K x W contiguous elements per stage; read transposed.
template <typename T, int W, int THREADS>
struct StridedOperand {
    static constexpr int KE = 128 / sizeof(T);                      // K per stage
    static constexpr int ROWB = W * sizeof(T);                      // bytes per K row
    static constexpr int CHUNKS = ROWB / 16;
    static constexpr int PASSES = KE * CHUNKS / THREADS;
    const char* base;
    long long pitch;
    uint32_t offset[PASSES];            // this lane's rows and columns of a stage, within 31 bits
    // Chunk permutation of K row k.  16-bit: a transposing read takes two neighbouring 32-byte pieces of four rows at a
    // time; they land in eight different bank groups.  fp32: two rows, four apart, 128 bytes each.
    static __device__ __forceinline__ int swizzle(int k) {
        if (sizeof(T) == 4) return ((k >> 2) & 1) << 3;
        return ROWB % 256 == 0 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
    }
    static __device__ __forceinline__ uint32_t column(int i, uint32_t first_byte, uint32_t last) {
        const int at = i * THREADS + threadIdx.x;
        const uint32_t c = first_byte + (((at % CHUNKS) ^ swizzle(at / CHUNKS)) << 4);
        return c < last ? c : last;                                 // columns past the end repeat the last chunk
    }
    uint32_t first_byte, last_byte;
    __device__ __forceinline__ void init(const char* b, long long p, long long first_col, long long cols) {
        base = b;
        pitch = p;
        first_byte = (uint32_t)(first_col * (long long)sizeof(T));
        last_byte = (uint32_t)(cols * (long long)sizeof(T)) - 16;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
            offset[i] = (uint32_t)((i * THREADS + threadIdx.x) / CHUNKS) * (uint32_t)p + column(i, first_byte, last_byte);
    }
    // K rows [k0, k0 + KE); rows past `last` repeat it
    __device__ __forceinline__ void stage(char* lds, long long k0, long long last) const {
        const char* from = base + k0 * pitch;
        if (k0 + KE - 1 <= last) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) stage16(from + offset[i], lds + i * THREADS * 16 + (threadIdx.x >> 6) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int r = min((i * THREADS + (int)threadIdx.x) / CHUNKS, (int)(last - k0));
                stage16(from + (r * pitch + column(i, first_byte, last_byte)),
                        lds + i * THREADS * 16 + (threadIdx.x >> 6) * 1024);
            }
        }
    }
    // fragment of columns [m0, m0 + 32), slab j of four
    static __device__ __forceinline__ u32x4 frag(const char* lds, int m0, int j, int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // a transposing read hands lane i of 16 the i-th element of the four rows that lanes 4r .. 4r+3 point at
            const int r = (lane & 15) >> 2;
            const int chunk = (m0 >> 3) + (((lane >> 4) & 1) << 1) + ((lane & 3) >> 1);
            const char* p = lds + (16 * j + 8 * h + r) * ROWB + ((chunk ^ swizzle(r)) << 4) + ((lane & 1) << 3);
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

// Order of a stage's instructions: `ahead` LDS reads first, then `steps` times `mfma` products and `reads` further reads.
template <int AHEAD, int STEPS, int PRODUCTS, int READS>
__device__ __forceinline__ void interleave() {
    constexpr int READ = 0x100, MFMA = 0x008;
    __builtin_amdgcn_sched_group_barrier(READ, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(MFMA, PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(READ, READS, 0);
    }
}

// Workgroup number -> work number such that each of the eight XCDs (hardware hands workgroups to them in turn) gets one
// contiguous range: neighbours share their operands in one L2.
__device__ __forceinline__ int xcd_range(int id, int total) {
    const int per = total / 8;
    return id < per * 8 ? (id % 8) * per + id / 8 : id;
}

// ---- preparation --------------------------------------------------------------------------------------------------
// Number of valid rows, their list and each row's place in it, in row order; clears row_loss.
// A row is valid if its flag is set (distillation) or its target is not negative.
struct RowLists {
    int* count;
    int* row_of;                        // [rows] valid rows in order
    int* place;                         // [rows] index into row_of, or -1
};

__device__ __forceinline__ bool row_counts(const long long* targets, const unsigned char* flags, long long r) {
    return flags ? flags[r] != 0 : targets[r] >= 0;
}

// PER * VT rows from `first` on, by one workgroup: lists them behind `before` others.  `write`: whether the lists are wanted in
// memory; s_row_of, if not null, gets them too.  Returns the number of valid ones.
template <int PER>
__device__ __forceinline__ int list_rows(const long long* targets, const unsigned char* flags, long long first, int rows,
                                         int before, const RowLists& lists, float* row_loss, bool write, int* s_row_of) {
    constexpr int WAVES = VT / 64;
    static_assert(PER * WAVES <= 64, "one lane per 64 rows");
    __shared__ int s_count[PER * WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned long long valid[PER];                                  // of 64 neighbouring rows
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long r = first + i * VT + threadIdx.x;
        valid[i] = __ballot(r < rows && row_counts(targets, flags, r));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane == 0) s_count[i * WAVES + wave] = __popcll(valid[i]);
    __syncthreads();
    const int n = lane < PER * WAVES ? s_count[lane] : 0;
    const int upto = (int)wave_scan_incl((uint32_t)n);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long r = first + i * VT + threadIdx.x;
        const int at = before + __shfl(upto - n, i * WAVES + wave, 64) + __popcll(valid[i] & ((1ull << lane) - 1));
        const bool on = (valid[i] >> lane) & 1;
        if (write && r < rows) {
            lists.place[r] = on ? at : -1;
            row_loss[r] = 0.0f;
        }
        if (on) {
            if (s_row_of) s_row_of[at] = (int)r;
            if (write) lists.row_of[at] = (int)r;
        }
    }
    return __shfl(upto, 63, 64);
}

// Many rows: 4096 per workgroup, counted by a first launch and listed by a second (32768 rows: 17 us; one workgroup for
// all of them took 99).
constexpr int LIST_ROWS = 16 * VT;

__global__ __launch_bounds__(VT) void count_rows_kernel(const long long* __restrict__ targets,
                                                        const unsigned char* __restrict__ flags, int rows,
                                                        int* __restrict__ counts) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < LIST_ROWS / VT; ++i) {
        const long long r = (long long)blockIdx.x * LIST_ROWS + i * VT + threadIdx.x;
        n += r < rows && row_counts(targets, flags, r) ? 1 : 0;
    }
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    __shared__ int s_sum[VT / 64];
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VT / 64; ++w) n += s_sum[w];
        counts[blockIdx.x] = n;
    }
}

__global__ __launch_bounds__(VT) void list_rows_kernel(const long long* __restrict__ targets,
                                                       const unsigned char* __restrict__ flags, int rows,
                                                       const int* __restrict__ counts, RowLists lists,
                                                       float* __restrict__ row_loss) {
    __shared__ int s_before;
    if (threadIdx.x == 0) s_before = 0;
    __syncthreads();
    int before = 0;
    for (int b = threadIdx.x; b < (int)blockIdx.x; b += VT) before += counts[b];
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
    if ((threadIdx.x & 63) == 0 && before > 0) atomicAdd(&s_before, before);
    __syncthreads();
    before = s_before;
    const int n = list_rows<LIST_ROWS / VT>(targets, flags, (long long)blockIdx.x * LIST_ROWS, rows, before, lists, row_loss,
                                            true, nullptr);
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *lists.count = before + n;
}

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Teacher's distribution of a row over its listed classes, one wave per row: p = softmax(t / T) over the entries with a
// class >= 0 and a logit above -inf.  Entries that name the same class are one class: the first of them gets the sum, the
// others 0, and the entropy term sum p log p is the merged distribution's.
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

// Scalars of a backward call, on the device.
struct Scales {
    float common;                       // largest |upstream| times share and temperature
    uint32_t features_max, weight_max;  // bits of the largest finite |weighted feature| and |weight|
};

// What the product reads, by one launch: features of the valid rows, weight rows where the caller's cannot be read in
// place, and the bias.
struct PrepareArgs {
    // features: dense, [rows rounded up to ROW_TILE][dim_pad], zero behind the last valid row and the last column
    const void* features;
    long long feature_pitch;
    void* packed;
    long long rows_pad;
    RowLists lists;
    // weight: [classes][dim_pad], zero behind the last column
    const void* weight;
    long long weight_pitch, classes;
    void* packed_weight;
    // bias in units of log2, -inf behind the last class: the tiles' tail then drops out of maxima and sums by itself
    const void* bias;
    int bias_len;
    float scale;
    float* bias2;
    int dim, dim_pad;
    unsigned feature_blocks, weight_blocks;
    // few rows: the lists are made here, by every workgroup for itself, instead of by a launch of their own
    const long long* targets;
    const unsigned char* flags;
    int rows;
    float* row_loss;
    // backward: the scalars of a call whose rows share one gradient
    Scales* scales;
    const float* upstream;
    int reduction;
    float temperature;
};

// 16 bytes of a packed row; a source that is not aligned for it is read element by element
template <typename T>
__device__ __forceinline__ void pack_chunk(const T* row, int c, int dim, T* dst) {
    constexpr int E = 16 / sizeof(T);
    alignas(16) T v[E];
    const T* p = row + c;
    if (row && c + E <= dim && ((uintptr_t)p & 15) == 0) {
        *reinterpret_cast<u32x4*>(v) = *reinterpret_cast<const u32x4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = row && c + i < dim ? p[i] : Elem<T>::from_float(0.0f);
    }
    *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(v);
}

// SCAN: rows per thread that a workgroup lists for itself; 0: they are listed already
template <typename T, int SCAN>
__global__ __launch_bounds__(VT) void prepare_kernel(PrepareArgs p) {
    constexpr int E = 16 / sizeof(T);
    const unsigned chunks = p.dim_pad / E;
    unsigned block = blockIdx.x;
    if (block < p.feature_blocks) {
        __shared__ int s_row_of[SCAN ? SCAN * VT : 1];
        int count;
        if constexpr (SCAN > 0) {
            count = list_rows<SCAN>(p.targets, p.flags, 0, p.rows, 0, p.lists, p.row_loss, block == 0, s_row_of);
            if (block == 0 && threadIdx.x == 0) *p.lists.count = count;
            __syncthreads();
        } else {
            count = *p.lists.count;
        }
        const unsigned at = block * VT + threadIdx.x;
        const long long r = at / chunks;
        if (r >= p.rows_pad || r >= up_to(count, ROW_TILE)) return;     // no tile reads behind the last one's end
        const int c = (int)(at % chunks) * E;
        const T* row = r < count ? (const T*)p.features + (long long)(SCAN ? s_row_of[r] : p.lists.row_of[r]) * p.feature_pitch
                                 : nullptr;
        pack_chunk<T>(row, c, p.dim, (T*)p.packed + r * p.dim_pad + c);
        return;
    }
    block -= p.feature_blocks;
    if (block < p.weight_blocks) {
        const unsigned at = block * VT + threadIdx.x;
        const long long r = at / chunks;
        if (r >= p.classes) return;
        const int c = (int)(at % chunks) * E;
        pack_chunk<T>((const T*)p.weight + r * p.weight_pitch, c, p.dim, (T*)p.packed_weight + r * p.dim_pad + c);
        return;
    }
    block -= p.weight_blocks;
    const int v = (int)block * VT + threadIdx.x;
    if (v < p.bias_len)
        p.bias2[v] = v >= p.classes ? -__builtin_inff() : p.bias ? Elem<T>::to_float(((const T*)p.bias)[v]) * p.scale : 0.0f;
    if (p.scales && v == 0) {
        const float share = p.reduction == OD_REDUCE_MEAN ? (float)max(1, *p.lists.count) : 1.0f;
        p.scales->common = p.upstream[0] * (p.temperature / share);
        p.scales->features_max = 0;
        p.scales->weight_max = 0;
    }
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
    int tiles, groups;                  // class tiles of the piece, groups of workgroups that share them out
    int row_tiles;                      // of all rows
    float scale;                        // log2(e) / temperature
    // forward
    float2* part;                       // [segment][rows of a tile] (maximum, sum) in log2 units, see Share
    int2* ends;                         // [groups][row_tiles]
    // backward
    const float* lse2;                  // [rows_pad] in log2 units
    void* dz;                           // rows_pad x piece, see Dz
    long long piece;
};

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
    return (long long)(((unsigned long long)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

constexpr int FIXED_TILES = 8;          // a segment of a product costs about so many of its tiles besides

// How the tiles of a product are shared out.  Only the device knows the number of valid rows, so the division is made
// there.  The class tiles fall to `groups` groups of workgroups (at most 8: one per XCD, whose L2 then sees an eighth of the
// weight).  The `units` of a group, its class tiles of one row tile after the other, are cut into equal runs, one for each
// of its workgroups (for nearly all of them, where runs then end with their row tile).  A run is one or more segments of
// neighbouring class tiles of one row tile.
// Against equal numbers of class tiles for every row tile, valid or not, with dF shared out alike, a training step of
// 16384 x 32000 x 256 bf16 takes 1050 us instead of 1204 with half the rows left out, 480 instead of 825 with nine tenths,
// 4096 x 5003 x 200 fp32 with 30 % kept 215 instead of 342; with no row left out the two differ by 2 % either way.
// Results of segments lie under number segment(group, worker, row tile): along a group's runs either the worker or the row
// tile or both advance, so that the sum of the two numbers names the segment.  The workers with a row tile's first and last
// tile write their segments' numbers to `ends`, for whoever joins them.
struct Share {
    long long units, workers;           // of the group; every worker has a unit at least
    int tiles, first_tile;              // of the group
    // row_tiles: with valid rows; most: workers at hand; fixed: what a segment costs beside its units, in units
    __device__ __forceinline__ Share(int all_tiles, int groups, int group, long long row_tiles, long long most, int fixed) {
        first_tile = (int)((long long)all_tiles * group / groups);
        tiles = (int)((long long)all_tiles * (group + 1) / groups) - first_tile;
        units = row_tiles * tiles;
        workers = min(units, most);
        if (workers < units && row_tiles <= workers) {              // the same number for every row tile: one segment each
            const int each = (int)quotient(workers, row_tiles);
            if (quotient(tiles, each) <= quotient(units, workers) + fixed) workers = each * row_tiles;
        }
    }
    // worker w has the units [start(w), start(w + 1))
    __device__ __forceinline__ long long start(long long w) const {
        return workers == units ? w : quotient(w * units, workers);
    }
    static __device__ __forceinline__ long long segment(int group, int per_group, int row_tiles, long long w,
                                                        long long row_tile) {
        return (long long)group * (per_group + row_tiles) + w + row_tile;
    }
    // segment of the tiles [t0, t1) of a row tile
    __device__ __forceinline__ void mark(int2* ends, long long segment, long long t0, long long t1) const {
        if (t0 == first_tile) ends->x = (int)segment;
        if (t1 == first_tile + tiles) ends->y = (int)segment;
    }
    static __device__ __forceinline__ long long quotient(long long a, long long b) {
        if (a < b) return 0;                                        // divisions are software: small calls do without
        return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
    }
};

// What the gradient products hold dz, weight and features in, and the power of two that dz is stored under.
template <typename T> struct GradOf { typedef _Float16 type; static constexpr int LOG2_DZ = 14; };
template <> struct GradOf<float> { typedef float type; static constexpr int LOG2_DZ = 0; };

// dz lies in blocks of 256 rows x 128 bytes of classes, [rows / 256][classes / DZ_CLASSES][256][DZ_CLASSES]: a tile of the
// product writes, and a stage of either gradient product reads, pieces of 8 KiB or more that are contiguous (rows of a
// plain layout lie a piece apart: writing 16384 x 8192 of them took 153 us instead of 110).
template <typename G> struct Dz {
    static constexpr int CLASSES = 128 / sizeof(G);                 // per block
    static constexpr long long BLOCK = 256 * CLASSES;               // elements
    // element (row, class) of a piece
    static __host__ __device__ __forceinline__ long long at(long long row, long long cls, long long piece) {
        return ((row >> 8) * (piece / CLASSES) + cls / CLASSES) * BLOCK + (row & 255) * CLASSES + cls % CLASSES;
    }
};

// Folds a tile's logits into the running maximum and sum of NF rows of this lane.  acc[f][g][i]: class 32 f + 16 h + i of
// the tile; bias: at class 16 h.
// A lane may sweep the whole vocabulary, and terms of one size are rounded to the same side again and again (a fresh head,
// whose logits are nearly equal, lost 1e-4 of its sum over 16384 terms): a tile's 16 or 32 terms are added in fp32, four by
// four, and the tiles in 64 bits, which costs 0.5 % at most (kd 16384 x 65001 x 256, a step 3328 -> 3345 us).
template <int CF, int NF>
__device__ __forceinline__ void fold(f32x16 (&acc)[CF][NF], const float* bias, float scale, float (&m)[NF], double (&s)[NF]) {
    float top[NF];
#pragma unroll
    for (int g = 0; g < NF; ++g) top[g] = m[g];
#pragma unroll
    for (int f = 0; f < CF; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const vec4f b = *reinterpret_cast<const vec4f*>(bias + f * 32 + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int g = 0; g < NF; ++g) {
                    const float z = fmaf(acc[f][g][4 * q + e], scale, b[e]);
                    acc[f][g][4 * q + e] = z;
                    top[g] = fmaxf(top[g], z);
                }
        }
#pragma unroll
    for (int g = 0; g < NF; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int f = 0; f < CF; ++f)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = __builtin_amdgcn_exp2f(acc[f][g][i + k] - top[g]);
                sum += (e[0] + e[1]) + (e[2] + e[3]);
            }
        s[g] = s[g] * (double)__builtin_amdgcn_exp2f(m[g] - top[g]) + (double)sum;
        m[g] = top[g];
    }
}

// Writes a tile of q times the power of two to dz, from class `first` (a multiple of 32) on; rows behind the last valid one
// get zeros.  shift: lse - LOG2_DZ;  out + lane_at: the first row's element of the piece's class 16 h,
// out the same in every lane.
template <typename G, int CF, int NF>
__device__ __forceinline__ void store_dz(const f32x16 (&acc)[CF][NF], const float* bias, float scale, const float (&shift)[NF],
                                         const bool (&on)[NF], G* out, uint32_t lane_at, int first) {
    constexpr int E = 16 / sizeof(G);
#pragma unroll
    for (int f = 0; f < CF; ++f) {
        G* const to = out + ((first + f * 32) / Dz<G>::CLASSES * Dz<G>::BLOCK + (first + f * 32) % Dz<G>::CLASSES);
#pragma unroll
        for (int c = 0; c < 16; c += E) {
            float b[E];
#pragma unroll
            for (int e = 0; e < E; ++e) b[e] = bias[f * 32 + c + e];
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[e] = __builtin_amdgcn_exp2f(fmaf(acc[f][g][c + e], scale, b[e] - shift[g]));
                    if (!on[g]) v[e] = 0.0f;
                }
                store_vec<G, E>(to + (lane_at + (uint32_t)(g * 32 * Dz<G>::CLASSES + c)), v);
            }
        }
    }
}

// (maximum, sum) of a row from the two lanes that share it; both get it.
__device__ __forceinline__ float2 join_halves(float m, double s) {
    const float sum = (float)s, om = __shfl_xor(m, 32, 64), os = __shfl_xor(sum, 32, 64);
    const float top = fmaxf(m, om);
    return make_float2(top, sum * __builtin_amdgcn_exp2f(m - top) + os * __builtin_amdgcn_exp2f(om - top));
}

// Rows of up to 1 KiB (fp32: 768 bytes, 1152 in three parts): a wave keeps the features of its 32 NF rows in registers for the
// whole sweep over the classes (at most 144 VGPRs), and only tiles of CT classes stream through LDS, two of them in turn.
// That takes 16 bytes per cycle and compute unit out of L2 at full matrix rate where a 128 x 128 tile that streams both
// operands takes 64, all that L2 gives.  Two workgroups per compute unit drift apart, so that one's exponentials run beside
// the other's products.  Forward, a tenth of the rows left out: 4096 x 32000 x 256 bf16 71 us (850 TFLOP/s of the valid rows),
// 32768 x 65536 x 512 1830 us (1080; the largest library products reach 1300).
// SMALL: calls of few tiles, whose time is that of one tile's loads, products and exponentials one after the other: forward
// with 64 x 1204 x 256 bf16 13.1 us instead of 15.9, 64 x 32000 (500 wide tiles) 18.8 instead of 22.5, 64 x 1204 x 128 fp32
// 13.9 instead of 15.0, but 1000 x 4000 x 128 fp32 (256 tiles) 21.6 instead of 19.4.
template <typename T, int KS, bool GRAD, bool SMALL>
struct Resident {
    static constexpr int ROW = KS * 32;                             // bytes of a row
    static constexpr int NF = !SMALL && KS <= (sizeof(T) == 4 ? 8 : 16) ? 2 : 1;    // row fragments per wave
    static constexpr int CT = !SMALL && KS <= 16 ? 64 : 32;         // classes per tile
    static constexpr int ROWS = 4 * 32 * NF;                        // rows per workgroup
    static constexpr int SLABS = Fragment<T>::SLABS, K = KS / SLABS;    // fragments of K
};

template <typename T, int KS, bool GRAD, bool SMALL>
__global__ __launch_bounds__(VT, 2) void resident_kernel(ProductArgs p) {
    typedef Resident<T, KS, GRAD, SMALL> S;
    typedef typename GradOf<T>::type G;
    constexpr int ROW = S::ROW, NF = S::NF, CT = S::CT, CF = CT / 32, CHUNKS = ROW / 16, PASSES = CT * CHUNKS / VT;
    __shared__ __align__(1024) char lds0[CT * ROW], lds1[CT * ROW];
    __shared__ __align__(16) float s_bias[2][CT];
    const int count = *p.count;
    if (count == 0) return;
    const int per_group = gridDim.x / p.groups;
    // hardware hands workgroups to the XCDs in turn; an XCD's workers are neighbours
    const int group = blockIdx.x % p.groups, worker = blockIdx.x % 8 / p.groups * (gridDim.x / 8) + blockIdx.x / 8;
    const Share share(p.tiles, p.groups, group, (count + S::ROWS - 1) / S::ROWS, per_group, FIXED_TILES);
    if (worker >= share.workers) return;
    long long unit = uniform(share.start(worker));
    const long long end = uniform(share.start(worker + 1));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;

    // This lane's source bytes within a class tile: chunk at % CHUNKS of row at / CHUNKS, at = i VT + thread.  Where a pass
    // covers a power of two of rows, the row's bits and so the permutation's come apart into the pass's and the thread's, and
    // one register serves all passes.
    constexpr bool APART = VT % CHUNKS == 0;
    constexpr int PASS_ROWS = VT / CHUNKS;
    const int my_row = threadIdx.x / CHUNKS;
    int my_chunk = ((threadIdx.x % CHUNKS) ^ class_swizzle<ROW>(my_row)) << 4;
    uint32_t offset[APART ? 1 : PASSES];
    if constexpr (APART) {
        offset[0] = my_row * (uint32_t)p.weight_pitch;
    } else {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int at = i * VT + threadIdx.x, r = at / CHUNKS;
            offset[i] = r * (uint32_t)p.weight_pitch + (((at % CHUNKS) ^ class_swizzle<ROW>(r)) << 4);
        }
    }
    const long long behind = p.last_class + 1 - p.first_class;      // classes of the piece that exist
    auto stage = [&](char* to, int t) {
        const long long c = (long long)t * CT;
        const char* from = p.weight + (p.first_class + c) * p.weight_pitch;
        if (c + CT <= behind) {
            asm volatile("" : "+v"(my_chunk));                      // formed anew in every step, as first_chunk below
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                if constexpr (APART)
                    stage16(from + i * PASS_ROWS * p.weight_pitch +
                                (offset[0] + (uint32_t)(my_chunk ^ (class_swizzle<ROW>(i * PASS_ROWS) << 4))),
                            to + i * VT * 16 + wave * 1024);
                else stage16(from + offset[i], to + i * VT * 16 + wave * 1024);
            }
        } else {                                                    // rows behind the last class repeat it
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int at = i * VT + threadIdx.x, r = at / CHUNKS;
                const long long cls = c + r < behind ? p.first_class + c + r : p.last_class;
                stage16(p.weight + cls * p.weight_pitch + (((at % CHUNKS) ^ class_swizzle<ROW>(r)) << 4),
                        to + i * VT * 16 + wave * 1024);
            }
        }
    };

    const int my_class = class_row(lane & 31);
    int first_chunk = my_class * ROW + ((h ^ class_swizzle<ROW>(my_class)) << 4);
    while (unit < end) {
        const long long row_tile = uniform(Share::quotient(unit, share.tiles));
        const int t0 = share.first_tile + (int)(unit - row_tile * share.tiles);
        const int t1 = min(share.first_tile + share.tiles, t0 + (int)min(end - unit, (long long)share.tiles));
        unit += t1 - t0;
        const long long mine = row_tile * S::ROWS + wave * 32 * NF + (lane & 31);       // this lane's first row
        float m[NF], shift[NF];
        double s[NF];
        bool on[NF];
#pragma unroll
        for (int g = 0; g < NF; ++g) {
            m[g] = LOWEST;
            s[g] = 0.0;
            if (GRAD) {
                shift[g] = p.lse2[mine + g * 32] - GradOf<T>::LOG2_DZ;
                on[g] = mine + g * 32 < count;
            }
        }
        G* const out = (G*)p.dz + Dz<G>::at(row_tile * S::ROWS, 0, p.piece);
        const uint32_t lane_at = (wave * 32 * NF + (lane & 31)) * Dz<G>::CLASSES + 16 * h;
        float tile_bias = 0.0f;
        auto fetch_bias = [&](int t) { if (threadIdx.x < CT && t < t1) tile_bias = p.bias2[(long long)t * CT + threadIdx.x]; };
        fetch_bias(t0);
        stage(lds0, t0);
        constexpr int SLABS = S::SLABS;
        Fragment<T> rows[NF][S::K];
#pragma unroll
        for (int g = 0; g < NF; ++g)
#pragma unroll
            for (int k = 0; k < S::K; ++k) {
                u32x4 slab[SLABS];
#pragma unroll
                for (int i = 0; i < SLABS; ++i)
                    slab[i] =
                        *reinterpret_cast<const u32x4*>(p.features + (mine + g * 32) * ROW + (k * SLABS + i) * 32 + 16 * h);
                rows[g][k].set(slab);
            }
        if (threadIdx.x < CT) s_bias[t0 & 1][threadIdx.x] = tile_bias;
        fetch_bias(t0 + 1);

        auto step = [&](const char* now, char* next, int t) __attribute__((always_inline)) {
            stage_barrier();
            if (threadIdx.x < CT) s_bias[(t + 1) & 1][threadIdx.x] = tile_bias;
            fetch_bias(t + 2);
            if (t + 1 < t1) stage(next, t + 1);
            f32x16 acc[CF][NF];
#pragma unroll
            for (int f = 0; f < CF; ++f)
#pragma unroll
                for (int g = 0; g < NF; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[f][g][i] = 0.0f;
            // chunk (2 k + h) ^ swizzle is chunk h ^ swizzle with the bits of 2 k flipped (rows of an odd multiple of 128
            // bytes: of its low three bits); formed anew in every step, since KS addresses held over the loop would not fit
            asm volatile("" : "+v"(first_chunk));
            constexpr int FLIP = ROW % 256 == 0 ? 15 : 7;
            // the wave that multiplies goes first, the one beside it fills in with its exponentials
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int k = 0; k < S::K; ++k) {
                u32x4 raw[CF][SLABS];
#pragma unroll
                for (int i = 0; i < SLABS; ++i) {
                    const int chunk = 2 * (k * SLABS + i);
                    const char* from = now + ((first_chunk ^ ((chunk & FLIP) << 4)) + ((chunk & ~FLIP) << 4));
#pragma unroll
                    for (int f = 0; f < CF; ++f) raw[f][i] = *reinterpret_cast<const u32x4*>(from + f * 32 * ROW);
                }
                Fragment<T> a[CF];
#pragma unroll
                for (int f = 0; f < CF; ++f) a[f].set(raw[f]);
#pragma unroll
                for (int f = 0; f < CF; ++f)
#pragma unroll
                    for (int g = 0; g < NF; ++g) acc[f][g] = mma(a[f], rows[g][k], acc[f][g]);
            }
            interleave<4 * CF, S::K, CF * NF * Fragment<T>::PRODUCTS, CF * SLABS>();
            __builtin_amdgcn_s_setprio(0);
            const float* bias = s_bias[t & 1] + 16 * h;
            if (GRAD) store_dz<G, CF, NF>(acc, bias, p.scale, shift, on, out, lane_at, t * CT);
            else fold<CF, NF>(acc, bias, p.scale, m, s);
        };
        int t = t0;
        while (t < t1) {
            step(lds0, lds1, t++);
            if (t == t1) break;
            step(lds1, lds0, t++);
        }
        if (!GRAD) {
            const long long segment = Share::segment(group, per_group, p.row_tiles, worker, row_tile);
            float2* part = p.part + segment * S::ROWS;
            if (threadIdx.x == 0) share.mark(p.ends + (long long)group * p.row_tiles + row_tile, segment, t0, t1);
#pragma unroll
            for (int g = 0; g < NF; ++g) {
                const float2 row = join_halves(m[g], s[g]);
                if (h == 0) part[wave * 32 * NF + g * 32 + lane] = row;
            }
        }
        __syncthreads();                                            // the next segment writes to LDS what others still read
    }
}

// Wider rows: both operands stream through LDS in stages of 128 bytes of K.  Four waves take 64 x 64 each of tiles of 128
// classes, or 32 x 32 of tiles of 32 where the wide ones would leave half the compute units without work (108 x 5992 x 736
// fp32: 24 us, by 47 workgroups of wide tiles 43; bf16 11 and 14).
template <typename T, bool GRAD, int CT>
__global__ __launch_bounds__(VT, 2) void product_kernel(ProductArgs p) {
    typedef typename GradOf<T>::type G;
    constexpr int F = CT == TILE ? 2 : 1, CLASS_STAGE = CT * 128;           // F x F fragments of 32 x 32 per wave
    __shared__ __align__(1024) char lds0[CLASS_STAGE + STAGE], lds1[CLASS_STAGE + STAGE];   // two stages of (classes, rows)
    __shared__ float2 joined[F][TILE];
    __shared__ __align__(16) float s_bias[CT];
    const int count = *p.count;
    if (count == 0) return;
    const int per_group = gridDim.x / p.groups;
    // hardware hands workgroups to the XCDs in turn; an XCD's workers are neighbours
    const int group = blockIdx.x % p.groups, worker = blockIdx.x % 8 / p.groups * (gridDim.x / 8) + blockIdx.x / 8;
    const Share share(p.tiles, p.groups, group, (count + TILE - 1) / TILE, per_group, FIXED_TILES);
    if (worker >= share.workers) return;
    long long unit = uniform(share.start(worker));
    const long long end = uniform(share.start(worker + 1));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
    // this wave's classes and rows of a tile
    const int wc = F == 2 ? (wave & 1) * 64 : 0, wr = F == 2 ? (wave >> 1) * 64 : wave * 32;
    constexpr int KE = 128 / sizeof(T);
    constexpr int SLABS = Fragment<T>::SLABS;
    const int ksteps = p.dim_pad / KE;                              // at least seven: narrower rows are resident
    typedef ChunkedOperand<CT, VT, true> Classes;
    typedef ChunkedOperand<TILE, VT, false> Rows;
    while (unit < end) {
        const long long row_tile = uniform(Share::quotient(unit, share.tiles)), r0 = row_tile * TILE;
        const int t0 = share.first_tile + (int)(unit - row_tile * share.tiles);
        const int t1 = min(share.first_tile + share.tiles, t0 + (int)min(end - unit, (long long)share.tiles));
        unit += t1 - t0;
        Rows rows;
        Classes cls;
        rows.init(p.features, (long long)p.dim_pad * sizeof(T), r0, r0 + TILE);

        float m[F], shift[F];
        double s[F];
        bool on[F];
#pragma unroll
        for (int g = 0; g < F; ++g) {
            m[g] = LOWEST;
            s[g] = 0.0;
            if (GRAD) {
                const long long row = r0 + wr + g * 32 + (lane & 31);
                shift[g] = p.lse2[row] - GradOf<T>::LOG2_DZ;
                on[g] = row < count;
            }
        }
        G* const out = (G*)p.dz + Dz<G>::at(r0, 0, p.piece);
        const uint32_t lane_at = (wr + (lane & 31)) * Dz<G>::CLASSES + 16 * h;

        f32x16 acc[F][F];
        auto clear = [&] {
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int g = 0; g < F; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[f][g][i] = 0.0f;
        };
        int next_t = t0, next_k = 0;                                    // what is staged next
        float tile_bias = 0.0f;
        auto fetch_bias = [&](int t) {
            if (threadIdx.x < CT && t < t1) tile_bias = p.bias2[(long long)t * CT + threadIdx.x];
        };
        auto stage_next = [&](char* to) {
            if (next_t >= t1) return;
            if (next_k == 0) cls.init(p.weight, p.weight_pitch, p.first_class + (long long)next_t * CT, p.last_class);
            cls.stage(to, (long long)next_k * 128);
            rows.stage(to + CLASS_STAGE, (long long)next_k * 128);
            if (++next_k == ksteps) {
                next_k = 0;
                ++next_t;
            }
        };
        auto multiply = [&](const char* now) __attribute__((always_inline)) {
            int at = lane;
            asm volatile("" : "+v"(at));                            // addresses are formed anew, see resident_kernel
#pragma unroll
            for (int j = 0; j < 4; j += SLABS) {
                Fragment<T> a[F], b[F];
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    u32x4 x[SLABS], y[SLABS];
#pragma unroll
                    for (int i = 0; i < SLABS; ++i) {
                        x[i] = Classes::frag(now, wc + f * 32, j + i, at);
                        y[i] = Rows::frag(now + CLASS_STAGE, wr + f * 32, j + i, at);
                    }
                    a[f].set(x);
                    b[f].set(y);
                }
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int g = 0; g < F; ++g) acc[f][g] = mma(a[f], b[g], acc[f][g]);
            }
            interleave<4 * F, 4 / SLABS, F * F * Fragment<T>::PRODUCTS, 2 * F * SLABS>();
        };
        // The bias of a tile is fetched ahead of the tile's first stage (waiting for it later would wait for the stages behind
        // it as well) and written to LDS in its first step.  The two stages are variables of their own, used by turns in
        // straight code: the compiler then knows that reading one need not wait for the loads into the other.
        auto step = [&](const char* now, char* next, int& t, int& k) __attribute__((always_inline)) {
            stage_barrier();
            if (k == 0 && threadIdx.x < CT) s_bias[threadIdx.x] = tile_bias;
            if (k + 1 == ksteps) fetch_bias(t + 1);
            stage_next(next);
            multiply(now);
            if (++k == ksteps) {
                const float* bias = s_bias + wc + 16 * h;
                if (GRAD) store_dz<G, F, F>(acc, bias, p.scale, shift, on, out, lane_at, t * CT + wc);
                else fold<F, F>(acc, bias, p.scale, m, s);
                clear();
                k = 0;
                ++t;
            }
        };
        clear();
        fetch_bias(t0);
        stage_next(lds0);
        int t = t0, k = 0;
        const int steps = (t1 - t0) * ksteps;
        for (int i = 0; i + 1 < steps; i += 2) {
            step(lds0, lds1, t, k);
            step(lds1, lds0, t, k);
        }
        if (steps & 1) step(lds0, lds1, t, k);
        if (!GRAD) {
            // a row's classes lie in two lanes and, of a wide tile, two waves
#pragma unroll
            for (int g = 0; g < F; ++g) {
                const float2 row = join_halves(m[g], s[g]);
                if (h == 0) joined[F == 2 ? wave & 1 : 0][wr + g * 32 + lane] = row;
            }
            __syncthreads();
            const long long segment = Share::segment(group, per_group, p.row_tiles, worker, row_tile);
            if (threadIdx.x == 0) share.mark(p.ends + (long long)group * p.row_tiles + row_tile, segment, t0, t1);
            if (threadIdx.x < TILE) {
                const float2 a = joined[0][threadIdx.x], b = joined[F - 1][threadIdx.x];
                const float top = fmaxf(a.x, b.x);
                const float sum = a.y * __builtin_amdgcn_exp2f(a.x - top) + b.y * __builtin_amdgcn_exp2f(b.x - top);
                p.part[segment * TILE + threadIdx.x] = F == 1 ? a : make_float2(top, sum);
            }
        }
        __syncthreads();                                            // the next segment writes to LDS what others still read
    }
}

// ---- forward's end -----------------------------------------------------------------------------------------------------
struct TargetArgs {
    const char* features;               // packed
    int dim_pad;
    const char* weight;                 // rows as the product reads them
    long long weight_pitch;             // bytes
    const void* bias;
    long long classes;
    const long long* targets;           // [rows] or [rows, top]
    int top;                            // 0: cross entropy
    const float* prob;                  // [rows, top]
    const float* entropy;               // [rows]
    RowLists lists;
    const float2* part;
    const int2* ends;
    int groups, row_tile, row_tiles;    // of the product, see Share
    long long rows_pad;
    float temperature;
    float* lse2;                        // [rows_pad]
    float* target_logit;                // [rows, max(top, 1)] by place, natural units, divided by the temperature
    float* row_loss;                    // [rows]
};

// One wave per valid row: joins the splits, forms the targets' logits (16 lanes a dot product), writes the row's loss.
// A class past the vocabulary makes the row's lse, and with it loss and gradient, NaN; it is not followed.
// UNROLL: sets of four entries taken together, so that their rows are in flight at once (16384 rows x 64 entries of 512 bytes:
// 77 us, one at a time 88; 10835 x 37 of 1824 bytes 56 and 77); 1 for cross entropy.
template <typename T, int UNROLL>
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
    const int lanes = 64 / p.groups, row_tile = (int)(place / p.row_tile);
    const int2 ends = p.ends[(long long)(lane / lanes) * p.row_tiles + row_tile];
    for (int k = ends.x + lane % lanes; k <= ends.y; k += lanes) {
        const float2 v = p.part[(long long)k * p.row_tile + place % p.row_tile];
        const float top = fmaxf(m, v.x);
        s = s * __builtin_amdgcn_exp2f(m - top) + v.y * __builtin_amdgcn_exp2f(v.x - top);
        m = top;
    }
    const float top = wave_max(m);
    s = wave_sum(s * __builtin_amdgcn_exp2f(m - top));
    float lse = (top + log2f(s)) * LN2;

    const int n = UNROLL > 1 ? p.top : 1;
    const float inv_temp = 1.0f / p.temperature;
    const T* f = (const T*)p.features + place * p.dim_pad;
    constexpr int E = 16 / sizeof(T);
    float dot_sum = 0.0f;                                           // sum p z over this group of 16 lanes' entries
    bool outside = false;
    for (int k0 = 0; k0 < n; k0 += 64) {                            // a lane fetches one entry of 64
        long long mine = -1;
        float mine_prob = 1.0f, mine_bias = 0.0f;
        if (k0 + lane < n) {
            mine = p.targets[row * n + k0 + lane];
            if (UNROLL > 1) mine_prob = p.prob[row * n + k0 + lane];
            if (mine >= p.classes) {
                outside = true;
                mine = -1;
            }
            if (p.bias && mine >= 0) mine_bias = Elem<T>::to_float(((const T*)p.bias)[mine]);
        }
        for (int k1 = 0; k1 < min(64, n - k0); k1 += 4 * UNROLL) {
            const T* w[UNROLL];
            float z[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int at = k1 + 4 * u + (lane >> 4);
                const long long c = ((long long)__shfl((int)(mine >> 32), at, 64) << 32) | (uint32_t)__shfl((int)mine, at, 64);
                w[u] = (const T*)(p.weight + max(c, 0ll) * p.weight_pitch);     // a missing entry's product goes nowhere
                z[u] = 0.0f;
            }
            for (int d = (lane & 15) * E; d < p.dim_pad; d += 16 * E) {
                float x[E], y[UNROLL][E];
                load_vec<T, E>(f + d, x);
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) load_vec<T, E>(w[u] + d, y[u]);
#pragma unroll
                for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                    for (int i = 0; i < E; ++i) z[u] = fmaf(x[i], y[u][i], z[u]);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int at = k1 + 4 * u + (lane >> 4);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) z[u] += __shfl_xor(z[u], o, 64);
                const float logit = (z[u] + __shfl(mine_bias, at, 64)) * inv_temp, prob = __shfl(mine_prob, at, 64);
                const bool there = __shfl((int)(mine >> 32), at, 64) >= 0;
                if (there && (lane & 15) == 0) {
                    p.target_logit[place * n + k0 + at] = logit;
                    if (!(prob == 0.0f)) dot_sum += prob * logit;   // an entry without weight takes no part: 0 * inf
                }
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
#pragma unroll 8
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
// Power of two under which an operand with this largest size lies in [2^13, 2^14): what is 2^27 times smaller is still a
// normal fp16 number, what is 2^37 times smaller vanishes.  From -114 to 162: no fp32 number for itself, an exponent to add.
__device__ __forceinline__ int exponent_of(uint32_t max_bits) {
    if (max_bits == 0) return 0;
    int e = 0;
    (void)frexpf(u2f(max_bits), &e);                                // max = f * 2^e, f in [0.5, 1)
    return 14 - e;
}

// A gradient per row, over the largest of them: g = mantissa * weight, mantissa in [1, 2) and weight a power of two with the
// gradient's sign.  The mantissa becomes part of dz (whose exponentials take it with lse) and is rounded with it; the power
// of two goes exactly onto the features (dW) and the results (dF), so that rows of small gradients keep their digits and no
// operand is rounded a second time.  Zero behind the last valid row.  And the scalars.
struct RowWeights {
    float *weight, *mantissa, *lse2;    // [rows_pad]; lse2 less log2 of the mantissa
};

__global__ __launch_bounds__(1024) void row_weights_kernel(const float* __restrict__ upstream, RowLists lists,
                                                           long long rows_pad, float temperature,
                                                           const float* __restrict__ lse2, RowWeights out,
                                                           Scales* __restrict__ scales) {
    __shared__ float red[1024];
    const int count = *lists.count;
    float top = 0.0f;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += 1024) {
        const float g = fabsf(upstream[lists.row_of[i]]);
        if (g < __builtin_inff()) top = fmaxf(top, g);             // infinities and NaN go through as they are
    }
    red[threadIdx.x] = top;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + o]);
        __syncthreads();
    }
    top = red[0] > 0.0f ? red[0] : 1.0f;
#pragma unroll 4
    for (long long i = threadIdx.x; i < rows_pad; i += 1024) {
        float g = i < count ? upstream[lists.row_of[i]] / top : 0.0f, m = 1.0f;
        if (g != 0.0f && fabsf(g) < __builtin_inff()) {
            int e;
            m = 2.0f * frexpf(fabsf(g), &e);
            g = copysignf(ldexpf(1.0f, e - 1), g);
        }
        out.weight[i] = g;
        out.mantissa[i] = m;
        out.lse2[i] = lse2[i] - log2f(m);
    }
    if (threadIdx.x == 0) {
        scales->common = top * temperature;
        scales->features_max = 0;
        scales->weight_max = 0;
    }
}

// An operand of the gradient products: rows of features (those valid, each times its weight) or of weight.
struct Operand {
    const void* x;
    long long pitch, rows;              // elements
    const float* weight;                // of the rows, or null: ones
    const int* count;                   // valid rows, or null: all
    uint32_t* max_bits;                 // null: no power of two
    void* out;                          // [rows][dim_pad]; null: not wanted
    unsigned blocks;
};
struct Operands {
    Operand part[2];
    int dim_pad;
};

// Largest finite |x| of an operand.  The maximum of integers does not depend on the order of the atomics.
template <typename T>
__global__ __launch_bounds__(VT) void max_kernel(Operands ops) {
    constexpr int E = 16 / sizeof(T);
    const bool second = blockIdx.x >= ops.part[0].blocks;
    const Operand& o = ops.part[second ? 1 : 0];
    const unsigned block = blockIdx.x - (second ? ops.part[0].blocks : 0);
    const unsigned chunks = ops.dim_pad / E;
    const unsigned total = (unsigned)(o.count ? *o.count : (int)o.rows) * chunks;
    constexpr int AHEAD = 4;                                        // loads in flight; behind the end the last chunk again
    float top = 0.0f;
    for (unsigned at = block * VT + threadIdx.x; at < total; at += AHEAD * o.blocks * VT) {
        float v[AHEAD][E], w[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const unsigned i = min(at + k * o.blocks * VT, total - 1), r = i / chunks;
            load_vec<T, E>((const T*)o.x + r * o.pitch + (i - r * chunks) * E, v[k]);
            w[k] = o.weight ? o.weight[r] : 1.0f;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float a = fabsf(v[k][i] * w[k]);
                if (a < __builtin_inff()) top = fmaxf(top, a);
            }
        }
    }
    __shared__ float red[VT / 64];
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {                                         // atomics on one address queue up: few workgroups
        for (int w = 1; w < VT / 64; ++w) top = fmaxf(top, red[w]);
        if (top > 0.0f) atomicMax(o.max_bits, f2u(top));
    }
}

// Rows in the gradient products' type: x times the row's weight times the operand's power of two; zero rows behind the
// last valid one up to a whole tile.
template <typename T>
__global__ __launch_bounds__(VT) void scale_kernel(Operands ops) {
    typedef typename GradOf<T>::type G;
    static_assert(sizeof(G) == sizeof(T), "operands change their type, not their size");
    constexpr int E = 16 / sizeof(T);
    const bool second = blockIdx.x >= ops.part[0].blocks;
    const Operand& o = ops.part[second ? 1 : 0];
    const unsigned chunks = ops.dim_pad / E;
    const unsigned at = (blockIdx.x - (second ? ops.part[0].blocks : 0)) * VT + threadIdx.x;
    const long long r = at / chunks;
    if (r >= o.rows) return;
    if (o.count && r >= up_to((long long)*o.count, ROW_TILE)) return;
    const int c = (int)(at % chunks) * E;
    float v[E];
    load_vec<T, E>((const T*)o.x + r * o.pitch + c, v);
    const int exponent = o.max_bits ? exponent_of(*o.max_bits) : 0;
    const float w = o.weight ? o.weight[r] : 1.0f;
    const bool on = !o.count || r < *o.count;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = on ? ldexpf(v[i], exponent) * w : 0.0f;
    store_vec<G, E>((G*)o.out + r * ops.dim_pad + c, v);
}

// The target entries of a piece of dz: q - p.  Next to p = 1 it is expm1(log q) + (1 - p), which keeps the digits of
// 1 - q of a confident row; for small p that sum would lose those of q and p.  Each (row, class) is written once: repeated
// classes carry their whole p in the first entry.
template <typename G>
__global__ __launch_bounds__(VT) void correct_targets_kernel(const long long* __restrict__ targets, int top,
                                                             const float* __restrict__ prob, RowLists lists,
                                                             const float* __restrict__ lse2,
                                                             const float* __restrict__ target_logit,
                                                             const float* __restrict__ mantissa, long long first_class,
                                                             long long piece, long long classes, float scale,
                                                             G* __restrict__ dz) {
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
    const float v = p > 0.5f ? expm1f(log_q) + (1.0f - p) : expf(log_q) - p;
    dz[Dz<G>::at(place, c - first_class, piece)] = Elem<G>::from_float(v * (mantissa ? mantissa[place] * scale : scale));
}

// 256 classes of KE rows of dz as an operand with K strided: four (fp32: eight) blocks side by side.
template <typename T, int THREADS>
struct DzOperand {
    typedef StridedOperand<T, ROW_TILE, THREADS> Tile;              // its place in LDS, and its fragments
    const char* base;
    long long row_block;                // bytes from 256 rows to the next
    uint32_t offset[Tile::PASSES];
    __device__ __forceinline__ void init(const char* dz, long long piece, long long first_class) {
        base = dz + Dz<T>::at(0, first_class, piece) * (long long)sizeof(T);
        row_block = Dz<T>::at(256, 0, piece) * (long long)sizeof(T);
#pragma unroll
        for (int i = 0; i < Tile::PASSES; ++i) {
            const int at = i * THREADS + threadIdx.x, k = at / Tile::CHUNKS;
            const int c = (at % Tile::CHUNKS) ^ Tile::swizzle(k);
            offset[i] = (c >> 3) * (uint32_t)(Dz<T>::BLOCK * sizeof(T)) + k * 128 + (c & 7) * 16;
        }
    }
    __device__ __forceinline__ void stage(char* lds, long long k0) const {
        const char* from = base + (k0 >> 8) * row_block + (k0 & 255) * 128;
#pragma unroll
        for (int i = 0; i < Tile::PASSES; ++i) stage16(from + offset[i], lds + i * THREADS * 16 + (threadIdx.x >> 6) * 1024);
    }
};

// Four elements of a result line: the sums of n partial results, and what they still lack: 2^-LOG2_DZ, the other operand's
// power of two, the common factor.  The powers of two are applied apart, so that no intermediate factor leaves the range.
__device__ __forceinline__ vec4f sum_parts(const float* part, long long step, int n) {
    vec4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int s = 0; s < n; ++s) v += *reinterpret_cast<const vec4f*>(part + s * step);
    return v;
}
template <typename T>
__device__ __forceinline__ void finish_line(vec4f v, int exponent, float factor, int dim, int d, T* out, T* line) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ldexpf(v[i], -exponent - GradOf<T>::LOG2_DZ) * factor;
    T* to = line + d;
    if (dim % 4 == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0) {
        const float f[4] = {v.x, v.y, v.z, v.w};
        store_vec<T, 4>(to, f);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < dim) to[i] = Elem<T>::from_float(v[i]);
    }
}

struct GradArgs {
    const char* a;                      // [K][a_pitch bytes], dim_pad columns: weight rows of the piece, or features
    long long a_pitch, a_last;          // last readable K row
    const char* dz;                     // rows_pad x piece, see Dz
    long long piece;
    int dim_pad;
    const int* count;
    long long cols;                     // columns of the result: rows_pad, or piece
    long long ksteps;                   // K steps of the piece (dF), or at most, see count (dW)
    int splits;                         // dW: of K;  dF: workgroups per tile of d, see RowShare
    float* out;                         // dW: [splits][cols][dim_pad];  dF: [segment][ROW_TILE][dim_pad]
    int2* ends;                         // dF: [rows_pad / ROW_TILE]
    int accumulate;
    float* bias_out;                    // [splits][cols] weighted sums of dz over K, or null
    const float* row_weight;            // [rows_pad], or null: ones
    // DIRECT: [classes][dim] instead of `out`, or null where only the bias is wanted
    void* result;
    int bf16_result, dim, scaled;
    long long classes;
    const Scales* scales;
};

// dF: the K steps of the valid rows' tiles, shared out as in Share.  A segment's sums are a partial result of their own,
// which costs as much as eight steps (fp32: as two): no worker gets fewer, and no tile more than 64 workers.
template <typename T> struct RowShare : Share {
    static constexpr int FIXED = sizeof(T) == 4 ? 2 : 8;
    __device__ __forceinline__ RowShare(int count, long long ksteps, int workgroups)
        : RowShare((long long)((count + ROW_TILE - 1) / ROW_TILE), ksteps, workgroups) {}
    __device__ __forceinline__ RowShare(long long row_tiles, long long ksteps, int workgroups)
        : Share((int)ksteps, 1, 0, row_tiles,
                min((long long)workgroups, min(64 * row_tiles, max(row_tiles, row_tiles * ksteps / FIXED))), FIXED) {}
};

// c plus both fp16 halves of a word, added in fp32
__device__ __forceinline__ float sum_pair(uint32_t w, float c) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), one, c, false);
}

// out[col][d] = sum_k dz(k, col) * a[k][d].  ROWS: columns are rows of dz and K runs over the classes of the piece (dF);
// otherwise columns are classes and K runs over the valid rows (dW).  A workgroup of eight waves takes 64 AF columns d and
// 256 columns of the result, 32 AF x 64 per wave: at AF = 4 a stage of 64 KiB feeds 2048 cycles of the matrix units, half
// of what L2 gives per cycle.  4096 x 32000 x 256 with a tenth of the rows left out: dF 94 us, dW 80 (640 and 750 TFLOP/s);
// reading 240 MB of dz takes 50, and waves wait half (dF) and a third (dW) of their cycles for loads, since a stage ends with
// a wait for all of them and no second workgroup fits beside 128 KiB of LDS.
// DIRECT: dW of one split, written as it leaves.
template <typename T, int AF, bool ROWS, bool DIRECT>
__global__ __launch_bounds__(2 * VT, 2) void grad_kernel(GradArgs p) {
    constexpr int THREADS = 2 * VT, DT = 64 * AF;
    constexpr int A_BYTES = DT * 128, B_BYTES = ROW_TILE * 128;
    __shared__ __align__(1024) char a0[A_BYTES], b0[B_BYTES], a1[A_BYTES], b1[B_BYTES];
    constexpr int KE = 128 / sizeof(T), SLABS = Fragment<T>::SLABS;
    const int dtiles = (p.dim_pad + DT - 1) / DT;
    const int id = xcd_range(blockIdx.x, gridDim.x);
    const int d0 = (id % dtiles) * DT, member = id / dtiles;
    const int count = *p.count;
    if (count == 0 && ROWS) return;
    long long unit = 0, end = 1;                                    // dW: one tile and split
    const RowShare<T> share(ROWS ? count : 1, ROWS ? p.ksteps : 1, ROWS ? p.splits : 1);
    if (ROWS) {
        if (member >= share.workers) return;
        unit = uniform(share.start(member));
        end = uniform(share.start(member + 1));
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
    const int wd = (wave & 1) * 32 * AF, wcol = (wave >> 1) * 64;

    typedef StridedOperand<T, DT, THREADS> A;
    typedef DzOperand<T, THREADS> BS;
    typedef ChunkedOperand<ROW_TILE, THREADS, false> BC;
    A a;
    a.init(p.a, p.a_pitch, d0, p.dim_pad);
    do {
        long long c0, k_first, k_end, line;                             // columns, K steps, and where the result goes
        if (ROWS) {
            const long long tile = uniform(Share::quotient(unit, share.tiles));
            k_first = unit - tile * share.tiles;
            k_end = min((long long)share.tiles, k_first + (end - unit));
            unit += k_end - k_first;
            c0 = tile * ROW_TILE;
            const long long segment = Share::segment(0, 0, 0, member, tile);
            line = segment * ROW_TILE;
            if (threadIdx.x == 0 && d0 == 0) share.mark(p.ends + tile, segment, k_first, k_end);
        } else {
            const long long ctiles = p.cols / ROW_TILE, ksteps = min(p.ksteps, (long long)(count + KE - 1) / KE);
            const int split = (int)(member / ctiles);
            c0 = member % ctiles * ROW_TILE;
            k_first = ksteps * split / p.splits;
            k_end = ksteps * (split + 1) / p.splits;
            line = split * p.cols + c0;
        }
        BS bs;
        BC bc;
        // 256 rows of dz times the classes of a stage are one block
        if (ROWS) bc.init(p.dz + Dz<T>::at(c0, 0, p.piece) * (long long)sizeof(T), 128, 0, ROW_TILE - 1);
        else bs.init(p.dz, p.piece, c0);

        f32x16 acc[AF][2];
#pragma unroll
        for (int f = 0; f < AF; ++f)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[f][g][i] = 0.0f;
        double bias = 0.0;                                          // a stage's rows are added in fp32, the stages in 64 bits
        const bool want_bias = !ROWS && p.bias_out && d0 == 0;

        auto stage = [&](char* to_a, char* to_b, long long k) {
            a.stage(to_a, k * KE, p.a_last);
            if (ROWS) bc.stage(to_b, k * Dz<T>::BLOCK * (long long)sizeof(T));
            else bs.stage(to_b, k * KE);
        };
        auto multiply = [&](const char* ta, const char* tb, long long k) __attribute__((always_inline)) {
            int at = lane;
            asm volatile("" : "+v"(at));                            // addresses are formed anew, see resident_kernel
            float stage_bias = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j += SLABS) {
                u32x4 y[2][SLABS];
                Fragment<T> b[2], x[AF];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
#pragma unroll
                    for (int i = 0; i < SLABS; ++i)
                        y[g][i] = ROWS ? BC::frag(tb, wcol + g * 32, j + i, at) : BS::Tile::frag(tb, wcol + g * 32, j + i, at);
                    b[g].set(y[g]);
                }
#pragma unroll
                for (int f = 0; f < AF; ++f) {
                    u32x4 raw[SLABS];
#pragma unroll
                    for (int i = 0; i < SLABS; ++i) raw[i] = A::frag(ta, wd + f * 32, j + i, at);
                    x[f].set(raw);
                }
#pragma unroll
                for (int f = 0; f < AF; ++f)
#pragma unroll
                    for (int g = 0; g < 2; ++g) acc[f][g] = mma(x[f], b[g], acc[f][g]);
                if (want_bias) {
                    constexpr int E = 16 / sizeof(T);               // a lane's K of slab j: E from (2 j + h) E on
#pragma unroll
                    for (int i = 0; i < SLABS; ++i) {
                        const u32x4 first = y[0][i], second = y[1][i];  // the two waves of these columns take one each
                        const u32x4 mine = (wave & 1) ? second : first;
                        if (p.row_weight) {
                            const float* weight = p.row_weight + k * KE + (2 * (j + i) + h) * E;
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                if constexpr (sizeof(T) == 2) {
                                    float lo, hi;
                                    unpack2(mine[w], lo, hi, (const T*)nullptr);
                                    stage_bias += lo * weight[2 * w] + hi * weight[2 * w + 1];
                                } else {
                                    stage_bias += u2f(mine[w]) * weight[w];
                                }
                            }
                        } else {
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                if constexpr (sizeof(T) == 2) stage_bias = sum_pair(mine[w], stage_bias);
                                else stage_bias += u2f(mine[w]);
                            }
                        }
                    }
                }
            }
            if (want_bias) bias += (double)stage_bias;
        };
        auto order = [&] {
            constexpr int PER = sizeof(T) == 4 ? 4 : 2;                 // LDS reads of a transposed fragment
            constexpr int READS = AF * PER + 2 * (ROWS ? 1 : PER);
            interleave<(sizeof(T) == 4 ? 1 : 2) * READS, 4 / SLABS, 2 * AF * Fragment<T>::PRODUCTS, READS * SLABS>();
        };
        if (k_first < k_end) stage(a0, b0, k_first);
        auto sweep = [&](auto works) __attribute__((always_inline)) {
            auto work = [&](const char* ta, const char* tb, long long k) __attribute__((always_inline)) {
                if constexpr (decltype(works)::value) {
                    multiply(ta, tb, k);
                    order();
                }
            };
            long long k = k_first;
            for (; k + 1 < k_end; k += 2) {
                stage_barrier();
                stage(a1, b1, k + 1);
                work(a0, b0, k);
                stage_barrier();
                if (k + 2 < k_end) stage(a0, b0, k + 2);
                work(a1, b1, k + 1);
            }
            if (k < k_end) {
                stage_barrier();
                work(a0, b0, k);
            }
        };
        // a wave without a valid row only takes part in the staging
        if (!ROWS || c0 + wcol < count) sweep(std::true_type());
        else sweep(std::false_type());
        // The result leaves through LDS, 32 columns of the wave at a time, so that a store covers whole lines: a lane holds 4
        // neighbouring d of one column, and stores of those reach memory in pieces of 32 bytes (25 us of 108 for dW of
        // 4096 x 32000 x 256).
        constexpr int WIDTH = 32 * AF, REGION = 32 * WIDTH * 4, ROW_CHUNKS = WIDTH / 4;
        static_assert(2 * REGION <= A_BYTES && 2 * REGION <= B_BYTES, "two waves' regions per stage");
        stage_barrier();
        int at_lane = lane;
        asm volatile("" : "+v"(at_lane));                           // formed here, not held over the loops
        char* region = (wave < 2 ? a0 : wave < 4 ? b0 : wave < 6 ? a1 : b1) + (wave & 1) * REGION;
        float* out = p.out + (line + wcol) * p.dim_pad + d0 + wd;
        const int exponent = DIRECT && p.scaled ? exponent_of(p.scales->features_max) : 0;
        const float common = DIRECT ? p.scales->common : 0.0f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int col = at_lane & 31;
#pragma unroll
            for (int f = 0; f < AF; ++f)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    vec4f v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[f][g][4 * q + e];
                    const int chunk = f * 8 + 2 * q + (at_lane >> 5);                // of 4 d; permuted against bank conflicts
                    *reinterpret_cast<vec4f*>(region + (col * ROW_CHUNKS + (chunk ^ (col & 7))) * 16) = v;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the region is this wave's own
#pragma unroll
            for (int i = 0; i < 32 * ROW_CHUNKS / 64; ++i) {
                const int at = i * 64 + at_lane, c = at / ROW_CHUNKS, chunk = at % ROW_CHUNKS;
                vec4f v = *reinterpret_cast<const vec4f*>(region + (c * ROW_CHUNKS + (chunk ^ (c & 7))) * 16);
                if constexpr (DIRECT) {
                    const long long cls = c0 + wcol + g * 32 + c;
                    const int d = d0 + wd + chunk * 4;
                    if (p.result && cls < p.classes && d < p.dim) {
                        if (sizeof(T) == 2 && p.bf16_result)
                            finish_line<bf16_t>(v, exponent, common, p.dim, d, (bf16_t*)p.result,
                                                (bf16_t*)p.result + cls * p.dim);
                        else finish_line<T>(v, exponent, common, p.dim, d, (T*)p.result, (T*)p.result + cls * p.dim);
                    }
                } else if (d0 + wd + chunk * 4 < p.dim_pad) {           // dim_pad is a multiple of four
                    vec4f* to = reinterpret_cast<vec4f*>(out + (long long)(g * 32 + c) * p.dim_pad + chunk * 4);
                    if (p.accumulate) v += *to;
                    *to = v;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (want_bias) {
            const float half = (float)bias, sum = half + __shfl_xor(half, 32, 64);
            if (h == 0) p.bias_out[line + wcol + (wave & 1) * 32 + lane] = sum;
        }
        if (ROWS) __syncthreads();                                  // the next segment writes to LDS what others still read
    } while (ROWS && unit < end);
}

// The partial results of the gradients, joined.
struct FinishArgs {
    const Scales* scales;
    int dim, dim_pad;
    // classes of a piece: out[class][0 .. dim) and bias[class], the splits' sums over the piece's columns
    const float *part_w, *part_b;
    long long piece, classes;
    int splits_w, scaled_f;
    void *dweight, *dbias;
    unsigned weight_blocks, bias_blocks;
    // rows, behind the last piece: out[row][0 .. dim) of line place[row], zero where there is none
    const float* part_f;
    long long rows;
    const int2* ends;                   // segments of part_f
    int scaled_w;
    const int* place;
    const float* row_weight;
    void* dfeatures;
};

template <typename T>
__global__ __launch_bounds__(VT) void finish_kernel(FinishArgs p) {
    const unsigned groups = (p.dim + 3) / 4;
    unsigned block = blockIdx.x;
    if (block < p.weight_blocks) {
        const unsigned at = block * VT + threadIdx.x;
        const long long c = at / groups;
        if (c >= p.classes) return;
        const int d = (int)(at % groups) * 4;
        finish_line<T>(sum_parts(p.part_w + c * p.dim_pad + d, p.piece * p.dim_pad, p.splits_w),
                       p.scaled_f ? exponent_of(p.scales->features_max) : 0, p.scales->common, p.dim, d, (T*)p.dweight,
                       (T*)p.dweight + c * p.dim);
        return;
    }
    block -= p.weight_blocks;
    if (block < p.bias_blocks) {
        const long long c = (long long)block * VT + threadIdx.x;
        if (c >= p.classes) return;
        float sum = 0.0f;
        for (int s = 0; s < p.splits_w; ++s) sum += p.part_b[s * p.piece + c];
        ((T*)p.dbias)[c] = Elem<T>::from_float(sum * ldexpf(1.0f, -GradOf<T>::LOG2_DZ) * p.scales->common);
        return;
    }
    block -= p.bias_blocks;
    const unsigned at = block * VT + threadIdx.x;
    const long long row = at / groups;
    if (row >= p.rows) return;
    const int line = p.place[row], d = (int)(at % groups) * 4;
    vec4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (line >= 0) {
        const int2 ends = p.ends[line / ROW_TILE];
        v = sum_parts(p.part_f + ((long long)ends.x * ROW_TILE + line % ROW_TILE) * p.dim_pad + d,
                      (long long)ROW_TILE * p.dim_pad, ends.y - ends.x + 1);
    }
    finish_line<T>(v, p.scaled_w ? exponent_of(p.scales->weight_max) : 0,
                   line < 0 ? 0.0f : p.scales->common * (p.row_weight ? p.row_weight[line] : 1.0f), p.dim, d, (T*)p.dfeatures,
                   (T*)p.dfeatures + row * p.dim);
}

// ---- host ---------------------------------------------------------------------------------------------------------
constexpr long long DZ_BYTES = 256ll << 20;     // size aimed at for a piece of dz
constexpr int SLOTS = 512;                      // workgroups of the products that run at once: two per compute unit
constexpr int GRAD_SLOTS = 256;                 // of the gradient products: one

long long up(long long v, long long to) { return (v + to - 1) / to * to; }
long long least(long long a, long long b) { return a < b ? a : b; }
long long most(long long a, long long b) { return a > b ? a : b; }
int elem_size(int dtype) { return dtype == OD_DTYPE_F32 ? 4 : 2; }

// Splits of `steps` steps of work, for each of `tiles` workgroups: the number with which the last workgroup ends first when
// `slots` run at once and each costs `fixed` steps beside its share.  Only numbers that fill the slots a whole number of
// times are worth a look.
int splits_for(long long tiles, long long steps, int slots, int fixed, int limit) {
    long long best = 1, best_cost = -1;
    for (int turns = 1; turns <= 4; ++turns) {
        long long s = most(1, least(turns * (long long)slots / tiles, least(steps, limit)));
        const long long share = (steps + s - 1) / s;
        s = (steps + share - 1) / share;                            // the fewest with this share
        const long long cost = (tiles * s + slots - 1) / slots * (share + fixed);
        if (best_cost < 0 || cost < best_cost) {
            best = s;
            best_cost = cost;
        }
    }
    return (int)best;
}

// Groups that share out the class tiles of a product, in each one or more XCDs: as many as there may be with enough tiles
// for an even division, and with a worker for every row tile unless runs are long (a run that passes from row tile to row
// tile loads its rows again: a piece of 4096 classes for 32768 rows of 512, 156 us in two groups, 158 in one, 171 in eight).
int groups_of(long long tiles, long long row_tiles) {
    int groups = 8;
    while (groups > 1 && (tiles < 8 * groups || (row_tiles * groups > SLOTS && tiles < 512))) groups /= 2;
    return groups;
}

// Everything that follows from the sizes.
struct Plan {
    long long rows, rows_pad, classes, classes_pad;
    int dim, dim_pad, size, n;                  // n: targets per row
    int slabs;                                  // 32-byte slabs of a row where the rows are resident, 0 where they stream
    int row_tile, class_tile, row_tiles;        // of the product
    bool small;                                 // see Resident
    int workgroups;                             // of the product
    long long piece;                            // classes per piece
    int pieces, grad_tile, workers_f, splits_w; // backward; grad_tile: columns of dim per workgroup, workers_f: for each
    // saved buffer
    size_t o_count, o_row_of, o_place, o_lse, o_logit, o_prob, o_packed, o_weight, saved;
    // forward's scratch
    size_t f_weight, f_bias, f_part, f_ends, f_entropy, f_flags, f_counts, forward;
    // backward's scratch
    size_t b_weight, b_bias, b_row_weight, b_scales, b_scaled_f, b_scaled_w, b_dz, b_part_f, b_ends, b_part_w, b_part_b;
    size_t backward;
};

size_t take(size_t& at, long long bytes) {
    const size_t o = at;
    at += (size_t)up(bytes, 256);
    return o;
}

bool plan_of(long long rows, long long classes, int dim, int top, int dtype, Plan& p) {
    p.size = elem_size(dtype);
    p.rows = rows;
    p.rows_pad = up(most(rows, 1), ROW_TILE);
    p.classes = classes;
    p.classes_pad = up(classes, ROW_TILE);
    p.dim = dim;
    // resident rows of 128, 256, 384, 512, 768 or (16-bit) 1024 bytes; wider ones stream in stages of 128
    long long bytes = up((long long)dim * p.size, 128);
    const int resident = dtype == OD_DTYPE_F32 ? 768 : 1024;        // three parts of 1 KiB do not fit the registers
    if (bytes > 512 && bytes <= resident) bytes = up(bytes, 256);
    p.dim_pad = (int)(bytes / p.size);
    p.slabs = bytes <= resident ? (int)(bytes / 32) : 0;
    const long long wide_tiles = (most(rows, 1) + 255) / 256 * (p.classes_pad / 64);
    p.small = p.slabs > 0 && p.slabs <= 16 && wide_tiles <= (p.size == 2 ? SLOTS : SLOTS / 4);
    p.row_tile = p.slabs > 0 && p.slabs <= (dtype == OD_DTYPE_F32 ? 8 : 16) && !p.small ? 256 : 128;
    p.row_tiles = (int)((most(rows, 1) + p.row_tile - 1) / p.row_tile);
    p.class_tile = p.slabs == 0 ? (p.row_tiles * (p.classes_pad / TILE) < SLOTS / 4 ? 32 : TILE)
                                : p.slabs <= 16 && !p.small ? 64 : 32;
    // one thread per 16 bytes of both packed operands, fewer than 2^32 threads in a launch
    if (most(p.rows_pad, p.classes_pad) * p.dim_pad * p.size / 16 > (1ll << 30)) return false;
    p.n = top > 0 ? top : 1;
    p.workgroups = (int)least(SLOTS, up(p.row_tiles * (p.classes_pad / p.class_tile), 8));
    long long piece = most(ROW_TILE, DZ_BYTES / (p.rows_pad * p.size) / ROW_TILE * ROW_TILE);
    p.pieces = (int)((p.classes_pad + piece - 1) / piece);
    p.piece = up((p.classes_pad + p.pieces - 1) / p.pieces, ROW_TILE);
    p.pieces = (int)((p.classes_pad + p.piece - 1) / p.piece);
    // columns of dim per workgroup of the gradient products: what leaves least unused, the widest of those
    p.grad_tile = 256;
    for (int t = 128; t >= 64; t /= 2)
        if (up(p.dim_pad, t) < up(p.dim_pad, p.grad_tile)) p.grad_tile = t;
    const long long dtiles = (p.dim_pad + p.grad_tile - 1) / p.grad_tile;
    const long long ke = 128 / p.size;
    p.workers_f = (int)most(1, GRAD_SLOTS / dtiles);
    // each split writes its own partial result, which costs about as much as eight steps (fp32: as two)
    p.splits_w = splits_for(p.piece / ROW_TILE * dtiles, p.rows_pad / ke, GRAD_SLOTS, p.size == 4 ? 2 : 8, 64);

    size_t at = 0;
    p.o_count = take(at, 4);
    p.o_row_of = take(at, 4 * p.rows_pad);
    p.o_place = take(at, 4 * p.rows_pad);
    p.o_lse = take(at, 4 * p.rows_pad);
    p.o_logit = take(at, 4 * p.rows_pad * p.n);
    p.o_prob = take(at, top > 0 ? 4 * p.rows_pad * p.n : 0);
    p.o_packed = take(at, p.rows_pad * p.dim_pad * p.size);
    p.o_weight = take(at, dim != p.dim_pad ? p.classes * p.dim_pad * p.size : 0);
    p.saved = at;

    at = 0;
    p.f_weight = take(at, dim == p.dim_pad ? p.classes * p.dim_pad * p.size : 0);
    p.f_bias = take(at, 4 * p.classes_pad);
    p.f_part = take(at, 8ll * p.row_tile * groups_of(p.classes_pad / p.class_tile, p.row_tiles) *
                            (p.workgroups / groups_of(p.classes_pad / p.class_tile, p.row_tiles) + p.row_tiles));
    p.f_ends = take(at, 8ll * groups_of(p.classes_pad / p.class_tile, p.row_tiles) * p.row_tiles);
    p.f_entropy = take(at, 4 * p.rows_pad);
    p.f_flags = take(at, p.rows_pad);
    p.f_counts = take(at, 4 * (p.rows / LIST_ROWS + 1));
    p.forward = at;

    at = 0;
    p.b_weight = take(at, dim == p.dim_pad ? p.classes * p.dim_pad * p.size : 0);
    p.b_bias = take(at, 4 * p.classes_pad + 4 * p.piece);
    p.b_row_weight = take(at, 3 * 4 * p.rows_pad);
    p.b_scales = take(at, sizeof(Scales));
    p.b_scaled_f = take(at, p.rows_pad * p.dim_pad * p.size);
    p.b_scaled_w = take(at, dtype == OD_DTYPE_BF16 ? p.classes * p.dim_pad * p.size : 0);
    p.b_dz = take(at, p.rows_pad * p.piece * p.size);
    p.b_part_f = take(at, 4 * (p.workers_f * (long long)ROW_TILE + p.rows_pad) * p.dim_pad);
    p.b_ends = take(at, 8 * (p.rows_pad / ROW_TILE));
    p.b_part_w = take(at, p.splits_w > 1 ? 4 * p.piece * p.dim_pad * p.splits_w : 0);
    p.b_part_b = take(at, 4 * p.piece * p.splits_w);
    p.backward = at;
    return true;
}

int check_call(int64_t rows, int64_t classes, int32_t dim, int32_t top, int32_t dtype, int32_t teacher_dtype,
               float temperature, int32_t reduction) {
    if (dtype < OD_DTYPE_F32 || dtype > OD_DTYPE_BF16 || teacher_dtype < OD_DTYPE_F32 || teacher_dtype > OD_DTYPE_BF16)
        return OD_ERR_ARG;
    if (rows < 0 || classes <= 0 || dim <= 0 || top < 0) return OD_ERR_ARG;
    // its square scales the loss: 2^-126 to 2^126
    if (!(temperature >= 0x1p-63f && temperature <= 0x1p63f) || (top == 0 && temperature != 1.0f)) return OD_ERR_ARG;
    if (reduction < OD_REDUCE_NONE || reduction > OD_REDUCE_SUM) return OD_ERR_ARG;
    if (rows > OD_MAX_VOCAB_ROWS || classes > OD_MAX_VOCAB_CLASSES || dim > OD_MAX_VOCAB_DIM || top > OD_MAX_TEACHER_TOP)
        return OD_ERR_LIMIT;
    return OD_OK;
}

unsigned blocks_of(long long n, int per) { return (unsigned)((n + per - 1) / per); }

// Whether tiles can be read from the caller's weight rows: whole stages of K, 16-byte chunks, and 64 rows within 31 bits.
bool weight_in_place(const Plan& p, const void* weight, long long pitch) {
    return p.dim == p.dim_pad && (pitch * p.size) % 16 == 0 && pitch * p.size <= (1 << 24) && ((uintptr_t)weight & 15) == 0;
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

RowLists lists_of(const Call& c) {
    return {(int*)(c.saved + c.p.o_count), (int*)(c.saved + c.p.o_row_of), (int*)(c.saved + c.p.o_place)};
}

// Packs what has to be packed and says where the product finds its weight rows.  `with_features`: forward.
template <typename T>
int prepare(const Call& c, bool with_features, const unsigned char* flags, size_t weight_at, size_t bias_at, long long bias_len,
            Scales* scales, const char** rows, long long* pitch) {
    const Plan& p = c.p;
    PrepareArgs a = {};
    const long long row_chunks = p.dim_pad * p.size / 16;
    a.lists = lists_of(c);
    a.dim = p.dim;
    a.dim_pad = p.dim_pad;
    int scan = 0;
    if (with_features) {
        a.features = c.features;
        a.feature_pitch = c.feature_pitch;
        a.packed = c.saved + p.o_packed;
        a.rows_pad = p.rows_pad;
        a.feature_blocks = blocks_of(p.rows_pad * row_chunks, VT);
        a.targets = c.targets;
        a.flags = flags;
        a.rows = (int)p.rows;
        a.row_loss = c.row_loss;
        scan = p.rows <= 4 * VT ? 4 : p.rows <= LIST_ROWS ? LIST_ROWS / VT : 0;
        if (scan == 0) {
            int* counts = (int*)(c.ws + p.f_counts);
            const dim3 grid(blocks_of(p.rows, LIST_ROWS));
            hipLaunchKernelGGL(count_rows_kernel, grid, dim3(VT), 0, c.stream, c.targets, flags, (int)p.rows, counts);
            OD_LAUNCH_CHECK();
            hipLaunchKernelGGL(list_rows_kernel, grid, dim3(VT), 0, c.stream, c.targets, flags, (int)p.rows, (const int*)counts,
                               a.lists, c.row_loss);
            OD_LAUNCH_CHECK();
        }
    }
    *rows = (const char*)c.weight;
    *pitch = c.weight_pitch * p.size;
    if (!weight_in_place(p, c.weight, c.weight_pitch)) {
        const bool keep = p.dim != p.dim_pad;                       // for the backward pass, which then need not pack again
        char* packed = keep ? c.saved + p.o_weight : c.ws + weight_at;
        if (with_features || !keep) {
            a.weight = c.weight;
            a.weight_pitch = c.weight_pitch;
            a.packed_weight = packed;
            a.weight_blocks = blocks_of(p.classes * row_chunks, VT);
        }
        *rows = packed;
        *pitch = (long long)p.dim_pad * p.size;
    }
    a.classes = p.classes;
    a.bias = c.bias;
    a.bias_len = (int)bias_len;
    a.scale = LOG2E / c.temperature;
    a.bias2 = (float*)(c.ws + bias_at);
    a.scales = scales;
    a.upstream = c.upstream;
    a.reduction = c.reduction;
    a.temperature = c.temperature;
    const dim3 grid(a.feature_blocks + a.weight_blocks + blocks_of(bias_len, VT));
    if (scan == 4) hipLaunchKernelGGL((prepare_kernel<T, 4>), grid, dim3(VT), 0, c.stream, a);
    else if (scan == 16) hipLaunchKernelGGL((prepare_kernel<T, 16>), grid, dim3(VT), 0, c.stream, a);
    else hipLaunchKernelGGL((prepare_kernel<T, 0>), grid, dim3(VT), 0, c.stream, a);
    OD_LAUNCH_CHECK();
    return OD_OK;
}

// The product by the kernel for its row width.
template <typename T, bool GRAD>
int launch_product(const Call& c, int kernel, const ProductArgs& a) {
    const dim3 grid((unsigned)c.p.workgroups);
    switch (c.p.slabs) {
#define OD_PRODUCT(KS)                                                                                        \
    case KS:                                                                                                  \
        if (c.p.small) OD_LAUNCH_KERNEL(kernel, (resident_kernel<T, KS, GRAD, true>), grid, dim3(VT), 0, c.stream, a); \
        else OD_LAUNCH_KERNEL(kernel, (resident_kernel<T, KS, GRAD, false>), grid, dim3(VT), 0, c.stream, a);  \
        break
        OD_PRODUCT(4);
        OD_PRODUCT(8);
        OD_PRODUCT(12);
        OD_PRODUCT(16);
#undef OD_PRODUCT
        case 24: OD_LAUNCH_KERNEL(kernel, (resident_kernel<T, 24, GRAD, false>), grid, dim3(VT), 0, c.stream, a); break;
        case 32:
            if constexpr (sizeof(T) == 2)
                OD_LAUNCH_KERNEL(kernel, (resident_kernel<T, 32, GRAD, false>), grid, dim3(VT), 0, c.stream, a);
            break;
        default:
            if (c.p.class_tile == TILE)
                OD_LAUNCH_KERNEL(kernel, (product_kernel<T, GRAD, TILE>), grid, dim3(VT), 0, c.stream, a);
            else OD_LAUNCH_KERNEL(kernel, (product_kernel<T, GRAD, 32>), grid, dim3(VT), 0, c.stream, a);
            break;
    }
    return OD_OK;
}

template <typename G, bool ROWS, bool DIRECT = false>
int launch_grad(const Call& c, int kernel, const GradArgs& g) {
    const Plan& p = c.p;
    const long long dtiles = (p.dim_pad + p.grad_tile - 1) / p.grad_tile;
    const dim3 grid((unsigned)(dtiles * (ROWS ? g.splits : g.cols / ROW_TILE * g.splits))), block(2 * VT);
    if (p.grad_tile == 256) OD_LAUNCH_KERNEL(kernel, (grad_kernel<G, 4, ROWS, DIRECT>), grid, block, 0, c.stream, g);
    else if (p.grad_tile == 128) OD_LAUNCH_KERNEL(kernel, (grad_kernel<G, 2, ROWS, DIRECT>), grid, block, 0, c.stream, g);
    else OD_LAUNCH_KERNEL(kernel, (grad_kernel<G, 1, ROWS, DIRECT>), grid, block, 0, c.stream, g);
    return OD_OK;
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
    ProductArgs a = {};
    int rc = prepare<T>(c, true, flags, p.f_weight, p.f_bias, p.classes_pad, nullptr, &a.weight, &a.weight_pitch);
    if (rc != OD_OK) return rc;
    a.features = c.saved + p.o_packed;
    a.dim_pad = p.dim_pad;
    a.first_class = 0;
    a.last_class = p.classes - 1;
    a.bias2 = (const float*)(c.ws + p.f_bias);
    a.count = lists.count;
    a.tiles = (int)(p.classes_pad / p.class_tile);
    a.groups = groups_of(a.tiles, p.row_tiles);
    a.row_tiles = p.row_tiles;
    a.scale = LOG2E / c.temperature;
    a.part = (float2*)(c.ws + p.f_part);
    a.ends = (int2*)(c.ws + p.f_ends);
    rc = launch_product<T, false>(c, OD_KERNEL_VOCAB_LSE, a);
    if (rc != OD_OK) return rc;
    TargetArgs t = {};
    t.features = a.features;
    t.dim_pad = p.dim_pad;
    t.weight = a.weight;
    t.weight_pitch = a.weight_pitch;
    t.bias = c.bias;
    t.classes = p.classes;
    t.targets = c.targets;
    t.top = c.top;
    t.prob = prob;
    t.entropy = entropy;
    t.lists = lists;
    t.part = a.part;
    t.ends = a.ends;
    t.groups = a.groups;
    t.row_tile = p.row_tile;
    t.row_tiles = p.row_tiles;
    t.rows_pad = p.rows_pad;
    t.temperature = c.temperature;
    t.lse2 = (float*)(c.saved + p.o_lse);
    t.target_logit = (float*)(c.saved + p.o_logit);
    t.row_loss = c.row_loss;
    const dim3 grid(blocks_of(p.rows_pad, VT / 64));
    if (c.top > 0) hipLaunchKernelGGL((targets_kernel<T, 4>), grid, dim3(VT), 0, c.stream, t);
    else hipLaunchKernelGGL((targets_kernel<T, 1>), grid, dim3(VT), 0, c.stream, t);
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
    typedef typename GradOf<T>::type G;
    constexpr bool BF16 = std::is_same<T, bf16_t>::value, WIDE = sizeof(T) == 4;
    const Plan& p = c.p;
    const RowLists lists = lists_of(c);
    const bool weighted = c.reduction == OD_REDUCE_NONE;
    float* row_weight = (float*)(c.ws + p.b_row_weight);
    const RowWeights weights = {row_weight, row_weight + p.rows_pad, row_weight + 2 * p.rows_pad};
    const float* lse2 = (const float*)(c.saved + p.o_lse);
    Scales* scales = (Scales*)(c.ws + p.b_scales);
    if (weighted) {
        hipLaunchKernelGGL(row_weights_kernel, dim3(1), dim3(1024), 0, c.stream, c.upstream, lists, p.rows_pad, c.temperature,
                           lse2, weights, scales);
        OD_LAUNCH_CHECK();
    }
    ProductArgs a = {};
    // the bias table: the last piece may reach past the last tile
    int rc = prepare<T>(c, false, nullptr, p.b_weight, p.b_bias, p.classes_pad + p.piece, weighted ? nullptr : scales,
                        &a.weight, &a.weight_pitch);
    if (rc != OD_OK) return rc;
    a.features = c.saved + p.o_packed;

    // operands of the gradient products: bf16 values and weighted rows change their form, the others stay what they are
    const char *grad_features = a.features, *grad_weight = a.weight;
    long long grad_weight_pitch = a.weight_pitch;
    const bool scale_f = !WIDE && (BF16 || weighted), scale_w = BF16;
    const long long row_chunks = p.dim_pad * p.size / 16;
    Operands ops = {};
    ops.dim_pad = p.dim_pad;
    if ((scale_f || weighted) && (c.dweight || c.dbias)) {
        ops.part[0] = {a.features, p.dim_pad, p.rows_pad, weighted ? row_weight : nullptr, lists.count,
                       scale_f ? &scales->features_max : nullptr, c.ws + p.b_scaled_f, 0};
        grad_features = c.ws + p.b_scaled_f;
    }
    if (scale_w && c.dfeatures) {
        ops.part[1] = {a.weight, a.weight_pitch / p.size, p.classes, nullptr, nullptr, &scales->weight_max, c.ws + p.b_scaled_w,
                       0};
        grad_weight = c.ws + p.b_scaled_w;
        grad_weight_pitch = (long long)p.dim_pad * p.size;
    }
    unsigned blocks = 0;
    for (Operand& o : ops.part) blocks += o.blocks = o.max_bits ? (unsigned)least(blocks_of(o.rows * row_chunks, VT), 256) : 0;
    if (blocks > 0) {
        hipLaunchKernelGGL(max_kernel<T>, dim3(blocks), dim3(VT), 0, c.stream, ops);
        OD_LAUNCH_CHECK();
    }
    blocks = 0;
    for (Operand& o : ops.part) blocks += o.blocks = o.out ? blocks_of(o.rows * row_chunks, VT) : 0;
    if (blocks > 0) {
        hipLaunchKernelGGL(scale_kernel<T>, dim3(blocks), dim3(VT), 0, c.stream, ops);
        OD_LAUNCH_CHECK();
    }

    a.dim_pad = p.dim_pad;
    a.last_class = p.classes - 1;
    a.count = lists.count;
    a.tiles = (int)(p.piece / p.class_tile);
    a.groups = groups_of(a.tiles, p.row_tiles);
    a.row_tiles = p.row_tiles;
    a.scale = LOG2E / c.temperature;
    a.lse2 = weighted ? weights.lse2 : lse2;
    a.dz = c.ws + p.b_dz;
    a.piece = p.piece;
    const int ke = 128 / p.size;
    for (int k = 0; k < p.pieces; ++k) {
        const long long first = k * p.piece;
        a.first_class = first;
        a.bias2 = (const float*)(c.ws + p.b_bias) + first;
        rc = launch_product<T, true>(c, OD_KERNEL_VOCAB_DZ, a);
        if (rc != OD_OK) return rc;
        hipLaunchKernelGGL(correct_targets_kernel<G>, dim3(blocks_of(p.rows * p.n, VT)), dim3(VT), 0, c.stream, c.targets,
                           c.top, (const float*)(c.saved + p.o_prob), lists, lse2, (const float*)(c.saved + p.o_logit),
                           weighted ? weights.mantissa : (const float*)nullptr, first, p.piece, p.classes,
                           (float)(1 << GradOf<T>::LOG2_DZ), (G*)(c.ws + p.b_dz));
        OD_LAUNCH_CHECK();
        GradArgs g = {};
        g.dz = c.ws + p.b_dz;
        g.piece = p.piece;
        g.dim_pad = p.dim_pad;
        g.count = lists.count;
        if (c.dfeatures) {
            g.a = grad_weight + first * grad_weight_pitch;
            g.a_pitch = grad_weight_pitch;
            g.a_last = p.classes - 1 - first;
            g.cols = p.rows_pad;
            g.ksteps = p.piece / ke;
            g.splits = p.workers_f;
            g.out = (float*)(c.ws + p.b_part_f);
            g.ends = (int2*)(c.ws + p.b_ends);
            g.accumulate = k > 0;
            rc = launch_grad<G, true>(c, OD_KERNEL_VOCAB_GRAD_ROWS, g);
            if (rc != OD_OK) return rc;
        }
        if (c.dweight || c.dbias) {
            g.a = grad_features;
            g.a_pitch = (long long)p.dim_pad * p.size;
            g.a_last = p.rows_pad - 1;
            g.cols = p.piece;
            g.ksteps = p.rows_pad / ke;
            g.splits = p.splits_w;
            g.out = (float*)(c.ws + p.b_part_w);
            g.accumulate = 0;
            g.bias_out = c.dbias ? (float*)(c.ws + p.b_part_b) : nullptr;
            g.row_weight = weighted ? row_weight : nullptr;
            const bool direct = p.splits_w == 1;
            if (direct) {
                g.result = c.dweight ? (T*)c.dweight + first * p.dim : nullptr;
                g.bf16_result = BF16;
                g.dim = p.dim;
                g.scaled = scale_f;
                g.classes = least(p.piece, p.classes - first);
                g.scales = scales;
            }
            rc = direct ? launch_grad<G, false, true>(c, OD_KERNEL_VOCAB_GRAD_CLASSES, g)
                        : launch_grad<G, false>(c, OD_KERNEL_VOCAB_GRAD_CLASSES, g);
            if (rc != OD_OK) return rc;
        }
        FinishArgs f = {};
        f.scales = scales;
        f.dim = p.dim;
        f.dim_pad = p.dim_pad;
        f.piece = p.piece;
        f.classes = least(p.piece, p.classes - first);
        const int groups = (p.dim + 3) / 4;
        unsigned finish_blocks = 0;
        if (c.dweight && p.splits_w > 1) {
            f.part_w = (const float*)(c.ws + p.b_part_w);
            f.dweight = (T*)c.dweight + first * p.dim;
            finish_blocks += f.weight_blocks = blocks_of(f.classes * groups, VT);
        }
        if (c.dbias) {
            f.part_b = (const float*)(c.ws + p.b_part_b);
            f.dbias = (T*)c.dbias + first;
            finish_blocks += f.bias_blocks = blocks_of(f.classes, VT);
        }
        f.splits_w = p.splits_w;
        f.scaled_f = scale_f;
        if (c.dfeatures && k == p.pieces - 1) {
            f.part_f = (const float*)(c.ws + p.b_part_f);
            f.rows = p.rows;
            f.ends = (const int2*)(c.ws + p.b_ends);
            f.scaled_w = scale_w;
            f.place = lists.place;
            f.row_weight = weighted ? row_weight : nullptr;
            f.dfeatures = c.dfeatures;
            finish_blocks += blocks_of(f.rows * groups, VT);
        }
        if (finish_blocks > 0) {
            hipLaunchKernelGGL(finish_kernel<T>, dim3(finish_blocks), dim3(VT), 0, c.stream, f);
            OD_LAUNCH_CHECK();
        }
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
