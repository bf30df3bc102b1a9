// state_fork.hip -- rows of recurrent states become copies of others, in place
// (beam search's reordering, forks of one prompt), in every buffer of a call.
//
// Row dst[i] of a buffer becomes row src[i] as it was.  In place: a workgroup
// takes a column (some bytes of every row) and has read it of all sources
// before it writes it to any destination, so that cycles and chains need no
// second copy of the states.  Each row that moves is read and written once, and
// rows that stay are not touched.  Bound by HBM: 24 rows, 24 layers' states and
// conv buffers, 442 us (the same bytes by a large copy 490).
#include "qm_device.h"
#include "qm_beam.h"

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

// The pairs whose rows differ, packed; -1: the list is refused (a row outside
// the buffers, a destination listed twice).  Every workgroup finds the same.
struct Moves {
    int32_t src[QMK_STATE_COUNT], dst[QMK_STATE_COUNT];
    int32_t n, bad;
    uint32_t seen[QMK_STATE_ROWS / 32];
};
QM_DEV int find_moves(const StateForkArgs& A, Moves& m, int threads) {
    const int tid = threadIdx.x;
    for (int i = tid; i < (A.rows + 31) / 32; i += threads) m.seen[i] = 0;
    if (tid == 0) m.n = m.bad = 0;
    __syncthreads();
    for (int i = tid; i < A.count; i += threads) {
        const int s = A.src[i], d = A.dst ? A.dst[i] : i;
        if ((uint32_t)s >= (uint32_t)A.rows || (uint32_t)d >= (uint32_t)A.rows) {
            m.bad = 1;
            continue;
        }
        if (atomicOr(&m.seen[d >> 5], 1u << (d & 31)) >> (d & 31) & 1) m.bad = 1;
        if (s != d) {
            const int at = atomicAdd(&m.n, 1);
            m.src[at] = s;
            m.dst[at] = d;
        }
    }
    __syncthreads();
    const int n = m.bad ? -1 : m.n;
    if (blockIdx.x == 0 && tid == 0) A.result[0] = n < 0 ? -1 : 0;
    return n;
}
// The buffer of column `at` (uniform).
QM_DEV int buffer_of(const StateForkArgs& A, int64_t at) {
    int lo = 0, hi = A.buffers - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (A.first[mid] <= at) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Up to N rows: a lane holds its 16 bytes of all of them, or 8 or 4 of more (in
// registers / by way of LDS, us, 24 layers' states: 8 rows 170 / 379, 16 348 /
// 715; 8 layers': 40 rows 280 / 630, 64 456 / 976, 128 952 / 1917; where 2 rows
// move, registers for 8 / for 32 34 / 54).
template <int N, class V>
QM_DEV void fork_few(const StateForkArgs& A) {
    __shared__ Moves m;
    const int n = __builtin_amdgcn_readfirstlane(find_moves(A, m, 256));
    if (n <= 0) return;
    for (int64_t at = blockIdx.x; at < A.first[A.buffers]; at += gridDim.x) {
        const int k = buffer_of(A, at);
        const int64_t stride = A.buffer[k].stride, off = (at - A.first[k]) * (256 * (int)sizeof(V)) + (int)sizeof(V) * (int64_t)threadIdx.x;
        if (off >= A.buffer[k].bytes) continue;
        uint8_t* base = A.buffer[k].rows + off;
        V x[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) x[i] = *reinterpret_cast<const V*>(base + (int64_t)__builtin_amdgcn_readfirstlane(m.src[i]) * stride);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) *reinterpret_cast<V*>(base + (int64_t)__builtin_amdgcn_readfirstlane(m.dst[i]) * stride) = x[i];
    }
}
extern "C" __global__ __launch_bounds__(256) void qm_state_fork_8(StateForkArgs A) { fork_few<8, uintx4>(A); }
extern "C" __global__ __launch_bounds__(256) void qm_state_fork_32(StateForkArgs A) { fork_few<32, uintx4>(A); }
extern "C" __global__ __launch_bounds__(256) void qm_state_fork_64(StateForkArgs A) { fork_few<64, uintx2>(A); }
extern "C" __global__ __launch_bounds__(256) void qm_state_fork_128(StateForkArgs A) { fork_few<128, uint32_t>(A); }

// More: in LDS.
extern "C" __global__ __launch_bounds__(256) void qm_state_fork_many(StateForkArgs A) {
    __shared__ Moves m;
    __shared__ __attribute__((aligned(16))) uintx4 held[QMK_STATE_LDS / 16];
    const int n = __builtin_amdgcn_readfirstlane(find_moves(A, m, 256));
    if (n <= 0) return;
    const int wide = A.column / 16, all = n * wide;        // 16-byte pieces of a row's column, of all
    for (int64_t at = blockIdx.x; at < A.first[A.buffers]; at += gridDim.x) {
        const int k = buffer_of(A, at);
        const int64_t stride = A.buffer[k].stride, off = (at - A.first[k]) * A.column, left = A.buffer[k].bytes - off;
        uint8_t* base = A.buffer[k].rows + off;
#pragma unroll 4
        for (int p = threadIdx.x; p < all; p += 256) {
            const int i = p / wide, c = 16 * (p - i * wide);
            if (c < left) held[p] = *reinterpret_cast<const uintx4*>(base + m.src[i] * stride + c);
        }
        __syncthreads();
#pragma unroll 4
        for (int p = threadIdx.x; p < all; p += 256) {
            const int i = p / wide, c = 16 * (p - i * wide);
            if (c < left) *reinterpret_cast<uintx4*>(base + m.dst[i] * stride + c) = held[p];
        }
        __syncthreads();
    }
}
