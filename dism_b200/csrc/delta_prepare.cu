// Chunk matrices of the gated delta rule: T = (I + L diag(b))^-1, P = scale tril(E * Q K^T) and the decay table of every
// chunk of 64 positions and every value head; all independent of one another and of the state.
#include "delta_common.cuh"

namespace dism {
namespace {

constexpr int PREPARE_THREADS = 128;

// Columns FIRST .. FIRST+31 of the inverse, one per lane, by forward substitution in 32 bits: row i of I - L diag(b) T.
// Rows above FIRST are zero in these columns.
template <int FIRST>
__device__ __forceinline__ void substitute(float (&x)[CHUNK], const float* a, int lane) {
#pragma unroll
    for (int i = FIRST; i < CHUNK; ++i) {
        float sum0 = lane == i - FIRST ? 1.f : 0.f, sum1 = 0.f, sum2 = 0.f, sum3 = 0.f;
#pragma unroll
        for (int s = FIRST; s < i; s += 4) {
            const float4 c = *reinterpret_cast<const float4*>(a + i * (CHUNK + 4) + s);  // zero from the diagonal on
            sum0 -= c.x * x[s];
            if (s + 1 < i) sum1 -= c.y * x[s + 1];
            if (s + 2 < i) sum2 -= c.z * x[s + 2];
            if (s + 3 < i) sum3 -= c.w * x[s + 3];
        }
        x[i] = (sum0 + sum1) + (sum2 + sum3);
    }
}

// Rows i and i+1 of a column pair leave as one 4-byte store per lane: even lanes take row i, odd lanes row i+1.
template <int FIRST>
__device__ __forceinline__ void store_columns(const float (&x)[CHUNK], __nv_bfloat16* t, __nv_bfloat16* rest, int lane) {
    const int column = FIRST + lane, odd = lane & 1;
    unsigned* out = reinterpret_cast<unsigned*>(t);
    unsigned* out_rest = reinterpret_cast<unsigned*>(rest);
#pragma unroll
    for (int i = FIRST; i < CHUNK; i += 2) {
        const float other = __shfl_xor_sync(FULL, odd ? x[i] : x[i + 1], 1);
        const float lo = odd ? other : x[i], hi = odd ? x[i + 1] : other;
        const unsigned value = pack2(lo, hi);
        const int row = i + odd, word = ((row >> 3) * (CHUNK / 8) + (column >> 3)) * 32 + (row & 7) * 4 + ((column & 7) >> 1);
        out[word] = value;
        if (rest) out_rest[word] = pack2_rest(lo, hi, value);
    }
}

template <int D>
__global__ void __launch_bounds__(PREPARE_THREADS) delta_prepare_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                        const __nv_bfloat16* __restrict__ k, const void* __restrict__ g,
                                                                        const void* __restrict__ beta, DeltaSaved saved) {
    constexpr int PITCH = 2 * D + 16;
    extern __shared__ __align__(16) unsigned char shared[];
    unsigned char *ks = shared, *qs = shared + CHUNK * PITCH;
    float* a = reinterpret_cast<float*>(shared + 2 * CHUNK * PITCH);  // L diag(b), [CHUNK][CHUNK + 4]
    float* table = a + CHUNK * (CHUNK + 4);                           // G as a pair, then b
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31, head = blockIdx.y;
    const int key_head = head / (shape.heads / shape.key_heads);
    int64_t row;
    int count;
    const int64_t slot = blockIdx.x;
    shape.layout.chunk(slot, row, count);
    if (count == 0) return;
    const int64_t stride = int64_t(shape.key_heads) * D * 2, at = (row * shape.key_heads + key_head) * D * 2;
    load_rows<2 * D, PREPARE_THREADS>(smem_address(ks), PITCH, reinterpret_cast<const char*>(k) + at, stride, count, thread);
    load_rows<2 * D, PREPARE_THREADS>(smem_address(qs), PITCH, reinterpret_cast<const char*>(q) + at, stride, count, thread);
    cp_async_commit();
    const int64_t place = slot * shape.heads + head;
    if (warp == 0) {
        // G in 64 bits, kept as two floats: its differences stay exact to 32 bits however far the sum has run.  A decay
        // of zero (g of minus infinity) becomes 2^-256, which is zero in 32 bits and leaves the sums finite.
        float* rows = saved.rows + place * ROW_VALUES;
        double sum[2];
        float b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = 2 * lane + e;
            const int64_t index = (row + t) * shape.heads + head;
            const double step = t < count ? double(gate(g, index, shape.gates_bf16)) * 1.4426950408889634 : 0.;
            sum[e] = step < -256. ? -256. : step;
            b[e] = t < count ? gate(beta, index, shape.gates_bf16) : 0.f;
        }
        sum[1] += sum[0];
        double before = sum[1];
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const double other = __shfl_up_sync(FULL, before, s);
            if (lane >= s) before += other;
        }
        const double total = __shfl_sync(FULL, before, 31);
        before -= sum[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = 2 * lane + e;
            const double here = before + sum[e];
            const float hi = float(here), lo = float(here - double(hi));
            table[t] = hi, table[CHUNK + t] = lo, table[2 * CHUNK + t] = b[e];
            rows[t] = ex2(hi) * (1.f + lo * .6931471805599453f);
            rows[CHUNK + t] = b[e];
            rows[2 * CHUNK + t] = ex2(float(total - here));
            rows[3 * CHUNK + t] = hi;
            rows[4 * CHUNK + t] = lo;
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // E * K K^T below the diagonal and P: warp w takes rows 16 w .. 16 w + 15 and the column tiles up to the diagonal
    {
        float kk[CHUNK / 8][4], qk[CHUNK / 8][4];
#pragma unroll
        for (int n = 0; n < CHUNK / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) kk[n][e] = qk[n][e] = 0.f;
        const unsigned own = smem_address(ks) + warp * 16 * PITCH + rows_first(lane, PITCH), own_q = own + CHUNK * PITCH;
        const unsigned all = smem_address(ks) + cols_first(lane, PITCH);
#pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) {
            unsigned ka[4], qa[4];
            ldsm4(ka, own + kb * 32);
            ldsm4(qa, own_q + kb * 32);
#pragma unroll
            for (int np = 0; np < CHUNK / 16; ++np) {
                if (np > warp) continue;
                unsigned b[4];
                ldsm4(b, all + np * 16 * PITCH + kb * 32);
                mma16816(kk[2 * np], ka, b[0], b[1]);
                mma16816(kk[2 * np + 1], ka, b[2], b[3]);
                mma16816(qk[2 * np], qa, b[0], b[1]);
                mma16816(qk[2 * np + 1], qa, b[2], b[3]);
            }
        }
        unsigned* p = reinterpret_cast<unsigned*>(saved.p + place * MATRIX);
#pragma unroll
        for (int n = 0; n < CHUNK / 8; ++n) {
            if (n > 2 * warp + 1) continue;
            const int s = 8 * n + 2 * (lane & 3);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int t = 16 * warp + 8 * half + (lane >> 2);
                float pv[2], av[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float between = ex2((table[t] - table[s + e]) + (table[CHUNK + t] - table[CHUNK + s + e]));
                    pv[e] = s + e <= t ? shape.scale * between * qk[n][2 * half + e] : 0.f;
                    av[e] = s + e < t ? between * kk[n][2 * half + e] * table[2 * CHUNK + s + e] : 0.f;
                }
                p[((2 * warp + half) * (CHUNK / 8) + n) * 32 + lane] = pack2(pv[0], pv[1]);
                *reinterpret_cast<float2*>(a + t * (CHUNK + 4) + s) = make_float2(av[0], av[1]);
            }
        }
    }
    __syncthreads();
    if (warp < 2) {
        float x[CHUNK];
        __nv_bfloat16* t = saved.t + place * MATRIX;
        __nv_bfloat16* rest = saved.t_rest ? saved.t_rest + place * MATRIX : nullptr;
        if (warp == 0) {
            substitute<0>(x, a, lane);
            store_columns<0>(x, t, rest, lane);
        } else {
            substitute<32>(x, a, lane);
            store_columns<32>(x, t, rest, lane);
        }
    }
}

template <int D>
cudaError_t launch(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const void* g, const void* beta,
                   const DeltaSaved& saved, cudaStream_t stream) {
    constexpr int BYTES = 2 * CHUNK * (2 * D + 16) + CHUNK * (CHUNK + 4) * 4 + 3 * CHUNK * 4;
    if (cudaError_t status = cudaFuncSetAttribute(delta_prepare_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES)) return status;
    KernelTimer timer("delta_prepare", stream);
    delta_prepare_kernel<D><<<dim3(unsigned(shape.layout.slots()), shape.heads), PREPARE_THREADS, BYTES, stream>>>(shape, q, k, g, beta, saved);
    return cudaGetLastError();
}
}  // namespace

cudaError_t launch_delta_prepare(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const void* g,
                                 const void* beta, const DeltaSaved& saved, cudaStream_t stream) {
    if (shape.d == 32) return launch<32>(shape, q, k, g, beta, saved, stream);
    if (shape.d == 64) return launch<64>(shape, q, k, g, beta, saved, stream);
    return launch<128>(shape, q, k, g, beta, saved, stream);
}

}  // namespace dism
