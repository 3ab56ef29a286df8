// linear.cu -- dense layers on the 5th-generation tensor cores.
//
//   forward    z = x W^T + b, y = act(z) + r
//   backward   dz = dy act'(z), dx = dz W + r, dW = dz^T x, db = column sums of dz
//
// All three products are one kernel, D[m][n] = sum_k A(m, k) B(n, k):
//   forward          A = x  [rows][in]   K-major   B = W  [out][in]   K-major
//   input gradient   A = dz [rows][out]  K-major   B = W  [out][in]   MN-major
//   weight gradient  A = dz [rows][out]  MN-major  B = x  [rows][in]  MN-major
// The tensor core reads either order from the same row-major boxes (tma.cuh),
// so nothing is transposed in memory.
//
// k_gemm: persistent CTAs, one 128 x BN tile (or one part of its K range) at
// a time.  Warp 0 copies operand boxes into a ring of shared-memory stages,
// one thread of warp 1 issues the MMAs into one of two tensor-memory
// accumulators, warps 4-7 drain the other one: the copies, the products and
// the epilogue of the tile before overlap.  Matrices whose rows do not start
// on 16-byte boundaries cannot be copied by the tensor copy unit; four more
// warps load them instead (plain_loads).
#include <cuda_bf16.h>

#include <atomic>

#include "linear.h"
#include "tma.cuh"

namespace nb {
namespace {

constexpr uint32_t kBM = kGemmBM, kBK = kGemmBK;
constexpr uint32_t kStageBytesA = kBM * 128u;
constexpr uint32_t kEpiWarps = 4;
constexpr uint32_t kSlabBytes = 32u * 128u;  // one epilogue warp's 32 rows x 128 bytes
constexpr uint32_t kMaxStages = 8;

__host__ __device__ constexpr uint32_t gemm_stages(uint32_t bn) { return bn >= 256u ? 4u : bn >= 128u ? 6u : 8u; }
__host__ __device__ constexpr uint32_t gemm_smem(uint32_t bn) {
    return 1024u + gemm_stages(bn) * (kStageBytesA + bn * 128u) + kEpiWarps * kSlabBytes + bn * 4u;
}
__host__ __device__ constexpr uint32_t tmem_cols(uint32_t n) { return n <= 32u ? 32u : n <= 64u ? 64u : n <= 128u ? 128u : n <= 256u ? 256u : 512u; }

// ------------------------------------------------------------ 16-bit values
NB_DEV float from_16(uint16_t v, bool bf16) {
    if (bf16) return __uint_as_float(static_cast<uint32_t>(v) << 16);
    return h2f_bits(v);
}
NB_DEV float2 unpack_16(uint32_t v, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return unpack_h2(v);
}
NB_DEV uint32_t pack_16(float lo, float hi, bool bf16) {
    if (bf16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    return pack_h2(lo, hi);
}
NB_DEV uint16_t to_16(float v, bool bf16) { return static_cast<uint16_t>(pack_16(v, 0.0f, bf16) & 0xffffu); }

// ------------------------------------------------------------- activations
NB_DEV float sigmoid_f(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }
NB_DEV float act_f(float z, uint32_t act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? z : 0.0f;
        case kActSilu: return z * sigmoid_f(z);
        case kActGelu: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case kActSigmoid: return sigmoid_f(z);
        default: return z;
    }
}
// One activation over a register row: the choice is made once, not per value.
template <int N>
NB_DEV void act_row(float (&v)[N], uint32_t act) {
    switch (act) {
#define NB_ACT_ROW(kind)                                   \
    case kind:                                             \
        _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = act_f(v[i], kind); \
        break;
        NB_ACT_ROW(kActRelu)
        NB_ACT_ROW(kActSilu)
        NB_ACT_ROW(kActGelu)
        NB_ACT_ROW(kActSigmoid)
#undef NB_ACT_ROW
        default: break;
    }
}
// dy act'(z).  ReLU selects: a closed unit passes nothing, whatever dy holds.
NB_DEV float dact_f(float dy, float z, uint32_t act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? dy : 0.0f;
        case kActSilu: {
            const float s = sigmoid_f(z);
            return dy * (s * (1.0f + z * (1.0f - s)));
        }
        case kActGelu:
            return dy * (0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __expf(-0.5f * z * z));
        case kActSigmoid: {
            const float s = sigmoid_f(z);
            return dy * (s * (1.0f - s));
        }
        default: return dy;
    }
}

// ------------------------------------------------- slabs: 32 rows x 128 bytes
// A warp's shared-memory slab, 16-byte pieces swizzled by the row so that both
// "one row a thread" and "eight threads a row" accesses are conflict-free.
NB_DEV uint32_t slab_at(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

// Global -> slab or back: `rows` rows of `cols` values of ES bytes (cols * ES
// <= 128) at g, ld values apart; vec: every row's first value is 16-byte aligned.
template <int ES, bool kStore>
NB_DEV void slab_copy(unsigned char* slab, unsigned char* g, uint64_t ld, uint32_t rows, uint32_t cols, bool vec, uint32_t lane) {
    constexpr uint32_t kPer = 16u / ES;
    if (vec) {
        const uint32_t p = lane & 7u;
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const uint32_t r = (lane >> 3) + 4u * i;
            if (r >= rows || p * kPer >= cols) continue;
            unsigned char* q = g + (r * ld + p * kPer) * ES;
            unsigned char* l = slab + slab_at(r, p);
            if ((p + 1u) * kPer <= cols) {
                if (kStore) *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(l);
                else *reinterpret_cast<uint4*>(l) = *reinterpret_cast<const uint4*>(q);
            } else {
                for (uint32_t e = 0; e < cols - p * kPer; ++e) {
                    if (ES == 2) {
                        if (kStore) reinterpret_cast<uint16_t*>(q)[e] = reinterpret_cast<const uint16_t*>(l)[e];
                        else reinterpret_cast<uint16_t*>(l)[e] = reinterpret_cast<const uint16_t*>(q)[e];
                    } else {
                        if (kStore) reinterpret_cast<uint32_t*>(q)[e] = reinterpret_cast<const uint32_t*>(l)[e];
                        else reinterpret_cast<uint32_t*>(l)[e] = reinterpret_cast<const uint32_t*>(q)[e];
                    }
                }
            }
        }
        return;
    }
    for (uint32_t r = 0; r < rows; ++r) {
        for (uint32_t c = lane; c < cols; c += 32u) {
            unsigned char* q = g + (r * ld + c) * ES;
            unsigned char* l = slab + slab_at(r, c / kPer) + (c % kPer) * ES;
            if (ES == 2) {
                if (kStore) *reinterpret_cast<uint16_t*>(q) = *reinterpret_cast<const uint16_t*>(l);
                else *reinterpret_cast<uint16_t*>(l) = *reinterpret_cast<const uint16_t*>(q);
            } else {
                if (kStore) *reinterpret_cast<uint32_t*>(q) = *reinterpret_cast<const uint32_t*>(l);
                else *reinterpret_cast<uint32_t*>(l) = *reinterpret_cast<const uint32_t*>(q);
            }
        }
    }
}
NB_DEV void slab_put(unsigned char* slab, uint32_t row, uint32_t piece, const uint32_t w[4]) {
    *reinterpret_cast<uint4*>(slab + slab_at(row, piece)) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------- operand boxes
// `rows` x 64 values at (row0, col0) of a matrix -> a swizzled box, zero
// outside the matrix, by 128 threads.
NB_DEV void fill_box(unsigned char* box, const MatrixView& m, uint32_t row0, uint32_t rows, uint32_t col0, uint32_t tid) {
    const uint16_t* base = static_cast<const uint16_t*>(m.ptr);
#pragma unroll 2
    for (uint32_t c = tid; c < rows * 8u; c += 128u) {
        const uint32_t r = c >> 3, p = c & 7u;
        const uint64_t gr = static_cast<uint64_t>(row0) + r;
        const uint32_t gc = col0 + 8u * p;
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (gr < m.rows && gc < m.cols) {
            const uint16_t* q = base + gr * m.ld + gc;
            const uint32_t have = min(8u, m.cols - gc);
            if (m.vec >= 8u && have == 8u) {
                const uint4 u = *reinterpret_cast<const uint4*>(q);
                w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            } else if (m.vec >= 2u && have == 8u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(q)[i];
            } else {
                uint16_t h[8];
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) h[i] = i < have ? q[i] : static_cast<uint16_t>(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(h[2 * i]) | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
            }
        }
        *reinterpret_cast<uint4*>(box + slab_at(r, p)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ------------------------------------------------------------------ the GEMM
struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
};

// Tile order: groups of 16 row tiles, column tiles slowest within a group, so
// that the CTAs of one wave share a few row and column panels in the L2 cache.
NB_DEV void tile_of(const GemmArgs& g, uint32_t t, uint32_t& tm, uint32_t& tn) {
    const uint32_t per = 16u * g.tiles_n, group = t / per, first = 16u * group;
    const uint32_t gm = min(16u, g.tiles_m - first), r = t - group * per;
    tm = first + r % gm;
    tn = r / gm;
}

template <uint32_t BN, int KIND, bool PLAIN>
__global__ void __launch_bounds__(PLAIN ? 384 : 256, 1)
    k_gemm(const GemmArgs g, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b) {
    constexpr uint32_t kStages = gemm_stages(BN);
    constexpr uint32_t kStageBytes = kStageBytesA + BN * 128u;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Barriers bar;
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* slabs = smem + kStages * kStageBytes;
    float* bias_s = reinterpret_cast<float*>(slabs + kEpiWarps * kSlabBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const bool bf16 = g.bf16 != 0u;

    if (threadIdx.x == 0u) {
        for (uint32_t i = 0; i < kStages; ++i) {
            umma::mbar_init(&bar.full[i], PLAIN ? 128u : 1u);
            umma::mbar_init(&bar.empty[i], 1u);
        }
        for (uint32_t i = 0; i < 2u; ++i) {
            umma::mbar_init(&bar.acc_full[i], 1u);
            umma::mbar_init(&bar.acc_empty[i], kEpiWarps);
        }
        umma::mbar_init(&bar.drain, 1u);
        umma::fence_mbar_init();
        if (!PLAIN) {
            tma::prefetch_map(&map_a);
            tma::prefetch_map(&map_b);
        }
    }
    if (warp == 2u) {
        umma::tmem_alloc(&bar.tmem_base, tmem_cols(2u * BN));
        umma::tmem_relinquish();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = bar.tmem_base;
    const uint32_t tiles = g.tiles_m * g.tiles_n, items = tiles * g.splits;

    if ((!PLAIN && warp == 0u && lane == 0u) || (PLAIN && warp >= 8u)) {
        // ---- producer: one thread issuing tensor copies, or four warps of plain loads
        uint32_t stage = 0, parity = 1u, issued = 0;
        bool ok = true;
        for (uint32_t it = blockIdx.x; it < items && ok; it += gridDim.x) {
            const uint32_t split = it / tiles;
            uint32_t tm, tn;
            tile_of(g, it - split * tiles, tm, tn);
            const uint32_t ks1 = min(g.k_steps, (split + 1u) * g.steps_per_split);
            for (uint32_t ks = split * g.steps_per_split; ks < ks1; ++ks) {
                if (!tma::wait(&bar.empty[stage], parity)) {
                    ok = false;
                    break;
                }
                unsigned char* sa = smem + stage * kStageBytes;
                unsigned char* sb = sa + kStageBytesA;
                const uint32_t k0 = ks * kBK, m0 = tm * kBM, n0 = tn * BN;
                if (PLAIN) {
                    const uint32_t tid = threadIdx.x - 256u;
                    if (g.a_mn) {
                        for (uint32_t j = 0; j < kBM / 64u; ++j) fill_box(sa + j * 8192u, g.a, k0, kBK, m0 + 64u * j, tid);
                    } else {
                        fill_box(sa, g.a, m0, kBM, k0, tid);
                    }
                    if (g.b_mn) {
                        for (uint32_t j = 0; j < BN / 64u; ++j) fill_box(sb + j * 8192u, g.b, k0, kBK, n0 + 64u * j, tid);
                    } else {
                        fill_box(sb, g.b, n0, BN, k0, tid);
                    }
                    umma::fence_async_smem();
                    tma::arrive(&bar.full[stage]);
                } else {
                    const uint32_t bytes_a = g.a_mn ? kStageBytesA : g.a_box_rows * 128u;
                    tma::expect_tx(&bar.full[stage], bytes_a + BN * 128u);
                    if (g.a_mn) {
                        for (uint32_t j = 0; j < kBM / 64u; ++j)
                            tma::load_2d(smem_u32(sa + j * 8192u), &map_a, m0 + 64u * j, k0, &bar.full[stage]);
                    } else {
                        tma::load_2d(smem_u32(sa), &map_a, k0, m0, &bar.full[stage]);
                    }
                    if (g.b_mn) {
                        for (uint32_t j = 0; j < BN / 64u; ++j)
                            tma::load_2d(smem_u32(sb + j * 8192u), &map_b, n0 + 64u * j, k0, &bar.full[stage]);
                    } else {
                        tma::load_2d(smem_u32(sb), &map_b, k0, n0, &bar.full[stage]);
                    }
                }
                ++issued;
                if (++stage == kStages) {
                    stage = 0;
                    parity ^= 1u;
                }
            }
        }
        if (!ok) {
            atomicOr(g.error, 1u);
            if (!PLAIN)  // this CTA's copies in flight: wait for them before its shared memory goes
                for (uint32_t i = issued > kStages ? issued - kStages : 0u; i < issued; ++i)
                    tma::wait(&bar.full[i % kStages], (i / kStages) & 1u);
        }
    } else if (warp == 1u && lane == 0u) {
        // ---- MMA issuer
        const uint32_t idesc = tma::idesc_16bit(kBM, BN, g.a_mn, g.b_mn, g.bf16);
        uint32_t stage = 0, parity = 0, acc = 0, acc_parity = 1u;
        bool ok = true;
        for (uint32_t it = blockIdx.x; it < items && ok; it += gridDim.x) {
            const uint32_t split = it / tiles;
            const uint32_t ks0 = split * g.steps_per_split, ks1 = min(g.k_steps, (split + 1u) * g.steps_per_split);
            if (!tma::wait(&bar.acc_empty[acc], acc_parity)) {
                ok = false;
                break;
            }
            umma::fence_after_sync();
            for (uint32_t ks = ks0; ks < ks1; ++ks) {
                if (!tma::wait(&bar.full[stage], parity)) {
                    ok = false;
                    break;
                }
                umma::fence_after_sync();
                const uint32_t sa = smem_u32(smem + stage * kStageBytes), sb = sa + kStageBytesA;
#pragma unroll
                for (uint32_t k = 0; k < kBK / 16u; ++k) {
                    const uint64_t da = g.a_mn ? tma::desc_sw128(sa + 2048u * k, 8192u, 1024u) : tma::desc_sw128(sa + 32u * k, 16u, 1024u);
                    const uint64_t db = g.b_mn ? tma::desc_sw128(sb + 2048u * k, 8192u, 1024u) : tma::desc_sw128(sb + 32u * k, 16u, 1024u);
                    umma::mma_f16(tmem + acc * BN, da, db, idesc, (ks > ks0 || k > 0u) ? 1u : 0u);
                }
                umma::commit(&bar.empty[stage]);
                if (++stage == kStages) {
                    stage = 0;
                    parity ^= 1u;
                }
            }
            if (ok) umma::commit(&bar.acc_full[acc]);
            acc ^= 1u;
            if (acc == 0u) acc_parity ^= 1u;
        }
        if (!ok) {  // the MMAs issued so far end before the tensor memory is freed
            atomicOr(g.error, 1u);
            umma::commit(&bar.drain);
            tma::wait(&bar.drain, 0u);
        }
    } else if (warp >= 4u && warp < 8u) {
        // ---- epilogue: warp q drains rows 32 q .. 32 q + 31 of the tile
        const uint32_t q = warp & 3u, row = 32u * q + lane;
        unsigned char* slab = slabs + q * kSlabBytes;
        uint32_t acc = 0, parity = 0;
        bool ok = true;  // after a wait that ran out the warp only keeps the named barriers' count
        for (uint32_t it = blockIdx.x; it < items; it += gridDim.x) {
            const uint32_t split = it / tiles, tile = it - split * tiles;
            uint32_t tm, tn;
            tile_of(g, tile, tm, tn);
            const uint32_t m0 = tm * kBM + 32u * q, n0 = tn * BN;
            const uint32_t rows = m0 < g.M ? min(32u, g.M - m0) : 0u;
            if (KIND == kGemmRows) {  // bias of the tile's columns, once per tile, shared by the four warps
                asm volatile("bar.sync 1, 128;\n" ::: "memory");
                for (uint32_t c = threadIdx.x & 127u; c < BN; c += 128u)
                    bias_s[c] = g.bias && n0 + c < g.N ? from_16(static_cast<const uint16_t*>(g.bias)[n0 + c], bf16) : 0.0f;
                asm volatile("bar.sync 1, 128;\n" ::: "memory");
            }
            if (ok && !tma::wait(&bar.acc_full[acc], parity)) {
                atomicOr(g.error, 1u);
                ok = false;
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            umma::fence_after_sync();
            const uint32_t taddr = tmem + acc * BN + ((32u * q) << 16);
            if (KIND == kGemmRows) {
                for (uint32_t c0 = 0; c0 < BN && n0 + c0 < g.N; c0 += 64u) {
                    const uint32_t cols = min(64u, g.N - n0 - c0);
                    float v[64];
                    umma::tmem_ld32(taddr + c0, v);
                    umma::tmem_ld32(taddr + c0 + 32u, v + 32);
#pragma unroll
                    for (uint32_t i = 0; i < 16u; ++i) {
                        const float4 b = *reinterpret_cast<const float4*>(bias_s + c0 + 4u * i);
                        v[4 * i] += b.x;
                        v[4 * i + 1] += b.y;
                        v[4 * i + 2] += b.z;
                        v[4 * i + 3] += b.w;
                    }
                    if (g.pre.ptr) {
#pragma unroll
                        for (uint32_t p = 0; p < 8u; ++p) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = pack_16(v[8 * p + 2 * i], v[8 * p + 2 * i + 1], bf16);
                            slab_put(slab, lane, p, w);
                        }
                        __syncwarp();
                        unsigned char* dst = static_cast<unsigned char*>(const_cast<void*>(g.pre.ptr)) + 2u * (m0 * g.pre.ld + n0 + c0);
                        slab_copy<2, true>(slab, dst, g.pre.ld, rows, cols, g.pre.vec >= 8u, lane);
                        __syncwarp();
                    }
                    act_row(v, g.act);
                    if (g.res.ptr) {
                        unsigned char* src = static_cast<unsigned char*>(const_cast<void*>(g.res.ptr)) + 2u * (m0 * g.res.ld + n0 + c0);
                        slab_copy<2, false>(slab, src, g.res.ld, rows, cols, g.res.vec >= 8u, lane);
                        __syncwarp();
#pragma unroll
                        for (uint32_t p = 0; p < 8u; ++p) {
                            const uint4 u = *reinterpret_cast<const uint4*>(slab + slab_at(lane, p));
                            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 f = unpack_16(w[i], bf16);
                                v[8 * p + 2 * i] += f.x;
                                v[8 * p + 2 * i + 1] += f.y;
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (uint32_t p = 0; p < 8u; ++p) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = pack_16(v[8 * p + 2 * i], v[8 * p + 2 * i + 1], bf16);
                        slab_put(slab, lane, p, w);
                    }
                    __syncwarp();
                    unsigned char* dst = static_cast<unsigned char*>(const_cast<void*>(g.y.ptr)) + 2u * (m0 * g.y.ld + n0 + c0);
                    slab_copy<2, true>(slab, dst, g.y.ld, rows, cols, g.y.vec >= 8u, lane);
                    __syncwarp();
                }
            } else if (g.splits > 1u) {
                // Partial tile, four columns of 128 rows at a time: 512 contiguous bytes a warp store.
                float4* dst = reinterpret_cast<float4*>(g.partials) + static_cast<uint64_t>(it) * (BN / 4u) * kBM + row;
                for (uint32_t c0 = 0; c0 < BN && n0 + c0 < g.N; c0 += 32u) {
                    float v[32];
                    umma::tmem_ld32(taddr + c0, v);
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i)
                        dst[(c0 / 4u + i) * kBM] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            } else {
                // The gradient itself: 32 fp32 or 64 16-bit columns (128 bytes) a slab.
                const uint32_t es = g.dw_f32 ? 4u : 2u, wide = 128u / es;
                for (uint32_t c0 = 0; c0 < BN && n0 + c0 < g.N; c0 += wide) {
                    const uint32_t cols = min(wide, g.N - n0 - c0);
                    unsigned char* at = static_cast<unsigned char*>(g.dw) + (static_cast<uint64_t>(m0) * g.N + n0 + c0) * es;
                    if (g.accumulate) {
                        if (g.dw_f32) slab_copy<4, false>(slab, at, g.N, rows, cols, g.dw_vec != 0u, lane);
                        else slab_copy<2, false>(slab, at, g.N, rows, cols, g.dw_vec != 0u, lane);
                        __syncwarp();
                    }
                    for (uint32_t h = 0; h < wide; h += 32u) {
                        float v[32];
                        umma::tmem_ld32(taddr + c0 + h, v);
                        if (g.dw_f32) {
#pragma unroll
                            for (uint32_t p = 0; p < 8u; ++p) {
                                float4* l = reinterpret_cast<float4*>(slab + slab_at(lane, p));
                                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (g.accumulate) o = *l;
                                *l = make_float4(o.x + v[4 * p], o.y + v[4 * p + 1], o.z + v[4 * p + 2], o.w + v[4 * p + 3]);
                            }
                        } else {
#pragma unroll
                            for (uint32_t p = 0; p < 4u; ++p) {
                                uint4* l = reinterpret_cast<uint4*>(slab + slab_at(lane, p + h / 8u));
                                uint4 o = make_uint4(0u, 0u, 0u, 0u);
                                if (g.accumulate) o = *l;
                                const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
                                uint32_t w[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float2 f = unpack_16(ow[i], bf16);
                                    w[i] = pack_16(f.x + v[8 * p + 2 * i], f.y + v[8 * p + 2 * i + 1], bf16);
                                }
                                *l = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    __syncwarp();
                    if (g.dw_f32) slab_copy<4, true>(slab, at, g.N, rows, cols, g.dw_vec != 0u, lane);
                    else slab_copy<2, true>(slab, at, g.N, rows, cols, g.dw_vec != 0u, lane);
                    __syncwarp();
                }
            }
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0u) tma::arrive(&bar.acc_empty[acc]);
            acc ^= 1u;
            if (acc == 0u) parity ^= 1u;
        }
    }
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (warp == 2u) umma::tmem_dealloc(tmem, tmem_cols(2u * BN));
}

// ------------------------------------------------- dz and its column sums
// 256 threads: 8 columns a thread, `cg` column groups side by side (a power of
// two up to 32), 256 / cg rows at a time.
__global__ void __launch_bounds__(256) k_dz(const DzArgs a, uint32_t cg_log2) {
    __shared__ float sums[256][8];
    const bool bf16 = a.bf16 != 0u;
    const uint32_t cg = 1u << cg_log2, gx = threadIdx.x & (cg - 1u), gy = threadIdx.x >> cg_log2, ny = 256u >> cg_log2;
    const uint32_t c0 = 8u * (blockIdx.x * cg + gx);
    const uint32_t have = c0 < a.dy.cols ? min(8u, a.dy.cols - c0) : 0u;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (have) {
        const uint64_t r0 = static_cast<uint64_t>(blockIdx.y) * a.rows_per_part;
        const uint64_t r1 = min(static_cast<uint64_t>(a.dy.rows), r0 + a.rows_per_part);
        for (uint64_t r = r0 + gy; r < r1; r += ny) {
            const uint16_t* qd = static_cast<const uint16_t*>(a.dy.ptr) + r * a.dy.ld + c0;
            uint32_t d[4] = {0u, 0u, 0u, 0u}, z[4] = {0u, 0u, 0u, 0u};
            if (have == 8u && a.dy.vec >= 8u) {
                const uint4 u = *reinterpret_cast<const uint4*>(qd);
                d[0] = u.x; d[1] = u.y; d[2] = u.z; d[3] = u.w;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i)
                    if (i < have) d[i / 2u] |= static_cast<uint32_t>(qd[i]) << (16u * (i & 1u));
            }
            if (a.act != kActNone) {
                const uint16_t* qz = static_cast<const uint16_t*>(a.pre.ptr) + r * a.pre.ld + c0;
                if (have == 8u && a.pre.vec >= 8u) {
                    const uint4 u = *reinterpret_cast<const uint4*>(qz);
                    z[0] = u.x; z[1] = u.y; z[2] = u.z; z[3] = u.w;
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i)
                        if (i < have) z[i / 2u] |= static_cast<uint32_t>(qz[i]) << (16u * (i & 1u));
                }
            }
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 f = unpack_16(d[i], bf16);
                if (a.act != kActNone) {
                    const float2 zz = unpack_16(z[i], bf16);
                    f.x = dact_f(f.x, zz.x, a.act);
                    f.y = dact_f(f.y, zz.y, a.act);
                }
                s[2 * i] += f.x;
                s[2 * i + 1] += f.y;
                o[i] = pack_16(f.x, f.y, bf16);  // the tensor cores take 16-bit operands
            }
            // dz rows are padded to a multiple of 8 values
            if (a.dz) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + r * a.dz_ld + c0) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    if (!a.db_part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[threadIdx.x][i] = s[i];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < 8u * cg; c += 256u) {
        const uint32_t col = 8u * blockIdx.x * cg + c;
        if (col >= a.dy.cols) break;
        float t = 0.0f;
        for (uint32_t y = 0; y < ny; ++y) t += sums[(y << cg_log2) + (c >> 3)][c & 7u];
        a.db_part[static_cast<uint64_t>(blockIdx.y) * a.dy.cols + col] = t;
    }
}

// -------------------------------------------- sums of the partial gradients
NB_DEV void grad_out(void* p, uint64_t i, float v, const GradReduceArgs& a) {
    if (a.f32) {
        float* q = static_cast<float*>(p) + i;
        *q = a.accumulate ? *q + v : v;
    } else {
        uint16_t* q = static_cast<uint16_t*>(p) + i;
        *q = to_16(a.accumulate ? from_16(*q, a.bf16 != 0u) + v : v, a.bf16 != 0u);
    }
}
// Blocks below n_dw: one row group of 128 x 4 columns of dw each, in split
// order; the others: 32 columns of db, eight warps each a range of the parts.
__global__ void __launch_bounds__(256) k_grad_reduce(const GradReduceArgs a, uint32_t n_dw) {
    if (blockIdx.x < n_dw) {
        const uint32_t per_tile = a.bn / 4u, idx = 2u * blockIdx.x + (threadIdx.x >> 7);
        const uint32_t tile = idx / per_tile, c4 = idx - tile * per_tile, row = threadIdx.x & 127u;
        const uint32_t tiles = a.tiles_m * a.tiles_n;
        if (tile >= tiles) return;
        const uint32_t per = 16u * a.tiles_n, group = tile / per, first = 16u * group;
        const uint32_t gm = min(16u, a.tiles_m - first), r = tile - group * per;
        const uint32_t m = (first + r % gm) * kBM + row, n = (r / gm) * a.bn + 4u * c4;
        if (m >= a.n_out || n >= a.n_in) return;
        const float4* src = reinterpret_cast<const float4*>(a.partials) + (static_cast<uint64_t>(tile) * per_tile + c4) * kBM + row;
        const uint64_t step = static_cast<uint64_t>(tiles) * per_tile * kBM;
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (uint32_t k = 0; k < a.splits; ++k) {
            const float4 v = __ldcs(src + k * step);
            t.x += v.x;
            t.y += v.y;
            t.z += v.z;
            t.w += v.w;
        }
        const float o[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (n + i < a.n_in) grad_out(a.dw, static_cast<uint64_t>(m) * a.n_in + n + i, o[i], a);
        return;
    }
    __shared__ float ws[8][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, c = 32u * (blockIdx.x - n_dw) + lane;
    const uint32_t per = (a.parts + 7u) / 8u, p0 = min(a.parts, warp * per), p1 = min(a.parts, p0 + per);
    float t = 0.0f;
    if (c < a.n_out) {
#pragma unroll 8
        for (uint32_t p = p0; p < p1; ++p) t += a.db_part[static_cast<uint64_t>(p) * a.n_out + c];
    }
    ws[warp][lane] = t;
    __syncthreads();
    if (warp == 0u && c < a.n_out) {
        t = ws[0][lane];
#pragma unroll
        for (uint32_t w = 1; w < 8u; ++w) t += ws[w][lane];
        grad_out(a.db, c, t, a);
    }
}

template <uint32_t BN, int KIND, bool PLAIN>
cudaError_t launch_gemm_t(const GemmArgs& g, const CUtensorMap& ma, const CUtensorMap& mb, uint32_t blocks, cudaStream_t s) {
    // The attribute belongs to the device: set once for each.
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev]) {
        e = cudaFuncSetAttribute(k_gemm<BN, KIND, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, gemm_smem(BN));
        if (e != cudaSuccess) return e;
        done[dev] = true;
    }
    k_gemm<BN, KIND, PLAIN><<<blocks, PLAIN ? 384u : 256u, gemm_smem(BN), s>>>(g, ma, mb);
    return cudaGetLastError();
}
template <int KIND, bool PLAIN>
cudaError_t launch_gemm_bn(const GemmArgs& g, uint32_t bn, const CUtensorMap& ma, const CUtensorMap& mb, uint32_t blocks, cudaStream_t s) {
    switch (bn) {
        case 64u: return launch_gemm_t<64u, KIND, PLAIN>(g, ma, mb, blocks, s);
        case 128u: return launch_gemm_t<128u, KIND, PLAIN>(g, ma, mb, blocks, s);
        case 256u: return launch_gemm_t<256u, KIND, PLAIN>(g, ma, mb, blocks, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_gemm(const GemmArgs& g, int kind, uint32_t bn, const CUtensorMap* map_a, const CUtensorMap* map_b,
                        bool plain_loads, uint32_t blocks, cudaStream_t s) {
    if (kind == kGemmRows)
        return plain_loads ? launch_gemm_bn<kGemmRows, true>(g, bn, *map_a, *map_b, blocks, s)
                           : launch_gemm_bn<kGemmRows, false>(g, bn, *map_a, *map_b, blocks, s);
    return plain_loads ? launch_gemm_bn<kGemmGrad, true>(g, bn, *map_a, *map_b, blocks, s)
                       : launch_gemm_bn<kGemmGrad, false>(g, bn, *map_a, *map_b, blocks, s);
}

cudaError_t launch_dz(const DzArgs& a, cudaStream_t s) {
    const uint32_t groups = (a.dy.cols + 7u) / 8u;
    uint32_t log2 = 0;
    while (log2 < 5u && (1u << log2) < groups) ++log2;
    const dim3 grid((groups + (1u << log2) - 1u) >> log2, a.parts);
    k_dz<<<grid, 256, 0, s>>>(a, log2);
    return cudaGetLastError();
}

cudaError_t launch_grad_reduce(const GradReduceArgs& a, cudaStream_t s) {
    const uint32_t n_dw = a.dw ? (a.tiles_m * a.tiles_n * (a.bn / 4u) + 1u) / 2u : 0u;
    const uint32_t n_db = a.db ? (a.n_out + 31u) / 32u : 0u;
    if (n_dw + n_db == 0u) return cudaSuccess;
    k_grad_reduce<<<n_dw + n_db, 256, 0, s>>>(a, n_dw);
    return cudaGetLastError();
}

}  // namespace nb
