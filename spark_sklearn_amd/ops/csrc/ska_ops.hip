// spark_sklearn_amd native kernels -- MI355X (gfx950, CDNA4) only.
//
// K1 (batched linear fit) + K4 (scoring) of SURVEY.md section 2.5: the
// worker-side compute the reference borrows from sklearn's Cython/BLAS
//  re-designed for CDNA4.  B candidate-columns (candidates x
// OVR classes) are fitted SIMULTANEOUSLY: the per-epoch work is two
// MFMA-shaped GEMMs over the resident bf16 matrix
//
//     Z = X[idx] . W^T          (fwd_d_kernel: fused elementwise d = dL/dz,
//                                per-column loss/db LDS reductions,
//                                transposed D write)
//     G = D^T . X[idx]          (bwd_g_kernel: split-K over row segments,
//                                atomic fp32 tile adds)
//
// followed by two tiny elementwise kernels (col_finalize_kernel: per-column
// bias/momentum/convergence state, fully on-device so the epoch loop never
// syncs the host; update_w_kernel: masked momentum update + bf16 mirror +
// G zeroing).  fp32 accumulation everywhere; bf16 is the storage/MFMA
// input dtype.
//
// Layout decisions (why everything is candidate-major):
//   X      [n][Fp]    bf16, row-major, Fp = roundup(F, 64) zero-padded
//   W,V,G  [Bp][Fp]   fp32, candidate-major -> update kernel fully
//                     coalesced, and the bf16 mirror Wt [Bp][Fp] stages
//                     into LDS with contiguous 16B reads as the MFMA
//                     B-operand (k-contiguous per column)
//   D^T    [Bp][NTp]  bf16 -- the fwd epilogue's C-fragment holds 4
//                     CONSECUTIVE rows per (lane, reg-quad) (C/D layout:
//                     col = lane&15, row = (lane>>4)*4 + reg), so the
//                     transposed store is a single 8-byte write; and the
//                     bwd kernel then reads D^T k-contiguously as its
//                     A-operand.  Zero-padded rows make split-K segments
//                     self-masking.
//
// MFMA fragment layout: C/D mapping is HW-verified in the programming
// guide; the A/B operand k-mapping (contiguous-8 vs two 4-blocks at k and
// k+16) is probed AT RUNTIME on first use (probe_kernel, all 4 A x B
// combinations) against a host reference -- see Common-mistake #3 /
// Guideline G9 (transpose-detecting checks with asymmetric inputs).

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <vector>

#define WAVE 64

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

#define HIP_CHECK(expr)                                                    \
  do {                                                                     \
    hipError_t _e = (expr);                                                \
    TORCH_CHECK(_e == hipSuccess, "HIP error: ", hipGetErrorString(_e));   \
  } while (0)

// ---------------------------------------------------------------------------
// fragment k-mapping (template param P = AMAP*2 + BMAP)
//   map 0: k = (lane>>4)*8 + i            (contiguous 8)
//   map 1: k = (lane>>4)*4 + (i&3) + (i>>2)*16   (two 4-blocks, +16 apart)
// ---------------------------------------------------------------------------
template <int MAP>
__device__ __forceinline__ int frag_k(int lane, int i) {
  if (MAP == 0) return ((lane >> 4) << 3) + i;
  return ((lane >> 4) << 2) + (i & 3) + ((i >> 2) << 4);
}

// Read an 8-element bf16 fragment from an LDS row `base` (element pointer to
// k=0 of that row).  map 0 -> one 16B read; map 1 -> two 8B reads.
template <int MAP>
__device__ __forceinline__ bf16x8 lds_frag(const __bf16* base, int lane) {
  bf16x8 out;
  if (MAP == 0) {
    const bf16x8* p =
        reinterpret_cast<const bf16x8*>(base + ((lane >> 4) << 3));
    out = *p;
  } else {
    const bf16x4* p0 =
        reinterpret_cast<const bf16x4*>(base + ((lane >> 4) << 2));
    const bf16x4* p1 =
        reinterpret_cast<const bf16x4*>(base + 16 + ((lane >> 4) << 2));
    bf16x4 a = *p0, b = *p1;
    out[0] = a[0]; out[1] = a[1]; out[2] = a[2]; out[3] = a[3];
    out[4] = b[0]; out[5] = b[1]; out[6] = b[2]; out[7] = b[3];
  }
  return out;
}


// ---------------------------------------------------------------------------
// Permuted + swizzled LDS tiles (fast path for the HW-probed layout P=3).
//
// The probe shows gfx950's mfma_f32_16x16x32_bf16 wants per-lane operand
// elements k = (lane>>4)*4 + (i&3) + (i>>2)*16 (two 4-blocks, +16 apart).
// Generic staging leaves those as 2 x 8B LDS reads with ~4-way bank
// aliasing (PMC: 25.6M SQ_LDS_BANK_CONFLICT/dispatch).  Fix: store each
// 64-k row PERMUTED so one lane's 8 fragment elements are contiguous
// (single ds_read_b128), row stride exactly 64 elements (128 B), and an
// XOR of the 16B-group index by (row&7) (guide T2, st-swizzle) so the 8
// groups x 4 banks tile all 32 banks with balanced load.
//   pos(k)  = (k>>5)*32 + (((k&15)>>2)<<3) + (((k>>4)&1)<<2) + (k&3)
//   addr(r,k) = r*64 + (pos(k) ^ ((r&7)<<3))
// ---------------------------------------------------------------------------
__device__ __forceinline__ int perm_pos(int k) {
  return ((k >> 5) << 5) + (((k & 15) >> 2) << 3) + (((k >> 4) & 1) << 2) +
         (k & 3);
}
__device__ __forceinline__ int swz8(int p, int r) {
  return p ^ ((r & 7) << 3);
}
// store 8 globally-contiguous elements (k0 % 8 == 0) into row r
__device__ __forceinline__ void store_row8(__bf16* row, int r, int k0,
                                           bf16x8 v) {
  bf16x4 lo = {v[0], v[1], v[2], v[3]};
  bf16x4 hi = {v[4], v[5], v[6], v[7]};
  *reinterpret_cast<bf16x4*>(row + swz8(perm_pos(k0), r)) = lo;
  *reinterpret_cast<bf16x4*>(row + swz8(perm_pos(k0 + 4), r)) = hi;
}
// read one lane's fragment: row pointer (r*64 into the tile), row index r,
// k-group g = lane>>4, half h = ks/32
__device__ __forceinline__ bf16x8 lds_frag_p(const __bf16* row, int r,
                                             int g, int h) {
  return *reinterpret_cast<const bf16x8*>(row + swz8(h * 32 + g * 8, r));
}

// ---------------------------------------------------------------------------
// v12 staging: async global->LDS (global_load_lds_dwordx4), no register
// round-trip.  LDS layout is LINEAR rows of 64 elements whose 16B granules
// are XOR-swizzled by (row&7); the swizzle is applied to the per-lane
// global SOURCE address (the LDS destination of global_load_lds is
// hardware-fixed at wave-uniform-base + lane*16, guide m104/m173), so LDS
// granule j of row r holds logical k-granule (j ^ (r&7)).  Fragment reads
// un-swizzle and deliver CONTIGUOUS logical k per lane-group (map 0).
// That differs from the HW-probed per-slot k map, but the GEMM contracts
// A and B slot-wise: feeding both operands through the SAME logical-k
// permutation leaves sum_k A[m][k]*B[n][k] unchanged, so no layout probe
// is needed on this path.  Bank math: 64 lanes of one ds_read_b128 hit
// (row, granule) pairs whose granule cycles over all 8 slots -> exactly
// 2 lanes/bank (free, guide m136).
// ---------------------------------------------------------------------------
__device__ __forceinline__ void gload_lds16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned int*)g,
      (__attribute__((address_space(3))) unsigned int*)lds, 16, 0, 0);
}
// fragment read: tile base, row r, logical granule gg (= h*4 + (lane>>4))
__device__ __forceinline__ bf16x8 frag12(const __bf16* tile, int r, int gg) {
  return *reinterpret_cast<const bf16x8*>(tile + r * 64 +
                                          ((gg ^ (r & 7)) << 3));
}

// ---------------------------------------------------------------------------
// v13: K=32 chunks, 4-buffer LDS ring, counted s_waitcnt vmcnt(N) with raw
// s_barrier (guide T3+T4) -- loads for chunks kc+1/kc+2 stay in flight
// across the barrier instead of draining to 0, which is the structural
// stall of the 2-phase schedule.  Rows are 32 elements = 4 granules of 16B;
// granule swizzle uses ((r>>1)&3) so a 16-row column read spreads over all
// 32 banks at 2 lanes/bank (parity bit of r supplies the 16-word offset).
// Iteration shape (one barrier per chunk):
//   wait own chunk-kc loads (vmcnt counted) -> s_barrier -> stage kc+3
//   (its buffer was last read at kc-1, before everyone's barrier) -> MFMA.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int swz32(int r) { return (r >> 1) & 3; }
// read logical granule g (= lane>>4) of row r; tile rows are 32 elements
__device__ __forceinline__ bf16x8 frag13(const __bf16* tile, int r, int g) {
  return *reinterpret_cast<const bf16x8*>(tile + r * 32 +
                                          ((g ^ swz32(r)) << 3));
}
#define SKA_WAIT_VMCNT(beyond)                                   \
  do {                                                           \
    if ((beyond) >= 2)                                           \
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");           \
    else if ((beyond) == 1)                                      \
      asm volatile("s_waitcnt vmcnt(2)" ::: "memory");           \
    else                                                         \
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           \
  } while (0)

// ---------------------------------------------------------------------------
// layout probe: D = A(16x32) . B(32x16), one wave, LDS-staged like the real
// kernels.  Host test compares all 4 (AMAP, BMAP) combos vs reference.
// ---------------------------------------------------------------------------
template <int AMAP, int BMAP>
__global__ void probe_kernel(const __bf16* __restrict__ A,   // [16][32]
                             const __bf16* __restrict__ B,   // [16][32] = B^T (col-major B: B[k][c] stored as Bt[c][k])
                             float* __restrict__ D) {        // [16][16]
  __shared__ __bf16 sA[16][32];
  __shared__ __bf16 sB[16][32];
  int lane = threadIdx.x & 63;
  for (int e = lane; e < 16 * 32; e += WAVE) {
    sA[e / 32][e % 32] = A[e];
    sB[e / 32][e % 32] = B[e];
  }
  __syncthreads();
  bf16x8 a, b;
  int row = lane & 15;
  for (int i = 0; i < 8; ++i) {
    a[i] = sA[row][frag_k<AMAP>(lane, i)];
    b[i] = sB[row][frag_k<BMAP>(lane, i)];   // row here = output col
  }
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  for (int r = 0; r < 4; ++r) {
    int orow = ((lane >> 4) << 2) + r;
    int ocol = lane & 15;
    D[orow * 16 + ocol] = acc[r];
  }
}

// ---------------------------------------------------------------------------
// mean squared row norm (auto-lr curvature bound)
// ---------------------------------------------------------------------------
__global__ void msq_kernel(const __bf16* __restrict__ X, long n, int Fp,
                           double* __restrict__ out) {
  long row = blockIdx.x * blockDim.x + threadIdx.x;
  double local = 0.0;
  for (; row < n; row += (long)gridDim.x * blockDim.x) {
    const __bf16* xr = X + row * Fp;
    float s = 0.f;
    for (int f = 0; f < Fp; f += 8) {
      bf16x8 v = *reinterpret_cast<const bf16x8*>(xr + f);
      for (int j = 0; j < 8; ++j) {
        float x = (float)v[j];
        s += x * x;
      }
    }
    local += (double)s;
  }
  // block-level reduce in LDS, one double atomic per block
  __shared__ double red[256];
  red[threadIdx.x] = local;
  __syncthreads();
  for (int s = blockDim.x / 2; s > 0; s >>= 1) {
    if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) atomicAdd(out, red[0]);
}

// ---------------------------------------------------------------------------
// loss elementwise: d = dL/dz and per-element loss
// ---------------------------------------------------------------------------
#define LOSS_LOGISTIC 0
#define LOSS_HINGE 1
#define LOSS_SQUARED 2

// 1-ulp hardware reciprocal: D is stored as bf16 (8 mantissa bits) and the
// loss sum is a convergence heuristic, so v_rcp_f32 replaces the
// correctly-rounded v_div_scale chain (~6 VALU ops saved per element in a
// 64x-unrolled epilogue).
__device__ __forceinline__ float fast_rcp(float x) {
  return __builtin_amdgcn_rcpf(x);
}

__device__ __forceinline__ void loss_grad(int lid, float z, float yv,
                                          int tgt, float* d, float* ls) {
  const float eps = 1e-12f;
  if (lid == LOSS_LOGISTIC) {
    float t = (yv == (float)tgt) ? 1.f : 0.f;
    float p = fast_rcp(1.f + __expf(-z));
    *d = p - t;
    *ls = -(t * __logf(p + eps) + (1.f - t) * __logf(1.f - p + eps));
  } else if (lid == LOSS_HINGE) {
    float s = (yv == (float)tgt) ? 1.f : -1.f;
    float m = s * z;
    *d = (m < 1.f) ? -s : 0.f;
    *ls = fmaxf(0.f, 1.f - m);
  } else {
    float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
    float r = z - t;
    *d = r;
    *ls = 0.5f * r * r;
  }
}

// ---------------------------------------------------------------------------
// fwd_d2_kernel: v2 of fwd_d -- block tile 64 rows x Bp cols (Bp<=256).
// 4 waves side-by-side over columns, each wave computes 64 x (Bp/4):
// 4 m-frags x nfrag n-frags -> 4x the MFMA work per staged byte of the
// 64x64 v1 tile, and W is staged once per k-chunk for ALL columns (no
// cross-block X re-reads within a row tile).
// ---------------------------------------------------------------------------
template <int P, int NF, int WT = 0>
__global__ __launch_bounds__(256)
void fwd_d2_kernel(const __bf16* __restrict__ X,       // [n][Fp]
                   const float* __restrict__ y,        // [n]
                   const int* __restrict__ idx,        // [NTp]
                   const __bf16* __restrict__ Wt,      // [Bp][Fp]
                   const float* __restrict__ bias,     // [Bp]
                   const int* __restrict__ loss_id,    // [Bp]
                   const int* __restrict__ target,     // [Bp]
                   __bf16* __restrict__ Dt,            // [Bp][NTp]
                   float* __restrict__ loss_sum,       // [Bp]
                   float* __restrict__ db_sum,         // [Bp]
                   const int* __restrict__ row_key,    // unused (generic)
                   const int* __restrict__ col_key,    // unused (generic)
                   int nt, int NTp, int Fp, int Bp, int want_loss,
                   const float* __restrict__ w = nullptr) {
  constexpr int AMAP = P >> 1, BMAP = P & 1;
  (void)want_loss;  // generic path always computes loss
  (void)row_key;
  (void)col_key;
  __shared__ __bf16 sX[64][72];
  __shared__ __bf16 sW[256][72];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[64];
  __shared__ float sY[64];
  __shared__ float sWgt[WT ? 64 : 1];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int rt = blockIdx.x;
  constexpr int cpw = NF * 16;        // cols per wave: 16/32/64

  if (tid < 64) {
    int r = rt * 64 + tid;
    int gi = idx[r];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    if (WT) sWgt[tid] = w[gi];
  }
  for (int i = tid; i < Bp; i += 256) { sLoss[i] = 0.f; sDb[i] = 0.f; }
  __syncthreads();

  f32x4 acc[4][4];
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const int srow = tid >> 2;
  const int sseg = tid & 3;
  for (int kc = 0; kc < Fp; kc += 64) {
    {
      const uint4* gx = reinterpret_cast<const uint4*>(
          X + (long)sIdx[srow] * Fp + kc + sseg * 16);
      uint4* lx = reinterpret_cast<uint4*>(&sX[srow][sseg * 16]);
      lx[0] = gx[0];
      lx[1] = gx[1];
    }
    for (int e = tid; e < Bp * 4; e += 256) {
      int c = e >> 2, seg = e & 3;
      const uint4* gw = reinterpret_cast<const uint4*>(
          Wt + (long)c * Fp + kc + seg * 16);
      uint4* lw = reinterpret_cast<uint4*>(&sW[c][seg * 16]);
      lw[0] = gw[0];
      lw[1] = gw[1];
    }
    __syncthreads();
    for (int ks = 0; ks < 64; ks += 32) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
        a[m] = lds_frag<AMAP>(&sX[m * 16 + (lane & 15)][ks], lane);
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        bf16x8 b = lds_frag<BMAP>(
            &sW[wave * cpw + fn * 16 + (lane & 15)][ks], lane);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], b, acc[m][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = wave * cpw + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    float lsum = 0.f, dsum = 0.f;
    for (int m = 0; m < 4; ++m) {
      int row_base = m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 64 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls;
        loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (WT) {
          float wt = sWgt[row_base + r];
          d *= wt;
          ls *= wt;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 64 + row_base) = dpack;
    }
    atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  for (int i = tid; i < Bp; i += 256) {
    atomicAdd(&loss_sum[i], sLoss[i]);
    atomicAdd(&db_sum[i], sDb[i]);
  }
}

// ---------------------------------------------------------------------------
// bwd_g2_kernel: v2 of bwd_g -- output tile Bp cands x 64 features, reading
// the RESIDENT TRANSPOSE Xt [Fp][n] so the B-operand stages coalesced
// (contiguity fast path: CV folds give contiguous index runs, so 16-element
// idx chunks are usually vector loads; scalar gather otherwise).
// grid (Fp/64, nseg).
// ---------------------------------------------------------------------------
template <int P, int NF>
__global__ __launch_bounds__(256)
void bwd_g2_kernel(const __bf16* __restrict__ Xt,    // [Fp][n]
                   const int* __restrict__ idx,      // [NTp]
                   const __bf16* __restrict__ Dt,    // [Bp][NTp]
                   float* __restrict__ Gt,           // [Bp][Fp]
                   long n_rows, int NTp, int Fp, int Bp, int seg_rows) {
  constexpr int AMAP = P >> 1, BMAP = P & 1;
  __shared__ __bf16 sD[256][72];
  __shared__ __bf16 sXt[64][72];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, NTp);
  constexpr int cpw = NF * 16;

  f32x4 acc[4][4];
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int rc = r0; rc < r1; rc += 64) {
    for (int e = tid; e < Bp * 4; e += 256) {
      int c = e >> 2, seg = e & 3;
      const uint4* gd = reinterpret_cast<const uint4*>(
          Dt + (long)c * NTp + rc + seg * 16);
      uint4* ld = reinterpret_cast<uint4*>(&sD[c][seg * 16]);
      ld[0] = gd[0];
      ld[1] = gd[1];
    }
    {
      // stage Xt rows (features) gathered over idx; 16-chunk contiguity
      // fast path (KFold folds are contiguous runs)
      int f = tid >> 2, seg = tid & 3;
      int rbase = rc + seg * 16;
      int i0 = idx[rbase];
      int i15 = idx[rbase + 15];
      const __bf16* src = Xt + (long)(ft * 64 + f) * n_rows;
      if (i15 - i0 == 15) {
        const uint4* gx = reinterpret_cast<const uint4*>(src + i0);
        // i0 may be unaligned for 16B vectors; use 8x2B fallback if so
        if (((unsigned long)(src + i0) & 15) == 0) {
          uint4* lx = reinterpret_cast<uint4*>(&sXt[f][seg * 16]);
          lx[0] = gx[0];
          lx[1] = gx[1];
        } else {
          for (int j = 0; j < 16; ++j) sXt[f][seg * 16 + j] = src[i0 + j];
        }
      } else {
        for (int j = 0; j < 16; ++j)
          sXt[f][seg * 16 + j] = src[idx[rbase + j]];
      }
    }
    __syncthreads();
    for (int ks = 0; ks < 64; ks += 32) {
      bf16x8 b[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn)
        b[fn] = lds_frag<BMAP>(&sXt[fn * 16 + (lane & 15)][ks], lane);
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        bf16x8 a = lds_frag<AMAP>(
            &sD[wave * cpw + m * 16 + (lane & 15)][ks], lane);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, b[fn], acc[m][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fn * 16 + (lane & 15);
      for (int r = 0; r < 4; ++r) {
        int c_in = wave * cpw + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 64 + f_in], acc[m][fn][r]);
      }
    }
  }
}


// ---------------------------------------------------------------------------
// fwd_d3_kernel: P=3 fast path -- permuted/swizzled LDS + 2-phase
// double-buffered staging (issue next k-chunk's global loads into
// registers while MFMA consumes the current LDS buffer; guide T3 minimum
// recipe) + want_loss gating.
// ---------------------------------------------------------------------------
template <int NF, int WT = 0>   // WT: per-row sample_weight (w != null)
__global__ __launch_bounds__(256)
void fwd_d3_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                   const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                   const float* __restrict__ bias,
                   const int* __restrict__ loss_id,
                   const int* __restrict__ target, __bf16* __restrict__ Dt,
                   float* __restrict__ loss_sum, float* __restrict__ db_sum,
                   const int* __restrict__ row_key,   // [n] or null
                   const int* __restrict__ col_key,   // [Bp] or null
                   int nt, int NTp, int Fp, int Bp, int want_loss,
                   const float* __restrict__ w = nullptr) {
  __shared__ __bf16 sX[2][64 * 64];
  __shared__ __bf16 sW[2][NF * 64 * 64];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[64];
  __shared__ float sY[64];
  __shared__ int sKey[64];
  __shared__ float sWgt[WT ? 64 : 1];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int rt = blockIdx.x;
  constexpr int cpw = NF * 16;
  const int g = lane >> 4;
  const int srow = tid >> 2;
  const int sseg = tid & 3;
  const int wrow = tid >> 2;        // W staging: base col row

  if (tid < 64) {
    int gi = idx[rt * 64 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    if (WT) sWgt[tid] = w[gi];
  }
  for (int i = tid; i < Bp; i += 256) { sLoss[i] = 0.f; sDb[i] = 0.f; }
  __syncthreads();

  bf16x8 rx[2], rw[2 * NF];
  auto issue = [&](int kc) {
    const bf16x8* gx = reinterpret_cast<const bf16x8*>(
        X + (long)sIdx[srow] * Fp + kc + sseg * 16);
    rx[0] = gx[0];
    rx[1] = gx[1];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      int c = wrow + i * 64;
      const bf16x8* gw = reinterpret_cast<const bf16x8*>(
          Wt + (long)c * Fp + kc + sseg * 16);
      rw[2 * i] = gw[0];
      rw[2 * i + 1] = gw[1];
    }
  };
  auto commit = [&](int b) {
    store_row8(&sX[b][srow * 64], srow, sseg * 16, rx[0]);
    store_row8(&sX[b][srow * 64], srow, sseg * 16 + 8, rx[1]);
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      int c = wrow + i * 64;
      store_row8(&sW[b][c * 64], c, sseg * 16, rw[2 * i]);
      store_row8(&sW[b][c * 64], c, sseg * 16 + 8, rw[2 * i + 1]);
    }
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  issue(0);
  commit(0);
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) issue((kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = m * 16 + (lane & 15);
        a[m] = lds_frag_p(&sX[b][r * 64], r, g, h);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = wave * cpw + fn * 16 + (lane & 15);
        bf16x8 bb = lds_frag_p(&sW[b][c * 64], c, g, h);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    if (kc + 1 < nkc) commit(b ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = wave * cpw + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 64 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = 1.f / (1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;          // keyed batching: column only sees its key
          ls = 0.f;
        }
        if (WT) {           // sample_weight: scale grad AND loss per row
          float wt = sWgt[row_base + r];
          d *= wt;
          ls *= wt;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 64 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  for (int i = tid; i < Bp; i += 256) {
    if (want_loss) atomicAdd(&loss_sum[i], sLoss[i]);
    atomicAdd(&db_sum[i], sDb[i]);
  }
}

// ---------------------------------------------------------------------------
// bwd_g3_kernel: P=3 fast path -- permuted/swizzled LDS + 2-phase
// double-buffered staging; reads the resident transpose Xt with a
// contiguity fast path for CV-fold index runs.
// ---------------------------------------------------------------------------
template <int NF>
__global__ __launch_bounds__(256)
void bwd_g3_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                   const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                   long n_rows, int NTp, int Fp, int Bp, int seg_rows) {
  __shared__ __bf16 sD[2][NF * 64 * 64];
  __shared__ __bf16 sXt[2][64 * 64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, NTp);
  constexpr int cpw = NF * 16;
  const int g = lane >> 4;
  const int drow = tid >> 2;
  const int sseg = tid & 3;
  const int xf = tid >> 2;           // Xt staging: feature row

  f32x4 acc[NF][4];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  bf16x8 rd[2 * NF], rxa, rxb;
  auto issue = [&](int rc) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      int c = drow + i * 64;
      const bf16x8* gd = reinterpret_cast<const bf16x8*>(
          Dt + (long)c * NTp + rc + sseg * 16);
      rd[2 * i] = gd[0];
      rd[2 * i + 1] = gd[1];
    }
    int rbase = rc + sseg * 16;
    const __bf16* src = Xt + (long)(ft * 64 + xf) * n_rows;
    int i0 = idx[rbase];
    if (idx[rbase + 15] - i0 == 15 &&
        (((unsigned long)(src + i0) & 15) == 0)) {
      const bf16x8* gx = reinterpret_cast<const bf16x8*>(src + i0);
      rxa = gx[0];
      rxb = gx[1];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) rxa[j] = src[idx[rbase + j]];
#pragma unroll
      for (int j = 0; j < 8; ++j) rxb[j] = src[idx[rbase + 8 + j]];
    }
  };
  auto commit = [&](int b) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      int c = drow + i * 64;
      store_row8(&sD[b][c * 64], c, sseg * 16, rd[2 * i]);
      store_row8(&sD[b][c * 64], c, sseg * 16 + 8, rd[2 * i + 1]);
    }
    store_row8(&sXt[b][xf * 64], xf, sseg * 16, rxa);
    store_row8(&sXt[b][xf * 64], xf, sseg * 16 + 8, rxb);
  };

  issue(r0);
  commit(0);
  __syncthreads();
  for (int rc = r0; rc < r1; rc += 64) {
    int b = (int)(((rc - r0) >> 6) & 1);
    if (rc + 64 < r1) issue(rc + 64);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fn * 16 + (lane & 15);
        bfr[fn] = lds_frag_p(&sXt[b][f * 64], f, g, h);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = wave * cpw + m * 16 + (lane & 15);
        bf16x8 a = lds_frag_p(&sD[b][c * 64], c, g, h);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
    if (rc + 64 < r1) commit(b ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = wave * cpw + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 64 + f_in], acc[m][fn][r]);
      }
    }
  }
}


// ---------------------------------------------------------------------------
// bwd_g5_kernel: Bp=256 wide-block variant -- 512 threads / 8 waves,
// output tile 256 cands x 128 features (waves 0-3: f 0-63, waves 4-7:
// f 64-127).  grid (Fp/128, nseg).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(512)
void bwd_g5_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                   const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                   long n_rows, int NTp, int Fp, int Bp, int seg_rows) {
  constexpr int NF = 4;
  __shared__ __bf16 sD[2][256 * 64];
  __shared__ __bf16 sXt[2][128 * 64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int fhalf = wave >> 2;
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, NTp);
  const int g = lane >> 4;
  const int sseg = tid & 3;
  const int xf = tid >> 2;            // Xt staging: feature 0..127

  f32x4 acc[NF][4];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  bf16x8 rd[4], rxa, rxb;
  auto issue = [&](int rc) {
    // D tile [256 c][64 r]: 1024 16-elem loads over 512 threads --
    // load l = tid + i*512 covers (c = l>>2, seg = l&3) COMPLETELY.
    // (The original drow/dseg2 mapping staged half the rows twice and
    // left the other half as LDS garbage.)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int l = tid + i * 512;
      int c = l >> 2, seg = l & 3;
      const bf16x8* gd = reinterpret_cast<const bf16x8*>(
          Dt + (long)c * NTp + rc + seg * 16);
      rd[2 * i] = gd[0];
      rd[2 * i + 1] = gd[1];
    }
    int rbase = rc + sseg * 16;
    const __bf16* src = Xt + (long)(ft * 128 + xf) * n_rows;
    int i0 = idx[rbase];
    if (idx[rbase + 15] - i0 == 15 &&
        (((unsigned long)(src + i0) & 15) == 0)) {
      const bf16x8* gx = reinterpret_cast<const bf16x8*>(src + i0);
      rxa = gx[0];
      rxb = gx[1];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) rxa[j] = src[idx[rbase + j]];
#pragma unroll
      for (int j = 0; j < 8; ++j) rxb[j] = src[idx[rbase + 8 + j]];
    }
  };
  auto commit = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int l = tid + i * 512;
      int c = l >> 2, seg = l & 3;
      store_row8(&sD[b][c * 64], c, seg * 16, rd[2 * i]);
      store_row8(&sD[b][c * 64], c, seg * 16 + 8, rd[2 * i + 1]);
    }
    store_row8(&sXt[b][xf * 64], xf, sseg * 16, rxa);
    store_row8(&sXt[b][xf * 64], xf, sseg * 16 + 8, rxb);
  };

  issue(r0);
  commit(0);
  __syncthreads();
  for (int rc = r0; rc < r1; rc += 64) {
    int b = (int)(((rc - r0) >> 6) & 1);
    if (rc + 64 < r1) issue(rc + 64);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fhalf * 64 + fn * 16 + (lane & 15);
        bfr[fn] = lds_frag_p(&sXt[b][f * 64], f, g, h);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = cwave * 64 + m * 16 + (lane & 15);
        bf16x8 a = lds_frag_p(&sD[b][c * 64], c, g, h);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
    if (rc + 64 < r1) commit(b ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fhalf * 64 + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cwave * 64 + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 128 + f_in], acc[m][fn][r]);
      }
    }
  }
}


// ---------------------------------------------------------------------------
// bwd_g8_kernel: 1024-thread bwd for Bp=256, Fp multiple of 256 -- each
// block owns the WHOLE 256x256 G tile for one split-K row segment
// (16 waves = 4 cand-quads x 4 feature-waves), so D and X^T are staged
// once per row chunk for all of G.  grid (Fp/256, nseg).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void bwd_g8_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                   const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                   long n_rows, int NTp, int n_take, int Fp, int Bp, int seg_rows) {
  constexpr int NF = 4;
  __shared__ __bf16 sD[2][256 * 64];
  __shared__ __bf16 sXt[2][256 * 64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cquad = wave >> 2;       // candidate quad 0..3
  const int fwave = wave & 3;        // feature wave 0..3
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, n_take);
  const int g = lane >> 4;
  const int srow = tid >> 2;         // staging row 0..255
  const int sseg = tid & 3;

  f32x4 acc[NF][4];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  bf16x8 rd[2], rxa, rxb;
  auto issue = [&](int rc) {
    const bf16x8* gd = reinterpret_cast<const bf16x8*>(
        Dt + (long)srow * NTp + rc + sseg * 16);
    rd[0] = gd[0];
    rd[1] = gd[1];
    int rbase = rc + sseg * 16;
    const __bf16* src = Xt + (long)(ft * 256 + srow) * n_rows;
    int i0 = idx[rbase];
    if (idx[rbase + 15] - i0 == 15 &&
        (((unsigned long)(src + i0) & 15) == 0)) {
      const bf16x8* gx = reinterpret_cast<const bf16x8*>(src + i0);
      rxa = gx[0];
      rxb = gx[1];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) rxa[j] = src[idx[rbase + j]];
#pragma unroll
      for (int j = 0; j < 8; ++j) rxb[j] = src[idx[rbase + 8 + j]];
    }
  };
  auto commit = [&](int b) {
    store_row8(&sD[b][srow * 64], srow, sseg * 16, rd[0]);
    store_row8(&sD[b][srow * 64], srow, sseg * 16 + 8, rd[1]);
    store_row8(&sXt[b][srow * 64], srow, sseg * 16, rxa);
    store_row8(&sXt[b][srow * 64], srow, sseg * 16 + 8, rxb);
  };

  issue(r0);
  commit(0);
  __syncthreads();
  for (int rc = r0; rc < r1; rc += 64) {
    int b = (int)(((rc - r0) >> 6) & 1);
    if (rc + 64 < r1) issue(rc + 64);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fwave * 64 + fn * 16 + (lane & 15);
        bfr[fn] = lds_frag_p(&sXt[b][f * 64], f, g, h);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = cquad * 64 + m * 16 + (lane & 15);
        bf16x8 a = lds_frag_p(&sD[b][c * 64], c, g, h);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
    if (rc + 64 < r1) commit(b ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fwave * 64 + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cquad * 64 + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 256 + f_in], acc[m][fn][r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// col_finalize_kernel: per-column bias update + convergence, on-device.
// ---------------------------------------------------------------------------
__global__ void col_finalize_kernel(
    float* __restrict__ loss_sum, float* __restrict__ db_sum,
    float* __restrict__ bias, float* __restrict__ Vb,
    float* __restrict__ prev_loss, float* __restrict__ cur_loss,
    int* __restrict__ active, int* __restrict__ epoch_mask,
    int* __restrict__ n_iter,
    const int* __restrict__ max_iter, const float* __restrict__ lr,
    const float* __restrict__ mom, const float* __restrict__ tol,
    const unsigned char* __restrict__ fit_ic,
    float inv_n, int epoch, int Bp, int want_loss,
    int* __restrict__ n_active) {
  int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= Bp) return;
  float cur = loss_sum[c] * inv_n;
  int ea = active[c] && (epoch < max_iter[c]);
  epoch_mask[c] = ea;
  if (ea) {
    n_iter[c] = epoch + 1;
    float gb = db_sum[c] * inv_n * (float)fit_ic[c];
    float vb = mom[c] * Vb[c] - lr[c] * gb;
    Vb[c] = vb;
    bias[c] += vb;
    if (want_loss) {
      cur_loss[c] = cur;
      if (fabsf(prev_loss[c] - cur) <= tol[c] * fmaxf(cur, 1.f))
        active[c] = 0;
      prev_loss[c] = cur;
    }
  }
  loss_sum[c] = 0.f;
  db_sum[c] = 0.f;
  if (active[c] && (epoch + 1) < max_iter[c]) atomicAdd(n_active, 1);
}

// ---------------------------------------------------------------------------
// update_w_kernel: masked momentum update, bf16 mirror, G zeroing.
// grid (Fp/256, Bp), block 256.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256)
void update_w_kernel(float* __restrict__ W, float* __restrict__ V,
                     float* __restrict__ Gt, __bf16* __restrict__ Wt,
                     const int* __restrict__ epoch_mask,
                     const float* __restrict__ lr,
                     const float* __restrict__ mom,
                     const float* __restrict__ l1v,
                     const float* __restrict__ l2v,
                     float inv_n, int Fp) {
  int c = blockIdx.y;
  long off = (long)c * Fp + blockIdx.x * 256 + threadIdx.x;
  float g = Gt[off];
  Gt[off] = 0.f;
  if (!epoch_mask[c]) return;
  float w = W[off];
  float grad = g * inv_n + l2v[c] * w +
               l1v[c] * ((w > 0.f) ? 1.f : ((w < 0.f) ? -1.f : 0.f));
  float v = mom[c] * V[off] - lr[c] * grad;
  V[off] = v;
  w += v;
  W[off] = w;
  Wt[off] = (__bf16)w;
}

// ---------------------------------------------------------------------------
// scores_kernel: per-candidate metric sums over idx rows.
// metric: 0=accuracy(correct count), 1=sum loglik, 2=sum squared residual.
// grid ceil(n_idx/32); block 256 (4 waves side by side over Bp cols).
// dynamic LDS: zbuf f32[32][Bp+8] + sX[32][72] + sW[Bp][72] + scand[ncand]
// ---------------------------------------------------------------------------
template <int P, int NF>
__global__ __launch_bounds__(256)
void scores_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                   const long* __restrict__ idx,   // [n_idx] (no padding)
                   const __bf16* __restrict__ Wt, const float* __restrict__ bias,
                   const int* __restrict__ loss_id,
                   const int* __restrict__ target,
                   int C, int metric, long n_idx, int Fp, int Bp, int n_cand,
                   double* __restrict__ out_sum) {
  constexpr int AMAP = P >> 1, BMAP = P & 1;
  const int scand_pad = (n_cand + 3) & ~3;   // keep sX 16B-aligned
  extern __shared__ char smem[];
  long* sRow = reinterpret_cast<long*>(smem);                // [32]
  float* zbuf = reinterpret_cast<float*>(sRow + 32);         // [32][Bp+8]
  float* scand = zbuf + 32 * (Bp + 8);                       // [scand_pad]
  __bf16* sX = reinterpret_cast<__bf16*>(scand + scand_pad); // [32][72]
  __bf16* sW = sX + 32 * 72;                                 // [Bp][72]

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int rt = blockIdx.x;
  constexpr int colsPerWave = NF * 16;       // Bp in {64,128,256}

  if (tid < 32) {
    long r = (long)rt * 32 + tid;
    sRow[tid] = (r < n_idx) ? idx[r] : idx[n_idx - 1];
  }
  for (int i = tid; i < n_cand; i += 256) scand[i] = 0.f;
  __syncthreads();

  // accumulators: 2 m-frags x nfrag n-frags (nfrag <= 4)
  f32x4 acc[2][4];
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int kc = 0; kc < Fp; kc += 64) {
    // stage 32 gathered X rows: 32 rows x 64 k = 2048 bf16; 256 thr x 8
    {
      int r = tid >> 3, seg = tid & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          X + sRow[r] * Fp + kc + seg * 8);
      *reinterpret_cast<bf16x8*>(&sX[r * 72 + seg * 8]) = v;
    }
    // stage Wt rows for all Bp cols: Bp x 64 bf16; thread strided
    for (int e = tid; e < Bp * 4; e += 256) {
      int c = e >> 2, seg = e & 3;
      const uint4* gw = reinterpret_cast<const uint4*>(
          Wt + (long)c * Fp + kc + seg * 16);
      uint4* lw = reinterpret_cast<uint4*>(&sW[c * 72 + seg * 16]);
      lw[0] = gw[0];
      lw[1] = gw[1];
    }
    __syncthreads();
    for (int ks = 0; ks < 64; ks += 32) {
      bf16x8 a0 = lds_frag<AMAP>(&sX[(lane & 15) * 72 + ks], lane);
      bf16x8 a1 = lds_frag<AMAP>(&sX[(16 + (lane & 15)) * 72 + ks], lane);
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int colbase = wave * colsPerWave + fn * 16 + (lane & 15);
        bf16x8 b = lds_frag<BMAP>(&sW[colbase * 72 + ks], lane);
        acc[0][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b, acc[0][fn], 0, 0, 0);
        acc[1][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b, acc[1][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

  // spill z to LDS (add bias)
#pragma unroll
  for (int fm = 0; fm < 2; ++fm) {
#pragma unroll
    for (int fn = 0; fn < NF; ++fn) {
      int col = wave * colsPerWave + fn * 16 + (lane & 15);
      float bia = bias[col];
      for (int r = 0; r < 4; ++r) {
        int row = fm * 16 + ((lane >> 4) << 2) + r;
        zbuf[row * (Bp + 8) + col] = acc[fm][fn][r] + bia;
      }
    }
  }
  __syncthreads();

  // score (row, cand) pairs
  const float eps = 1e-12f;
  for (int p = tid; p < 32 * n_cand; p += 256) {
    int row = p & 31;
    int cand = p >> 5;
    long gr = (long)rt * 32 + row;
    if (gr >= n_idx) continue;
    float yv = y[sRow[row]];
    const float* zr = &zbuf[row * (Bp + 8) + cand * C];
    float val = 0.f;
    if (metric == 2) {                       // r2: squared residual
      float r = yv - zr[0];
      val = r * r;
    } else if (C == 1) {
      float z = zr[0];
      if (metric == 0) {
        int pred = (z > 0.f) ? 1 : 0;
        val = (pred == (int)yv) ? 1.f : 0.f;
      } else {
        float pr = 1.f / (1.f + __expf(-z));
        float t = (yv == 1.f) ? 1.f : 0.f;
        val = t * __logf(pr + eps) + (1.f - t) * __logf(1.f - pr + eps);
      }
    } else {
      if (metric == 0) {
        int best = 0;
        float bz = zr[0];
        for (int c = 1; c < C; ++c)
          if (zr[c] > bz) { bz = zr[c]; best = c; }
        val = (best == (int)yv) ? 1.f : 0.f;
      } else {
        float ssum = 0.f, sy = 0.f;
        for (int c = 0; c < C; ++c) {
          float s = 1.f / (1.f + __expf(-zr[c]));
          ssum += s;
          if (c == (int)yv) sy = s;
        }
        val = __logf(sy / fmaxf(ssum, eps) + eps);
      }
    }
    atomicAdd(&scand[cand], val);
  }
  __syncthreads();
  for (int cand = tid; cand < n_cand; cand += 256)
    atomicAdd(&out_sum[cand], (double)scand[cand]);
}


// ===========================================================================
// K2: KMeans (Lloyd) -- centroid-block batched.  P=3 permuted LDS only
// (the HW-probed layout; host refuses other layouts for this family).
// ===========================================================================

// per-row squared norms (assign-phase distance completion)
__global__ void row_norms_kernel(const __bf16* __restrict__ X, long n,
                                 int Fp, float* __restrict__ out) {
  long row = blockIdx.x * blockDim.x + threadIdx.x;
  for (; row < n; row += (long)gridDim.x * blockDim.x) {
    const __bf16* xr = X + row * Fp;
    float s = 0.f;
    for (int f = 0; f < Fp; f += 8) {
      bf16x8 v = *reinterpret_cast<const bf16x8*>(xr + f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = (float)v[j];
        s += x * x;
      }
    }
    out[row] = s;
  }
}

// assign: S = X[idx] . Ct^T; per (row, block) argmin of cn - 2S -> labels,
// inertia partials.  32-row tiles, Kp <= 256 centroid columns, NF = Kp/64.
template <int NF>
__global__ __launch_bounds__(256)
void kmeans_assign_kernel(const __bf16* __restrict__ X,
                          const int* __restrict__ idx,      // [NTp]
                          const __bf16* __restrict__ Ct,    // [Kp][Fp]
                          const float* __restrict__ cnorm,  // [Kp]
                          const float* __restrict__ xnorm,  // [n]
                          const int* __restrict__ cstart,   // [nb+1]
                          unsigned char* __restrict__ labels,  // [nb][NTp]
                          float* __restrict__ inertia,      // [nb]
                          float* __restrict__ counts,       // [Kp] or null
                          int nt, int NTp, int Fp, int Kp, int nb,
                          int want_labels,
                          const float* __restrict__ w) {
  constexpr int cpw = NF * 16;
  const int Kpad = NF * 64;
  extern __shared__ char km_smem[];
  float* zbuf = reinterpret_cast<float*>(km_smem);          // [32][Kpad+8]
  float* sIn = zbuf + 32 * (Kpad + 8);                      // [nb<=256]
  float* sCnt = sIn + 256;                                  // [Kpad]
  int* sIdx = reinterpret_cast<int*>(sCnt + Kpad);          // [32]
  __bf16* sX = reinterpret_cast<__bf16*>(sIdx + 32);        // [32][64]
  __bf16* sC = sX + 32 * 64;                                // [Kpad][64]

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int rt = blockIdx.x;
  const int g = lane >> 4;

  if (tid < 32) sIdx[tid] = idx[rt * 32 + tid];
  for (int i = tid; i < nb; i += 256) sIn[i] = 0.f;
  for (int i = tid; i < Kpad; i += 256) sCnt[i] = 0.f;
  __syncthreads();

  f32x4 acc[2][NF];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int kc = 0; kc < Fp; kc += 64) {
    {
      int r = tid >> 3, seg = tid & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          X + (long)sIdx[r] * Fp + kc + seg * 8);
      store_row8(&sX[r * 64], r, seg * 8, v);
    }
    for (int e = tid; e < Kpad * 8; e += 256) {
      int c = e >> 3, seg = e & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          Ct + (long)c * Fp + kc + seg * 8);
      store_row8(&sC[c * 64], c, seg * 8, v);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a0 = lds_frag_p(&sX[(lane & 15) * 64], lane & 15, g, h);
      bf16x8 a1 = lds_frag_p(&sX[(16 + (lane & 15)) * 64],
                             16 + (lane & 15), g, h);
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = wave * cpw + fn * 16 + (lane & 15);
        bf16x8 b = lds_frag_p(&sC[c * 64], c, g, h);
        acc[0][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a0, b, acc[0][fn], 0, 0, 0);
        acc[1][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a1, b, acc[1][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

  // spill q = cn - 2S to zbuf
#pragma unroll
  for (int fm = 0; fm < 2; ++fm) {
#pragma unroll
    for (int fn = 0; fn < NF; ++fn) {
      int col = wave * cpw + fn * 16 + (lane & 15);
      float cn = cnorm[col];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int row = fm * 16 + ((lane >> 4) << 2) + r;
        zbuf[row * (Kpad + 8) + col] = cn - 2.f * acc[fm][fn][r];
      }
    }
  }
  __syncthreads();

  for (int p = tid; p < 32 * nb; p += 256) {
    int row = p & 31;
    int b = p >> 5;
    int gr = rt * 32 + row;
    if (gr >= nt) continue;
    int lo = cstart[b], hi = cstart[b + 1];
    const float* q = &zbuf[row * (Kpad + 8)];
    float best = q[lo];
    int bj = 0;
    for (int j = lo + 1; j < hi; ++j)
      if (q[j] < best) { best = q[j]; bj = j - lo; }
    if (want_labels)
      labels[(long)b * NTp + gr] = (unsigned char)bj;
    float wt = (w != nullptr) ? w[sIdx[row]] : 1.f;
    if (counts != nullptr) atomicAdd(&sCnt[lo + bj], wt);
    atomicAdd(&sIn[b], wt * (xnorm[sIdx[row]] + best));
  }
  __syncthreads();
  for (int b = tid; b < nb; b += 256) atomicAdd(&inertia[b], sIn[b]);
  if (counts != nullptr)
    for (int i = tid; i < Kp; i += 256)
      if (sCnt[i] != 0.f) atomicAdd(&counts[i], sCnt[i]);
}


// wide assign: 128-row tiles, 512 threads (2 row-halves x 4 col-waves),
// for Kp <= 128 (zbuf LDS bound).  4x the MFMA per staged byte of the
// 32-row kernel.
template <int NF>   // col-frags per wave: Kp = NF * 64
__global__ __launch_bounds__(512)
void kmeans_assign_w_kernel(const __bf16* __restrict__ X,
                            const int* __restrict__ idx,    // [NTp]
                            const __bf16* __restrict__ Ct,  // [Kp][Fp]
                            const float* __restrict__ cnorm,
                            const float* __restrict__ xnorm,
                            const int* __restrict__ cstart,
                            unsigned char* __restrict__ labels,
                            float* __restrict__ inertia,
                            float* __restrict__ counts,
                            int nt, int NTp, int Fp, int Kp, int nb,
                            int want_labels,
                            const float* __restrict__ w) {
  constexpr int cpw = NF * 16;
  const int Kpad = NF * 64;
  extern __shared__ char kw_smem[];
  float* zbuf = reinterpret_cast<float*>(kw_smem);           // [128][Kpad+8]
  float* sIn = zbuf + 128 * (Kpad + 8);                      // [256]
  float* sCnt = sIn + 256;                                   // [Kpad]
  int* sIdx = reinterpret_cast<int*>(sCnt + Kpad);           // [128]
  __bf16* sX = reinterpret_cast<__bf16*>(sIdx + 128);        // [128][64]
  __bf16* sC = sX + 128 * 64;                                // [Kpad][64]

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rhalf = wave >> 2;
  const int rt = blockIdx.x;
  const int g = lane >> 4;

  if (tid < 128) sIdx[tid] = idx[rt * 128 + tid];
  for (int i = tid; i < nb; i += 512) sIn[i] = 0.f;
  for (int i = tid; i < Kpad; i += 512) sCnt[i] = 0.f;
  __syncthreads();

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int kc = 0; kc < Fp; kc += 64) {
    {
      int r = tid >> 2, seg = tid & 3;
      const bf16x8* gx = reinterpret_cast<const bf16x8*>(
          X + (long)sIdx[r] * Fp + kc + seg * 16);
      store_row8(&sX[r * 64], r, seg * 16, gx[0]);
      store_row8(&sX[r * 64], r, seg * 16 + 8, gx[1]);
    }
    for (int e = tid; e < Kpad * 8; e += 512) {
      int c = e >> 3, seg = e & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          Ct + (long)c * Fp + kc + seg * 8);
      store_row8(&sC[c * 64], c, seg * 8, v);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rhalf * 64 + m * 16 + (lane & 15);
        a[m] = lds_frag_p(&sX[r * 64], r, g, h);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * cpw + fn * 16 + (lane & 15);
        bf16x8 b = lds_frag_p(&sC[c * 64], c, g, h);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], b, acc[m][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col = cwave * cpw + fn * 16 + (lane & 15);
    float cn = cnorm[col];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int rowb = rhalf * 64 + m * 16 + ((lane >> 4) << 2);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        zbuf[(rowb + r) * (Kpad + 8) + col] = cn - 2.f * acc[m][fn][r];
    }
  }
  __syncthreads();

  for (int p = tid; p < 128 * nb; p += 512) {
    int row = p & 127;
    int b = p >> 7;
    int gr = rt * 128 + row;
    if (gr >= nt) continue;
    int lo = cstart[b], hi = cstart[b + 1];
    const float* q = &zbuf[row * (Kpad + 8)];
    float best = q[lo];
    int bj = 0;
    for (int j = lo + 1; j < hi; ++j)
      if (q[j] < best) { best = q[j]; bj = j - lo; }
    if (want_labels)
      labels[(long)b * NTp + gr] = (unsigned char)bj;
    float wt = (w != nullptr) ? w[sIdx[row]] : 1.f;
    if (counts != nullptr) atomicAdd(&sCnt[lo + bj], wt);
    atomicAdd(&sIn[b], wt * (xnorm[sIdx[row]] + best));
  }
  __syncthreads();
  for (int b = tid; b < nb; b += 512) atomicAdd(&inertia[b], sIn[b]);
  if (counts != nullptr)
    for (int i = tid; i < Kp; i += 512)
      if (sCnt[i] != 0.f) atomicAdd(&counts[i], sCnt[i]);
}

// one-hot membership matrix: D[cstart[b]+label_b(r)][r] = 1 for train
// rows.  Feeds the MFMA bwd kernel: sums = X^T . onehot -- replaces the
// LDS-atomic update kernel (same-label rows serialized its atomics).
__global__ void kmeans_onehot_kernel(const unsigned char* __restrict__ labels,
                                     const int* __restrict__ cstart,
                                     __bf16* __restrict__ Dt,  // [Kp][NTp]
                                     long nt, long NTp, int nb,
                                     const int* __restrict__ idx,
                                     const float* __restrict__ w) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    // sample_weight: the one-hot entry becomes w (pre-quantized to a
    // bf16-representable value on the host, so the cast is exact and
    // the weighted-count denominator matches the GEMM numerator)
    float wt = (w != nullptr) ? w[idx[r]] : 1.f;
    for (int b = 0; b < nb; ++b) {
      int c = cstart[b] + labels[(long)b * NTp + r];
      Dt[(long)c * NTp + r] = (__bf16)wt;
    }
  }
}

// center update: new = count>0 ? sum/count : old; accumulate shift^2 per
// block and refresh the bf16 mirror + cnorm; zero sums.
__global__ void kmeans_center_kernel(float* __restrict__ C,      // [Kp][Fp]
                                     __bf16* __restrict__ Ct,    // [Kp][Fp]
                                     float* __restrict__ cnorm,  // [Kp]
                                     float* __restrict__ sums,
                                     float* __restrict__ counts,
                                     const int* __restrict__ cen_block,
                                     const int* __restrict__ block_active,
                                     float* __restrict__ shift2,  // [nb]
                                     int Fp, int Kp) {
  int c = blockIdx.x;
  int b = cen_block[c];
  float cntv = counts[c];
  __shared__ float sh[256];
  __shared__ float nrm[256];
  float local_sh = 0.f, local_nrm = 0.f;
  bool upd = block_active[b] && cntv > 0.f;
  for (int f = threadIdx.x; f < Fp; f += blockDim.x) {
    long off = (long)c * Fp + f;
    float oldv = C[off];
    float newv = upd ? sums[off] / cntv : oldv;
    sums[off] = 0.f;
    float d = newv - oldv;
    local_sh += d * d;
    __bf16 nb16 = (__bf16)newv;
    float rv = (float)nb16;       // cnorm must match the bf16 GEMM operand
    local_nrm += rv * rv;
    C[off] = newv;
    Ct[off] = nb16;
  }
  sh[threadIdx.x] = local_sh;
  nrm[threadIdx.x] = local_nrm;
  __syncthreads();
  for (int s2 = blockDim.x / 2; s2 > 0; s2 >>= 1) {
    if (threadIdx.x < s2) {
      sh[threadIdx.x] += sh[threadIdx.x + s2];
      nrm[threadIdx.x] += nrm[threadIdx.x + s2];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    cnorm[c] = nrm[0];
    if (block_active[b]) atomicAdd(&shift2[b], sh[0]);
    counts[c] = 0.f;
  }
}

// per-block convergence bookkeeping
__global__ void kmeans_block_finalize_kernel(
    float* __restrict__ shift2, int* __restrict__ active,
    int* __restrict__ n_iter, const int* __restrict__ max_iter,
    const float* __restrict__ tol, int epoch, int nb,
    int* __restrict__ n_active) {
  int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= nb) return;
  int ea = active[b] && (epoch < max_iter[b]);
  if (ea) {
    n_iter[b] = epoch + 1;
    if (shift2[b] <= tol[b]) active[b] = 0;
  }
  shift2[b] = 0.f;
  if (active[b] && (epoch + 1) < max_iter[b]) atomicAdd(n_active, 1);
}


// ===========================================================================
// K3: histogram gradient boosting (depth-wise heap trees)
// ===========================================================================

__global__ void gbt_grad_kernel(const float* __restrict__ raw,
                                const float* __restrict__ y,
                                float* __restrict__ g, float* __restrict__ h,
                                long nt, int loss,
                                const float* __restrict__ w) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    float wt = (w != nullptr) ? w[r] : 1.f;
    if (loss == LOSS_LOGISTIC) {
      float p = 1.f / (1.f + __expf(-raw[r]));
      g[r] = wt * (p - y[r]);
      h[r] = wt * (p * (1.f - p));
    } else {
      g[r] = wt * (raw[r] - y[r]);
      h[r] = wt;
    }
  }
}

// quantile binning on device: bin = searchsorted(edges[f], x, 'left')
// (first edge >= x).  Edges live in global memory (F x 255 floats, hot in
// L2); one thread per element, 8-step binary search -- replaces a
// 10+-second host bin_data pass at 1M x 128.
__global__ void gbt_bin_kernel(const float* __restrict__ X,
                               const float* __restrict__ edges,  // [F][255]
                               const int* __restrict__ ecnt,     // [F]
                               unsigned char* __restrict__ Xb,
                               long total, int F) {
  long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  for (; i < total; i += (long)gridDim.x * blockDim.x) {
    int f = (int)(i % F);
    float x = X[i];
    const float* e = edges + (long)f * 255;
    int lo = 0, hi = ecnt[f];
    while (lo < hi) {
      int mid = (lo + hi) >> 1;
      if (e[mid] < x) lo = mid + 1; else hi = mid;
    }
    Xb[i] = (unsigned char)lo;
  }
}

// per-(node, feature, bin) histograms in LDS: g as float atomics, (h,
// count) packed into ONE u64 atomic -- h fixed-point in the high half
// (hscale chosen on the host so the sum cannot overflow 32 bits), exact
// count in the low half.  2 LDS atomics per (row, feature) instead of 3;
// LDS atomic throughput is the bound (profiles/r01_families_kernels.md).
// Rows keep a heap node_id; settled rows are skipped by the level range
// check; odd nodes are skipped under the sibling-subtraction trick.
// gscale > 0 selects the DETERMINISTIC mode: g is accumulated as a
// biased fixed-point u64 (g+1 >= 0, so plain unsigned adds; unbiased at
// flush using the exact count) -- integer atomics commute exactly, so
// tree structures are bit-stable run to run.  gscale == 0 keeps the
// default float-atomic g (faster: 12 B/cell vs 16 B).
template <int MULTI,    // 0: single plane, loop-free (the hot path: a
                        // runtime class loop cost ~30% at KP == 1)
          int TBT>      // 1: TREE-BATCHED small-n mode -- grid.z carries
                        // (tree, node-group): the launch-bound digits-
                        // style forests fold a whole tree chunk's level
                        // into ONE launch (per-tree buffer strides below)
__global__ __launch_bounds__(512)
void gbt_hist_kernel(const unsigned char* __restrict__ Xbt,  // [F][n]
                     const int* __restrict__ idxmap,          // [nt]
                     const int* __restrict__ node_id,         // [nt]
                     const float* __restrict__ g,
                     const float* __restrict__ h,
                     float* __restrict__ hist,  // [lvl_nodes][F][256][3]
                     long nt, long n_rows, int F, int lvl_lo,
                     int lvl_nodes, int f_pb, long rows_pb, int even_only,
                     int ng_nodes, int g01, float hscale, float gscale,
                     float gbias, int KP, long g_stride,
                     long hist_stride, int n_tgroups, long idx_tstride,
                     long g_tstride, long hist_tstride, int store_flush,
                     int cellw) {
  extern __shared__ char smem[];
  // under sibling subtraction only EVEN nodes are histogrammed: LDS
  // covers lvl_nodes/2 node slots, doubling resident blocks at deep
  // levels (round-1 PMC: 11.8% occupancy, WAIT-bound on LDS atomics).
  // Deeper levels than LDS can hold are split into node GROUPS of
  // ng_nodes along grid.z (each z-block scans the rows, histogramming
  // only its nodes) -- this is what lifts the device tree-depth cap
  // from 6 to 10.
  if (TBT) {
    const int t = (int)blockIdx.z / n_tgroups;
    idxmap += (long)t * idx_tstride;    // 0 when all trees share the map
    node_id += (long)t * nt;
    g += (long)t * g_tstride;
    hist += (long)t * hist_tstride;
  }
  const int ng0 =
      (TBT ? ((int)blockIdx.z % n_tgroups) : (int)blockIdx.z) * ng_nodes;
  const int cellsg = ng_nodes * f_pb * 256;
  const bool gfix = gscale > 0.f;
  unsigned long long* lhc = reinterpret_cast<unsigned long long*>(smem);
  unsigned long long* lgq = lhc + cellsg;            // gfix mode only
  float* lg = reinterpret_cast<float*>(smem + (size_t)cellsg * 8);
  const int tid = threadIdx.x;
  const int nthr = blockDim.x;
  const int f0 = blockIdx.y * f_pb;
  const long r0 = (long)blockIdx.x * rows_pb;
  const long r1 = min(r0 + rows_pb, nt);

  // KP > 1: one launch histograms ALL class planes (g + c*g_stride ->
  // hist + c*hist_stride) with the block's row range cache-hot across
  // classes -- replaces K separate launches (the digits-style K=10
  // forests were launch-bound, and the row-metadata HBM re-read was xK)
  for (int cls = 0; cls < (MULTI ? KP : 1); ++cls) {
  const float* gcls = MULTI ? g + (long)cls * g_stride : g;
  float* hist_c = MULTI ? hist + (long)cls * hist_stride : hist;
  if (gfix) {
    for (int i = tid; i < 2 * cellsg; i += nthr) lhc[i] = 0ull;
  } else if (g01) {
    // g values are 0/1 integers and h == 1: (g-sum, count) pack into the
    // ONE u64 cell (h derived as count) -- halves the LDS atomics and
    // shrinks cells from 12 to 8 bytes (RandomForest classification)
    for (int i = tid; i < cellsg; i += nthr) lhc[i] = 0ull;
  } else {
    for (int i = tid; i < cellsg; i += nthr) { lhc[i] = 0ull; lg[i] = 0.f; }
  }
  __syncthreads();

  const bool vec8 = (F % 8 == 0) && (f_pb == 8);
  for (long r = r0 + tid; r < r1; r += nthr) {
    int nd = node_id[r];
    if (nd < lvl_lo || nd >= lvl_lo + lvl_nodes) continue;
    if (even_only && ((nd - lvl_lo) & 1)) continue;   // sibling trick
    int local = (nd - lvl_lo) >> even_only;
    if (local < ng0 || local >= ng0 + ng_nodes) continue;
    long gi = idxmap[r];
    float gr = gcls[r];
    unsigned long long gq = 0ull;
    if (gfix) gq = (unsigned long long)((double)(gr + gbias) *
                                        (double)gscale + 0.5);
    unsigned long long hpack;
    if (g01 == 1) {
      hpack = ((unsigned long long)(gr != 0.f ? 1u : 0u) << 32) | 1ull;
    } else if (g01 == 2) {
      // (g+1) in [0,2] at 2^-13; h in [0,0.25] at 2^-11; count 14 bits
      unsigned gq28 = __float2uint_rn((gr + 1.f) * 8192.f);
      unsigned hq22 = __float2uint_rn(h[r] * 2048.f);
      hpack = ((unsigned long long)gq28 << 36) |
              ((unsigned long long)hq22 << 14) | 1ull;
    } else {
      unsigned hfx = __float2uint_rn(h[r] * hscale);
      hpack = ((unsigned long long)hfx << 32) | 1ull;
    }
    const int base = (local - ng0) * f_pb;
    // feature-major bins: each feature is a contiguous [n_rows] stream,
    // so a wave's consecutive-ish gi values coalesce into full 64B
    // lines per feature chunk (the row-major layout pulled a line per
    // row PER FEATURE-CHUNK BLOCK -- F/f_pb-fold read amplification)
    const unsigned char* xcol = Xbt + gi;
    if (vec8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int cell = (base + j) * 256 + (int)xcol[(long)(f0 + j) * n_rows];
        if (gfix) atomicAdd(&lgq[cell], gq);
        else if (!g01) atomicAdd(&lg[cell], gr);
        atomicAdd(&lhc[cell], hpack);
      }
    } else {
      for (int ff = 0; ff < f_pb; ++ff) {
        int cell = (base + ff) * 256 + (int)xcol[(long)(f0 + ff) * n_rows];
        if (gfix) atomicAdd(&lgq[cell], gq);
        else if (!g01) atomicAdd(&lg[cell], gr);
        atomicAdd(&lhc[cell], hpack);
      }
    }
  }
  __syncthreads();
  const float hinv = 1.f / hscale;
  for (int i = tid; i < cellsg; i += nthr) {
    int ndl = ((i / (256 * f_pb)) + ng0) << even_only;  // full-level slot
    // the last node group can overrun the level (lvl_eff % ng_nodes):
    // those LDS cells are necessarily empty, but the store flush below
    // must not write them
    if (ndl >= lvl_nodes) continue;
    unsigned long long p = lhc[i];
    // count==0 -> cell never touched.  store_flush (host-guaranteed: ONE
    // block owns every global cell) writes zeros instead, replacing the
    // pre-launch global memset -- the 2D fill was 27% of device time on
    // launch-bound small-n forests.
    if (p == 0ull && !store_flush) continue;
    float hv = 0.f, gv = 0.f;
    unsigned cnt = 0;
    if (p != 0ull) {
      if (g01 == 2) {
        cnt = (unsigned)(p & 0x3fffull);
        hv = (float)((p >> 14) & 0x3fffffull) * (1.f / 2048.f);
        gv = (float)(p >> 36) * (1.f / 8192.f) - (float)cnt;
      } else if (g01 == 1) {
        cnt = (unsigned)(p & 0xffffffffull);
        gv = (float)(p >> 32);          // integer class-1 count
        hv = (float)cnt;                // h == 1 per row
      } else {
        cnt = (unsigned)(p & 0xffffffffull);
        hv = (float)(p >> 32) * hinv;
        gv = gfix ? (float)((double)lgq[i] / (double)gscale -
                            (double)cnt * (double)gbias)
                  : lg[i];
      }
    }
    int bin = i & 255;
    int ff = (i >> 8) % f_pb;
    if (cellw) {
      // COMPACT layout [node][F][256][cellw]: per-class g at +cls, ONE
      // shared count at +cellw-1 (written by class 0; the count channel
      // is identical across classes, and RF's h IS the count).  Cuts
      // the dominant hist/sibling/split-scan traffic 2.7x for K=10.
      float* cell = &hist[((((long)ndl * F + f0 + ff) * 256 + bin)) *
                          cellw + (MULTI ? cls : 0)];
      float* ccnt = &hist[((((long)ndl * F + f0 + ff) * 256 + bin)) *
                          cellw + (cellw - 1)];
      if (store_flush) {
        cell[0] = gv;
        if (!MULTI || cls == 0) *ccnt = (float)cnt;
      } else {
        atomicAdd(cell, gv);
        if (!MULTI || cls == 0) atomicAdd(ccnt, (float)cnt);
      }
    } else {
      float* cell = &hist_c[(((long)ndl * F + f0 + ff) * 256 + bin) * 3];
      if (store_flush) {
        cell[0] = gv;
        cell[1] = hv;
        cell[2] = (float)cnt;
      } else {
        atomicAdd(cell, gv);
        atomicAdd(cell + 1, hv);
        atomicAdd(cell + 2, (float)cnt);
      }
    }
  }
  if (MULTI) __syncthreads();    // LDS reuse across class planes
  }
}

// host helper: one level's histogram launch, shared by gbt_fit and
// gbt_fit_multi.  Picks features-per-block to fit 96 KB LDS, row
// segments >=8192 rows (amortizes the global flush), and the largest
// power-of-two h scale whose worst-case sum stays under 2^31.
// SKA_DETERMINISTIC_GBT=1 selects bit-stable histograms for losses with
// |g| <= 1 (logistic, softmax): g accumulates as biased fixed-point u64,
// so integer-add commutativity makes tree structures identical run to
// run.  Costs 16 B/LDS cell instead of 12 (fewer features per block at
// deep levels) -- opt-in.
static bool det_gbt_mode() {
  // read per call (cheap, once per level launch) so tests can toggle
  // the env var inside one process
  const char* e = getenv("SKA_DETERMINISTIC_GBT");
  return e != nullptr && e[0] == '1';
}

static float det_fix_scale(long nt, float gbias = 1.f) {
  // biased g in [0, 2*gbias]: keep nt*(2*gbias*gs + 1) well under 2^62
  double cap = 4.0e18 / (2.0 * (double)gbias * (double)nt + 1.0);
  float gs = 1.f;
  while ((double)gs * 2.0 < cap && gs < 1.0e12f) gs *= 2.f;
  while ((double)gs > cap && gs > 1e-12f) gs *= 0.5f;
  return gs;
}

// deterministic per-round |g| bound for the squared-loss det mode:
// bit-level atomicMax on non-negative floats is order-independent
__global__ void absmax_kernel(const float* __restrict__ g, long n,
                              unsigned* __restrict__ out_bits) {
  float m = 0.f;
  for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    m = fmaxf(m, fabsf(g[i]));
  for (int off = 32; off > 0; off >>= 1)
    m = fmaxf(m, __shfl_down(m, off));
  __shared__ float wm[16];
  int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) wm[wave] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) m = fmaxf(m, wm[w]);
    atomicMax(out_bits, __float_as_uint(m));
  }
}

static void launch_hist_level(const unsigned char* Xtp, const int* idxmap,
                              const int* node_id, const float* g,
                              const float* h, float* hist, long nt,
                              long n_rows, int F, int d, float hmax,
                              bool g_bounded, bool g01, hipStream_t s,
                              int KP = 1, long g_stride = 0,
                              long hist_stride = 0, float gbias = 1.f,
                              bool packed_ok = false, int n_trees = 1,
                              long idx_tstride = 0, long g_tstride = 0,
                              long hist_tstride = 0, int cellw = 0) {
  int lvl_lo = (1 << d) - 1;
  int lvl_nodes = 1 << d;
  int lvl_eff = (d > 0) ? (lvl_nodes >> 1) : lvl_nodes;  // even nodes only
  bool gfix = g_bounded && det_gbt_mode();
  // cell mode: 1 = RF 0/1-g single-atomic; 2 = bounded-g (logistic/
  // softmax) fixed-point single-atomic; 0 = float g channel.
  // mode 2's packed fields (count 14 b, h-sum 22 b at 2^11 scale) bound
  // the rows a block may scan to 8192 -- the block cap below can push
  // rows_pb beyond that at large nt, so mode 2 only engages when the
  // resulting segmentation stays within the field widths.
  // packed_ok gates mode 2: its 2^-13/2^-11 fixed-point resolution
  // flips near-tie splits relative to the f64 reference, so the binary
  // GBT path keeps exact f32 g (structure-identical trees is a test
  // guarantee there); the softmax-multiclass path opts in (+75%
  // measured, its structure tests hold).
  int mode = gfix ? 0 : (g01 ? 1 : ((g_bounded && packed_ok) ? 2 : 0));
  if (mode == 2) {
    long fp2 = std::min(16, std::max(1, (48 * 1024) /
                                     (8 * 256 * std::min(lvl_eff, 16))));
    while (F % fp2 != 0) fp2 /= 2;
    long fch2 = F / fp2;
    long rs2 = std::max<long>(1, std::min<long>(2048 / fch2,
                                                (nt + 8191) / 8192));
    long rpb2 = (nt + rs2 - 1) / rs2;
    if (rpb2 > 8192) mode = 0;
  }
  int cell_b = gfix ? 16 : (mode ? 8 : 12);
  // feature-major bins have no per-row vector-load constraint: f_pb up
  // to 16 halves the (node_id, idxmap, g, h) re-reads per level vs 8
  int f_pb = std::min(16, std::max(1, (48 * 1024) /
                                   (cell_b * 256 * std::min(lvl_eff, 16))));
  while (F % f_pb != 0) f_pb /= 2;       // F is a multiple of f_pb
  int fchunks = F / f_pb;
  int ng_nodes = std::min(lvl_eff,
                          std::max(1, (48 * 1024) / (cell_b * 256 * f_pb)));
  int ngroups = (lvl_eff + ng_nodes - 1) / ng_nodes;
  long rowsegs = std::max<long>(
      1, std::min<long>(2048 / fchunks, (nt + 8191) / 8192));
  if (gfix) rowsegs = 1;   // one writer per global cell: the float flush
                           // adds stay single-sourced, so bit-stable
  long rows_pb = (nt + rowsegs - 1) / rowsegs;
  rowsegs = (nt + rows_pb - 1) / rows_pb;
  size_t lsm = (size_t)ng_nodes * f_pb * 256 * cell_b;
  int even_only = (d > 0) ? 1 : 0;       // sibling subtraction
  float hs = 1.f;
  while (hs * 2.f * hmax * (float)nt + (float)nt < 1.8e9f &&
         hs < 65536.f)
    hs *= 2.f;
  // biased g in [0,2]: keep nt*(2*gs + 1) well under 2^62
  float gs = gfix ? det_fix_scale(nt, gbias) : 0.f;
  long lvlcells = (long)lvl_nodes * F * 256 * (cellw ? cellw : 3);
  // rowsegs == 1 means exactly ONE block owns every global cell: the
  // flush can plain-store (empty cells write zeros), and the pre-launch
  // zeroing of the level is skipped entirely
  int store_flush = (rowsegs == 1) ? 1 : 0;
  if (!store_flush) {
    if (cellw) {
      HIP_CHECK(hipMemset2DAsync(hist, (size_t)hist_tstride * 4, 0,
                                 (size_t)lvlcells * 4, (size_t)n_trees,
                                 s));
    } else if (n_trees > 1) {
      // zero exactly the level's cells of EVERY (tree, class) plane with
      // one strided memset (planes are contiguous: hist_tstride == KP *
      // hist_stride)
      long planes = (long)n_trees * std::max(1, KP);
      long pitch = (KP > 1) ? hist_stride : hist_tstride;
      HIP_CHECK(hipMemset2DAsync(hist, (size_t)pitch * 4, 0,
                                 (size_t)lvlcells * 4, (size_t)planes, s));
    } else {
      HIP_CHECK(hipMemsetAsync(
          hist, 0,
          ((size_t)std::max(0L, (long)(KP - 1)) * (size_t)hist_stride +
           (size_t)lvlcells) * 4, s));
    }
  }
  auto hl = [&](auto kern) {
    HIP_CHECK(hipFuncSetAttribute(
        reinterpret_cast<const void*>(kern),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lsm));
    hipLaunchKernelGGL(kern,
                       dim3((unsigned)rowsegs, (unsigned)fchunks,
                            (unsigned)(ngroups * n_trees)), dim3(512),
                       lsm, s, Xtp, idxmap, node_id, g, h, hist, nt,
                       n_rows, F, lvl_lo, lvl_nodes, f_pb, rows_pb,
                       even_only, ng_nodes, mode, hs, gs, gbias,
                       KP, g_stride, hist_stride, ngroups, idx_tstride,
                       g_tstride, hist_tstride, store_flush, cellw);
  };
  if (n_trees > 1) {
    if (KP > 1) hl(gbt_hist_kernel<1, 1>);
    else hl(gbt_hist_kernel<0, 1>);
  } else {
    if (KP > 1) hl(gbt_hist_kernel<1, 0>);
    else hl(gbt_hist_kernel<0, 0>);
  }
}

// sibling subtraction: right-child histogram = parent - left.  Parents
// that became leaves have no descending rows: both children zero.
__global__ void gbt_sibling_kernel(const float* __restrict__ prev,
                                   float* __restrict__ cur,
                                   const int* __restrict__ feat,
                                   int prev_lo, int F, int lvl_nodes) {
  int pair = blockIdx.y;                   // local parent index
  long cells = (long)F * 256 * 3;
  long base_l = (long)(2 * pair) * cells;
  long base_r = (long)(2 * pair + 1) * cells;
  long base_p = (long)pair * cells;
  bool split = feat[prev_lo + pair] >= 0;
  for (long i = blockIdx.x * blockDim.x + threadIdx.x; i < cells;
       i += (long)gridDim.x * blockDim.x) {
    cur[base_r + i] = split ? prev[base_p + i] - cur[base_l + i] : 0.f;
  }
}

// best split per node: one WAVE per feature.  Each lane owns 4
// consecutive bins; cumulative (G,H,C) up to every threshold comes from a
// wave-level shfl prefix scan, so the 256-bin walk that used to run
// serially per thread is 64-lane parallel and the histogram is read ONCE
// (totals = last prefix element).  Deterministic tie-break: lowest
// feature, then lowest threshold, within a +-1e-12 gain band.
// ---------------------------------------------------------------------------
// RandomForest (K3b) device pieces.  Shares the binned matrix, histogram,
// sibling-subtraction, split-apply and leaf kernels with GBT; RF adds a
// stateless-hash bootstrap resample, exact-k per-node feature subsampling
// inside the split finder, and (for K>2) a summed-per-class gini gain.
// Binary-gini and MSE split criteria are EXACTLY the xgboost-style gain
// with g=y, h=1, lam=0 (the -2n1+n terms telescope in the gain
// difference), so the single-channel path reuses gbt_split_find verbatim;
// leaf value = mean(y) falls out of -g/(h)*lr with lr=-1.
// The numpy reference (models/_rf_ref.py) replicates rf_hash bit-for-bit.
// ---------------------------------------------------------------------------
__host__ __device__ __forceinline__ unsigned rf_hash(unsigned s) {
  s ^= s >> 16;
  s *= 0x7feb352dU;
  s ^= s >> 15;
  s *= 0x846ca68bU;
  s ^= s >> 16;
  return s;
}
__device__ __forceinline__ unsigned rf_feat_hash(unsigned fseed, int nd,
                                                 int f) {
  return rf_hash(fseed ^ (unsigned)(nd * 2654435761u) ^
                 (unsigned)(f * 40503u));
}
// ExtraTrees random-threshold stream (distinct from the selection stream)
__device__ __forceinline__ unsigned rf_thr_hash(unsigned fseed, int nd,
                                                int f) {
  return rf_hash(rf_feat_hash(fseed, nd, f) ^ 0x9E3779B9u);
}

// bootstrap resample: position i draws source position (hash * nt) >> 32
__global__ void rf_bootstrap_kernel(const int* __restrict__ idx_in,
                                    const float* __restrict__ y_in,
                                    int* __restrict__ idx_out,
                                    float* __restrict__ y_out, long nt,
                                    unsigned seed,
                                    const float* __restrict__ w_in,
                                    float* __restrict__ w_out) {
  long i = blockIdx.x * (long)blockDim.x + threadIdx.x;
  for (; i < nt; i += (long)gridDim.x * blockDim.x) {
    unsigned r = rf_hash(seed ^ (unsigned)i);
    long p = (long)(((unsigned long long)r * (unsigned long long)nt) >> 32);
    idx_out[i] = idx_in[p];
    y_out[i] = y_in[p];
    if (w_in != nullptr) w_out[i] = w_in[p];
  }
}

// per-class indicator planes for multiclass gini
__global__ void rf_planes_kernel(const float* __restrict__ y_boot,
                                 float* __restrict__ G, long nt, int K,
                                 const float* __restrict__ w) {
  long i = blockIdx.x * (long)blockDim.x + threadIdx.x;
  for (; i < nt; i += (long)gridDim.x * blockDim.x) {
    int cls = (int)y_boot[i];
    float wt = (w != nullptr) ? w[i] : 1.f;
    for (int c = 0; c < K; ++c)
      G[(long)c * nt + i] = (c == cls) ? wt : 0.f;
  }
}

// exact-k feature selection: block-wide binary search for the largest
// 32-bit threshold t with |{f : rf_feat_hash(f) < t}| <= kfeat; with
// collision-free hashes the selected set is exactly the kfeat smallest.
__device__ unsigned rf_feat_threshold(int F, int kfeat, unsigned fseed,
                                      int nd, int* sred) {
  unsigned t = 0;
  const int tid = threadIdx.x;
  for (int bit = 31; bit >= 0; --bit) {
    unsigned cand = t | (1u << bit);
    int cnt = 0;
    for (int f = tid; f < F; f += (int)blockDim.x)
      cnt += (rf_feat_hash(fseed, nd, f) < cand) ? 1 : 0;
    for (int off = 32; off > 0; off >>= 1) cnt += __shfl_down(cnt, off);
    if ((tid & 63) == 0) sred[tid >> 6] = cnt;
    __syncthreads();
    if (tid == 0) {
      int tot = 0;
      for (int w = 0; w < (int)(blockDim.x >> 6); ++w) tot += sred[w];
      sred[4] = tot;
    }
    __syncthreads();
    if (sred[4] <= kfeat) t = cand;
    __syncthreads();
  }
  return t;
}

template <int CH>   // cell floats: 3 = (g,h,c); 2 = compact RF (g,c) with
                    // h == count (the batched small-n layout)
__device__ __forceinline__
void gbt_split_find_body(const float* __restrict__ nh, int F, int nd,
                         float lam, float lr, int min_leaf,
                         int force_leaf, int* __restrict__ feat,
                         int* __restrict__ thr, float* __restrict__ val,
                         int kfeat, unsigned fseed, int etr) {
  // dead subtree: a non-split parent leaves no rows (and, under the
  // store-flush + skipped-sibling scheme, garbage cells) here.  feat
  // buffers are -1-initialized, so returning IS the leaf/dead marking.
  if (nd > 0 && feat[(nd - 1) >> 1] < 0) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;

  __shared__ float sGain[4];
  __shared__ int sFt[4], sTt[4];
  __shared__ float sG, sH;
  __shared__ int sRed[5];

  unsigned fthr = 0xffffffffu;
  if (kfeat < F) fthr = rf_feat_threshold(F, kfeat, fseed, nd, sRed);

  float bgain = 0.f;
  int bf = -1, bt = 0;

  for (int f = wave; f < F; f += 4) {
    const float* fh = nh + (long)f * 256 * CH;
    float g[4], h[4], c[4];
    float lg = 0.f, lh = 0.f, lc = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int b = 4 * lane + j;
      g[j] = fh[b * CH];
      c[j] = fh[b * CH + CH - 1];
      h[j] = (CH == 2) ? c[j] : fh[b * CH + 1];
      lg += g[j]; lh += h[j]; lc += c[j];
    }
    // inclusive prefix over lanes of the per-lane chunk sums
    float pg = lg, ph = lh, pc = lc;
    for (int off = 1; off < 64; off <<= 1) {
      float tg = __shfl_up(pg, off);
      float th = __shfl_up(ph, off);
      float tc = __shfl_up(pc, off);
      if (lane >= off) { pg += tg; ph += th; pc += tc; }
    }
    float G = __shfl(pg, 63), H = __shfl(ph, 63), C = __shfl(pc, 63);
    if (f == 0 && lane == 0) { sG = G; sH = H; }
    // ExtraTrees: one RANDOM threshold bin per (node, feature), drawn
    // uniformly over the node's occupied bin range [minbin, maxbin)
    int tstar = -1;
    if (etr) {
      int lmin = 256, lmax = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c[j] > 0.f) {
          int b = 4 * lane + j;
          if (b < lmin) lmin = b;
          if (b > lmax) lmax = b;
        }
      }
      for (int off = 32; off > 0; off >>= 1) {
        lmin = min(lmin, __shfl_down(lmin, off));
        lmax = max(lmax, __shfl_down(lmax, off));
      }
      lmin = __shfl(lmin, 0);
      lmax = __shfl(lmax, 0);
      if (lmax > lmin)
        tstar = lmin + (int)(rf_thr_hash(fseed, nd, f) %
                             (unsigned)(lmax - lmin));
    }
    if (!force_leaf &&
        (kfeat >= F || rf_feat_hash(fseed, nd, f) < fthr)) {
      float ps = G * G / (H + lam + 1e-12f);
      float gl = pg - lg, hl = ph - lh, cl = pc - lc;   // exclusive base
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int b = 4 * lane + j;
        gl += g[j]; hl += h[j]; cl += c[j];
        if (b >= 255) continue;
        if (etr && b != tstar) continue;
        float cr = C - cl;
        if (cl < (float)min_leaf || cr < (float)min_leaf) continue;
        float gr2 = G - gl, hr2 = H - hl;
        float gain = gl * gl / (hl + lam + 1e-12f) +
                     gr2 * gr2 / (hr2 + lam + 1e-12f) - ps;
        if (gain > bgain + 1e-12f ||
            (gain > bgain - 1e-12f &&
             (bf < 0 || f < bf || (f == bf && b < bt)))) {
          bgain = gain; bf = f; bt = b;
        }
      }
    }
  }
  // wave argmax (same tie-break), then cross-wave via LDS
  for (int off = 32; off > 0; off >>= 1) {
    float og = __shfl_down(bgain, off);
    int of = __shfl_down(bf, off);
    int ot = __shfl_down(bt, off);
    if (og > bgain + 1e-12f ||
        (og > bgain - 1e-12f && of >= 0 &&
         (bf < 0 || of < bf || (of == bf && ot < bt)))) {
      bgain = og; bf = of; bt = ot;
    }
  }
  if (lane == 0) { sGain[wave] = bgain; sFt[wave] = bf; sTt[wave] = bt; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 4; ++w) {
      if (sGain[w] > sGain[0] + 1e-12f ||
          (sGain[w] > sGain[0] - 1e-12f && sFt[w] >= 0 &&
           (sFt[0] < 0 || sFt[w] < sFt[0] ||
            (sFt[w] == sFt[0] && sTt[w] < sTt[0])))) {
        sGain[0] = sGain[w]; sFt[0] = sFt[w]; sTt[0] = sTt[w];
      }
    }
    if (sFt[0] < 0 || sGain[0] <= 1e-12f) {
      feat[nd] = -1;
      if (sH > 0.f || sG != 0.f)
        val[nd] = -sG / (sH + lam + 1e-12f) * lr;
    } else {
      feat[nd] = sFt[0];
      thr[nd] = sTt[0];
      val[nd] = 0.f;
    }
  }
}

__global__ __launch_bounds__(256)
void gbt_split_find_kernel(const float* __restrict__ hist, int F,
                           int lvl_lo, float lam, float lr, int min_leaf,
                           int force_leaf, int* __restrict__ feat,
                           int* __restrict__ thr, float* __restrict__ val,
                           int kfeat, unsigned fseed, int etr) {
  const int nd_local = blockIdx.x;
  gbt_split_find_body<3>(hist + (long)nd_local * F * 256 * 3, F,
                         lvl_lo + nd_local, lam, lr, min_leaf, force_leaf,
                         feat, thr, val, kfeat, fseed, etr);
}

// tree-batched split find (small-n RF): grid.y = tree within the chunk;
// the per-tree feature-selection seed is recomputed from the forest seed
// exactly as the host loop does, so trees match the per-tree path (and
// the numpy reference) bit for bit.
__global__ __launch_bounds__(256)
void rf_bsplit_find_kernel(const float* __restrict__ hist,
                           long tree_hstride, int F, int lvl_lo,
                           int min_leaf, int* __restrict__ feat,
                           int* __restrict__ thr, float* __restrict__ val,
                           long plane_tstride, int kfeat, unsigned seed,
                           int etr, int t0) {
  const int tl = blockIdx.y;
  const unsigned st =
      rf_hash(seed ^ (unsigned)((t0 + tl) * 0x9e3779b9u));
  const unsigned fs = rf_hash(st ^ 0x85ebca6bu);
  const long po = (long)tl * plane_tstride;
  gbt_split_find_body<2>(
      hist + (long)tl * tree_hstride + (long)blockIdx.x * F * 256 * 2, F,
      lvl_lo + (int)blockIdx.x, 0.f, -1.f, min_leaf, 0, feat + po,
      thr + po, val + po, kfeat, fs, etr);
}

__global__ void gbt_split_apply_kernel(const unsigned char* __restrict__ Xb,
                                       const int* __restrict__ idxmap,
                                       int* __restrict__ node_id,
                                       const int* __restrict__ feat,
                                       const int* __restrict__ thr,
                                       long nt, int F, int lvl_lo,
                                       int lvl_hi) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    int nd = node_id[r];
    if (nd < lvl_lo || nd >= lvl_hi) continue;
    int f = feat[nd];
    if (f < 0) continue;
    int bin = Xb[(long)idxmap[r] * F + f];
    node_id[r] = 2 * nd + 1 + (bin > thr[nd] ? 1 : 0);
  }
}

// bottom-level leaf values: per-node g/h sums.  LDS-staged per block --
// direct global atomics serialized 1M adds onto <=64 node addresses
// (4.8 ms/tree measured; this form is ~100x cheaper).
// gscale > 0 selects deterministic fixed-point accumulation (biased g,
// exact count to unbias; integer atomics commute) -- launched with a
// single block in that mode so the global add has one writer.
__global__ void gbt_node_sums_kernel(const int* __restrict__ node_id,
                                     const float* __restrict__ g,
                                     const float* __restrict__ h,
                                     float* __restrict__ gsum,
                                     float* __restrict__ hsum,
                                     long nt, int lvl_lo_full, int lvl_hi_full,
                                     float gscale, float hscale,
                                     float gbias) {
  __shared__ float lg[128], lh[128];
  __shared__ unsigned long long lgq[128], lhq[128], lcq[128];
  const bool fix = gscale > 0.f;
  // grid.y chunks the node range in 128s (depth > 7 levels)
  const int lvl_lo = lvl_lo_full + (int)blockIdx.y * 128;
  const int lvl_hi = min(lvl_hi_full, lvl_lo + 128);
  int nn = lvl_hi - lvl_lo;
  for (int i = threadIdx.x; i < nn; i += blockDim.x) {
    if (fix) { lgq[i] = 0ull; lhq[i] = 0ull; lcq[i] = 0ull; }
    else { lg[i] = 0.f; lh[i] = 0.f; }
  }
  __syncthreads();
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    int nd = node_id[r];
    if (nd < lvl_lo || nd >= lvl_hi) continue;
    if (fix) {
      atomicAdd(&lgq[nd - lvl_lo],
                (unsigned long long)((double)(g[r] + gbias) *
                                     (double)gscale + 0.5));
      atomicAdd(&lhq[nd - lvl_lo],
                (unsigned long long)((double)h[r] *
                                     (double)hscale + 0.5));
      atomicAdd(&lcq[nd - lvl_lo], 1ull);
    } else {
      atomicAdd(&lg[nd - lvl_lo], g[r]);
      atomicAdd(&lh[nd - lvl_lo], h[r]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nn; i += blockDim.x) {
    if (fix) {
      if (lcq[i] != 0ull) {
        atomicAdd(&gsum[lvl_lo + i],
                  (float)((double)lgq[i] / (double)gscale -
                          (double)lcq[i] * (double)gbias));
        atomicAdd(&hsum[lvl_lo + i],
                  (float)((double)lhq[i] / (double)hscale));
      }
    } else {
      if (lg[i] != 0.f) atomicAdd(&gsum[lvl_lo + i], lg[i]);
      if (lh[i] != 0.f) atomicAdd(&hsum[lvl_lo + i], lh[i]);
    }
  }
}

__global__ void gbt_leaf_vals_kernel(const float* __restrict__ gsum,
                                     const float* __restrict__ hsum,
                                     float* __restrict__ val,
                                     int* __restrict__ feat, float lam,
                                     float lr, int lvl_lo, int lvl_hi) {
  int nd = lvl_lo + blockIdx.x * blockDim.x + threadIdx.x;
  if (nd >= lvl_hi) return;
  if (hsum[nd] > 0.f) {
    feat[nd] = -1;
    val[nd] = -gsum[nd] / (hsum[nd] + lam + 1e-12f) * lr;
  }
}

__global__ void gbt_leaf_apply_kernel(float* __restrict__ raw,
                                      int* __restrict__ node_id,
                                      const float* __restrict__ val,
                                      long nt) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    raw[r] += val[node_id[r]];
    node_id[r] = 0;
  }
}

// predict: walk all trees for arbitrary rows
__global__ void gbt_predict_kernel(const unsigned char* __restrict__ Xb,
                                   const int* __restrict__ idx,  // [n_idx]
                                   const int* __restrict__ feats,  // [T][NN]
                                   const int* __restrict__ thrs,
                                   const float* __restrict__ vals,
                                   int T, int NN, int F, long n_idx,
                                   float f0, float* __restrict__ out) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < n_idx; r += (long)gridDim.x * blockDim.x) {
    const unsigned char* xrow = Xb + (long)idx[r] * F;
    float acc = f0;
    for (int t = 0; t < T; ++t) {
      const int* tf = feats + (long)t * NN;
      const int* tt = thrs + (long)t * NN;
      int nd = 0;
      int guard = 0;
      while (tf[nd] >= 0 && guard++ < 16) {
        nd = 2 * nd + 1 + (xrow[tf[nd]] > tt[nd] ? 1 : 0);
        if (nd >= NN) { nd = (nd - 1) / 2; break; }
      }
      acc += vals[(long)t * NN + nd];
    }
    out[r] = acc;
  }
}

// multiclass predict: ONE launch walks every class plane (grid.y = c)
// directly in the interleaved [T*K][NN] layout -- replaces K separate
// gbt_predict launches on K .contiguous() plane copies (the digits-style
// K=10 scoring was launch/copy bound)
__global__ void gbt_predict_multi_kernel(
    const unsigned char* __restrict__ Xb, const int* __restrict__ idx,
    const int* __restrict__ feats, const int* __restrict__ thrs,
    const float* __restrict__ vals, int T, int K, int NN, int F,
    long n_idx, const float* __restrict__ f0s,
    float* __restrict__ out) {
  const int c = blockIdx.y;
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < n_idx; r += (long)gridDim.x * blockDim.x) {
    const unsigned char* xrow = Xb + (long)idx[r] * F;
    float acc = f0s[c];
    for (int t = 0; t < T; ++t) {
      const long pl = ((long)t * K + c) * NN;
      const int* tf = feats + pl;
      const int* tt = thrs + pl;
      int nd = 0;
      int guard = 0;
      while (tf[nd] >= 0 && guard++ < 16) {
        nd = 2 * nd + 1 + (xrow[tf[nd]] > tt[nd] ? 1 : 0);
        if (nd >= NN) { nd = (nd - 1) / 2; break; }
      }
      acc += vals[pl + nd];
    }
    out[(long)c * n_idx + r] = acc;
  }
}

// metric sums: [0] = correct count (accuracy), [1] = squared residual
__global__ void gbt_metric_kernel(const float* __restrict__ raw,
                                  const float* __restrict__ y,
                                  const int* __restrict__ idx, long n_idx,
                                  int metric, double* __restrict__ out) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  double local = 0.0;
  for (; r < n_idx; r += (long)gridDim.x * blockDim.x) {
    float yv = y[idx[r]];
    if (metric == 0) {
      local += ((raw[r] > 0.f) == (yv > 0.5f)) ? 1.0 : 0.0;
    } else {
      float d = yv - raw[r];
      local += (double)d * d;
    }
  }
  __shared__ double red[256];
  red[threadIdx.x] = local;
  __syncthreads();
  for (int s2 = blockDim.x / 2; s2 > 0; s2 >>= 1) {
    if (threadIdx.x < s2) red[threadIdx.x] += red[threadIdx.x + s2];
    __syncthreads();
  }
  if (threadIdx.x == 0) atomicAdd(out, red[0]);
}


// ---------------------------------------------------------------------------
// fwd_d7_kernel: 1024-thread fwd for Bp=256 -- block tile 256 rows x 256
// cols, 16 waves (4 row-quads x 4 col-waves, each 64x64 like fwd_d5's
// waves).  16 waves/CU at 1 block/CU doubles occupancy over fwd_d5 and
// halves the per-row staging overhead.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void fwd_d7_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                   const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                   const float* __restrict__ bias,
                   const int* __restrict__ loss_id,
                   const int* __restrict__ target, __bf16* __restrict__ Dt,
                   float* __restrict__ loss_sum, float* __restrict__ db_sum,
                   const int* __restrict__ row_key,
                   const int* __restrict__ col_key,
                   int nt, int NTp, int Fp, int Bp, int want_loss) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[256];
  __shared__ float sY[256];
  __shared__ int sKey[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;        // row quad 0..3
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int srow = tid >> 2;          // staging row/col 0..255
  const int sseg = tid & 3;

  if (tid < 256) {
    int gi = idx[rt * 256 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  bf16x8 rx[2], rw[2];
  auto issue = [&](int kc) {
    const bf16x8* gx = reinterpret_cast<const bf16x8*>(
        X + (long)sIdx[srow] * Fp + kc + sseg * 16);
    rx[0] = gx[0];
    rx[1] = gx[1];
    const bf16x8* gw = reinterpret_cast<const bf16x8*>(
        Wt + (long)srow * Fp + kc + sseg * 16);
    rw[0] = gw[0];
    rw[1] = gw[1];
  };
  auto commit = [&](int b) {
    store_row8(&sX[b][srow * 64], srow, sseg * 16, rx[0]);
    store_row8(&sX[b][srow * 64], srow, sseg * 16 + 8, rx[1]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16, rw[0]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16 + 8, rw[1]);
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  issue(0);
  commit(0);
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) issue((kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rquad * 64 + m * 16 + (lane & 15);
        a[m] = lds_frag_p(&sX[b][r * 64], r, g, h);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = lds_frag_p(&sW[b][c * 64], c, g, h);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    if (kc + 1 < nkc) commit(b ^ 1);
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 256 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = 1.f / (1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 256 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// fwd_d12_kernel: fwd_d7 with async global->LDS staging (gload_lds16 +
// frag12 layout; see the v12 comment block up top).  Removes the register
// round-trip + perm_pos VALU path that made fwd_d7 VALU-bound
// (PMC round 1: MfmaUtil 10.8, VALUBusy 47.9).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void fwd_d12_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target, __bf16* __restrict__ Dt,
                    float* __restrict__ loss_sum, float* __restrict__ db_sum,
                    const int* __restrict__ row_key,
                    const int* __restrict__ col_key,
                    int nt, int NTp, int Fp, int Bp, int want_loss) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[256];
  __shared__ float sY[256];
  __shared__ int sKey[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;        // row quad 0..3
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int rl8 = lane >> 3;          // staging: row-in-group 0..7
  const int slot = lane & 7;          // staging: 16B granule 0..7

  if (tid < 256) {
    int gi = idx[rt * 256 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  auto stage = [&](int b, int kc) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int rbase = q * 128 + wave * 8;
      int r = rbase + rl8;
      int ksw = kc + ((slot ^ (r & 7)) << 3);
      gload_lds16(X + (long)sIdx[r] * Fp + ksw, &sX[b][rbase * 64]);
      gload_lds16(Wt + (long)r * Fp + ksw, &sW[b][rbase * 64]);
    }
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)");
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) stage(b ^ 1, (kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rquad * 64 + m * 16 + (lane & 15);
        a[m] = frag12(sX[b], r, h * 4 + g);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = frag12(sW[b], c, h * 4 + g);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)");
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 256 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = 1.f / (1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 256 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// bwd_g12_kernel: bwd_g8 with async global->LDS staging (same v12 layout).
// The Xt tile is gathered by train-row index; when the 64-sample window is
// contiguous and 16B-aligned (the common KFold case away from the single
// fold boundary) it streams through global_load_lds, otherwise a register
// gather writes the identical LDS layout.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void bwd_g12_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                    const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                    long n_rows, int NTp, int n_take, int Fp, int Bp, int seg_rows) {
  constexpr int NF = 4;
  __shared__ __bf16 sD[2][256 * 64];
  __shared__ __bf16 sXt[2][256 * 64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cquad = wave >> 2;       // candidate quad 0..3
  const int fwave = wave & 3;        // feature wave 0..3
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, n_take);
  const int g = lane >> 4;
  const int rl8 = lane >> 3;
  const int slot = lane & 7;

  f32x4 acc[NF][4];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  auto stage = [&](int b, int rc) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int cbase = q * 128 + wave * 8;
      int c = cbase + rl8;
      gload_lds16(Dt + (long)c * NTp + rc + ((slot ^ (c & 7)) << 3),
                  &sD[b][cbase * 64]);
    }
    int i0 = idx[rc];
    if ((idx[rc + 63] - i0) == 63 && (((i0 | (int)n_rows) & 7) == 0)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        int fbase = q * 128 + wave * 8;
        int f = fbase + rl8;
        gload_lds16(Xt + (long)(ft * 256 + f) * n_rows + i0 +
                        ((slot ^ (f & 7)) << 3),
                    &sXt[b][fbase * 64]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        int gi = tid + (q << 10);
        int f = gi >> 3, sl = gi & 7;
        int kb = rc + ((sl ^ (f & 7)) << 3);
        const __bf16* src = Xt + (long)(ft * 256 + f) * n_rows;
        bf16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = src[idx[kb + j]];
        *reinterpret_cast<bf16x8*>(&sXt[b][f * 64 + (sl << 3)]) = v;
      }
    }
  };

  stage(0, r0);
  asm volatile("s_waitcnt vmcnt(0)");
  __syncthreads();
  for (int rc = r0; rc < r1; rc += 64) {
    int b = (int)(((rc - r0) >> 6) & 1);
    if (rc + 64 < r1) stage(b ^ 1, rc + 64);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fwave * 64 + fn * 16 + (lane & 15);
        bfr[fn] = frag12(sXt[b], f, h * 4 + g);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = cquad * 64 + m * 16 + (lane & 15);
        bf16x8 a = frag12(sD[b], c, h * 4 + g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)");
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fwave * 64 + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cquad * 64 + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 256 + f_in], acc[m][fn][r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// fwd_d16_kernel: the measured-ablation rework of the fwd kernel.  The
// round-2 ablation (flagship_ablate) showed the kernel is throughput-
// additive -- X stream ~90us, W staging ~57us, MFMA+LDS reads ~65us,
// epilogue VALU ~77us, D store ~36us of a 355us launch -- so this variant
// REMOVES work instead of pipelining it:
//  * W fragments are read DIRECTLY from global memory.  W is 128 KB and
//    L2/L3-resident (every XCD caches it), a 4-lane group reads one full
//    64 B line per fragment, and this deletes the whole W staging path
//    (2 global_load_lds + 32 KB LDS write + 8 LDS fragment reads per
//    chunk) -- LDS read traffic halves.
//  * The epilogue's tail (gr >= nt) and row-key masks are hoisted into a
//    block-uniform fast path: interior blocks of key-less fits skip 4+
//    VALU ops per element (210M elements/epoch).
//  * X keeps the v12 async global->LDS staging (one buffer pair).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void fwd_d16_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target, __bf16* __restrict__ Dt,
                    float* __restrict__ loss_sum, float* __restrict__ db_sum,
                    const int* __restrict__ row_key,
                    const int* __restrict__ col_key,
                    int nt, int NTp, int Fp, int Bp, int want_loss) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[256];
  __shared__ float sY[256];
  __shared__ int sKey[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int rl8 = lane >> 3;
  const int slot = lane & 7;

  if (tid < 256) {
    int gi = idx[rt * 256 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  auto stage = [&](int b, int kc) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int rbase = q * 128 + wave * 8;
      int r = rbase + rl8;
      int ksw = kc + ((slot ^ (r & 7)) << 3);
      gload_lds16(X + (long)sIdx[r] * Fp + ksw, &sX[b][rbase * 64]);
      gload_lds16(Wt + (long)r * Fp + ksw, &sW[b][rbase * 64]);
    }
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) stage(b ^ 1, (kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rquad * 64 + m * 16 + (lane & 15);
        a[m] = frag12(sX[b], r, h * 4 + g);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = frag12(sW[b], c, h * 4 + g);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  const bool interior =
      (rt * 256 + 256 <= nt) && (row_key == nullptr) && !want_loss;
#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
      if (interior) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float z = acc[m][fn][r] + bia;
          float yv = sY[row_base + r];
          float d;
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
          dpack[r] = (__bf16)d;
          dsum += d;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int gr = rt * 256 + row_base + r;
          float z = acc[m][fn][r] + bia;
          float d, ls = 0.f;
          if (want_loss) {
            loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
          } else {
            float yv = sY[row_base + r];
            if (lid == LOSS_LOGISTIC) {
              float t = (yv == (float)tgt) ? 1.f : 0.f;
              d = fast_rcp(1.f + __expf(-z)) - t;
            } else if (lid == LOSS_HINGE) {
              float sg = (yv == (float)tgt) ? 1.f : -1.f;
              d = (sg * z < 1.f) ? -sg : 0.f;
            } else {
              float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
              d = z - t;
            }
          }
          if (gr >= nt) { d = 0.f; ls = 0.f; }
          if (row_key != nullptr && sKey[row_base + r] != ck) {
            d = 0.f;
            ls = 0.f;
          }
          dpack[r] = (__bf16)d;
          lsum += ls;
          dsum += d;
        }
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 256 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// fwd_d13_kernel: fwd with the v13 counted-vmcnt 4-ring pipeline (see the
// v13 comment block up top).  K=32 chunks, one raw s_barrier per chunk,
// chunk kc+1/kc+2 loads stay in flight across it.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void fwd_d13_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target, __bf16* __restrict__ Dt,
                    float* __restrict__ loss_sum, float* __restrict__ db_sum,
                    const int* __restrict__ row_key,
                    const int* __restrict__ col_key,
                    int nt, int NTp, int Fp, int Bp, int want_loss) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[4][256 * 32];
  __shared__ __bf16 sW[4][256 * 32];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[256];
  __shared__ float sY[256];
  __shared__ int sKey[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;        // row quad 0..3
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int srow = wave * 16 + (lane >> 2);   // staging row 0..255
  const int slot = lane & 3;                  // staging 16B granule 0..3

  if (tid < 256) {
    int gi = idx[rt * 256 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  auto stage = [&](int buf, int kc) {
    int ksw = (kc << 5) + ((slot ^ swz32(srow)) << 3);
    gload_lds16(X + (long)sIdx[srow] * Fp + ksw, &sX[buf][wave * 16 * 32]);
    gload_lds16(Wt + (long)srow * Fp + ksw, &sW[buf][wave * 16 * 32]);
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const int nkc = Fp >> 5;
  stage(0, 0);
  if (nkc > 1) stage(1, 1);
  if (nkc > 2) stage(2, 2);
  for (int kc = 0; kc < nkc; ++kc) {
    SKA_WAIT_VMCNT(min(nkc - 1 - kc, 2));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (kc + 3 < nkc) stage((kc + 3) & 3, kc + 3);
    const __bf16* bx = sX[kc & 3];
    const __bf16* bw = sW[kc & 3];
    bf16x8 a[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int r = rquad * 64 + m * 16 + (lane & 15);
      a[m] = frag13(bx, r, g);
    }
#pragma unroll
    for (int fn = 0; fn < NF; ++fn) {
      int c = cwave * 64 + fn * 16 + (lane & 15);
      bf16x8 bb = frag13(bw, c, g);
#pragma unroll
      for (int m = 0; m < 4; ++m)
        acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a[m], bb, acc[m][fn], 0, 0, 0);
    }
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 256 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 256 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[col_in], lsum);
    atomicAdd(&sDb[col_in], dsum);
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// bwd_g13_kernel: bwd with the v13 counted-vmcnt 4-ring pipeline.  The
// pipelined path requires the segment's train indices to be one contiguous
// aligned run (the common KFold case); other segments (one per fold
// boundary) take a single-buffer gather loop.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void bwd_g13_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                    const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                    long n_rows, int NTp, int n_take, int Fp, int Bp, int seg_rows) {
  constexpr int NF = 4;
  __shared__ __bf16 sD[4][256 * 32];
  __shared__ __bf16 sXt[4][256 * 32];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cquad = wave >> 2;       // candidate quad 0..3
  const int fwave = wave & 3;        // feature wave 0..3
  const int ft = blockIdx.x;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, n_take);
  const int g = lane >> 4;
  const int srow = wave * 16 + (lane >> 2);
  const int slot = lane & 3;

  f32x4 acc[NF][4];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const int ibase = idx[r0];
  bool seg_cont = (idx[r1 - 1] - ibase == r1 - 1 - r0) &&
                  (((ibase | (int)n_rows) & 7) == 0);
  if (seg_cont) {
    auto stage = [&](int buf, int rc) {
      int gsw = ((slot ^ swz32(srow)) << 3);
      gload_lds16(Dt + (long)srow * NTp + rc + gsw,
                  &sD[buf][wave * 16 * 32]);
      gload_lds16(Xt + (long)(ft * 256 + srow) * n_rows + ibase + (rc - r0) +
                      gsw,
                  &sXt[buf][wave * 16 * 32]);
    };
    const int nkc = (r1 - r0) >> 5;
    stage(0, r0);
    if (nkc > 1) stage(1, r0 + 32);
    if (nkc > 2) stage(2, r0 + 64);
    for (int i = 0; i < nkc; ++i) {
      SKA_WAIT_VMCNT(min(nkc - 1 - i, 2));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (i + 3 < nkc) stage((i + 3) & 3, r0 + ((i + 3) << 5));
      const __bf16* bd = sD[i & 3];
      const __bf16* bx = sXt[i & 3];
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fwave * 64 + fn * 16 + (lane & 15);
        bfr[fn] = frag13(bx, f, g);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = cquad * 64 + m * 16 + (lane & 15);
        bf16x8 a = frag13(bd, c, g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
  } else {
    // gather fallback: 1024 threads cover 256 rows x 4 granules for both
    // tiles; full-drain single buffer (fold-boundary segments only).
    const int fr = tid >> 2, sl = tid & 3;
    for (int rc = r0; rc < r1; rc += 32) {
      int kb = rc + ((sl ^ swz32(fr)) << 3);
      const __bf16* srcx = Xt + (long)(ft * 256 + fr) * n_rows;
      bf16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = srcx[idx[kb + j]];
      *reinterpret_cast<bf16x8*>(&sXt[0][fr * 32 + (sl << 3)]) = v;
      bf16x8 vd = *reinterpret_cast<const bf16x8*>(Dt + (long)fr * NTp + kb);
      *reinterpret_cast<bf16x8*>(&sD[0][fr * 32 + (sl << 3)]) = vd;
      __syncthreads();
      const __bf16* bd = sD[0];
      const __bf16* bx = sXt[0];
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fwave * 64 + fn * 16 + (lane & 15);
        bfr[fn] = frag13(bx, f, g);
      }
#pragma unroll
      for (int m = 0; m < NF; ++m) {
        int c = cquad * 64 + m * 16 + (lane & 15);
        bf16x8 a = frag13(bd, c, g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
      __syncthreads();
    }
  }

#pragma unroll
  for (int m = 0; m < NF; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = fwave * 64 + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cquad * 64 + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + ft * 256 + f_in], acc[m][fn][r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// fused_fb14_kernel: ONE kernel per epoch computing the fwd GEMM, the loss
// epilogue AND the gradient GEMM, with the D (dual/residual) tile resident
// in LDS between the two -- the bf16 D matrix (Bp x NTp, ~0.4 GB at the
// flagship shape) is never written to HBM.  PMC round 2 measured the
// separate fwd/bwd pair moving 1.64 GB/epoch of which 0.82 GB was the D
// write + re-read; fusing nearly halves the HBM traffic and removes the
// scatter write that stalled fwd.
//   Per block: loop over S subtiles of 64 rows.  Per subtile:
//     fwd   : acc_f[4] = X[64r x Fp] . Wt^T       (K=64 chunks via LDS)
//     epilog: d = dloss(z), transposed store into sD[256c][64r] (frag12
//             swizzle), loss/db partial sums into LDS
//     bwd   : acc_g[4][NFW] += D^T . Xt           (two r-chunks of 32)
//   Block end: one atomicAdd flush of G (and loss/db) -- G atomic traffic
//   is 256 KB per block, amortized over S subtiles.
// The 64-row subtile keeps live registers at acc_g(64) + acc_f(16) +
// fragments, inside the 128-VGPR budget __launch_bounds__(1024) implies
// (the 128-row variant spilled to scratch in the hot loop).
// NFW = Fp/64 (1, 2 or 4); requires Bp==256, NTp%256==0, Fp in {64,128,256}.
// ---------------------------------------------------------------------------
template <int NFW>
__global__ __launch_bounds__(1024)
void fused_fb14_kernel(const __bf16* __restrict__ X,
                       const __bf16* __restrict__ Xt,
                       const float* __restrict__ y,
                       const int* __restrict__ idx,
                       const __bf16* __restrict__ Wt,
                       const float* __restrict__ bias,
                       const int* __restrict__ loss_id,
                       const int* __restrict__ target,
                       float* __restrict__ Gt,
                       float* __restrict__ loss_sum,
                       float* __restrict__ db_sum,
                       const int* __restrict__ row_key,
                       const int* __restrict__ col_key,
                       int nt, int NTp, int Fp, int Bp, int want_loss,
                       int S, long n_rows) {
  __shared__ __bf16 sD[256 * 64];         // D^T tile [cand][row], 32 KB
  __shared__ __bf16 sA[64 * 64];          // X chunk [64r][64k], 8 KB
  __shared__ __bf16 sW[256 * 64];         // W chunk [256c][64k] / Xt chunk
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[64];
  __shared__ float sY[64];
  __shared__ int sKey[64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;         // fwd: candidate wave (64 cols)
  const int rquad = wave >> 2;        // fwd: row quad (16 rows)
  const int cquad = wave >> 2;        // bwd: candidate quad (64 cands)
  const int fwave = wave & 3;         // bwd: feature wave (16*NFW feats)
  const int g = lane >> 4;

  if (tid < 256) {
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }

  f32x4 acc_g[4][NFW];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NFW; ++j) acc_g[i][j] = {0.f, 0.f, 0.f, 0.f};

  const long row0 = (long)blockIdx.x * S * 64;
  const int nsub = (int)min((long)S, (NTp - row0 + 63) / 64);

  for (int s = 0; s < nsub; ++s) {
    const int rbase = (int)row0 + s * 64;
    __syncthreads();     // sIdx/sA/sW reuse vs previous subtile
    if (tid < 64) {
      int gi = idx[rbase + tid];
      sIdx[tid] = gi;
      sY[tid] = y[gi];
      sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    }
    __syncthreads();

    // ---- fwd GEMM: acc_f = X . W^T -------------------------------------
    f32x4 acc_f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc_f[j] = {0.f, 0.f, 0.f, 0.f};

    for (int kc = 0; kc < Fp; kc += 64) {
      if (tid < 512) {  // stage X chunk [64r][64k]: waves 0-7
        int r = tid >> 3, sl = tid & 7;
        gload_lds16(X + (long)sIdx[r] * Fp + kc + ((sl ^ (r & 7)) << 3),
                    &sA[wave * 8 * 64]);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // stage W chunk [256c][64k]: 2/thread
        int l = tid + (q << 10);
        int c = l >> 3, sl = l & 7;
        gload_lds16(Wt + (long)c * Fp + kc + ((sl ^ (c & 7)) << 3),
                    &sW[(q * 128 + wave * 8) * 64]);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int r = rquad * 16 + (lane & 15);
        bf16x8 a = frag12(sA, r, h * 4 + g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn) {
          int c = cwave * 64 + fn * 16 + (lane & 15);
          bf16x8 bb = frag12(sW, c, h * 4 + g);
          acc_f[fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bb, acc_f[fn], 0, 0, 0);
        }
      }
      __syncthreads();
    }

    // ---- epilogue: d values -> sD (transposed, swizzled) + loss/db -----
#pragma unroll 1
    for (int fn = 0; fn < 4; ++fn) {
      int col_in = cwave * 64 + fn * 16 + (lane & 15);
      float bia = bias[col_in];
      int lid = loss_id[col_in];
      int tgt = target[col_in];
      int ck = (col_key != nullptr) ? col_key[col_in] : 0;
      float lsum = 0.f, dsum = 0.f;
      int row_base = rquad * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rbase + row_base + r;
        float z = acc_f[fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      {
        int j = row_base >> 3, half = (row_base >> 2) & 1;
        *reinterpret_cast<bf16x4*>(
            &sD[col_in * 64 + ((j ^ (col_in & 7)) << 3) + (half << 2)]) =
            dpack;
      }
      if (want_loss) atomicAdd(&sLoss[col_in], lsum);
      atomicAdd(&sDb[col_in], dsum);
    }
    __syncthreads();

    // ---- bwd GEMM: acc_g += D^T . Xt (two r-chunks of 32) --------------
    for (int rc = 0; rc < 64; rc += 32) {
      {  // stage Xt chunk [Fp f][32 r] into sW (16 KB at NFW=4)
        int i0 = sIdx[rc];
        bool cont = (sIdx[rc + 31] - i0 == 31) &&
                    (((i0 | (int)n_rows) & 7) == 0);
        if (cont) {
          int fr = wave * 16 + (lane >> 2), sl = lane & 3;
          if (fr < NFW * 64)
            gload_lds16(Xt + (long)fr * n_rows + i0 + ((sl ^ swz32(fr)) << 3),
                        &sW[(wave * 16) * 32]);
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
          int fr = tid >> 2, sl = tid & 3;
          if (fr < NFW * 64) {
            int kb = rc + ((sl ^ swz32(fr)) << 3);
            const __bf16* src = Xt + (long)fr * n_rows;
            bf16x8 v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = src[idx[rbase + kb + j]];
            *reinterpret_cast<bf16x8*>(&sW[fr * 32 + (sl << 3)]) = v;
          }
        }
        __syncthreads();
        constexpr int FH = NFW > 2 ? 2 : NFW;   // bfr regs held at once
#pragma unroll
        for (int fh = 0; fh < NFW / FH; ++fh) {
          bf16x8 bfr[FH];
#pragma unroll
          for (int fj = 0; fj < FH; ++fj) {
            int f = fwave * (16 * NFW) + (fh * FH + fj) * 16 + (lane & 15);
            bfr[fj] = frag13(sW, f, g);
          }
#pragma unroll
          for (int mm = 0; mm < 4; ++mm) {
            int c = cquad * 64 + mm * 16 + (lane & 15);
            bf16x8 a = frag12(sD, c, (rc >> 3) + g);
#pragma unroll
            for (int fj = 0; fj < FH; ++fj)
              acc_g[mm][fh * FH + fj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  a, bfr[fj], acc_g[mm][fh * FH + fj], 0, 0, 0);
          }
        }
        __syncthreads();
      }
    }
  }

  // ---- block end: flush G, loss, db ------------------------------------
#pragma unroll
  for (int mm = 0; mm < 4; ++mm) {
#pragma unroll
    for (int fn = 0; fn < NFW; ++fn) {
      int f_in = fwave * (16 * NFW) + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cquad * 64 + mm * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + f_in], acc_g[mm][fn][r]);
      }
    }
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss && sLoss[tid] != 0.f) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// v15: block-level latency hiding.  Every earlier flagship variant (2-phase
// register staging, async staging, counted-vmcnt ring, fused) ran at ONE
// resident 16-wave block per CU (LDS 96-136 KB), so each barrier-
// synchronized stage burst was latency-exposed with nothing to overlap it
// -- measured ~4-7 us per phase across all of them.  v15 shrinks to
// 512-thread blocks with 128x128 tiles and ~34 KB LDS / ~100 VGPR so TWO+
// independent blocks are resident per CU: one block's MFMA phase overlaps
// the other's staging drain, no intra-block pipelining needed.
// fwd grid: (NTp/128, Bp/128); bwd grid: ((Fp/128)*(Bp/128), nseg).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(512, 4)
void fwd_d15_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target, __bf16* __restrict__ Dt,
                    float* __restrict__ loss_sum, float* __restrict__ db_sum,
                    const int* __restrict__ row_key,
                    const int* __restrict__ col_key,
                    int nt, int NTp, int Fp, int Bp, int want_loss) {
  __shared__ __bf16 sX[128 * 64];
  __shared__ __bf16 sW[128 * 64];
  __shared__ float sLoss[128];
  __shared__ float sDb[128];
  __shared__ int sIdx[128];
  __shared__ float sY[128];
  __shared__ int sKey[128];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;          // 0..7
  const int rquad = wave >> 1;        // 32-row quad 0..3
  const int cwave = wave & 1;         // 64-col wave 0..1
  const int rt = blockIdx.x;
  const int col0 = blockIdx.y * 128;
  const int g = lane >> 4;

  if (tid < 128) {
    int gi = idx[rt * 128 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  auto stage = [&](int kc) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int l = tid + (q << 9);
      int r = l >> 3, sl = l & 7;
      gload_lds16(X + (long)sIdx[r] * Fp + kc + ((sl ^ (r & 7)) << 3),
                  &sX[((q << 6) + wave * 8) * 64]);
      gload_lds16(Wt + (long)(col0 + r) * Fp + kc + ((sl ^ (r & 7)) << 3),
                  &sW[((q << 6) + wave * 8) * 64]);
    }
  };

  f32x4 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int kc = 0; kc < Fp; kc += 64) {
    stage(kc);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        int r = rquad * 32 + m * 16 + (lane & 15);
        a[m] = frag12(sX, r, h * 4 + g);
      }
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = frag12(sW, c, h * 4 + g);
#pragma unroll
        for (int m = 0; m < 2; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll 1
  for (int fn = 0; fn < 4; ++fn) {
    int c_loc = cwave * 64 + fn * 16 + (lane & 15);
    int col_in = col0 + c_loc;
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    int ck = (col_key != nullptr) ? col_key[col_in] : 0;
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      int row_base = rquad * 32 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 128 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      *reinterpret_cast<bf16x4*>(
          Dt + (long)col_in * NTp + rt * 128 + row_base) = dpack;
    }
    if (want_loss) atomicAdd(&sLoss[c_loc], lsum);
    atomicAdd(&sDb[c_loc], dsum);
  }
  __syncthreads();
  if (tid < 128) {
    if (want_loss) atomicAdd(&loss_sum[col0 + tid], sLoss[tid]);
    atomicAdd(&db_sum[col0 + tid], sDb[tid]);
  }
}

__global__ __launch_bounds__(512, 4)
void bwd_g15_kernel(const __bf16* __restrict__ Xt, const int* __restrict__ idx,
                    const __bf16* __restrict__ Dt, float* __restrict__ Gt,
                    long n_rows, int NTp, int Fp, int Bp, int seg_rows) {
  __shared__ __bf16 sD[128 * 64];
  __shared__ __bf16 sXt[128 * 64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cquad = wave >> 1;       // 32-cand quad 0..3
  const int fwave = wave & 1;        // 64-feature wave 0..1
  const int nft = Fp >> 7;
  const int f0 = (blockIdx.x % nft) * 128;
  const int c0 = (blockIdx.x / nft) * 128;
  const int r0 = blockIdx.y * seg_rows;
  const int r1 = min(r0 + seg_rows, NTp);
  const int g = lane >> 4;

  f32x4 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  auto stage = [&](int rc) {
    int i0 = idx[rc];
    bool cont = (idx[rc + 63] - i0 == 63) && (((i0 | (int)n_rows) & 7) == 0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int l = tid + (q << 9);
      int r = l >> 3, sl = l & 7;
      gload_lds16(Dt + (long)(c0 + r) * NTp + rc + ((sl ^ (r & 7)) << 3),
                  &sD[((q << 6) + wave * 8) * 64]);
    }
    if (cont) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        int l = tid + (q << 9);
        int r = l >> 3, sl = l & 7;
        gload_lds16(Xt + (long)(f0 + r) * n_rows + i0 + ((sl ^ (r & 7)) << 3),
                    &sXt[((q << 6) + wave * 8) * 64]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        int l = tid + (q << 9);
        int f = l >> 3, sl = l & 7;
        int kb = rc + ((sl ^ (f & 7)) << 3);
        const __bf16* src = Xt + (long)(f0 + f) * n_rows;
        bf16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = src[idx[kb + j]];
        *reinterpret_cast<bf16x8*>(&sXt[f * 64 + (sl << 3)]) = v;
      }
    }
  };

  for (int rc = r0; rc < r1; rc += 64) {
    stage(rc);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 bfr[4];
#pragma unroll
      for (int fn = 0; fn < 4; ++fn) {
        int f = fwave * 64 + fn * 16 + (lane & 15);
        bfr[fn] = frag12(sXt, f, h * 4 + g);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        int c = cquad * 32 + m * 16 + (lane & 15);
        bf16x8 a = frag12(sD, c, h * 4 + g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bfr[fn], acc[m][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int f_in = f0 + fwave * 64 + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = c0 + cquad * 32 + m * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + f_in], acc[m][fn][r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// fused_fb18_kernel: fused_fb14 with double-buffered async staging -- the
// v14 measurement showed the fused epoch is correct and moves ~45% less
// HBM but loses 1.4x to serialized stage->drain phases; v18 overlaps
// chunk k+1's loads with chunk k's MFMA (fwd) and the first Xt chunk
// with the loss epilogue (bwd), keeping the traffic win without the
// drain serialization.
// ---------------------------------------------------------------------------
template <int NFW>
__global__ __launch_bounds__(1024)
void fused_fb18_kernel(const __bf16* __restrict__ X,
                       const __bf16* __restrict__ Xt,
                       const float* __restrict__ y,
                       const int* __restrict__ idx,
                       const __bf16* __restrict__ Wt,
                       const float* __restrict__ bias,
                       const int* __restrict__ loss_id,
                       const int* __restrict__ target,
                       float* __restrict__ Gt,
                       float* __restrict__ loss_sum,
                       float* __restrict__ db_sum,
                       const int* __restrict__ row_key,
                       const int* __restrict__ col_key,
                       int nt, int NTp, int Fp, int Bp, int want_loss,
                       int S, long n_rows) {
  __shared__ __bf16 sD[256 * 64];         // D^T tile [cand][row], 32 KB
  __shared__ __bf16 sA[2][64 * 64];       // X chunk dbuf, 2 x 8 KB
  __shared__ __bf16 sW[2][256 * 64];      // W chunk dbuf / Xt chunks
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[64];
  __shared__ float sY[64];
  __shared__ int sKey[64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;
  const int cquad = wave >> 2;
  const int fwave = wave & 3;
  const int g = lane >> 4;

  if (tid < 256) {
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }

  f32x4 acc_g[4][NFW];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NFW; ++j) acc_g[i][j] = {0.f, 0.f, 0.f, 0.f};

  const long row0 = (long)blockIdx.x * S * 64;
  const int nsub = (int)min((long)S, (NTp - row0 + 63) / 64);
  const int nkc = Fp >> 6;

  auto stage_fwd = [&](int buf, int kc) {
    if (tid < 512) {
      int r = tid >> 3, sl = tid & 7;
      gload_lds16(X + (long)sIdx[r] * Fp + kc + ((sl ^ (r & 7)) << 3),
                  &sA[buf][wave * 8 * 64]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int l = tid + (q << 10);
      int c = l >> 3, sl = l & 7;
      gload_lds16(Wt + (long)c * Fp + kc + ((sl ^ (c & 7)) << 3),
                  &sW[buf][(q * 128 + wave * 8) * 64]);
    }
  };
  auto stage_xt = [&](int buf, int rbase, int rc) {
    int i0 = sIdx[rc];
    bool cont = (sIdx[rc + 31] - i0 == 31) &&
                (((i0 | (int)n_rows) & 7) == 0);
    if (cont) {
      int fr = wave * 16 + (lane >> 2), sl = lane & 3;
      if (fr < NFW * 64)
        gload_lds16(Xt + (long)fr * n_rows + i0 + ((sl ^ swz32(fr)) << 3),
                    &sW[buf][(wave * 16) * 32]);
    } else {
      int fr = tid >> 2, sl = tid & 3;
      if (fr < NFW * 64) {
        int kb = rc + ((sl ^ swz32(fr)) << 3);
        const __bf16* src = Xt + (long)fr * n_rows;
        bf16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = src[idx[rbase + kb + j]];
        *reinterpret_cast<bf16x8*>(&sW[buf][fr * 32 + (sl << 3)]) = v;
      }
    }
  };

  for (int s = 0; s < nsub; ++s) {
    const int rbase = (int)row0 + s * 64;
    __syncthreads();
    if (tid < 64) {
      int gi = idx[rbase + tid];
      sIdx[tid] = gi;
      sY[tid] = y[gi];
      sKey[tid] = (row_key != nullptr) ? row_key[gi] : 0;
    }
    __syncthreads();

    // ---- fwd GEMM, chunk k+1 staged during chunk k's MFMA -------------
    f32x4 acc_f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc_f[j] = {0.f, 0.f, 0.f, 0.f};

    stage_fwd(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kc = 0; kc < nkc; ++kc) {
      int b = kc & 1;
      if (kc + 1 < nkc) stage_fwd(b ^ 1, (kc + 1) << 6);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int r = rquad * 16 + (lane & 15);
        bf16x8 a = frag12(sA[b], r, h * 4 + g);
#pragma unroll
        for (int fn = 0; fn < 4; ++fn) {
          int c = cwave * 64 + fn * 16 + (lane & 15);
          bf16x8 bb = frag12(sW[b], c, h * 4 + g);
          acc_f[fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, bb, acc_f[fn], 0, 0, 0);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }

    // first Xt chunk flies during the loss epilogue (reuses the W buffer
    // the last fwd chunk did NOT occupy)
    const int xb0 = nkc & 1;
    stage_xt(xb0, rbase, 0);

    // ---- epilogue: d values -> sD + loss/db ----------------------------
#pragma unroll
    for (int fn = 0; fn < 4; ++fn) {
      int col_in = cwave * 64 + fn * 16 + (lane & 15);
      float bia = bias[col_in];
      int lid = loss_id[col_in];
      int tgt = target[col_in];
      int ck = (col_key != nullptr) ? col_key[col_in] : 0;
      float lsum = 0.f, dsum = 0.f;
      int row_base = rquad * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rbase + row_base + r;
        float z = acc_f[fn][r] + bia;
        float d, ls = 0.f;
        if (want_loss) {
          loss_grad(lid, z, sY[row_base + r], tgt, &d, &ls);
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
            d = z - t;
          }
        }
        if (gr >= nt) { d = 0.f; ls = 0.f; }
        if (row_key != nullptr && sKey[row_base + r] != ck) {
          d = 0.f;
          ls = 0.f;
        }
        dpack[r] = (__bf16)d;
        lsum += ls;
        dsum += d;
      }
      {
        int j = row_base >> 3, half = (row_base >> 2) & 1;
        *reinterpret_cast<bf16x4*>(
            &sD[col_in * 64 + ((j ^ (col_in & 7)) << 3) + (half << 2)]) =
            dpack;
      }
      if (want_loss) atomicAdd(&sLoss[col_in], lsum);
      atomicAdd(&sDb[col_in], dsum);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();

    // ---- bwd GEMM: second Xt chunk staged during the first's MFMA ------
    for (int rc = 0; rc < 64; rc += 32) {
      int xb = xb0 ^ ((rc >> 5) & 1);
      if (rc + 32 < 64) stage_xt(xb ^ 1, rbase, rc + 32);
      constexpr int FH = NFW > 2 ? 2 : NFW;
#pragma unroll
      for (int fh = 0; fh < NFW / FH; ++fh) {
        bf16x8 bfr[FH];
#pragma unroll
        for (int fj = 0; fj < FH; ++fj) {
          int f = fwave * (16 * NFW) + (fh * FH + fj) * 16 + (lane & 15);
          bfr[fj] = frag13(sW[xb], f, g);
        }
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) {
          int c = cquad * 64 + mm * 16 + (lane & 15);
          bf16x8 a = frag12(sD, c, (rc >> 3) + g);
#pragma unroll
          for (int fj = 0; fj < FH; ++fj)
            acc_g[mm][fh * FH + fj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                a, bfr[fj], acc_g[mm][fh * FH + fj], 0, 0, 0);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }

  // ---- block end: flush G, loss, db ------------------------------------
#pragma unroll
  for (int mm = 0; mm < 4; ++mm) {
#pragma unroll
    for (int fn = 0; fn < NFW; ++fn) {
      int f_in = fwave * (16 * NFW) + fn * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int c_in = cquad * 64 + mm * 16 + ((lane >> 4) << 2) + r;
        atomicAdd(&Gt[(long)c_in * Fp + f_in], acc_g[mm][fn][r]);
      }
    }
  }
  __syncthreads();
  if (tid < 256) {
    if (want_loss && sLoss[tid] != 0.f) atomicAdd(&loss_sum[tid], sLoss[tid]);
    atomicAdd(&db_sum[tid], sDb[tid]);
  }
}

// ---------------------------------------------------------------------------
// scores3_kernel: permuted-LDS (P=3) port of scores_kernel -- removes the
// 22M bank conflicts per dispatch of the generic [72]-stride tiles.
// ---------------------------------------------------------------------------
template <int NF>
__global__ __launch_bounds__(256)
void scores3_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const long* __restrict__ idx,
                    const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target,
                    int C, int metric, long n_idx, int Fp, int Bp,
                    int n_cand, double* __restrict__ out_sum) {
  constexpr int colsPerWave = NF * 16;
  const int scand_pad = (n_cand + 3) & ~3;
  extern __shared__ char smem[];
  long* sRow = reinterpret_cast<long*>(smem);                // [32]
  float* zbuf = reinterpret_cast<float*>(sRow + 32);         // [32][Bp+8]
  float* scand = zbuf + 32 * (Bp + 8);                       // [scand_pad]
  __bf16* sX = reinterpret_cast<__bf16*>(scand + scand_pad); // [32][64]
  __bf16* sW = sX + 32 * 64;                                 // [Bp][64]

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int rt = blockIdx.x;
  const int g = lane >> 4;

  if (tid < 32) {
    long r = (long)rt * 32 + tid;
    sRow[tid] = (r < n_idx) ? idx[r] : idx[n_idx - 1];
  }
  for (int i = tid; i < n_cand; i += 256) scand[i] = 0.f;
  __syncthreads();

  f32x4 acc[2][NF];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  for (int kc = 0; kc < Fp; kc += 64) {
    {
      int r = tid >> 3, seg = tid & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          X + sRow[r] * Fp + kc + seg * 8);
      store_row8(&sX[r * 64], r, seg * 8, v);
    }
    for (int e = tid; e < Bp * 8; e += 256) {
      int c = e >> 3, seg = e & 7;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(
          Wt + (long)c * Fp + kc + seg * 8);
      store_row8(&sW[c * 64], c, seg * 8, v);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a0 = lds_frag_p(&sX[(lane & 15) * 64], lane & 15, g, h);
      bf16x8 a1 = lds_frag_p(&sX[(16 + (lane & 15)) * 64],
                             16 + (lane & 15), g, h);
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = wave * colsPerWave + fn * 16 + (lane & 15);
        bf16x8 b = lds_frag_p(&sW[c * 64], c, g, h);
        acc[0][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a0, b, acc[0][fn], 0, 0, 0);
        acc[1][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            a1, b, acc[1][fn], 0, 0, 0);
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int fm = 0; fm < 2; ++fm) {
#pragma unroll
    for (int fn = 0; fn < NF; ++fn) {
      int col = wave * colsPerWave + fn * 16 + (lane & 15);
      float bia = bias[col];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int row = fm * 16 + ((lane >> 4) << 2) + r;
        zbuf[row * (Bp + 8) + col] = acc[fm][fn][r] + bia;
      }
    }
  }
  __syncthreads();

  const float eps = 1e-12f;
  for (int p = tid; p < 32 * n_cand; p += 256) {
    int row = p & 31;
    int cand = p >> 5;
    long gr = (long)rt * 32 + row;
    if (gr >= n_idx) continue;
    float yv = y[sRow[row]];
    const float* zr = &zbuf[row * (Bp + 8) + cand * C];
    float val = 0.f;
    if (metric == 2) {
      float r = yv - zr[0];
      val = r * r;
    } else if (C == 1) {
      float z = zr[0];
      if (metric == 0) {
        int pred = (z > 0.f) ? 1 : 0;
        val = (pred == (int)yv) ? 1.f : 0.f;
      } else {
        float pr = 1.f / (1.f + __expf(-z));
        float t = (yv == 1.f) ? 1.f : 0.f;
        val = t * __logf(pr + eps) + (1.f - t) * __logf(1.f - pr + eps);
      }
    } else {
      if (metric == 0) {
        int best = 0;
        float bz = zr[0];
        for (int c = 1; c < C; ++c)
          if (zr[c] > bz) { bz = zr[c]; best = c; }
        val = (best == (int)yv) ? 1.f : 0.f;
      } else {
        float ssum = 0.f, sy = 0.f;
        for (int c = 0; c < C; ++c) {
          float s2 = 1.f / (1.f + __expf(-zr[c]));
          ssum += s2;
          if (c == (int)yv) sy = s2;
        }
        val = __logf(sy / fmaxf(ssum, eps) + eps);
      }
    }
    atomicAdd(&scand[cand], val);
  }
  __syncthreads();
  for (int cand = tid; cand < n_cand; cand += 256)
    atomicAdd(&out_sum[cand], (double)scand[cand]);
}



// ---------------------------------------------------------------------------
// scores7_kernel: 1024-thread scoring for C==1 candidates at Bp=256 --
// fwd_d7's 256x256 GEMM tile with a metric-reduction epilogue instead of
// the D write.  scores3's 32-row tiles re-read the whole W per block
// (~800 MB of L2 traffic per dispatch at 200k test rows); 256-row tiles
// cut that 8x.  Multiclass (C>1) needs the per-row zbuf for argmax and
// stays on scores3.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void scores7_kernel(const __bf16* __restrict__ X,
                    const float* __restrict__ y,
                    const long* __restrict__ idx,
                    const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    int metric, long n_idx, int Fp, int Bp, int n_cand,
                    double* __restrict__ out_sum) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sVal[256];
  __shared__ long sRow[256];
  __shared__ float sY[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int srow = tid >> 2;
  const int sseg = tid & 3;

  if (tid < 256) {
    long r = (long)rt * 256 + tid;
    long gi = (r < n_idx) ? idx[r] : idx[n_idx - 1];
    sRow[tid] = gi;
    sY[tid] = y[gi];
    sVal[tid] = 0.f;
  }
  __syncthreads();

  bf16x8 rx[2], rw[2];
  auto issue = [&](int kc) {
    const bf16x8* gx = reinterpret_cast<const bf16x8*>(
        X + sRow[srow] * Fp + kc + sseg * 16);
    rx[0] = gx[0];
    rx[1] = gx[1];
    const bf16x8* gw = reinterpret_cast<const bf16x8*>(
        Wt + (long)srow * Fp + kc + sseg * 16);
    rw[0] = gw[0];
    rw[1] = gw[1];
  };
  auto commit = [&](int b) {
    store_row8(&sX[b][srow * 64], srow, sseg * 16, rx[0]);
    store_row8(&sX[b][srow * 64], srow, sseg * 16 + 8, rx[1]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16, rw[0]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16 + 8, rw[1]);
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  issue(0);
  commit(0);
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) issue((kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rquad * 64 + m * 16 + (lane & 15);
        a[m] = lds_frag_p(&sX[b][r * 64], r, g, h);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = lds_frag_p(&sW[b][c * 64], c, g, h);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    if (kc + 1 < nkc) commit(b ^ 1);
    __syncthreads();
  }

  const float eps = 1e-12f;
#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    float vsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        long gr = (long)rt * 256 + row_base + r;
        if (gr >= n_idx) continue;
        float z = acc[m][fn][r] + bia;
        float yv = sY[row_base + r];
        float val;
        if (metric == 2) {
          float d = yv - z;
          val = d * d;
        } else if (metric == 0) {
          int pred = (z > 0.f) ? 1 : 0;
          val = (pred == (int)yv) ? 1.f : 0.f;
        } else {
          float pr = 1.f / (1.f + __expf(-z));
          float t = (yv == 1.f) ? 1.f : 0.f;
          val = t * __logf(pr + eps) +
                (1.f - t) * __logf(1.f - pr + eps);
        }
        vsum += val;
      }
    }
    if (col_in < n_cand) atomicAdd(&sVal[col_in], vsum);
  }
  __syncthreads();
  if (tid < n_cand)
    atomicAdd(&out_sum[tid], (double)sVal[tid]);
}


// ---------------------------------------------------------------------------
// scores8_kernel: wide-tile MULTICLASS scoring --
// scores7's 256x256 GEMM tile, with the per-row argmax/OVR epilogue done
// through a z-tile that REUSES the staging LDS (the 2x32 KB sX buffers
// become a [64][256] f32 z chunk after the GEMM loop; 4 row-chunks).
// Replaces the 32-row scores3 tiles that re-read all of W per block.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024)
void scores8_kernel(const __bf16* __restrict__ X,
                    const float* __restrict__ y,
                    const long* __restrict__ idx,
                    const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    int C, int metric, long n_idx, int Fp, int Bp,
                    int n_cand, double* __restrict__ out_sum) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sVal[256];
  __shared__ long sRow[256];
  __shared__ float sY[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int srow = tid >> 2;
  const int sseg = tid & 3;

  if (tid < 256) {
    long r = (long)rt * 256 + tid;
    long gi = (r < n_idx) ? idx[r] : idx[n_idx - 1];
    sRow[tid] = gi;
    sY[tid] = y[gi];
    sVal[tid] = 0.f;
  }
  __syncthreads();

  bf16x8 rx[2], rw[2];
  auto issue = [&](int kc) {
    const bf16x8* gx = reinterpret_cast<const bf16x8*>(
        X + sRow[srow] * Fp + kc + sseg * 16);
    rx[0] = gx[0];
    rx[1] = gx[1];
    const bf16x8* gw = reinterpret_cast<const bf16x8*>(
        Wt + (long)srow * Fp + kc + sseg * 16);
    rw[0] = gw[0];
    rw[1] = gw[1];
  };
  auto commit = [&](int b) {
    store_row8(&sX[b][srow * 64], srow, sseg * 16, rx[0]);
    store_row8(&sX[b][srow * 64], srow, sseg * 16 + 8, rx[1]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16, rw[0]);
    store_row8(&sW[b][srow * 64], srow, sseg * 16 + 8, rw[1]);
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  issue(0);
  commit(0);
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) issue((kc + 1) << 6);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int r = rquad * 64 + m * 16 + (lane & 15);
        a[m] = lds_frag_p(&sX[b][r * 64], r, g, h);
      }
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int c = cwave * 64 + fn * 16 + (lane & 15);
        bf16x8 bb = lds_frag_p(&sW[b][c * 64], c, g, h);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a[m], bb, acc[m][fn], 0, 0, 0);
      }
    }
    if (kc + 1 < nkc) commit(b ^ 1);
    __syncthreads();
  }

  // z-tile through the retired staging LDS, 64 rows per pass
  float* zbuf = reinterpret_cast<float*>(sX);   // [64][256] f32 = 64 KB
  const float eps = 1e-12f;
  for (int q = 0; q < 4; ++q) {
    __syncthreads();      // previous pass's reads complete
    if (rquad == q) {
#pragma unroll
      for (int fn = 0; fn < NF; ++fn) {
        int col = cwave * 64 + fn * 16 + (lane & 15);
        float bia = bias[col];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          int rb = m * 16 + ((lane >> 4) << 2);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            zbuf[(rb + r) * 256 + col] = acc[m][fn][r] + bia;
        }
      }
    }
    __syncthreads();
    for (int p = tid; p < 64 * n_cand; p += 1024) {
      int cd = p % n_cand;      // cand fastest: spreads LDS banks
      int row = p / n_cand;
      long gr = (long)rt * 256 + q * 64 + row;
      if (gr >= n_idx) continue;
      float yv = sY[q * 64 + row];
      const float* zr = &zbuf[row * 256 + cd * C];
      float val;
      if (metric == 0) {
        int best = 0;
        float bz = zr[0];
        for (int c = 1; c < C; ++c)
          if (zr[c] > bz) { bz = zr[c]; best = c; }
        val = (best == (int)yv) ? 1.f : 0.f;
      } else {
        float ssum = 0.f, sy = 0.f;
        for (int c = 0; c < C; ++c) {
          float s2 = 1.f / (1.f + __expf(-zr[c]));
          ssum += s2;
          if (c == (int)yv) sy = s2;
        }
        val = __logf(sy / fmaxf(ssum, eps) + eps);
      }
      atomicAdd(&sVal[cd], val);
    }
  }
  __syncthreads();
  if (tid < n_cand)
    atomicAdd(&out_sum[tid], (double)sVal[tid]);
}

// multiclass softmax gradients: raw [K][nt] class-major
__global__ void gbt_softmax_grad_kernel(const float* __restrict__ raw,
                                        const float* __restrict__ y,
                                        float* __restrict__ g,
                                        float* __restrict__ h,
                                        long nt, int K,
                                        const float* __restrict__ w) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    float mx = raw[r];
    for (int c = 1; c < K; ++c) mx = fmaxf(mx, raw[(long)c * nt + r]);
    float sum = 0.f;
    for (int c = 0; c < K; ++c) sum += __expf(raw[(long)c * nt + r] - mx);
    int yc = (int)y[r];
    float wt = (w != nullptr) ? w[r] : 1.f;
    for (int c = 0; c < K; ++c) {
      float p = __expf(raw[(long)c * nt + r] - mx) / sum;
      g[(long)c * nt + r] = wt * (p - ((c == yc) ? 1.f : 0.f));
      h[(long)c * nt + r] = wt * (p * (1.f - p));
    }
  }
}

// per-class leaf apply into class-major raw
__global__ void gbt_leaf_apply_c_kernel(float* __restrict__ raw_c,
                                        int* __restrict__ node_id,
                                        const float* __restrict__ val,
                                        long nt) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    raw_c[r] += val[node_id[r]];
    node_id[r] = 0;
  }
}

// multiclass accuracy: argmax over K class-major raw planes
__global__ void gbt_argmax_acc_kernel(const float* __restrict__ raws,
                                      const float* __restrict__ y,
                                      const int* __restrict__ idx,
                                      long n_idx, int K,
                                      double* __restrict__ out) {
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  double local = 0.0;
  for (; r < n_idx; r += (long)gridDim.x * blockDim.x) {
    int best = 0;
    float bz = raws[r];
    for (int c = 1; c < K; ++c) {
      float z = raws[(long)c * n_idx + r];
      if (z > bz) { bz = z; best = c; }
    }
    local += (best == (int)y[idx[r]]) ? 1.0 : 0.0;
  }
  __shared__ double red[256];
  red[threadIdx.x] = local;
  __syncthreads();
  for (int s2 = blockDim.x / 2; s2 > 0; s2 >>= 1) {
    if (threadIdx.x < s2) red[threadIdx.x] += red[threadIdx.x + s2];
    __syncthreads();
  }
  if (threadIdx.x == 0) atomicAdd(out, red[0]);
}

// ===========================================================================
// K5: CSR-resident linear fits -- for matrices too large or too sparse to
// densify into HBM.  Layouts:
//   X CSR:   indptr i32 [n+1], cols i32 [nnz], vals bf16 [nnz]
//   bwd:     transpose entries sorted by (4096-row chunk, feature, row):
//            consecutive entries share a feature (register-accumulated
//            runs, ONE coalesced flush per run) and a row chunk (the dense
//            D rows they touch stay L2-resident)
//   Wf/Gf:   feature-major mirrors [Fp][Bp] -- a wave reads/flushes one
//            contiguous 64*CPL-column slice per nnz
//   D:       ROW-major bf16 [nt][Bp]; lane owns columns
//            [lane*CPL, lane*CPL + CPL)
// ===========================================================================

template <int CPL>   // columns per lane; Bp = 64 * CPL
__global__ __launch_bounds__(256)
void csr_fwd_d_kernel(const int* __restrict__ indptr,
                      const int* __restrict__ cols,
                      const __bf16* __restrict__ vals,
                      const float* __restrict__ y,
                      const int* __restrict__ idx,     // [nt] train rows
                      const __bf16* __restrict__ Wf,   // [Fp][Bp]
                      const float* __restrict__ bias,
                      const int* __restrict__ loss_id,
                      const int* __restrict__ target,
                      __bf16* __restrict__ D,          // [nt][Bp]
                      float* __restrict__ loss_sum,
                      float* __restrict__ db_sum,
                      long nt, int Bp, int want_loss) {
  const int lane = threadIdx.x & 63;
  const long gwave = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 6;
  const long nwaves = ((long)gridDim.x * blockDim.x) >> 6;
  const int c0 = lane * CPL;

  float ls[CPL], db[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j) { ls[j] = 0.f; db[j] = 0.f; }

  for (long i = gwave; i < nt; i += nwaves) {
    long r = idx[i];
    float z[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) z[j] = 0.f;
    int k1 = indptr[r + 1];
    for (int k = indptr[r]; k < k1; ++k) {
      float v = (float)vals[k];            // lane-uniform broadcast reads
      const __bf16* wrow = Wf + (long)cols[k] * Bp + c0;
#pragma unroll
      for (int j = 0; j < CPL; ++j) z[j] += v * (float)wrow[j];
    }
    float yv = y[r];
    __bf16* drow = D + i * Bp + c0;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      int c = c0 + j;
      float zz = z[j] + bias[c];
      float d, l = 0.f;
      if (want_loss) {
        loss_grad(loss_id[c], zz, yv, target[c], &d, &l);
      } else {
        int lid = loss_id[c];
        int tgt = target[c];
        if (lid == LOSS_LOGISTIC) {
          float t = (yv == (float)tgt) ? 1.f : 0.f;
          d = 1.f / (1.f + __expf(-zz)) - t;
        } else if (lid == LOSS_HINGE) {
          float sg = (yv == (float)tgt) ? 1.f : -1.f;
          d = (sg * zz < 1.f) ? -sg : 0.f;
        } else {
          float t = (tgt < 0) ? yv : ((yv == (float)tgt) ? 1.f : -1.f);
          d = zz - t;
        }
      }
      drow[j] = (__bf16)d;
      ls[j] += l;
      db[j] += d;
    }
  }
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    if (want_loss) atomicAdd(&loss_sum[c0 + j], ls[j]);
    atomicAdd(&db_sum[c0 + j], db[j]);
  }
}

template <int CPL>
__global__ __launch_bounds__(256)
void csr_bwd_g_kernel(const int* __restrict__ tf,    // [nnz] feature
                      const int* __restrict__ tr,    // [nnz] global row
                      const __bf16* __restrict__ tv, // [nnz] value
                      const long* __restrict__ chunk_off,  // [nchunks+1]
                      const int* __restrict__ inv,   // [n] -> local / -1
                      const __bf16* __restrict__ D,  // [nt][Bp]
                      float* __restrict__ Gf,        // [Fp][Bp]
                      int Bp) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int c0 = lane * CPL;
  long lo = chunk_off[blockIdx.x], hi = chunk_off[blockIdx.x + 1];
  long per = (hi - lo + 3) / 4;
  long s0 = lo + wave * per;
  long s1 = min(s0 + per, hi);

  float acc[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j) acc[j] = 0.f;
  int curf = -1;
  for (long k = s0; k < s1; ++k) {
    int f = tf[k];
    if (f != curf) {
      if (curf >= 0) {
#pragma unroll
        for (int j = 0; j < CPL; ++j)
          if (acc[j] != 0.f)
            atomicAdd(&Gf[(long)curf * Bp + c0 + j], acc[j]);
      }
      curf = f;
#pragma unroll
      for (int j = 0; j < CPL; ++j) acc[j] = 0.f;
    }
    int dl = inv[tr[k]];
    if (dl < 0) continue;
    float v = (float)tv[k];
    const __bf16* drow = D + (long)dl * Bp + c0;
#pragma unroll
    for (int j = 0; j < CPL; ++j) acc[j] += v * (float)drow[j];
  }
  if (curf >= 0) {
#pragma unroll
    for (int j = 0; j < CPL; ++j)
      if (acc[j] != 0.f)
        atomicAdd(&Gf[(long)curf * Bp + c0 + j], acc[j]);
  }
}

// sparse-mode weight update: f-major gradient/mirror, c-major master
__global__ void update_w_sparse_kernel(
    float* __restrict__ W,    // [Bp][Fp]
    float* __restrict__ V,    // [Bp][Fp]
    float* __restrict__ Gf,   // [Fp][Bp]
    __bf16* __restrict__ Wf,  // [Fp][Bp]
    const int* __restrict__ epoch_mask, const float* __restrict__ lr,
    const float* __restrict__ mom, const float* __restrict__ l1v,
    const float* __restrict__ l2v, float inv_n, int Fp, int Bp) {
  int c = blockIdx.y;
  int f = blockIdx.x * blockDim.x + threadIdx.x;
  if (f >= Fp) return;
  long cf = (long)c * Fp + f;
  long fc = (long)f * Bp + c;
  float g = Gf[fc];
  Gf[fc] = 0.f;
  if (!epoch_mask[c]) return;
  float w = W[cf];
  float grad = g * inv_n + l2v[c] * w +
               l1v[c] * ((w > 0.f) ? 1.f : ((w < 0.f) ? -1.f : 0.f));
  float v = mom[c] * V[cf] - lr[c] * grad;
  V[cf] = v;
  w += v;
  W[cf] = w;
  Wf[fc] = (__bf16)w;
}

// scores over CSR rows: binary / regression metrics (C == 1 only; the
// engine densifies multiclass sparse searches)
template <int CPL>
__global__ __launch_bounds__(256)
void csr_scores_kernel(const int* __restrict__ indptr,
                       const int* __restrict__ cols,
                       const __bf16* __restrict__ vals,
                       const float* __restrict__ y,
                       const long* __restrict__ idx,  // [n_idx]
                       const __bf16* __restrict__ Wf,
                       const float* __restrict__ bias,
                       const int* __restrict__ loss_id,
                       const int* __restrict__ target,
                       int metric, long n_idx, int Bp, int n_cand,
                       double* __restrict__ out_sum) {
  const int lane = threadIdx.x & 63;
  const long gwave = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 6;
  const long nwaves = ((long)gridDim.x * blockDim.x) >> 6;
  const int c0 = lane * CPL;
  const float eps = 1e-12f;

  float accm[CPL];
#pragma unroll
  for (int j = 0; j < CPL; ++j) accm[j] = 0.f;

  for (long i = gwave; i < n_idx; i += nwaves) {
    long r = idx[i];
    float z[CPL];
#pragma unroll
    for (int j = 0; j < CPL; ++j) z[j] = 0.f;
    int k1 = indptr[r + 1];
    for (int k = indptr[r]; k < k1; ++k) {
      float v = (float)vals[k];
      const __bf16* wrow = Wf + (long)cols[k] * Bp + c0;
#pragma unroll
      for (int j = 0; j < CPL; ++j) z[j] += v * (float)wrow[j];
    }
    float yv = y[r];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      int c = c0 + j;
      if (c >= n_cand) continue;
      float zz = z[j] + bias[c];
      if (metric == 2) {
        float d = yv - zz;
        accm[j] += d * d;
      } else if (metric == 0) {
        int pred = (zz > 0.f) ? 1 : 0;
        accm[j] += (pred == (int)yv) ? 1.f : 0.f;
      } else {
        float pr = 1.f / (1.f + __expf(-zz));
        float t = (yv == 1.f) ? 1.f : 0.f;
        accm[j] += t * __logf(pr + eps) +
                   (1.f - t) * __logf(1.f - pr + eps);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    int c = c0 + j;
    if (c < n_cand && accm[j] != 0.f)
      atomicAdd(&out_sum[c], (double)accm[j]);
  }
}

// multiclass OVR scores over CSR rows: per candidate (= C adjacent
// columns) argmax for accuracy / normalized OVR log-likelihood.  A wave
// stages one row's Bp z-values in LDS (wave-lockstep, no barrier), then
// lanes reduce candidate groups.
__global__ __launch_bounds__(256)
void csr_scores_multi_kernel(const int* __restrict__ indptr,
                             const int* __restrict__ cols,
                             const __bf16* __restrict__ vals,
                             const float* __restrict__ y,
                             const long* __restrict__ idx,
                             const __bf16* __restrict__ Wf,
                             const float* __restrict__ bias,
                             int C, int metric, long n_idx, int Bp,
                             int n_cand, double* __restrict__ out_sum) {
  __shared__ float zrow[4][256];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const long gwave = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 6;
  const long nwaves = ((long)gridDim.x * blockDim.x) >> 6;
  const int cpl = Bp >> 6;
  const float eps = 1e-12f;

  float accm[2] = {0.f, 0.f};
  for (long i = gwave; i < n_idx; i += nwaves) {
    long r = idx[i];
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    int k1 = indptr[r + 1];
    for (int k = indptr[r]; k < k1; ++k) {
      float v = (float)vals[k];
      const __bf16* wrow = Wf + (long)cols[k] * Bp + lane * cpl;
      for (int j = 0; j < cpl; ++j) z[j] += v * (float)wrow[j];
    }
    for (int j = 0; j < cpl; ++j) {
      int c = lane * cpl + j;
      zrow[wave][c] = z[j] + bias[c];
    }
    float yv = y[r];
    for (int q = 0; q < 2; ++q) {
      int cd = lane + (q << 6);
      if (cd >= n_cand) continue;
      const float* zr = &zrow[wave][cd * C];
      if (metric == 0) {
        int best = 0;
        float bz = zr[0];
        for (int c = 1; c < C; ++c)
          if (zr[c] > bz) { bz = zr[c]; best = c; }
        accm[q] += (best == (int)yv) ? 1.f : 0.f;
      } else {
        float ssum = 0.f, sy = 0.f;
        for (int c = 0; c < C; ++c) {
          float s2 = 1.f / (1.f + __expf(-zr[c]));
          ssum += s2;
          if (c == (int)yv) sy = s2;
        }
        accm[q] += __logf(sy / fmaxf(ssum, eps) + eps);
      }
    }
  }
  for (int q = 0; q < 2; ++q) {
    int cd = lane + (q << 6);
    if (cd < n_cand && accm[q] != 0.f)
      atomicAdd(&out_sum[cd], (double)accm[q]);
  }
}

// ===========================================================================
// host wrappers
// ===========================================================================

static int g_layout = -1;   // P = AMAP*2+BMAP chosen by the runtime probe

// Flagship fwd/bwd kernel version selector (SKA_FLAGSHIP_V; the round-2
// measured ladder lives in profiles/r02_flagship_ablation.md):
//   16 (DEFAULT) fwd_d16 + bwd_g12: async-staged 2-phase, block-uniform
//      fast epilogue -- 17.0-17.2k candidate-fits/s
//   7  round-1 register-staged kernels (baseline)
//   12 async global->LDS staging only
//   13 counted-vmcnt 4-buffer ring      (measured slower; kept for A/B)
//   14 fused epoch, D resident in LDS   (measured slower; kept for A/B)
//   15 512-thread 128x128 multi-block   (measured slower; kept for A/B)
//   17 pass-pipelined epoch, side stream(measured slower; kept for A/B)
//   18 fused + double-buffered staging  (measured slower; kept for A/B)
static int flagship_v() {
  static int v = [] {
    const char* e = getenv("SKA_FLAGSHIP_V");
    return (e && *e) ? atoi(e) : 16;
  }();
  return v;
}
static auto* flagship_fwd() {
  int v = flagship_v();
  if (v >= 16) return fwd_d16_kernel;
  return v == 13 ? fwd_d13_kernel : (v == 12 ? fwd_d12_kernel : fwd_d7_kernel);
}
static auto* flagship_bwd() {
  int v = flagship_v();
  if (v >= 16) return bwd_g12_kernel;
  return v == 13 ? bwd_g13_kernel : (v == 12 ? bwd_g12_kernel : bwd_g8_kernel);
}

// Side stream for overlapped bwd passes (v17 pipelined epoch).
static hipStream_t side_stream() {
  static hipStream_t t = [] {
    hipStream_t s2;
    HIP_CHECK(hipStreamCreateWithFlags(&s2, hipStreamNonBlocking));
    return s2;
  }();
  return t;
}

// Launch the flagship fwd+bwd pair for the current SKA_FLAGSHIP_V.
static void launch_flagship_pair(
    hipStream_t s, const __bf16* Xp, const __bf16* Xtp, const float* yp,
    const int* idxp, const __bf16* Wtp, float* biasp, const int* lossp,
    const int* tgtp, __bf16* Dtp, float* losssum, float* dbsum,
    const int* rkp, const int* ckp, long nt, long NTp, int Fp, int Bp,
    int want_loss, float* Gtp, long n_rows, long nseg, int seg_rows) {
  if (flagship_v() >= 17 && Bp == 256 && NTp % 256 == 0 && Fp % 256 == 0 &&
      NTp > 2 * (long)seg_rows) {
    // v17: epoch split into row passes small enough that each pass's D
    // stripe (256 cands x pass_rows bf16) stays L3-resident between its
    // fwd (producer) and bwd (consumer); bwd pass k runs on a side stream
    // concurrently with fwd pass k+1.  PMC round 2: the D re-read was
    // ~25% of epoch HBM traffic and the two kernels' pipe usage is
    // complementary (fwd VALU-heavy epilogue, bwd pure streams).
    hipStream_t sb = side_stream();
    long segs_per_pass =
        std::max<long>(1, (96L << 20) / (512L * (long)seg_rows));
    long pass_rows = segs_per_pass * (long)seg_rows;
    for (long off = 0; off < NTp; off += pass_rows) {
      long rows = std::min<long>(pass_rows, NTp - off);
      long nsegp = (rows + seg_rows - 1) / seg_rows;
      long nt_loc = std::max<long>(0, nt - off);
      hipLaunchKernelGGL(fwd_d16_kernel, dim3((unsigned)(rows / 256)),
                         dim3(1024), 0, s, Xp, yp, idxp + off, Wtp, biasp,
                         lossp, tgtp, Dtp + off, losssum, dbsum, rkp, ckp,
                         (int)nt_loc, (int)NTp, Fp, Bp, want_loss);
      hipEvent_t ev;
      HIP_CHECK(hipEventCreateWithFlags(&ev, hipEventDisableTiming));
      HIP_CHECK(hipEventRecord(ev, s));
      HIP_CHECK(hipStreamWaitEvent(sb, ev, 0));
      HIP_CHECK(hipEventDestroy(ev));
      hipLaunchKernelGGL(flagship_bwd(),
                         dim3((unsigned)(Fp / 256), (unsigned)nsegp),
                         dim3(1024), 0, sb, Xtp, idxp + off, Dtp + off, Gtp,
                         n_rows, (int)NTp, (int)rows, Fp, Bp, seg_rows);
    }
    hipEvent_t evb;
    HIP_CHECK(hipEventCreateWithFlags(&evb, hipEventDisableTiming));
    HIP_CHECK(hipEventRecord(evb, sb));
    HIP_CHECK(hipStreamWaitEvent(s, evb, 0));
    HIP_CHECK(hipEventDestroy(evb));
    return;
  }
  if (flagship_v() == 15 && Bp % 128 == 0 && NTp % 128 == 0) {
    hipLaunchKernelGGL(fwd_d15_kernel,
                       dim3((unsigned)(NTp / 128), (unsigned)(Bp / 128)),
                       dim3(512), 0, s, Xp, yp, idxp, Wtp, biasp, lossp,
                       tgtp, Dtp, losssum, dbsum, rkp, ckp, (int)nt,
                       (int)NTp, Fp, Bp, want_loss);
    hipLaunchKernelGGL(bwd_g15_kernel,
                       dim3((unsigned)((Fp / 128) * (Bp / 128)),
                            (unsigned)nseg),
                       dim3(512), 0, s, Xtp, idxp, Dtp, Gtp, n_rows,
                       (int)NTp, Fp, Bp, seg_rows);
    return;
  }
  hipLaunchKernelGGL(flagship_fwd(), dim3((unsigned)(NTp / 256)), dim3(1024),
                     0, s, Xp, yp, idxp, Wtp, biasp, lossp, tgtp, Dtp,
                     losssum, dbsum, rkp, ckp, (int)nt, (int)NTp, Fp, Bp,
                     want_loss);
  if (Fp % 256 == 0) {
    hipLaunchKernelGGL(flagship_bwd(),
                       dim3((unsigned)(Fp / 256), (unsigned)nseg), dim3(1024),
                       0, s, Xtp, idxp, Dtp, Gtp, n_rows, (int)NTp, (int)NTp,
                       Fp, Bp, seg_rows);
  } else {
    hipLaunchKernelGGL(bwd_g5_kernel,
                       dim3((unsigned)(Fp / 128), (unsigned)nseg), dim3(512),
                       0, s, Xtp, idxp, Dtp, Gtp, n_rows, (int)NTp, Fp, Bp,
                       seg_rows);
  }
}


static hipStream_t cur_stream() {
  return at::cuda::getCurrentCUDAStream().stream();
}

// run all 4 layout combos; returns tensor [4][16][16] of probe outputs
torch::Tensor gemm_probe(torch::Tensor A, torch::Tensor B) {
  TORCH_CHECK(A.is_cuda() && A.dtype() == torch::kBFloat16);
  TORCH_CHECK(A.sizes() == std::vector<int64_t>({16, 32}));
  TORCH_CHECK(B.sizes() == std::vector<int64_t>({16, 32}));
  auto D = torch::zeros({4, 16, 16},
                        A.options().dtype(torch::kFloat32));
  const __bf16* a = reinterpret_cast<const __bf16*>(A.data_ptr());
  const __bf16* b = reinterpret_cast<const __bf16*>(B.data_ptr());
  float* d = D.data_ptr<float>();
  hipStream_t s = cur_stream();
  hipLaunchKernelGGL((probe_kernel<0, 0>), dim3(1), dim3(64), 0, s, a, b, d);
  hipLaunchKernelGGL((probe_kernel<0, 1>), dim3(1), dim3(64), 0, s, a, b, d + 256);
  hipLaunchKernelGGL((probe_kernel<1, 0>), dim3(1), dim3(64), 0, s, a, b, d + 512);
  hipLaunchKernelGGL((probe_kernel<1, 1>), dim3(1), dim3(64), 0, s, a, b, d + 768);
  HIP_CHECK(hipGetLastError());
  return D;
}

void set_layout(int64_t p) {
  TORCH_CHECK(p >= 0 && p < 4, "layout in [0,4)");
  g_layout = (int)p;
}

int64_t get_layout() { return g_layout; }

double msq_rows(torch::Tensor X) {
  TORCH_CHECK(X.is_cuda() && X.dtype() == torch::kBFloat16 &&
              X.dim() == 2 && X.stride(1) == 1);
  long n = X.size(0);
  int Fp = (int)X.size(1);
  TORCH_CHECK(Fp % 8 == 0);
  auto out = torch::zeros({1}, X.options().dtype(torch::kFloat64));
  int blocks = (int)std::min<long>((n + 255) / 256, 2048);
  hipLaunchKernelGGL(msq_kernel, dim3(blocks), dim3(256), 0, cur_stream(),
                     reinterpret_cast<const __bf16*>(X.data_ptr()), n, Fp,
                     out.data_ptr<double>());
  HIP_CHECK(hipGetLastError());
  return out.item<double>() / (double)n;
}

// linear_fit: the full epoch loop on device.
// Returns (W [Bp][Fp] f32, bias [Bp], n_iter [Bp] i32, cur_loss [Bp] f32,
//          Wt [Bp][Fp] bf16 -- kept on device for the scores kernel).
std::vector<torch::Tensor> linear_fit(
    torch::Tensor X, torch::Tensor Xt, torch::Tensor y, torch::Tensor idx,
    torch::Tensor loss_id, torch::Tensor lr, torch::Tensor l1,
    torch::Tensor l2, torch::Tensor mom, torch::Tensor tol,
    torch::Tensor max_iter, torch::Tensor target, torch::Tensor fit_ic,
    torch::Tensor row_key, torch::Tensor col_key,
    int64_t nt, int64_t max_epochs, int64_t check_every,
    torch::Tensor sw) {
  TORCH_CHECK(g_layout >= 0, "MFMA layout not probed; call ensure_layout()");
  TORCH_CHECK(X.is_cuda() && X.dtype() == torch::kBFloat16 && X.dim() == 2);
  TORCH_CHECK(X.stride(1) == 1 && X.stride(0) == X.size(1));
  TORCH_CHECK(Xt.is_cuda() && Xt.dtype() == torch::kBFloat16 &&
              Xt.size(0) == X.size(1) && Xt.size(1) == X.size(0) &&
              Xt.stride(1) == 1);
  const at::cuda::CUDAGuard guard(X.device());
  int Fp = (int)X.size(1);
  TORCH_CHECK(Fp % 64 == 0, "Fp must be a multiple of 64");
  int Bp = (int)loss_id.size(0);
  TORCH_CHECK(Bp % 64 == 0 && Bp <= 256,
              "Bp must be 64, 128 or 256 (chunk larger batches)");
  long NTp = idx.size(0);
  TORCH_CHECK(NTp % 64 == 0 && nt <= NTp);
  TORCH_CHECK(idx.dtype() == torch::kInt32);
  TORCH_CHECK(y.dtype() == torch::kFloat32);

  auto optF = X.options().dtype(torch::kFloat32);
  auto optI = X.options().dtype(torch::kInt32);
  // sample_weight: per-row weight over the FULL resident matrix (kernels
  // index it by the global row id).  Weighted fits run the generic
  // fwd_d3/fwd_d2 epoch path with the WT=1 epilogue (the fused/flagship
  // variants stay weight-free).
  const bool weighted = sw.numel() > 0;
  const float* wp = nullptr;
  if (weighted) {
    TORCH_CHECK(sw.dtype() == torch::kFloat32 && sw.is_cuda() &&
                sw.size(0) == X.size(0),
                "sample_weight must be float32 [n_rows] on device");
    wp = sw.data_ptr<float>();
  }
  auto W = torch::zeros({Bp, Fp}, optF);
  auto V = torch::zeros({Bp, Fp}, optF);
  auto Gt = torch::zeros({Bp, Fp}, optF);
  auto Wt = torch::zeros({Bp, Fp}, X.options());
  bool use_fused14 = (flagship_v() == 14 || flagship_v() >= 18) &&
                     !weighted &&
                     Bp == 256 && NTp % 256 == 0 &&
                     (Fp == 64 || Fp == 128 || Fp == 256);
  auto Dt = torch::zeros({(long)Bp, use_fused14 ? 1L : NTp}, X.options());
  auto bias = torch::zeros({Bp}, optF);
  auto Vb = torch::zeros({Bp}, optF);
  auto loss_sum = torch::zeros({Bp}, optF);
  auto db_sum = torch::zeros({Bp}, optF);
  auto prev_loss = torch::full({Bp}, 3.0e38, optF);
  auto cur_loss = torch::zeros({Bp}, optF);
  auto active = torch::ones({Bp}, optI);
  auto epoch_mask = torch::zeros({Bp}, optI);
  auto n_iter = torch::zeros({Bp}, optI);
  auto n_active = torch::zeros({1}, optI);

  const __bf16* Xp = reinterpret_cast<const __bf16*>(X.data_ptr());
  float inv_n = 1.0f / (float)nt;
  hipStream_t s = cur_stream();

  // split-K segmentation: target ~1024 blocks for the bwd launch
  int ftiles = Fp / 64;
  long rtiles = NTp / 64;
  long want_nseg = std::max<long>(1, 1024 / ftiles);
  long seg_tiles = std::max<long>(1, (rtiles + want_nseg - 1) / want_nseg);
  long nseg = (rtiles + seg_tiles - 1) / seg_tiles;
  int seg_rows = (int)(seg_tiles * 64);

  dim3 fwd_grid((unsigned)(NTp / 64));
  dim3 bwd_grid((unsigned)ftiles, (unsigned)nseg);
  dim3 fin_grid((unsigned)((Bp + 255) / 256));
  TORCH_CHECK(Fp % 256 == 0 || Fp == 64 || Fp == 128,
              "Fp must be 64, 128 or a multiple of 256");
  int upd_threads = Fp >= 256 ? 256 : Fp;
  dim3 upd_grid2((unsigned)(Fp / upd_threads), (unsigned)Bp);

  const __bf16* Xtp = reinterpret_cast<const __bf16*>(Xt.data_ptr());
  long n_rows = X.size(0);
  const int* rkp = row_key.numel() ? row_key.data_ptr<int>() : nullptr;
  const int* ckp = col_key.numel() ? col_key.data_ptr<int>() : nullptr;
  bool any_tol = tol.max().item<float>() > 0.f;
  int want_loss_cur = 1;
  auto launch_epoch = [&](int epoch, auto fwd_k, auto bwd_k) {
    hipLaunchKernelGGL(fwd_k, fwd_grid, dim3(256), 0, s, Xp,
                       y.data_ptr<float>(), idx.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                       bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                       target.data_ptr<int>(),
                       reinterpret_cast<__bf16*>(Dt.data_ptr()),
                       loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(),
                       rkp, ckp, (int)nt, (int)NTp, Fp, Bp, want_loss_cur,
                       wp);
    hipLaunchKernelGGL(bwd_k, bwd_grid, dim3(256), 0, s, Xtp,
                       idx.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(Dt.data_ptr()),
                       Gt.data_ptr<float>(), n_rows, (int)NTp, Fp, Bp,
                       seg_rows);
    hipLaunchKernelGGL(col_finalize_kernel, fin_grid, dim3(256), 0, s,
                       loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(),
                       bias.data_ptr<float>(), Vb.data_ptr<float>(),
                       prev_loss.data_ptr<float>(), cur_loss.data_ptr<float>(),
                       active.data_ptr<int>(), epoch_mask.data_ptr<int>(),
                       n_iter.data_ptr<int>(), max_iter.data_ptr<int>(),
                       lr.data_ptr<float>(), mom.data_ptr<float>(),
                       tol.data_ptr<float>(),
                       fit_ic.data_ptr<unsigned char>(), inv_n, epoch, Bp,
                       want_loss_cur, n_active.data_ptr<int>());
    hipLaunchKernelGGL(update_w_kernel, upd_grid2, dim3(upd_threads), 0, s,
                       W.data_ptr<float>(), V.data_ptr<float>(),
                       Gt.data_ptr<float>(),
                       reinterpret_cast<__bf16*>(Wt.data_ptr()),
                       epoch_mask.data_ptr<int>(), lr.data_ptr<float>(),
                       mom.data_ptr<float>(), l1.data_ptr<float>(),
                       l2.data_ptr<float>(), inv_n, Fp);
  };

  int nf = Bp / 64;   // fragments per wave: 1, 2 or 4
  for (int epoch = 0; epoch < (int)max_epochs; ++epoch) {
    want_loss_cur = (any_tol || epoch == (int)max_epochs - 1) ? 1 : 0;
    if (g_layout == 3) {   // HW-probed fast path: permuted/swizzled LDS
      bool fused = use_fused14 && nf == 4;
      if (fused) {
        long subt = NTp / 64;
        long Ssub = (subt + 255) / 256;
        unsigned nblk = (unsigned)((subt + Ssub - 1) / Ssub);
        auto* fk = flagship_v() >= 18
                       ? (Fp == 256   ? fused_fb18_kernel<4>
                          : Fp == 128 ? fused_fb18_kernel<2>
                                      : fused_fb18_kernel<1>)
                       : (Fp == 256   ? fused_fb14_kernel<4>
                          : Fp == 128 ? fused_fb14_kernel<2>
                                      : fused_fb14_kernel<1>);
        hipLaunchKernelGGL(fk, dim3(nblk), dim3(1024), 0, s, Xp, Xtp,
                           y.data_ptr<float>(), idx.data_ptr<int>(),
                           reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                           bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                           target.data_ptr<int>(), Gt.data_ptr<float>(),
                           loss_sum.data_ptr<float>(),
                           db_sum.data_ptr<float>(), rkp, ckp, (int)nt,
                           (int)NTp, Fp, Bp, want_loss_cur, (int)Ssub,
                           n_rows);
        hipLaunchKernelGGL(col_finalize_kernel, fin_grid, dim3(256), 0, s,
                           loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(),
                           bias.data_ptr<float>(), Vb.data_ptr<float>(),
                           prev_loss.data_ptr<float>(), cur_loss.data_ptr<float>(),
                           active.data_ptr<int>(), epoch_mask.data_ptr<int>(),
                           n_iter.data_ptr<int>(), max_iter.data_ptr<int>(),
                           lr.data_ptr<float>(), mom.data_ptr<float>(),
                           tol.data_ptr<float>(),
                           fit_ic.data_ptr<unsigned char>(), inv_n, epoch, Bp,
                           want_loss_cur, n_active.data_ptr<int>());
        hipLaunchKernelGGL(update_w_kernel, upd_grid2, dim3(upd_threads), 0, s,
                           W.data_ptr<float>(), V.data_ptr<float>(),
                           Gt.data_ptr<float>(),
                           reinterpret_cast<__bf16*>(Wt.data_ptr()),
                           epoch_mask.data_ptr<int>(), lr.data_ptr<float>(),
                           mom.data_ptr<float>(), l1.data_ptr<float>(),
                           l2.data_ptr<float>(), inv_n, Fp);
        HIP_CHECK(hipGetLastError());
        if (check_every > 0 && (epoch + 1) % check_every == 0 &&
            epoch + 1 < max_epochs) {
          int na = n_active.item<int>();
          if (na == 0) break;
          n_active.zero_();
        } else {
          HIP_CHECK(hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s));
        }
        continue;
      }
      if (!weighted && nf == 4 && NTp % 256 == 0 && Fp % 128 == 0) {
        launch_flagship_pair(
            s, Xp, Xtp, y.data_ptr<float>(), idx.data_ptr<int>(),
            reinterpret_cast<const __bf16*>(Wt.data_ptr()),
            bias.data_ptr<float>(), loss_id.data_ptr<int>(),
            target.data_ptr<int>(), reinterpret_cast<__bf16*>(Dt.data_ptr()),
            loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(), rkp, ckp,
            nt, NTp, Fp, Bp, want_loss_cur, Gt.data_ptr<float>(), n_rows,
            nseg, seg_rows);
        hipLaunchKernelGGL(col_finalize_kernel, fin_grid, dim3(256), 0, s,
                           loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(),
                           bias.data_ptr<float>(), Vb.data_ptr<float>(),
                           prev_loss.data_ptr<float>(), cur_loss.data_ptr<float>(),
                           active.data_ptr<int>(), epoch_mask.data_ptr<int>(),
                           n_iter.data_ptr<int>(), max_iter.data_ptr<int>(),
                           lr.data_ptr<float>(), mom.data_ptr<float>(),
                           tol.data_ptr<float>(),
                           fit_ic.data_ptr<unsigned char>(), inv_n, epoch, Bp,
                           want_loss_cur, n_active.data_ptr<int>());
        hipLaunchKernelGGL(update_w_kernel, upd_grid2, dim3(upd_threads), 0, s,
                           W.data_ptr<float>(), V.data_ptr<float>(),
                           Gt.data_ptr<float>(),
                           reinterpret_cast<__bf16*>(Wt.data_ptr()),
                           epoch_mask.data_ptr<int>(), lr.data_ptr<float>(),
                           mom.data_ptr<float>(), l1.data_ptr<float>(),
                           l2.data_ptr<float>(), inv_n, Fp);
      } else if (weighted) switch (nf) {
        case 1:
          launch_epoch(epoch, fwd_d3_kernel<1, 1>, bwd_g3_kernel<1>);
          break;
        case 2:
          launch_epoch(epoch, fwd_d3_kernel<2, 1>, bwd_g3_kernel<2>);
          break;
        default:
          launch_epoch(epoch, fwd_d3_kernel<4, 1>, bwd_g3_kernel<4>);
          break;
      } else switch (nf) {
        case 1: launch_epoch(epoch, fwd_d3_kernel<1>, bwd_g3_kernel<1>); break;
        case 2: launch_epoch(epoch, fwd_d3_kernel<2>, bwd_g3_kernel<2>); break;
        default: launch_epoch(epoch, fwd_d3_kernel<4>, bwd_g3_kernel<4>); break;
      }
      HIP_CHECK(hipGetLastError());
      if (check_every > 0 && (epoch + 1) % check_every == 0 &&
          epoch + 1 < max_epochs) {
        int na = n_active.item<int>();
        if (na == 0) break;
        n_active.zero_();
      } else {
        HIP_CHECK(hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s));
      }
      continue;
    }
    if (weighted) switch (g_layout * 4 + (nf == 4 ? 2 : nf - 1)) {
      case 0:  launch_epoch(epoch, fwd_d2_kernel<0, 1, 1>, bwd_g2_kernel<0, 1>); break;
      case 1:  launch_epoch(epoch, fwd_d2_kernel<0, 2, 1>, bwd_g2_kernel<0, 2>); break;
      case 2:  launch_epoch(epoch, fwd_d2_kernel<0, 4, 1>, bwd_g2_kernel<0, 4>); break;
      case 4:  launch_epoch(epoch, fwd_d2_kernel<1, 1, 1>, bwd_g2_kernel<1, 1>); break;
      case 5:  launch_epoch(epoch, fwd_d2_kernel<1, 2, 1>, bwd_g2_kernel<1, 2>); break;
      case 6:  launch_epoch(epoch, fwd_d2_kernel<1, 4, 1>, bwd_g2_kernel<1, 4>); break;
      case 8:  launch_epoch(epoch, fwd_d2_kernel<2, 1, 1>, bwd_g2_kernel<2, 1>); break;
      case 9:  launch_epoch(epoch, fwd_d2_kernel<2, 2, 1>, bwd_g2_kernel<2, 2>); break;
      case 10: launch_epoch(epoch, fwd_d2_kernel<2, 4, 1>, bwd_g2_kernel<2, 4>); break;
      case 12: launch_epoch(epoch, fwd_d2_kernel<3, 1, 1>, bwd_g2_kernel<3, 1>); break;
      case 13: launch_epoch(epoch, fwd_d2_kernel<3, 2, 1>, bwd_g2_kernel<3, 2>); break;
      default: launch_epoch(epoch, fwd_d2_kernel<3, 4, 1>, bwd_g2_kernel<3, 4>); break;
    } else switch (g_layout * 4 + (nf == 4 ? 2 : nf - 1)) {
      case 0:  launch_epoch(epoch, fwd_d2_kernel<0, 1>, bwd_g2_kernel<0, 1>); break;
      case 1:  launch_epoch(epoch, fwd_d2_kernel<0, 2>, bwd_g2_kernel<0, 2>); break;
      case 2:  launch_epoch(epoch, fwd_d2_kernel<0, 4>, bwd_g2_kernel<0, 4>); break;
      case 4:  launch_epoch(epoch, fwd_d2_kernel<1, 1>, bwd_g2_kernel<1, 1>); break;
      case 5:  launch_epoch(epoch, fwd_d2_kernel<1, 2>, bwd_g2_kernel<1, 2>); break;
      case 6:  launch_epoch(epoch, fwd_d2_kernel<1, 4>, bwd_g2_kernel<1, 4>); break;
      case 8:  launch_epoch(epoch, fwd_d2_kernel<2, 1>, bwd_g2_kernel<2, 1>); break;
      case 9:  launch_epoch(epoch, fwd_d2_kernel<2, 2>, bwd_g2_kernel<2, 2>); break;
      case 10: launch_epoch(epoch, fwd_d2_kernel<2, 4>, bwd_g2_kernel<2, 4>); break;
      case 12: launch_epoch(epoch, fwd_d2_kernel<3, 1>, bwd_g2_kernel<3, 1>); break;
      case 13: launch_epoch(epoch, fwd_d2_kernel<3, 2>, bwd_g2_kernel<3, 2>); break;
      default: launch_epoch(epoch, fwd_d2_kernel<3, 4>, bwd_g2_kernel<3, 4>); break;
    }
    HIP_CHECK(hipGetLastError());
    if (check_every > 0 && (epoch + 1) % check_every == 0 &&
        epoch + 1 < max_epochs) {
      int na = n_active.item<int>();   // syncs the stream
      if (na == 0) break;
      n_active.zero_();
    } else {
      // zero without sync: n_active is recomputed every finalize
      hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s);
    }
  }
  return {W, bias, n_iter, cur_loss, Wt};
}

// linear_scores: per-candidate sums; host finalizes means/r2.
torch::Tensor linear_scores(torch::Tensor X, torch::Tensor y,
                            torch::Tensor idx, torch::Tensor Wt_bf16,
                            torch::Tensor bias, torch::Tensor loss_id,
                            torch::Tensor target, int64_t C, int64_t metric,
                            int64_t n_cand) {
  TORCH_CHECK(g_layout >= 0, "MFMA layout not probed");
  const at::cuda::CUDAGuard guard(X.device());
  int Fp = (int)X.size(1);
  int Bp = (int)Wt_bf16.size(0);
  TORCH_CHECK(Bp == 64 || Bp == 128 || Bp == 256,
              "scores kernel supports Bp in {64,128,256}");
  TORCH_CHECK(idx.dtype() == torch::kInt64);
  long n_idx = idx.size(0);
  auto out = torch::zeros({n_cand}, X.options().dtype(torch::kFloat64));

  size_t scand_pad = ((size_t)n_cand + 3) & ~(size_t)3;
  size_t smem = 32 * 8 + 32 * (Bp + 8) * 4 + scand_pad * 4 +
                32 * 72 * 2 + (size_t)Bp * 72 * 2;
  dim3 grid((unsigned)((n_idx + 31) / 32));
  hipStream_t s = cur_stream();

  auto launch = [&](auto k) {
    HIP_CHECK(hipFuncSetAttribute(
        reinterpret_cast<const void*>(k),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    hipLaunchKernelGGL(k, grid, dim3(256), smem, s,
                       reinterpret_cast<const __bf16*>(X.data_ptr()),
                       y.data_ptr<float>(), idx.data_ptr<long>(),
                       reinterpret_cast<const __bf16*>(Wt_bf16.data_ptr()),
                       bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                       target.data_ptr<int>(), (int)C, (int)metric, n_idx,
                       Fp, Bp, (int)n_cand, out.data_ptr<double>());
  };
  size_t smem3 = 32 * 8 + 32 * (Bp + 8) * 4 + scand_pad * 4 +
                 32 * 64 * 2 + (size_t)Bp * 64 * 2;
  auto launch3 = [&](auto k) {
    HIP_CHECK(hipFuncSetAttribute(
        reinterpret_cast<const void*>(k),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem3));
    hipLaunchKernelGGL(k, grid, dim3(256), smem3, s,
                       reinterpret_cast<const __bf16*>(X.data_ptr()),
                       y.data_ptr<float>(), idx.data_ptr<long>(),
                       reinterpret_cast<const __bf16*>(Wt_bf16.data_ptr()),
                       bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                       target.data_ptr<int>(), (int)C, (int)metric, n_idx,
                       Fp, Bp, (int)n_cand, out.data_ptr<double>());
  };
  int nf = Bp / 64;
  if (g_layout == 3) {
    if (C > 1 && Bp == 256 && n_idx >= 4096 && Fp % 128 == 0) {
      // wide multiclass tile (z chunk through the retired staging LDS)
      hipLaunchKernelGGL(scores8_kernel,
                         dim3((unsigned)((n_idx + 255) / 256)), dim3(1024),
                         0, s,
                         reinterpret_cast<const __bf16*>(X.data_ptr()),
                         y.data_ptr<float>(), idx.data_ptr<long>(),
                         reinterpret_cast<const __bf16*>(
                             Wt_bf16.data_ptr()),
                         bias.data_ptr<float>(), (int)C, (int)metric,
                         n_idx, Fp, Bp, (int)n_cand,
                         out.data_ptr<double>());
      HIP_CHECK(hipGetLastError());
      return out;
    }
    if (C == 1 && Bp == 256 && n_idx >= 4096 && Fp % 128 == 0) {
      // wide tile: 8x less W traffic than the 32-row scores3 blocks
      hipLaunchKernelGGL(scores7_kernel,
                         dim3((unsigned)((n_idx + 255) / 256)), dim3(1024),
                         0, s,
                         reinterpret_cast<const __bf16*>(X.data_ptr()),
                         y.data_ptr<float>(), idx.data_ptr<long>(),
                         reinterpret_cast<const __bf16*>(
                             Wt_bf16.data_ptr()),
                         bias.data_ptr<float>(), (int)metric, n_idx, Fp,
                         Bp, (int)n_cand, out.data_ptr<double>());
      HIP_CHECK(hipGetLastError());
      return out;
    }
    switch (nf) {
      case 1: launch3(scores3_kernel<1>); break;
      case 2: launch3(scores3_kernel<2>); break;
      default: launch3(scores3_kernel<4>); break;
    }
    HIP_CHECK(hipGetLastError());
    return out;
  }
  switch (g_layout * 4 + (nf == 4 ? 2 : nf - 1)) {
    case 0:  launch(scores_kernel<0, 1>); break;
    case 1:  launch(scores_kernel<0, 2>); break;
    case 2:  launch(scores_kernel<0, 4>); break;
    case 4:  launch(scores_kernel<1, 1>); break;
    case 5:  launch(scores_kernel<1, 2>); break;
    case 6:  launch(scores_kernel<1, 4>); break;
    case 8:  launch(scores_kernel<2, 1>); break;
    case 9:  launch(scores_kernel<2, 2>); break;
    case 10: launch(scores_kernel<2, 4>); break;
    case 12: launch(scores_kernel<3, 1>); break;
    case 13: launch(scores_kernel<3, 2>); break;
    default: launch(scores_kernel<3, 4>); break;
  }
  HIP_CHECK(hipGetLastError());
  return out;
}


// ---------------------------------------------------------------------------
// KMeans host wrappers
// ---------------------------------------------------------------------------

static void launch_kmeans_assign(const __bf16* X, const int* idx,
                                 const __bf16* Ct, const float* cnorm,
                                 const float* xnorm, const int* cstart,
                                 unsigned char* labels, float* inertia,
                                 float* counts, int nt, int NTp, int Fp,
                                 int Kp, int nb, int want_labels,
                                 hipStream_t s,
                                 const float* w = nullptr) {
  if (Kp <= 128 && NTp % 128 == 0) {
    size_t wsm = (size_t)128 * (Kp + 8) * 4 + 256 * 4 + (size_t)Kp * 4 +
                 128 * 4 + (size_t)128 * 64 * 2 + (size_t)Kp * 64 * 2;
    dim3 wgrid((unsigned)(NTp / 128));
    auto gow = [&](auto k) {
      HIP_CHECK(hipFuncSetAttribute(
          reinterpret_cast<const void*>(k),
          hipFuncAttributeMaxDynamicSharedMemorySize, (int)wsm));
      hipLaunchKernelGGL(k, wgrid, dim3(512), wsm, s, X, idx, Ct, cnorm,
                         xnorm, cstart, labels, inertia, counts, nt, NTp,
                         Fp, Kp, nb, want_labels, w);
    };
    if (Kp == 64) gow(kmeans_assign_w_kernel<1>);
    else gow(kmeans_assign_w_kernel<2>);
    HIP_CHECK(hipGetLastError());
    return;
  }
  size_t smem = (size_t)32 * (Kp + 8) * 4 + 256 * 4 + (size_t)Kp * 4 +
                32 * 4 + (size_t)32 * 64 * 2 + (size_t)Kp * 64 * 2;
  dim3 grid((unsigned)(NTp / 32));
  auto go = [&](auto k) {
    HIP_CHECK(hipFuncSetAttribute(
        reinterpret_cast<const void*>(k),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    hipLaunchKernelGGL(k, grid, dim3(256), smem, s, X, idx, Ct, cnorm,
                       xnorm, cstart, labels, inertia, counts, nt, NTp,
                       Fp, Kp, nb, want_labels, w);
  };
  switch (Kp / 64) {
    case 1: go(kmeans_assign_kernel<1>); break;
    case 2: go(kmeans_assign_kernel<2>); break;
    case 3: go(kmeans_assign_kernel<3>); break;
    default: go(kmeans_assign_kernel<4>); break;
  }
  HIP_CHECK(hipGetLastError());
}

// Full Lloyd loop on device.  Returns (C [Kp][Fp] f32, n_iter [nb],
// inertia_final [nb] f32, Ct bf16, cnorm f32) -- Ct/cnorm stay resident for
// the scores pass.
std::vector<torch::Tensor> kmeans_fit(
    torch::Tensor X, torch::Tensor Xt, torch::Tensor idx, torch::Tensor C0,
    torch::Tensor cstart, torch::Tensor cen_block, torch::Tensor max_iter,
    torch::Tensor tol, torch::Tensor xnorm, int64_t nt, int64_t max_epochs,
    int64_t check_every, torch::Tensor sw) {
  TORCH_CHECK(g_layout == 3,
              "kmeans kernels require the probed layout P=3 (MI355X)");
  // sample_weight [n_rows] (bf16-representable values, engine-normalized):
  // weighted counts/sums/inertia; assignment is weight-free
  const float* wp = nullptr;
  if (sw.numel() > 0) {
    TORCH_CHECK(sw.dtype() == torch::kFloat32 && sw.size(0) == X.size(0));
    wp = sw.data_ptr<float>();
  }
  const at::cuda::CUDAGuard guard(X.device());
  int Fp = (int)X.size(1);
  int Kp = (int)C0.size(0);
  int nb = (int)max_iter.size(0);
  long NTp = idx.size(0);
  TORCH_CHECK(Kp % 64 == 0 && Kp <= 256);
  TORCH_CHECK(NTp % 32 == 0);
  TORCH_CHECK(C0.dtype() == torch::kFloat32 && C0.size(1) == Fp);

  auto optF = X.options().dtype(torch::kFloat32);
  auto optI = X.options().dtype(torch::kInt32);
  auto C = C0.clone();
  auto Ct = torch::empty({Kp, Fp}, X.options());
  auto cnorm = torch::empty({Kp}, optF);
  auto sums = torch::zeros({Kp, Fp}, optF);
  auto counts = torch::zeros({Kp}, optF);
  auto labels = torch::zeros({(long)nb, NTp},
                             X.options().dtype(torch::kUInt8));
  auto shift2 = torch::zeros({nb + 1}, optF);
  auto active = torch::ones({nb + 1}, optI);
  active[nb] = 0;
  auto n_iter = torch::zeros({nb}, optI);
  auto inertia = torch::zeros({nb}, optF);
  auto n_active = torch::zeros({1}, optI);

  hipStream_t s = cur_stream();
  const __bf16* Xp = reinterpret_cast<const __bf16*>(X.data_ptr());
  const __bf16* Xtp = reinterpret_cast<const __bf16*>(Xt.data_ptr());
  long n_rows = X.size(0);
  auto Dhot = torch::zeros({Kp, NTp}, X.options());

  // init pass: counts==0 everywhere -> keeps C, fills Ct + cnorm
  hipLaunchKernelGGL(kmeans_center_kernel, dim3(Kp), dim3(256), 0, s,
                     C.data_ptr<float>(),
                     reinterpret_cast<__bf16*>(Ct.data_ptr()),
                     cnorm.data_ptr<float>(), sums.data_ptr<float>(),
                     counts.data_ptr<float>(), cen_block.data_ptr<int>(),
                     active.data_ptr<int>(), shift2.data_ptr<float>(),
                     Fp, Kp);

  // split-K geometry for the sums GEMM (bwd_g3 generic tiles)
  int ftiles = Fp / 64;
  long rtiles = NTp / 64;
  long want_nseg = std::max<long>(1, 1024 / ftiles);
  long seg_tiles = std::max<long>(1, (rtiles + want_nseg - 1) / want_nseg);
  long nseg = (rtiles + seg_tiles - 1) / seg_tiles;
  int seg_rows = (int)(seg_tiles * 64);
  int onehot_blocks = (int)std::min<long>((nt + 255) / 256, 2048);

  for (int epoch = 0; epoch < (int)max_epochs; ++epoch) {
    HIP_CHECK(hipMemsetAsync(inertia.data_ptr(), 0, nb * sizeof(float), s));
    launch_kmeans_assign(Xp, idx.data_ptr<int>(),
                         reinterpret_cast<const __bf16*>(Ct.data_ptr()),
                         cnorm.data_ptr<float>(), xnorm.data_ptr<float>(),
                         cstart.data_ptr<int>(),
                         labels.data_ptr<unsigned char>(),
                         inertia.data_ptr<float>(),
                         counts.data_ptr<float>(), (int)nt, (int)NTp, Fp,
                         Kp, nb, 1, s, wp);
    // sums = X^T . onehot(labels): the same MFMA bwd kernel as the
    // linear family (one-hot rows are exact in bf16)
    HIP_CHECK(hipMemsetAsync(Dhot.data_ptr(), 0,
                             (size_t)Kp * NTp * 2, s));
    hipLaunchKernelGGL(kmeans_onehot_kernel, dim3(onehot_blocks),
                       dim3(256), 0, s, labels.data_ptr<unsigned char>(),
                       cstart.data_ptr<int>(),
                       reinterpret_cast<__bf16*>(Dhot.data_ptr()), nt,
                       (long)NTp, nb, idx.data_ptr<int>(), wp);
    switch (Kp / 64) {
      case 1:
        hipLaunchKernelGGL(bwd_g3_kernel<1>, dim3(ftiles, (unsigned)nseg),
                           dim3(256), 0, s, Xtp, idx.data_ptr<int>(),
                           reinterpret_cast<const __bf16*>(Dhot.data_ptr()),
                           sums.data_ptr<float>(), n_rows, (int)NTp, Fp,
                           Kp, seg_rows);
        break;
      case 2:
        hipLaunchKernelGGL(bwd_g3_kernel<2>, dim3(ftiles, (unsigned)nseg),
                           dim3(256), 0, s, Xtp, idx.data_ptr<int>(),
                           reinterpret_cast<const __bf16*>(Dhot.data_ptr()),
                           sums.data_ptr<float>(), n_rows, (int)NTp, Fp,
                           Kp, seg_rows);
        break;
      case 3:
        hipLaunchKernelGGL(bwd_g3_kernel<3>, dim3(ftiles, (unsigned)nseg),
                           dim3(256), 0, s, Xtp, idx.data_ptr<int>(),
                           reinterpret_cast<const __bf16*>(Dhot.data_ptr()),
                           sums.data_ptr<float>(), n_rows, (int)NTp, Fp,
                           Kp, seg_rows);
        break;
      default:
        hipLaunchKernelGGL(bwd_g3_kernel<4>, dim3(ftiles, (unsigned)nseg),
                           dim3(256), 0, s, Xtp, idx.data_ptr<int>(),
                           reinterpret_cast<const __bf16*>(Dhot.data_ptr()),
                           sums.data_ptr<float>(), n_rows, (int)NTp, Fp,
                           Kp, seg_rows);
        break;
    }
    hipLaunchKernelGGL(kmeans_center_kernel, dim3(Kp), dim3(256), 0, s,
                       C.data_ptr<float>(),
                       reinterpret_cast<__bf16*>(Ct.data_ptr()),
                       cnorm.data_ptr<float>(), sums.data_ptr<float>(),
                       counts.data_ptr<float>(), cen_block.data_ptr<int>(),
                       active.data_ptr<int>(), shift2.data_ptr<float>(),
                       Fp, Kp);
    hipLaunchKernelGGL(kmeans_block_finalize_kernel,
                       dim3((nb + 255) / 256), dim3(256), 0, s,
                       shift2.data_ptr<float>(), active.data_ptr<int>(),
                       n_iter.data_ptr<int>(), max_iter.data_ptr<int>(),
                       tol.data_ptr<float>(), epoch, nb,
                       n_active.data_ptr<int>());
    HIP_CHECK(hipGetLastError());
    if (check_every > 0 && (epoch + 1) % check_every == 0 &&
        epoch + 1 < max_epochs) {
      int na = n_active.item<int>();
      if (na == 0) break;
      n_active.zero_();
    } else {
      HIP_CHECK(hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s));
    }
  }
  // final inertia under the final centers
  HIP_CHECK(hipMemsetAsync(inertia.data_ptr(), 0, nb * sizeof(float), s));
  launch_kmeans_assign(Xp, idx.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(Ct.data_ptr()),
                       cnorm.data_ptr<float>(), xnorm.data_ptr<float>(),
                       cstart.data_ptr<int>(),
                       labels.data_ptr<unsigned char>(),
                       inertia.data_ptr<float>(), nullptr, (int)nt,
                       (int)NTp, Fp, Kp, nb, 1, s, wp);
  return {C, n_iter, inertia, Ct, cnorm, labels};
}

// assignment / inertia of arbitrary rows under given centers (scores +
// labels_ paths)
std::vector<torch::Tensor> kmeans_assign(
    torch::Tensor X, torch::Tensor idx, torch::Tensor Ct,
    torch::Tensor cnorm, torch::Tensor xnorm, torch::Tensor cstart,
    int64_t nt, int64_t want_labels) {
  TORCH_CHECK(g_layout == 3, "kmeans kernels require layout P=3");
  const at::cuda::CUDAGuard guard(X.device());
  int Fp = (int)X.size(1);
  int Kp = (int)Ct.size(0);
  int nb = (int)cstart.size(0) - 1;
  long NTp = idx.size(0);
  auto labels = torch::zeros({(long)nb, NTp},
                             X.options().dtype(torch::kUInt8));
  auto inertia = torch::zeros({nb}, X.options().dtype(torch::kFloat32));
  launch_kmeans_assign(
      reinterpret_cast<const __bf16*>(X.data_ptr()), idx.data_ptr<int>(),
      reinterpret_cast<const __bf16*>(Ct.data_ptr()),
      cnorm.data_ptr<float>(), xnorm.data_ptr<float>(),
      cstart.data_ptr<int>(), labels.data_ptr<unsigned char>(),
      inertia.data_ptr<float>(), nullptr, (int)nt, (int)NTp, Fp, Kp, nb,
      (int)want_labels, cur_stream());
  return {inertia, labels};
}

torch::Tensor row_norms(torch::Tensor X) {
  const at::cuda::CUDAGuard guard(X.device());
  long n = X.size(0);
  int Fp = (int)X.size(1);
  auto out = torch::empty({n}, X.options().dtype(torch::kFloat32));
  int blocks = (int)std::min<long>((n + 255) / 256, 2048);
  hipLaunchKernelGGL(row_norms_kernel, dim3(blocks), dim3(256), 0,
                     cur_stream(),
                     reinterpret_cast<const __bf16*>(X.data_ptr()), n, Fp,
                     out.data_ptr<float>());
  HIP_CHECK(hipGetLastError());
  return out;
}


// ---------------------------------------------------------------------------
// GBT host wrappers
// ---------------------------------------------------------------------------

// One full boosting fit on device.  Returns (feats [T][NN] i32,
// thrs [T][NN] i32, vals [T][NN] f32).
torch::Tensor gbt_bin(torch::Tensor X, torch::Tensor edges,
                      torch::Tensor ecnt) {
  const at::cuda::CUDAGuard guard(X.device());
  TORCH_CHECK(X.is_contiguous() && X.dtype() == torch::kFloat32);
  long n = X.size(0), F = X.size(1);
  auto Xb = torch::empty({n, F}, X.options().dtype(torch::kUInt8));
  long total = n * F;
  hipStream_t s = cur_stream();
  int blocks = (int)std::min<long>((total + 255) / 256, 4096);
  hipLaunchKernelGGL(gbt_bin_kernel, dim3(blocks), dim3(256), 0, s,
                     X.data_ptr<float>(), edges.data_ptr<float>(),
                     ecnt.data_ptr<int>(),
                     Xb.data_ptr<unsigned char>(), total, (int)F);
  HIP_CHECK(hipGetLastError());
  return Xb;
}

std::vector<torch::Tensor> gbt_fit(torch::Tensor Xb, torch::Tensor Xbt,
                                   torch::Tensor idxmap,
                                   torch::Tensor y_tr, int64_t loss,
                                   int64_t n_estimators, double lrate,
                                   int64_t max_depth, int64_t min_leaf,
                                   double lam, double f0,
                                   torch::Tensor sw) {
  const at::cuda::CUDAGuard guard(Xb.device());
  TORCH_CHECK(Xb.dtype() == torch::kUInt8 && Xb.dim() == 2);
  TORCH_CHECK(max_depth >= 1 && max_depth <= 10,
              "device GBT supports max_depth in [1, 10]");
  // sample_weight (fold-sliced [nt], engine-normalized): scales g and h
  // in the grad kernel; the packed/deterministic histogram modes assume
  // unweighted gradient bounds and are disabled under weighting
  const bool weighted = sw.numel() > 0;
  const float* wp = nullptr;
  float wmax = 1.f;
  if (weighted) {
    TORCH_CHECK(sw.dtype() == torch::kFloat32 &&
                sw.size(0) == idxmap.size(0));
    wp = sw.data_ptr<float>();
    wmax = sw.max().item<float>();
  }
  int F = (int)Xb.size(1);
  long nt = idxmap.size(0);
  int T = (int)n_estimators;
  int NN = (1 << (max_depth + 1)) - 1;

  auto optF = y_tr.options().dtype(torch::kFloat32);
  auto optI = y_tr.options().dtype(torch::kInt32);
  auto raw = torch::full({nt}, f0, optF);
  auto g = torch::empty({nt}, optF);
  auto h = torch::empty({nt}, optF);
  auto node_id = torch::zeros({nt}, optI);
  auto feats = torch::full({(long)T, NN}, -1,
                           optI);
  auto thrs = torch::zeros({(long)T, NN}, optI);
  auto vals = torch::zeros({(long)T, NN}, optF);
  int max_lvl_nodes = 1 << (max_depth - 1);
  auto hist = torch::empty({(long)max_lvl_nodes * F * 256 * 3}, optF);
  auto hist_prev = torch::empty({(long)std::max(1, max_lvl_nodes / 2) *
                                 F * 256 * 3}, optF);
  auto gsum = torch::zeros({NN}, optF);
  auto hsum = torch::zeros({NN}, optF);

  hipStream_t s = cur_stream();
  const unsigned char* Xp = Xb.data_ptr<unsigned char>();
  TORCH_CHECK(Xbt.dtype() == torch::kUInt8 && Xbt.size(0) == Xb.size(1) &&
              Xbt.size(1) == Xb.size(0) && Xbt.stride(1) == 1);
  const unsigned char* Xtp = Xbt.data_ptr<unsigned char>();
  long n_rows = Xb.size(0);
  int blocks = (int)std::min<long>((nt + 255) / 256, 2048);
  // deterministic squared loss: g is unbounded, so each round measures
  // max|g| (bit-level atomicMax, order-independent) to set the
  // fixed-point bias/scale; the one host sync per round is the price of
  // the opt-in mode
  bool det_sq = det_gbt_mode() && loss == LOSS_SQUARED && !weighted;
  auto gmax_bits = torch::zeros({1}, optI);
  float gbias_r = 1.f;

  for (int t = 0; t < T; ++t) {
    int* feat_t = feats.data_ptr<int>() + (long)t * NN;
    int* thr_t = thrs.data_ptr<int>() + (long)t * NN;
    float* val_t = vals.data_ptr<float>() + (long)t * NN;
    hipLaunchKernelGGL(gbt_grad_kernel, dim3(blocks), dim3(256), 0, s,
                       raw.data_ptr<float>(), y_tr.data_ptr<float>(),
                       g.data_ptr<float>(), h.data_ptr<float>(), nt,
                       (int)loss, wp);
    if (det_sq) {
      HIP_CHECK(hipMemsetAsync(gmax_bits.data_ptr(), 0, 4, s));
      hipLaunchKernelGGL(absmax_kernel, dim3(blocks), dim3(256), 0, s,
                         g.data_ptr<float>(), nt,
                         reinterpret_cast<unsigned*>(
                             gmax_bits.data_ptr<int>()));
      int bits = gmax_bits.item<int>();            // syncs the stream
      float gm;
      memcpy(&gm, &bits, 4);
      gbias_r = std::max(gm, 1e-3f);
    }
    for (int d = 0; d < (int)max_depth; ++d) {
      int lvl_lo = (1 << d) - 1;
      int lvl_nodes = 1 << d;
      int even_only = (d > 0) ? 1 : 0;    // sibling subtraction
      launch_hist_level(Xtp, idxmap.data_ptr<int>(),
                        node_id.data_ptr<int>(), g.data_ptr<float>(),
                        h.data_ptr<float>(), hist.data_ptr<float>(), nt, n_rows,
                        F, d,
                        ((loss == LOSS_LOGISTIC) ? 0.25f : 1.f) * wmax,
                        (loss == LOSS_LOGISTIC && !weighted) || det_sq,
                        false, s, 1, 0, 0, det_sq ? gbias_r : 1.f);
      if (even_only) {
        int prev_lo = (1 << (d - 1)) - 1;
        long cells = (long)F * 256 * 3;
        unsigned gx = (unsigned)std::min<long>((cells + 255) / 256, 1024);
        hipLaunchKernelGGL(gbt_sibling_kernel,
                           dim3(gx, (unsigned)(lvl_nodes / 2)), dim3(256),
                           0, s, hist_prev.data_ptr<float>(),
                           hist.data_ptr<float>(), feat_t, prev_lo, F,
                           lvl_nodes);
      }
      hipLaunchKernelGGL(gbt_split_find_kernel, dim3(lvl_nodes), dim3(256),
                         0, s, hist.data_ptr<float>(), F, lvl_lo,
                         (float)lam, (float)lrate, (int)min_leaf, 0,
                         feat_t, thr_t, val_t, 1 << 30, 0u, 0);
      if (d + 1 < (int)max_depth)
        hist_prev.narrow(0, 0, (long)lvl_nodes * F * 256 * 3)
            .copy_(hist.narrow(0, 0, (long)lvl_nodes * F * 256 * 3),
                   /*non_blocking=*/true);
      hipLaunchKernelGGL(gbt_split_apply_kernel, dim3(blocks), dim3(256),
                         0, s, Xp, idxmap.data_ptr<int>(),
                         node_id.data_ptr<int>(), feat_t, thr_t, nt, F,
                         lvl_lo, lvl_lo + lvl_nodes);
      HIP_CHECK(hipGetLastError());
    }
    // bottom-level leaves
    int bl_lo = (1 << max_depth) - 1;
    HIP_CHECK(hipMemsetAsync(gsum.data_ptr(), 0, NN * 4, s));
    HIP_CHECK(hipMemsetAsync(hsum.data_ptr(), 0, NN * 4, s));
    {
      bool fix = det_gbt_mode() && !weighted &&
                 (loss == LOSS_LOGISTIC || loss == LOSS_SQUARED);
      float gb = det_sq ? gbias_r : 1.f;
      float fsc = fix ? det_fix_scale(nt, gb) : 0.f;
      hipLaunchKernelGGL(gbt_node_sums_kernel,
                         dim3(fix ? 1 : blocks,
                              (unsigned)(((NN - bl_lo) + 127) / 128)), dim3(256), 0, s,
                         node_id.data_ptr<int>(), g.data_ptr<float>(),
                         h.data_ptr<float>(), gsum.data_ptr<float>(),
                         hsum.data_ptr<float>(), nt, bl_lo, NN, fsc, fsc,
                         gb);
    }
    hipLaunchKernelGGL(gbt_leaf_vals_kernel,
                       dim3(((NN - bl_lo) + 255) / 256), dim3(256), 0, s,
                       gsum.data_ptr<float>(), hsum.data_ptr<float>(),
                       val_t, feat_t, (float)lam, (float)lrate, bl_lo, NN);
    hipLaunchKernelGGL(gbt_leaf_apply_kernel, dim3(blocks), dim3(256), 0, s,
                       raw.data_ptr<float>(), node_id.data_ptr<int>(),
                       val_t, nt);
    HIP_CHECK(hipGetLastError());
  }
  return {feats, thrs, vals};
}

torch::Tensor gbt_predict(torch::Tensor Xb, torch::Tensor idx,
                          torch::Tensor feats, torch::Tensor thrs,
                          torch::Tensor vals, double f0) {
  const at::cuda::CUDAGuard guard(Xb.device());
  int T = (int)feats.size(0);
  int NN = (int)feats.size(1);
  int F = (int)Xb.size(1);
  long n_idx = idx.size(0);
  auto out = torch::empty({n_idx},
                          vals.options().dtype(torch::kFloat32));
  int blocks = (int)std::min<long>((n_idx + 255) / 256, 2048);
  hipLaunchKernelGGL(gbt_predict_kernel, dim3(blocks), dim3(256), 0,
                     cur_stream(), Xb.data_ptr<unsigned char>(),
                     idx.data_ptr<int>(), feats.data_ptr<int>(),
                     thrs.data_ptr<int>(), vals.data_ptr<float>(), T, NN,
                     F, n_idx, (float)f0, out.data_ptr<float>());
  HIP_CHECK(hipGetLastError());
  return out;
}

torch::Tensor gbt_predict_multi(torch::Tensor Xb, torch::Tensor idx,
                                torch::Tensor feats, torch::Tensor thrs,
                                torch::Tensor vals, int64_t K,
                                torch::Tensor f0s) {
  const at::cuda::CUDAGuard guard(Xb.device());
  TORCH_CHECK(f0s.size(0) == K && f0s.dtype() == torch::kFloat32);
  int T = (int)(feats.size(0) / K);
  int NN = (int)feats.size(1);
  int F = (int)Xb.size(1);
  long n_idx = idx.size(0);
  auto out = torch::empty({(long)K, n_idx},
                          vals.options().dtype(torch::kFloat32));
  int blocks = (int)std::min<long>((n_idx + 255) / 256, 2048);
  hipLaunchKernelGGL(gbt_predict_multi_kernel,
                     dim3(blocks, (unsigned)K), dim3(256), 0,
                     cur_stream(), Xb.data_ptr<unsigned char>(),
                     idx.data_ptr<int>(), feats.data_ptr<int>(),
                     thrs.data_ptr<int>(), vals.data_ptr<float>(), T,
                     (int)K, NN, F, n_idx, f0s.data_ptr<float>(),
                     out.data_ptr<float>());
  HIP_CHECK(hipGetLastError());
  return out;
}

torch::Tensor gbt_metric(torch::Tensor raw, torch::Tensor y,
                         torch::Tensor idx, int64_t metric) {
  const at::cuda::CUDAGuard guard(raw.device());
  long n_idx = idx.size(0);
  auto out = torch::zeros({1}, raw.options().dtype(torch::kFloat64));
  int blocks = (int)std::min<long>((n_idx + 255) / 256, 2048);
  hipLaunchKernelGGL(gbt_metric_kernel, dim3(blocks), dim3(256), 0,
                     cur_stream(), raw.data_ptr<float>(),
                     y.data_ptr<float>(), idx.data_ptr<int>(), n_idx,
                     (int)metric, out.data_ptr<double>());
  HIP_CHECK(hipGetLastError());
  return out;
}


// ---------------------------------------------------------------------------
// linear_search_run: the whole (fold x candidate-chunk) loop natively.
//
// One call executes an entire search shard on the device -- for each fold:
// for each 256-column candidate chunk: reset state, run the epoch loop
// (fwd/bwd/finalize/update), then score the test (and optionally train)
// fold -- with NO host synchronization between batches.  Per-(fold, chunk)
// fit/score times come from HIP events and populate cv_results_'s
// *_fit_time / *_score_time.  This is the C++ engine core of SURVEY.md
// section 7.1 (the Python layer builds plans and assembles cv_results_).
//
// Requirements: Bp_total % 256 == 0 (pad with max_iter=0 dummy columns),
// layout P=3 (probed), candidate chunks aligned to candidate boundaries.
// Returns {test_sums [n_folds][n_cand], train_sums or empty,
//          fit_ms [n_folds][n_chunks], score_ms [n_folds][n_chunks],
//          n_iter [n_folds][Bp_total]}.
// ---------------------------------------------------------------------------
std::vector<torch::Tensor> linear_search_run(
    torch::Tensor X, torch::Tensor Xt, torch::Tensor y,
    std::vector<torch::Tensor> train_idx,   // i32 [NTp_f], 256-padded
    std::vector<int64_t> nt_list,
    std::vector<torch::Tensor> test_idx,    // i64 [n_test_f]
    torch::Tensor loss_id, torch::Tensor lr, torch::Tensor l1,
    torch::Tensor l2, torch::Tensor mom, torch::Tensor tol,
    torch::Tensor max_iter, torch::Tensor target, torch::Tensor fit_ic,
    int64_t C, int64_t metric, int64_t n_cand_total,
    int64_t want_train_scores, int64_t check_every) {
  TORCH_CHECK(g_layout == 3, "linear_search_run requires probed layout P=3");
  const at::cuda::CUDAGuard guard(X.device());
  int Fp = (int)X.size(1);
  TORCH_CHECK(Fp % 128 == 0, "Fp must be a multiple of 128");
  long Bt = loss_id.size(0);
  TORCH_CHECK(Bt % 256 == 0, "total columns must be 256-padded");
  int n_chunks = (int)(Bt / 256);
  int n_folds = (int)train_idx.size();
  constexpr int Bp = 256;

  auto optF = X.options().dtype(torch::kFloat32);
  auto optI = X.options().dtype(torch::kInt32);
  long max_NTp = 0;
  for (auto& t : train_idx) max_NTp = std::max(max_NTp, t.size(0));
  auto W = torch::empty({Bp, Fp}, optF);
  auto V = torch::empty({Bp, Fp}, optF);
  auto Gt = torch::zeros({Bp, Fp}, optF);
  auto Wt = torch::empty({Bp, Fp}, X.options());
  // fused v14 epoch kernel keeps D in LDS -- no global D buffer needed
  bool use_fused = (flagship_v() == 14 || flagship_v() >= 18) &&
                   (Fp == 64 || Fp == 128 || Fp == 256);
  auto Dt = torch::empty({(long)Bp, use_fused ? 1L : max_NTp}, X.options());
  auto bias = torch::empty({Bp}, optF);
  auto Vb = torch::empty({Bp}, optF);
  auto loss_sum = torch::zeros({Bp}, optF);
  auto db_sum = torch::zeros({Bp}, optF);
  auto prev_loss = torch::empty({Bp}, optF);
  auto cur_loss = torch::zeros({Bp}, optF);
  auto active = torch::empty({Bp}, optI);
  auto epoch_mask = torch::zeros({Bp}, optI);
  auto n_iter = torch::zeros({(long)n_folds, Bt}, optI);
  auto n_active = torch::zeros({1}, optI);
  auto test_sums = torch::zeros({(long)n_folds, n_cand_total},
                                X.options().dtype(torch::kFloat64));
  auto train_sums = torch::zeros(
      {want_train_scores ? (long)n_folds : 0, n_cand_total},
      X.options().dtype(torch::kFloat64));

  const __bf16* Xp = reinterpret_cast<const __bf16*>(X.data_ptr());
  const __bf16* Xtp = reinterpret_cast<const __bf16*>(Xt.data_ptr());
  long n_rows = X.size(0);
  hipStream_t s = cur_stream();

  // host copies of per-column max_iter/tol for chunk planning (one sync)
  auto mi_cpu = max_iter.cpu();
  auto tol_cpu = tol.cpu();
  const int* mi_h = mi_cpu.data_ptr<int>();
  const float* tol_h = tol_cpu.data_ptr<float>();

  std::vector<hipEvent_t> evs(4 * n_folds * n_chunks);
  for (auto& e : evs) HIP_CHECK(hipEventCreate(&e));
  int cands_per_chunk = 256 / (int)C;

  for (int f = 0; f < n_folds; ++f) {
    long NTp = train_idx[f].size(0);
    long nt = nt_list[f];
    float inv_n = 1.0f / (float)nt;
    dim3 fin_grid(1);
    int upd_threads = Fp >= 256 ? 256 : Fp;
    dim3 upd_grid2((unsigned)(Fp / upd_threads), (unsigned)Bp);
    int ftiles = Fp / 64;
    long rtiles = NTp / 64;
    long want_nseg = std::max<long>(1, 1024 / ftiles);
    long seg_tiles = std::max<long>(1, (rtiles + want_nseg - 1) / want_nseg);
    long nseg = (rtiles + seg_tiles - 1) / seg_tiles;
    int seg_rows = (int)(seg_tiles * 64);
    const int* idxp = train_idx[f].data_ptr<int>();

    for (int c = 0; c < n_chunks; ++c) {
      long off = (long)c * 256;
      int max_ep = 0;
      bool any_tol = false;
      for (int j = 0; j < 256; ++j) {
        max_ep = std::max(max_ep, mi_h[off + j]);
        any_tol = any_tol || tol_h[off + j] > 0.f;
      }
      hipEvent_t ev_f0 = evs[(f * n_chunks + c) * 4 + 0];
      hipEvent_t ev_f1 = evs[(f * n_chunks + c) * 4 + 1];
      hipEvent_t ev_s0 = evs[(f * n_chunks + c) * 4 + 2];
      hipEvent_t ev_s1 = evs[(f * n_chunks + c) * 4 + 3];
      HIP_CHECK(hipEventRecord(ev_f0, s));
      // reset per-chunk fit state
      HIP_CHECK(hipMemsetAsync(W.data_ptr(), 0, (size_t)Bp * Fp * 4, s));
      HIP_CHECK(hipMemsetAsync(V.data_ptr(), 0, (size_t)Bp * Fp * 4, s));
      HIP_CHECK(hipMemsetAsync(Wt.data_ptr(), 0, (size_t)Bp * Fp * 2, s));
      HIP_CHECK(hipMemsetAsync(bias.data_ptr(), 0, Bp * 4, s));
      HIP_CHECK(hipMemsetAsync(Vb.data_ptr(), 0, Bp * 4, s));
      prev_loss.fill_(3.0e38f);
      active.fill_(1);

      const int* loss_p = loss_id.data_ptr<int>() + off;
      const float* lr_p = lr.data_ptr<float>() + off;
      const float* l1_p = l1.data_ptr<float>() + off;
      const float* l2_p = l2.data_ptr<float>() + off;
      const float* mom_p = mom.data_ptr<float>() + off;
      const float* tol_p = tol.data_ptr<float>() + off;
      const int* mi_p = max_iter.data_ptr<int>() + off;
      const int* tgt_p = target.data_ptr<int>() + off;
      const unsigned char* ic_p =
          fit_ic.data_ptr<unsigned char>() + off;
      int* ni_p = n_iter.data_ptr<int>() + (long)f * Bt + off;

      bool fused = use_fused && NTp % 256 == 0;
      long subt = NTp / 64;
      long Ssub = (subt + 255) / 256;
      unsigned fnblk = (unsigned)((subt + Ssub - 1) / Ssub);
      auto* fk = flagship_v() >= 18
                     ? (Fp == 256   ? fused_fb18_kernel<4>
                        : Fp == 128 ? fused_fb18_kernel<2>
                                    : fused_fb18_kernel<1>)
                     : (Fp == 256   ? fused_fb14_kernel<4>
                        : Fp == 128 ? fused_fb14_kernel<2>
                                    : fused_fb14_kernel<1>);
      for (int epoch = 0; epoch < max_ep; ++epoch) {
        int want_loss = (any_tol || epoch == max_ep - 1) ? 1 : 0;
        if (fused) {
          hipLaunchKernelGGL(fk, dim3(fnblk), dim3(1024), 0, s, Xp, Xtp,
                             y.data_ptr<float>(), idxp,
                             reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                             bias.data_ptr<float>(), loss_p, tgt_p,
                             Gt.data_ptr<float>(),
                             loss_sum.data_ptr<float>(),
                             db_sum.data_ptr<float>(), nullptr, nullptr,
                             (int)nt, (int)NTp, Fp, Bp, want_loss,
                             (int)Ssub, n_rows);
        } else {
          launch_flagship_pair(
              s, Xp, Xtp, y.data_ptr<float>(), idxp,
              reinterpret_cast<const __bf16*>(Wt.data_ptr()),
              bias.data_ptr<float>(), loss_p, tgt_p,
              reinterpret_cast<__bf16*>(Dt.data_ptr()),
              loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(), nullptr,
              nullptr, nt, NTp, Fp, Bp, want_loss, Gt.data_ptr<float>(),
              n_rows, nseg, seg_rows);
        }
        hipLaunchKernelGGL(col_finalize_kernel, fin_grid, dim3(256), 0, s,
                           loss_sum.data_ptr<float>(),
                           db_sum.data_ptr<float>(), bias.data_ptr<float>(),
                           Vb.data_ptr<float>(), prev_loss.data_ptr<float>(),
                           cur_loss.data_ptr<float>(), active.data_ptr<int>(),
                           epoch_mask.data_ptr<int>(), ni_p,
                           mi_p, lr_p, mom_p, tol_p, ic_p, inv_n, epoch, Bp,
                           want_loss, n_active.data_ptr<int>());
        hipLaunchKernelGGL(update_w_kernel, upd_grid2, dim3(upd_threads), 0,
                           s, W.data_ptr<float>(), V.data_ptr<float>(),
                           Gt.data_ptr<float>(),
                           reinterpret_cast<__bf16*>(Wt.data_ptr()),
                           epoch_mask.data_ptr<int>(), lr_p, mom_p, l1_p,
                           l2_p, inv_n, Fp);
        HIP_CHECK(hipGetLastError());
        if (check_every > 0 && (epoch + 1) % check_every == 0 &&
            epoch + 1 < max_ep) {
          int na = n_active.item<int>();
          if (na == 0) break;
          n_active.zero_();
        } else {
          HIP_CHECK(hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s));
        }
      }
      HIP_CHECK(hipEventRecord(ev_f1, s));
      HIP_CHECK(hipEventRecord(ev_s0, s));
      // scores (permuted kernel): test fold, then train if requested
      int n_cand_chunk = std::min<long>(cands_per_chunk,
                                        n_cand_total - (long)c * cands_per_chunk);
      if (n_cand_chunk > 0) {
        long n_t = test_idx[f].size(0);
        size_t scand_pad = ((size_t)n_cand_chunk + 3) & ~(size_t)3;
        size_t smem3 = 32 * 8 + 32 * (Bp + 8) * 4 + scand_pad * 4 +
                       32 * 64 * 2 + (size_t)Bp * 64 * 2;
        bool wide = (C == 1 && Bp == 256 && Fp % 128 == 0);
        bool wide_mc = (C > 1 && Bp == 256 && Fp % 128 == 0);
        auto score_one = [&](torch::Tensor& it, long ni, double* outp) {
          if (wide && ni >= 4096) {
            hipLaunchKernelGGL(scores7_kernel,
                               dim3((unsigned)((ni + 255) / 256)),
                               dim3(1024), 0, s,
                               reinterpret_cast<const __bf16*>(
                                   X.data_ptr()),
                               y.data_ptr<float>(), it.data_ptr<long>(),
                               reinterpret_cast<const __bf16*>(
                                   Wt.data_ptr()),
                               bias.data_ptr<float>(), (int)metric, ni,
                               Fp, Bp, n_cand_chunk, outp);
            return;
          }
          if (wide_mc && ni >= 4096) {
            hipLaunchKernelGGL(scores8_kernel,
                               dim3((unsigned)((ni + 255) / 256)),
                               dim3(1024), 0, s,
                               reinterpret_cast<const __bf16*>(
                                   X.data_ptr()),
                               y.data_ptr<float>(), it.data_ptr<long>(),
                               reinterpret_cast<const __bf16*>(
                                   Wt.data_ptr()),
                               bias.data_ptr<float>(), (int)C,
                               (int)metric, ni, Fp, Bp, n_cand_chunk,
                               outp);
            return;
          }
          HIP_CHECK(hipFuncSetAttribute(
              reinterpret_cast<const void*>(scores3_kernel<4>),
              hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem3));
          hipLaunchKernelGGL(scores3_kernel<4>,
                             dim3((unsigned)((ni + 31) / 32)), dim3(256),
                             smem3, s,
                             reinterpret_cast<const __bf16*>(X.data_ptr()),
                             y.data_ptr<float>(), it.data_ptr<long>(),
                             reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                             bias.data_ptr<float>(), loss_p, tgt_p, (int)C,
                             (int)metric, ni, Fp, Bp, n_cand_chunk, outp);
        };
        score_one(test_idx[f], n_t,
                  test_sums.data_ptr<double>() + (long)f * n_cand_total +
                      (long)c * cands_per_chunk);
        if (want_train_scores) {
          long n_tr = test_idx[n_folds + f].size(0);
          score_one(test_idx[n_folds + f], n_tr,
                    train_sums.data_ptr<double>() +
                        (long)f * n_cand_total +
                        (long)c * cands_per_chunk);
        }
      }
      HIP_CHECK(hipEventRecord(ev_s1, s));
      HIP_CHECK(hipGetLastError());
    }
  }
  HIP_CHECK(hipStreamSynchronize(s));
  auto fit_ms = torch::empty({n_folds, n_chunks},
                             torch::dtype(torch::kFloat32));
  auto score_ms = torch::empty({n_folds, n_chunks},
                               torch::dtype(torch::kFloat32));
  for (int f = 0; f < n_folds; ++f)
    for (int c = 0; c < n_chunks; ++c) {
      float ms;
      HIP_CHECK(hipEventElapsedTime(&ms, evs[(f * n_chunks + c) * 4 + 0],
                                    evs[(f * n_chunks + c) * 4 + 1]));
      fit_ms[f][c] = ms;
      HIP_CHECK(hipEventElapsedTime(&ms, evs[(f * n_chunks + c) * 4 + 2],
                                    evs[(f * n_chunks + c) * 4 + 3]));
      score_ms[f][c] = ms;
    }
  for (auto& e : evs) HIP_CHECK(hipEventDestroy(e));
  // W/bias of the LAST chunk fitted -- debugging/refit aid
  return {test_sums, train_sums, fit_ms, score_ms, n_iter, W, bias};
}


// ---------------------------------------------------------------------------
// K5 host wrappers
// ---------------------------------------------------------------------------

std::vector<torch::Tensor> csr_linear_fit(
    torch::Tensor indptr, torch::Tensor ccols, torch::Tensor vals,
    torch::Tensor tf, torch::Tensor tr, torch::Tensor tv,
    torch::Tensor chunk_off, torch::Tensor inv, torch::Tensor y,
    torch::Tensor idx,   // i32 [nt], exact (no padding)
    torch::Tensor loss_id, torch::Tensor lr, torch::Tensor l1,
    torch::Tensor l2, torch::Tensor mom, torch::Tensor tol,
    torch::Tensor max_iter, torch::Tensor target, torch::Tensor fit_ic,
    int64_t Fp, int64_t max_epochs, int64_t check_every) {
  const at::cuda::CUDAGuard guard(vals.device());
  int Bp = (int)loss_id.size(0);
  TORCH_CHECK(Bp == 64 || Bp == 128 || Bp == 256);
  long nt = idx.size(0);
  int nchunks = (int)chunk_off.size(0) - 1;

  auto optF = y.options().dtype(torch::kFloat32);
  auto optI = y.options().dtype(torch::kInt32);
  auto W = torch::zeros({Bp, Fp}, optF);
  auto V = torch::zeros({Bp, Fp}, optF);
  auto Gf = torch::zeros({Fp, Bp}, optF);
  auto Wf = torch::zeros({Fp, Bp}, vals.options());
  auto D = torch::empty({nt, (long)Bp}, vals.options());
  auto bias = torch::zeros({Bp}, optF);
  auto Vb = torch::zeros({Bp}, optF);
  auto loss_sum = torch::zeros({Bp}, optF);
  auto db_sum = torch::zeros({Bp}, optF);
  auto prev_loss = torch::full({Bp}, 3.0e38, optF);
  auto cur_loss = torch::zeros({Bp}, optF);
  auto active = torch::ones({Bp}, optI);
  auto epoch_mask = torch::zeros({Bp}, optI);
  auto n_iter = torch::zeros({Bp}, optI);
  auto n_active = torch::zeros({1}, optI);

  hipStream_t s = cur_stream();
  float inv_n = 1.0f / (float)nt;
  bool any_tol = tol.max().item<float>() > 0.f;
  int fwd_blocks = (int)std::min<long>((nt + 3) / 4, 4096);
  int upd_threads = Fp >= 256 ? 256 : (int)Fp;
  dim3 upd_grid((unsigned)((Fp + upd_threads - 1) / upd_threads),
                (unsigned)Bp);
  int CPL = Bp / 64;

  auto fwd = [&](auto k, int want_loss) {
    hipLaunchKernelGGL(k, dim3(fwd_blocks), dim3(256), 0, s,
                       indptr.data_ptr<int>(), ccols.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(vals.data_ptr()),
                       y.data_ptr<float>(), idx.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(Wf.data_ptr()),
                       bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                       target.data_ptr<int>(),
                       reinterpret_cast<__bf16*>(D.data_ptr()),
                       loss_sum.data_ptr<float>(), db_sum.data_ptr<float>(),
                       nt, Bp, want_loss);
  };
  auto bwd = [&](auto k) {
    hipLaunchKernelGGL(k, dim3(nchunks), dim3(256), 0, s,
                       tf.data_ptr<int>(), tr.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(tv.data_ptr()),
                       chunk_off.data_ptr<long>(), inv.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(D.data_ptr()),
                       Gf.data_ptr<float>(), Bp);
  };

  for (int epoch = 0; epoch < (int)max_epochs; ++epoch) {
    int want_loss = (any_tol || epoch == (int)max_epochs - 1) ? 1 : 0;
    switch (CPL) {
      case 1: fwd(csr_fwd_d_kernel<1>, want_loss); bwd(csr_bwd_g_kernel<1>); break;
      case 2: fwd(csr_fwd_d_kernel<2>, want_loss); bwd(csr_bwd_g_kernel<2>); break;
      default: fwd(csr_fwd_d_kernel<4>, want_loss); bwd(csr_bwd_g_kernel<4>); break;
    }
    hipLaunchKernelGGL(col_finalize_kernel, dim3((Bp + 255) / 256),
                       dim3(256), 0, s, loss_sum.data_ptr<float>(),
                       db_sum.data_ptr<float>(), bias.data_ptr<float>(),
                       Vb.data_ptr<float>(), prev_loss.data_ptr<float>(),
                       cur_loss.data_ptr<float>(), active.data_ptr<int>(),
                       epoch_mask.data_ptr<int>(), n_iter.data_ptr<int>(),
                       max_iter.data_ptr<int>(), lr.data_ptr<float>(),
                       mom.data_ptr<float>(), tol.data_ptr<float>(),
                       fit_ic.data_ptr<unsigned char>(), inv_n, epoch, Bp,
                       want_loss, n_active.data_ptr<int>());
    hipLaunchKernelGGL(update_w_sparse_kernel, upd_grid, dim3(upd_threads),
                       0, s, W.data_ptr<float>(), V.data_ptr<float>(),
                       Gf.data_ptr<float>(),
                       reinterpret_cast<__bf16*>(Wf.data_ptr()),
                       epoch_mask.data_ptr<int>(), lr.data_ptr<float>(),
                       mom.data_ptr<float>(), l1.data_ptr<float>(),
                       l2.data_ptr<float>(), inv_n, (int)Fp, Bp);
    HIP_CHECK(hipGetLastError());
    if (check_every > 0 && (epoch + 1) % check_every == 0 &&
        epoch + 1 < max_epochs) {
      int na = n_active.item<int>();
      if (na == 0) break;
      n_active.zero_();
    } else {
      HIP_CHECK(hipMemsetAsync(n_active.data_ptr(), 0, sizeof(int), s));
    }
  }
  return {W, bias, n_iter, cur_loss, Wf};
}

torch::Tensor csr_linear_scores(
    torch::Tensor indptr, torch::Tensor ccols, torch::Tensor vals,
    torch::Tensor y, torch::Tensor idx, torch::Tensor Wf,
    torch::Tensor bias, torch::Tensor loss_id, torch::Tensor target,
    int64_t metric, int64_t n_cand, int64_t C) {
  const at::cuda::CUDAGuard guard(vals.device());
  int Bp = (int)Wf.size(1);
  long n_idx = idx.size(0);
  auto out = torch::zeros({n_cand}, y.options().dtype(torch::kFloat64));
  int blocks = (int)std::min<long>((n_idx + 3) / 4, 4096);
  if (C > 1) {   // multiclass OVR: per-candidate argmax over C columns
    hipLaunchKernelGGL(csr_scores_multi_kernel, dim3(blocks), dim3(256), 0,
                       cur_stream(), indptr.data_ptr<int>(),
                       ccols.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(vals.data_ptr()),
                       y.data_ptr<float>(), idx.data_ptr<long>(),
                       reinterpret_cast<const __bf16*>(Wf.data_ptr()),
                       bias.data_ptr<float>(), (int)C, (int)metric, n_idx,
                       Bp, (int)n_cand, out.data_ptr<double>());
    HIP_CHECK(hipGetLastError());
    return out;
  }
  auto go = [&](auto k) {
    hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, cur_stream(),
                       indptr.data_ptr<int>(), ccols.data_ptr<int>(),
                       reinterpret_cast<const __bf16*>(vals.data_ptr()),
                       y.data_ptr<float>(), idx.data_ptr<long>(),
                       reinterpret_cast<const __bf16*>(Wf.data_ptr()),
                       bias.data_ptr<float>(), loss_id.data_ptr<int>(),
                       target.data_ptr<int>(), (int)metric, n_idx, Bp,
                       (int)n_cand, out.data_ptr<double>());
  };
  switch (Bp / 64) {
    case 1: go(csr_scores_kernel<1>); break;
    case 2: go(csr_scores_kernel<2>); break;
    default: go(csr_scores_kernel<4>); break;
  }
  HIP_CHECK(hipGetLastError());
  return out;
}


// multiclass boosting fit: trees [T*K][NN], class-major raw.
std::vector<torch::Tensor> gbt_fit_multi(
    torch::Tensor Xb, torch::Tensor Xbt, torch::Tensor idxmap,
    torch::Tensor y_tr,
    torch::Tensor f0, torch::Tensor sw,
    int64_t K, int64_t n_estimators, double lrate,
    int64_t max_depth, int64_t min_leaf, double lam) {
  const at::cuda::CUDAGuard guard(Xb.device());
  TORCH_CHECK(max_depth >= 1 && max_depth <= 10);
  TORCH_CHECK(K >= 2 && K <= 64);
  int F = (int)Xb.size(1);
  const unsigned char* Xtp = Xbt.data_ptr<unsigned char>();
  long n_rows = Xb.size(0);
  long nt = idxmap.size(0);
  int T = (int)n_estimators;
  int NN = (1 << (max_depth + 1)) - 1;

  auto optF = y_tr.options().dtype(torch::kFloat32);
  auto optI = y_tr.options().dtype(torch::kInt32);
  auto raw = f0.to(optF).reshape({K, 1}).repeat({1, nt}).contiguous();
  auto g = torch::empty({K, nt}, optF);
  auto h = torch::empty({K, nt}, optF);
  auto node_id = torch::zeros({nt}, optI);
  auto feats = torch::full({(long)T * K, NN}, -1, optI);
  auto thrs = torch::zeros({(long)T * K, NN}, optI);
  auto vals = torch::zeros({(long)T * K, NN}, optF);
  int max_lvl_nodes = 1 << (max_depth - 1);
  auto hist = torch::empty({(long)max_lvl_nodes * F * 256 * 3}, optF);
  auto hist_prev = torch::empty({(long)std::max(1, max_lvl_nodes / 2) *
                                 F * 256 * 3}, optF);
  auto gsum = torch::zeros({NN}, optF);
  auto hsum = torch::zeros({NN}, optF);

  hipStream_t s = cur_stream();
  const unsigned char* Xp = Xb.data_ptr<unsigned char>();
  int blocks = (int)std::min<long>((nt + 255) / 256, 2048);
  const bool weighted = sw.numel() > 0;
  const float* wp = nullptr;
  float wmax = 1.f;
  if (weighted) {
    TORCH_CHECK(sw.dtype() == torch::kFloat32 && sw.size(0) == nt);
    wp = sw.data_ptr<float>();
    wmax = sw.max().item<float>();
  }

  for (int t = 0; t < T; ++t) {
    hipLaunchKernelGGL(gbt_softmax_grad_kernel, dim3(blocks), dim3(256), 0,
                       s, raw.data_ptr<float>(), y_tr.data_ptr<float>(),
                       g.data_ptr<float>(), h.data_ptr<float>(), nt,
                       (int)K, wp);
    for (int c = 0; c < (int)K; ++c) {
      float* gc = g.data_ptr<float>() + (long)c * nt;
      float* hc = h.data_ptr<float>() + (long)c * nt;
      int* feat_t = feats.data_ptr<int>() + ((long)t * K + c) * NN;
      int* thr_t = thrs.data_ptr<int>() + ((long)t * K + c) * NN;
      float* val_t = vals.data_ptr<float>() + ((long)t * K + c) * NN;
      for (int d = 0; d < (int)max_depth; ++d) {
        int lvl_lo = (1 << d) - 1;
        int lvl_nodes = 1 << d;
        int even_only = (d > 0) ? 1 : 0;
        launch_hist_level(Xtp, idxmap.data_ptr<int>(),
                          node_id.data_ptr<int>(), gc, hc,
                          hist.data_ptr<float>(), nt, n_rows, F, d,
                          0.25f * wmax, /*g_bounded=*/!weighted, false, s,
                          1, 0, 0, 1.f, /*packed_ok=*/!weighted);
        if (even_only) {
          int prev_lo = (1 << (d - 1)) - 1;
          long cells = (long)F * 256 * 3;
          unsigned gx = (unsigned)std::min<long>((cells + 255) / 256,
                                                 1024);
          hipLaunchKernelGGL(gbt_sibling_kernel,
                             dim3(gx, (unsigned)(lvl_nodes / 2)),
                             dim3(256), 0, s, hist_prev.data_ptr<float>(),
                             hist.data_ptr<float>(), feat_t, prev_lo, F,
                             lvl_nodes);
        }
        hipLaunchKernelGGL(gbt_split_find_kernel, dim3(lvl_nodes),
                           dim3(256), 0, s, hist.data_ptr<float>(), F,
                           lvl_lo, (float)lam, (float)lrate,
                           (int)min_leaf, 0, feat_t, thr_t, val_t,
                           1 << 30, 0u, 0);
        if (d + 1 < (int)max_depth)
          hist_prev.narrow(0, 0, (long)lvl_nodes * F * 256 * 3)
              .copy_(hist.narrow(0, 0, (long)lvl_nodes * F * 256 * 3),
                     true);
        hipLaunchKernelGGL(gbt_split_apply_kernel, dim3(blocks), dim3(256),
                           0, s, Xp, idxmap.data_ptr<int>(),
                           node_id.data_ptr<int>(), feat_t, thr_t, nt, F,
                           lvl_lo, lvl_lo + lvl_nodes);
        HIP_CHECK(hipGetLastError());
      }
      int bl_lo = (1 << max_depth) - 1;
      HIP_CHECK(hipMemsetAsync(gsum.data_ptr(), 0, NN * 4, s));
      HIP_CHECK(hipMemsetAsync(hsum.data_ptr(), 0, NN * 4, s));
      {
        bool fix = det_gbt_mode() && !weighted;
        float fsc = fix ? det_fix_scale(nt) : 0.f;
        hipLaunchKernelGGL(gbt_node_sums_kernel,
                           dim3(fix ? 1 : blocks,
                                (unsigned)(((NN - bl_lo) + 127) / 128)), dim3(256), 0, s,
                           node_id.data_ptr<int>(), gc, hc,
                           gsum.data_ptr<float>(), hsum.data_ptr<float>(),
                           nt, bl_lo, NN, fsc, fsc, 1.f);
      }
      hipLaunchKernelGGL(gbt_leaf_vals_kernel,
                         dim3(((NN - bl_lo) + 255) / 256), dim3(256), 0, s,
                         gsum.data_ptr<float>(), hsum.data_ptr<float>(),
                         val_t, feat_t, (float)lam, (float)lrate, bl_lo,
                         NN);
      hipLaunchKernelGGL(gbt_leaf_apply_c_kernel, dim3(blocks), dim3(256),
                         0, s, raw.data_ptr<float>() + (long)c * nt,
                         node_id.data_ptr<int>(), val_t, nt);
      HIP_CHECK(hipGetLastError());
    }
  }
  return {feats, thrs, vals};
}

torch::Tensor gbt_metric_multi(torch::Tensor raws, torch::Tensor y,
                               torch::Tensor idx, int64_t K) {
  const at::cuda::CUDAGuard guard(raws.device());
  long n_idx = idx.size(0);
  auto out = torch::zeros({1}, raws.options().dtype(torch::kFloat64));
  int blocks = (int)std::min<long>((n_idx + 255) / 256, 2048);
  hipLaunchKernelGGL(gbt_argmax_acc_kernel, dim3(blocks), dim3(256), 0,
                     cur_stream(), raws.data_ptr<float>(),
                     y.data_ptr<float>(), idx.data_ptr<int>(), n_idx,
                     (int)K, out.data_ptr<double>());
  HIP_CHECK(hipGetLastError());
  return out;
}

// ---------------------------------------------------------------------------
// rf_split_find_multi_kernel: summed per-class gini gain over K histogram
// copies (class c's g-channel = count of class c; the count channel is
// identical in every copy, class 0's is used).  Writes the winning
// (feature, threshold) into all K planes of the tree so gbt_predict can
// walk each plane unchanged; no-split nodes get per-class leaf
// probabilities G_c / C.
// ---------------------------------------------------------------------------
template <int FMT>  // 0: classic per-class (g,h,c) planes (cstride apart)
                    // 1: compact [256][K+1] cells (per-class g + count)
__device__ __forceinline__
void rf_split_find_multi_body(const float* __restrict__ ndh, long cstride,
                              int K, int F, int nd, int min_leaf,
                              int kfeat, unsigned fseed, int etr,
                              int* __restrict__ feats,
                              int* __restrict__ thrs,
                              float* __restrict__ vals, long NN) {
  // dead subtree (see gbt_split_find_body): plane-0 feat carries the
  // tree structure for every class
  if (nd > 0 && feats[(nd - 1) >> 1] < 0) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;

  __shared__ float sGain[4];
  __shared__ int sFt[4], sTt[4];
  __shared__ int sRed[5];
  __shared__ float sCnt;
  __shared__ float sH;
  __shared__ float sPC[64];

  unsigned fthr = 0xffffffffu;
  if (kfeat < F) fthr = rf_feat_threshold(F, kfeat, fseed, nd, sRed);

  float bgain = 0.f;
  int bf = -1, bt = 0;
  const float eps = 1e-12f;

  for (int f = wave; f < F; f += 4) {
    bool active = (kfeat >= F) || (rf_feat_hash(fseed, nd, f) < fthr);
    const int cw = FMT ? (K + 1) : 3;
    const float* fh0 = ndh + (long)f * 256 * cw;
    float c4[4];
    float lc = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c4[j] = fh0[(4 * lane + j) * cw + (FMT ? K : 2)];
      lc += c4[j];
    }
    float pc = lc;
    for (int off = 1; off < 64; off <<= 1) {
      float t = __shfl_up(pc, off);
      if (lane >= off) pc += t;
    }
    float C = __shfl(pc, 63);
    float cl[4];
    {
      float a = pc - lc;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a += c4[j];
        cl[j] = a;
      }
    }
    if (f == 0 && lane == 0) sCnt = C;
    // weighted mass per threshold: DERIVED as the sum of the class-g
    // prefixes (classes partition the mass: sum_c w*1{y=c} == w).
    // Reading a separate h channel instead would mix float-atomic g
    // sums with fixed-point h sums -- pure nodes then get tiny nonzero
    // gains and split spuriously.  Unweighted fits have integer-exact
    // class counts, so this equals the count channel bit-for-bit.
    // ONE pass accumulates mass hl, sum-of-squares A (left) / B
    // (right) and SG2: the gini denominators are class-INDEPENDENT,
    // so the division factors out of the class loop (2 divisions per
    // threshold instead of 2K, and the g channels are read once).
    float hl[4] = {0.f, 0.f, 0.f, 0.f};
    float A[4] = {0.f, 0.f, 0.f, 0.f};
    float B[4] = {0.f, 0.f, 0.f, 0.f};
    float H = 0.f, SG2 = 0.f;
    for (int c = 0; c < K; ++c) {
      const float* fhc = FMT ? (fh0 + c) : (fh0 + (long)c * cstride);
      float g4[4];
      float lg = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g4[j] = fhc[(4 * lane + j) * cw];
        lg += g4[j];
      }
      float pg = lg;
      for (int off = 1; off < 64; off <<= 1) {
        float t = __shfl_up(pg, off);
        if (lane >= off) pg += t;
      }
      float G = __shfl(pg, 63);
      H += G;
      SG2 += G * G;
      if (f == 0 && lane == 0) sPC[c] = G;
      float a = pg - lg;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a += g4[j];
        float gl = a, gr = G - gl;
        hl[j] += gl;
        A[j] += gl * gl;
        B[j] += gr * gr;
      }
    }
    if (f == 0 && lane == 0) sH = H;
    int tstar = -1;
    if (etr) {
      int lmin = 256, lmax = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c4[j] > 0.f) {
          int b = 4 * lane + j;
          if (b < lmin) lmin = b;
          if (b > lmax) lmax = b;
        }
      }
      for (int off = 32; off > 0; off >>= 1) {
        lmin = min(lmin, __shfl_down(lmin, off));
        lmax = max(lmax, __shfl_down(lmax, off));
      }
      lmin = __shfl(lmin, 0);
      lmax = __shfl(lmax, 0);
      if (lmax > lmin)
        tstar = lmin + (int)(rf_thr_hash(fseed, nd, f) %
                             (unsigned)(lmax - lmin));
    }
    float gainsum[4];
    const float parent = SG2 / (H + eps);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      gainsum[j] = A[j] / (hl[j] + eps) + B[j] / ((H - hl[j]) + eps);
    if (active) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int b = 4 * lane + j;
        if (b >= 255) continue;
        if (etr && b != tstar) continue;
        if (cl[j] < (float)min_leaf || C - cl[j] < (float)min_leaf)
          continue;
        float gain = gainsum[j] - parent;
        if (gain > bgain + 1e-12f ||
            (gain > bgain - 1e-12f &&
             (bf < 0 || f < bf || (f == bf && b < bt)))) {
          bgain = gain;
          bf = f;
          bt = b;
        }
      }
    }
  }
  for (int off = 32; off > 0; off >>= 1) {
    float og = __shfl_down(bgain, off);
    int of = __shfl_down(bf, off);
    int ot = __shfl_down(bt, off);
    if (og > bgain + 1e-12f ||
        (og > bgain - 1e-12f && of >= 0 &&
         (bf < 0 || of < bf || (of == bf && ot < bt)))) {
      bgain = og;
      bf = of;
      bt = ot;
    }
  }
  if (lane == 0) { sGain[wave] = bgain; sFt[wave] = bf; sTt[wave] = bt; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 4; ++w) {
      if (sGain[w] > sGain[0] + 1e-12f ||
          (sGain[w] > sGain[0] - 1e-12f && sFt[w] >= 0 &&
           (sFt[0] < 0 || sFt[w] < sFt[0] ||
            (sFt[w] == sFt[0] && sTt[w] < sTt[0])))) {
        sGain[0] = sGain[w];
        sFt[0] = sFt[w];
        sTt[0] = sTt[w];
      }
    }
    // PURE node: one class holds the whole mass (exact in fp32: the
    // other class sums are sums of 0.0f).  The reference's f64 eps
    // makes pure-node gains negative; fp32's x*x/x rounding noise can
    // make them spuriously positive under weighted masses, so decide
    // purity explicitly.
    float gmx = 0.f;
    for (int c = 0; c < K; ++c) gmx = fmaxf(gmx, sPC[c]);
    if (sFt[0] < 0 || sGain[0] <= 1e-12f || gmx == sH) {
      for (int c = 0; c < K; ++c) {
        feats[(long)c * NN + nd] = -1;
        if (sCnt > 0.f)
          vals[(long)c * NN + nd] = sPC[c] / (sH + eps);
      }
    } else {
      for (int c = 0; c < K; ++c) {
        feats[(long)c * NN + nd] = sFt[0];
        thrs[(long)c * NN + nd] = sTt[0];
        vals[(long)c * NN + nd] = 0.f;
      }
    }
  }
}

__global__ __launch_bounds__(256)
void rf_split_find_multi_kernel(const float* __restrict__ hist, long cstride,
                                int K, int F, int lvl_lo, int min_leaf,
                                int kfeat, unsigned fseed, int etr,
                                int* __restrict__ feats,
                                int* __restrict__ thrs,
                                float* __restrict__ vals, long NN) {
  const int nd_local = blockIdx.x;
  rf_split_find_multi_body<0>(hist + (long)nd_local * F * 256 * 3,
                              cstride, K, F, lvl_lo + nd_local, min_leaf,
                              kfeat, fseed, etr, feats, thrs, vals, NN);
}

// tree-batched multiclass split find: grid.y = tree within the chunk
// (COMPACT hist layout [tree][nodes][F][256][K+1]; outputs offset by
// the tree's K*NN plane block)
__global__ __launch_bounds__(256)
void rf_bsplit_find_multi_kernel(const float* __restrict__ hist,
                                 long tree_hstride, int K,
                                 int F, int lvl_lo, int min_leaf,
                                 int kfeat, unsigned seed, int etr,
                                 int* __restrict__ feats,
                                 int* __restrict__ thrs,
                                 float* __restrict__ vals, long NN,
                                 int t0) {
  const int tl = blockIdx.y;
  const unsigned st =
      rf_hash(seed ^ (unsigned)((t0 + tl) * 0x9e3779b9u));
  const unsigned fs = rf_hash(st ^ 0x85ebca6bu);
  const long po = (long)tl * (long)K * NN;
  rf_split_find_multi_body<1>(
      hist + (long)tl * tree_hstride +
          (long)blockIdx.x * F * 256 * (K + 1),
      0, K, F, lvl_lo + (int)blockIdx.x, min_leaf, kfeat, fs, etr,
      feats + po, thrs + po, vals + po, NN);
}

// ---------------------------------------------------------------------------
// tree-batched small-n RF pieces: for launch-bound forests (digits-scale
// nt) a chunk of TB whole trees advances one level per kernel launch.
// grid.y carries the tree (bootstrap/planes/apply), grid.z carries
// (tree, class) (sibling/sums) or (tree, node-group) (histograms, see
// gbt_hist_kernel<MULTI, 1>).
// ---------------------------------------------------------------------------
__global__ void rf_bbootstrap_kernel(const int* __restrict__ idx_in,
                                     const float* __restrict__ y_in,
                                     int* __restrict__ idx_out,
                                     float* __restrict__ y_out, long nt,
                                     unsigned seed, int t0) {
  const int tl = blockIdx.y;
  const unsigned st =
      rf_hash(seed ^ (unsigned)((t0 + tl) * 0x9e3779b9u));
  idx_out += (long)tl * nt;
  y_out += (long)tl * nt;
  long i = blockIdx.x * (long)blockDim.x + threadIdx.x;
  for (; i < nt; i += (long)gridDim.x * blockDim.x) {
    unsigned r = rf_hash(st ^ (unsigned)i);
    long p = (long)(((unsigned long long)r * (unsigned long long)nt) >> 32);
    idx_out[i] = idx_in[p];
    y_out[i] = y_in[p];
  }
}

__global__ void rf_bplanes_kernel(const float* __restrict__ y_boot,
                                  float* __restrict__ G, long nt, int K) {
  const int tl = blockIdx.y;
  y_boot += (long)tl * nt;
  G += (long)tl * (long)K * nt;
  long i = blockIdx.x * (long)blockDim.x + threadIdx.x;
  for (; i < nt; i += (long)gridDim.x * blockDim.x) {
    int cls = (int)y_boot[i];
    for (int c = 0; c < K; ++c) G[(long)c * nt + i] = (c == cls) ? 1.f : 0.f;
  }
}

// sibling subtraction, one launch per level for the whole tree chunk:
// grid.z = tree (compact layout: all classes share the tree's cells);
// prev/cur are SAME-SHAPE alternating full-level buffers ([TB][ccells])
__global__ void rf_bsibling_kernel(const float* __restrict__ prev,
                                   float* __restrict__ cur,
                                   const int* __restrict__ feat,
                                   int prev_lo, int F, int lvl_nodes,
                                   long ccells, long plane_tstride,
                                   int cellw) {
  const int z = blockIdx.z;
  prev += (long)z * ccells;
  cur += (long)z * ccells;
  feat += (long)z * plane_tstride;            // plane 0 of the tree
  int pair = blockIdx.y;
  long cells = (long)F * 256 * cellw;
  long base_l = (long)(2 * pair) * cells;
  long base_r = (long)(2 * pair + 1) * cells;
  long base_p = (long)pair * cells;
  // non-split parents are skipped outright (instead of zero-filling the
  // right child): the split finders early-out on dead subtrees, so the
  // stale cells are never read
  if (feat[prev_lo + pair] < 0) return;
  for (long i = blockIdx.x * blockDim.x + threadIdx.x; i < cells;
       i += (long)gridDim.x * blockDim.x) {
    cur[base_r + i] = prev[base_p + i] - cur[base_l + i];
  }
}

__global__ void rf_bapply_kernel(const unsigned char* __restrict__ Xb,
                                 const int* __restrict__ idxmap,
                                 int* __restrict__ node_id,
                                 const int* __restrict__ feat,
                                 const int* __restrict__ thr, long nt,
                                 int F, int lvl_lo, int lvl_hi,
                                 long idx_tstride, long plane_tstride) {
  const int tl = blockIdx.y;
  idxmap += (long)tl * idx_tstride;
  node_id += (long)tl * nt;
  feat += (long)tl * plane_tstride;
  thr += (long)tl * plane_tstride;
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    int nd = node_id[r];
    if (nd < lvl_lo || nd >= lvl_hi) continue;
    int f = feat[nd];
    if (f < 0) continue;
    int bin = Xb[(long)idxmap[r] * F + f];
    node_id[r] = 2 * nd + 1 + (bin > thr[nd] ? 1 : 0);
  }
}

// bottom-level (g, count) sums per (tree, class): h == 1 in RF, so the
// count IS the h channel.  grid (row blocks, 128-node chunks, tl*KP+c).
__global__ void rf_bsums_kernel(const int* __restrict__ node_id,
                                const float* __restrict__ g,
                                float* __restrict__ gsum,
                                float* __restrict__ hsum, long nt,
                                int lvl_lo_full, int lvl_hi_full,
                                long g_tstride, long g_cstride, int KP,
                                int NN) {
  __shared__ float lg[128], lc[128];
  const int z = blockIdx.z;
  node_id += (long)(z / KP) * nt;
  g += (long)(z / KP) * g_tstride + (long)(z % KP) * g_cstride;
  gsum += (long)z * NN;
  hsum += (long)z * NN;
  const int lvl_lo = lvl_lo_full + (int)blockIdx.y * 128;
  const int lvl_hi = min(lvl_hi_full, lvl_lo + 128);
  int nn = lvl_hi - lvl_lo;
  for (int i = threadIdx.x; i < nn; i += blockDim.x) {
    lg[i] = 0.f;
    lc[i] = 0.f;
  }
  __syncthreads();
  long r = blockIdx.x * blockDim.x + threadIdx.x;
  for (; r < nt; r += (long)gridDim.x * blockDim.x) {
    int nd = node_id[r];
    if (nd < lvl_lo || nd >= lvl_hi) continue;
    atomicAdd(&lg[nd - lvl_lo], g[r]);
    atomicAdd(&lc[nd - lvl_lo], 1.f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nn; i += blockDim.x) {
    if (lc[i] != 0.f) {
      atomicAdd(&gsum[lvl_lo + i], lg[i]);
      atomicAdd(&hsum[lvl_lo + i], lc[i]);
    }
  }
}

// bottom-level leaf values for every (tree, class) plane in one launch;
// vals/feats offset per plane (z = tl*KP + c matches the [T*KP][NN]
// output layout when the host pre-offsets by t0*KP*NN)
__global__ void rf_bleafs_kernel(const float* __restrict__ gsum,
                                 const float* __restrict__ hsum,
                                 float* __restrict__ vals,
                                 int* __restrict__ feats, int lvl_lo,
                                 int lvl_hi, int NN) {
  const int z = blockIdx.y;
  const long po = (long)z * NN;
  int nd = lvl_lo + blockIdx.x * blockDim.x + threadIdx.x;
  if (nd >= lvl_hi) return;
  float h = hsum[po + nd];
  if (h > 0.f) {
    feats[po + nd] = -1;
    vals[po + nd] = gsum[po + nd] / (h + 1e-12f);
  }
}

// ---------------------------------------------------------------------------
// rf_fit: RandomForest fit over the shared binned matrix.  Trees are
// independent: per tree a stateless-hash bootstrap resample of the train
// positions, level-wise growth with gini (classification) / MSE
// (regression) splits and exact-k per-node feature subsampling.  Returns
// (feats, thrs, vals) in the gbt_fit layout ([T*planes][NN]); leaf values
// are class probabilities / means ALREADY divided by n_estimators so the
// summing gbt_predict yields the forest average.
// ---------------------------------------------------------------------------
std::vector<torch::Tensor> rf_fit(torch::Tensor Xb, torch::Tensor Xbt,
                                  torch::Tensor idxmap0,
                                  torch::Tensor y_tr, int64_t K,
                                  int64_t n_estimators, int64_t max_depth,
                                  int64_t min_leaf, int64_t max_features,
                                  int64_t seed, int64_t bootstrap,
                                  int64_t splitter_random,
                                  torch::Tensor sw) {
  const at::cuda::CUDAGuard guard(Xb.device());
  TORCH_CHECK(Xb.dtype() == torch::kUInt8 && Xb.dim() == 2);
  TORCH_CHECK(max_depth >= 1 && max_depth <= 10,
              "device RF supports max_depth in [1, 10]");
  TORCH_CHECK(K <= 64, "device RF supports at most 64 classes");
  // sample_weight (fold-sliced [nt]): weighted gini/MSE via w-scaled g
  // planes + an h channel carrying sum(w) (min_samples_leaf keeps plain
  // counts).  Weighted fits run the per-tree CLASSIC-layout path: the
  // tree-batched compact cells have no h channel.
  const bool weighted = sw.numel() > 0;
  float wmax = 1.f;
  if (weighted) {
    TORCH_CHECK(sw.dtype() == torch::kFloat32 &&
                sw.size(0) == idxmap0.size(0));
    wmax = sw.max().item<float>();
  }
  int F = (int)Xb.size(1);
  long nt = idxmap0.size(0);
  int T = (int)n_estimators;
  int NN = (1 << (max_depth + 1)) - 1;
  int KP = K > 2 ? (int)K : 1;          // histogram / tree planes
  int kfeat = (max_features <= 0 || max_features >= F) ? (1 << 30)
                                                       : (int)max_features;

  auto optF = y_tr.options().dtype(torch::kFloat32);
  auto optI = y_tr.options().dtype(torch::kInt32);
  auto feats = torch::full({(long)T * KP, (long)NN}, -1, optI);
  auto thrs = torch::zeros({(long)T * KP, (long)NN}, optI);
  auto vals = torch::zeros({(long)T * KP, (long)NN}, optF);
  int max_lvl_nodes = 1 << (max_depth - 1);
  long ccells = (long)max_lvl_nodes * F * 256 * 3;

  hipStream_t s = cur_stream();
  const unsigned char* Xp = Xb.data_ptr<unsigned char>();
  const unsigned char* Xtp = Xbt.data_ptr<unsigned char>();
  long n_rows = Xb.size(0);
  int blocks = (int)std::min<long>((nt + 255) / 256, 2048);
  int bl_lo = (1 << max_depth) - 1;

  if (nt <= 65536 && !weighted) {
    // ---- tree-batched small-n path (digits-scale forests are LAUNCH
    // bound: ~4 launches per tree-LEVEL here vs ~4 launches per tree-
    // level PER TREE in the large-n loop below).  A chunk of TB whole
    // trees shares every launch; per-tree seeds are recomputed inside
    // the kernels, so trees are identical to the per-tree path.  Two
    // full-size histogram buffers alternate as (current, parent) so the
    // sibling subtraction needs no parent copy.  The coalescing sort of
    // the large-n path is skipped: at <=64k rows the binned matrix is
    // L2-resident and gather order does not matter.
    // Histograms use the COMPACT cell layout ([256][K+1] per (node,
    // feature) for K-class, [256][2] binary: per-class g + one shared
    // count) -- the dense hist stream bounds the small-n hist/sibling/
    // split kernels, and RF's h IS the count. ----
    const int cellw = (KP > 1) ? KP + 1 : 2;
    const long ccells_b = (long)max_lvl_nodes * F * 256 * cellw;
    double per_tree = 2.0 * (double)ccells_b * 4.0;
    int TB = (int)std::max<long>(
        1, std::min<long>({(long)T, 2048L,
                           (long)(6.0e9 / std::max(per_tree, 1.0))}));
    auto hista = torch::empty({(long)TB * ccells_b}, optF);
    auto histb = torch::empty({(long)TB * ccells_b}, optF);
    auto node_id = torch::empty({(long)TB * nt}, optI);
    auto gsum = torch::zeros({(long)TB * KP, (long)NN}, optF);
    auto hsum = torch::zeros({(long)TB * KP, (long)NN}, optF);
    auto ones = torch::ones({nt}, optF);
    torch::Tensor idx_b, y_b, G;
    long idx_ts = 0, g_ts = 0;
    if (bootstrap) {
      idx_b = torch::empty({(long)TB * nt}, optI);
      y_b = torch::empty({(long)TB * nt}, optF);
      idx_ts = nt;
      g_ts = (KP > 1) ? (long)KP * nt : nt;
    }
    if (KP > 1) {
      G = torch::empty({(long)(bootstrap ? TB : 1) * KP, nt}, optF);
      if (!bootstrap)      // identical planes for every tree: share them
        hipLaunchKernelGGL(rf_planes_kernel, dim3(blocks), dim3(256), 0,
                           s, y_tr.data_ptr<float>(), G.data_ptr<float>(),
                           nt, KP, nullptr);
    }
    for (int t0 = 0; t0 < T; t0 += TB) {
      int tb = std::min(TB, T - t0);
      if (bootstrap) {
        hipLaunchKernelGGL(rf_bbootstrap_kernel,
                           dim3(blocks, (unsigned)tb), dim3(256), 0, s,
                           idxmap0.data_ptr<int>(),
                           y_tr.data_ptr<float>(), idx_b.data_ptr<int>(),
                           y_b.data_ptr<float>(), nt, (unsigned)seed, t0);
        if (KP > 1)
          hipLaunchKernelGGL(rf_bplanes_kernel,
                             dim3(blocks, (unsigned)tb), dim3(256), 0, s,
                             y_b.data_ptr<float>(), G.data_ptr<float>(),
                             nt, KP);
      }
      HIP_CHECK(hipMemsetAsync(node_id.data_ptr(), 0,
                               (size_t)tb * nt * 4, s));
      const int* idxp = bootstrap ? idx_b.data_ptr<int>()
                                  : idxmap0.data_ptr<int>();
      const float* gp = (KP > 1)
                            ? G.data_ptr<float>()
                            : (bootstrap ? y_b.data_ptr<float>()
                                         : y_tr.data_ptr<float>());
      int* feat_t = feats.data_ptr<int>() + (long)t0 * KP * NN;
      int* thr_t = thrs.data_ptr<int>() + (long)t0 * KP * NN;
      float* val_t = vals.data_ptr<float>() + (long)t0 * KP * NN;
      for (int d = 0; d < (int)max_depth; ++d) {
        int lvl_lo = (1 << d) - 1;
        int lvl_nodes = 1 << d;
        float* cur = (d & 1) ? histb.data_ptr<float>()
                             : hista.data_ptr<float>();
        float* prev = (d & 1) ? hista.data_ptr<float>()
                              : histb.data_ptr<float>();
        launch_hist_level(Xtp, idxp, node_id.data_ptr<int>(), gp,
                          ones.data_ptr<float>(), cur, nt, n_rows, F, d,
                          1.f, false, K != 0, s, KP, nt, 0, 1.f,
                          false, tb, idx_ts, g_ts, ccells_b, cellw);
        if (d > 0) {
          long cells = (long)F * 256 * cellw;
          unsigned gx =
              (unsigned)std::min<long>((cells + 255) / 256, 256);
          hipLaunchKernelGGL(rf_bsibling_kernel,
                             dim3(gx, (unsigned)(lvl_nodes / 2),
                                  (unsigned)tb), dim3(256), 0, s,
                             prev, cur, feat_t, (1 << (d - 1)) - 1, F,
                             lvl_nodes, ccells_b, (long)KP * NN, cellw);
        }
        if (KP > 1) {
          hipLaunchKernelGGL(rf_bsplit_find_multi_kernel,
                             dim3((unsigned)lvl_nodes, (unsigned)tb),
                             dim3(256), 0, s, cur, ccells_b,
                             KP, F, lvl_lo, (int)min_leaf, kfeat,
                             (unsigned)seed, (int)splitter_random,
                             feat_t, thr_t, val_t, (long)NN, t0);
        } else {
          hipLaunchKernelGGL(rf_bsplit_find_kernel,
                             dim3((unsigned)lvl_nodes, (unsigned)tb),
                             dim3(256), 0, s, cur, ccells_b, F, lvl_lo,
                             (int)min_leaf, feat_t, thr_t, val_t,
                             (long)KP * NN, kfeat, (unsigned)seed,
                             (int)splitter_random, t0);
        }
        hipLaunchKernelGGL(rf_bapply_kernel,
                           dim3(blocks, (unsigned)tb), dim3(256), 0, s,
                           Xp, idxp, node_id.data_ptr<int>(), feat_t,
                           thr_t, nt, F, lvl_lo, lvl_lo + lvl_nodes,
                           idx_ts, (long)KP * NN);
        HIP_CHECK(hipGetLastError());
      }
      HIP_CHECK(hipMemsetAsync(gsum.data_ptr(), 0,
                               (size_t)tb * KP * NN * 4, s));
      HIP_CHECK(hipMemsetAsync(hsum.data_ptr(), 0,
                               (size_t)tb * KP * NN * 4, s));
      hipLaunchKernelGGL(
          rf_bsums_kernel,
          dim3(blocks, (unsigned)(((NN - bl_lo) + 127) / 128),
               (unsigned)(tb * KP)), dim3(256), 0, s,
          node_id.data_ptr<int>(), gp, gsum.data_ptr<float>(),
          hsum.data_ptr<float>(), nt, bl_lo, NN, g_ts,
          (KP > 1) ? nt : 0L, KP, NN);
      hipLaunchKernelGGL(rf_bleafs_kernel,
                         dim3((unsigned)(((NN - bl_lo) + 255) / 256),
                              (unsigned)(tb * KP)), dim3(256), 0, s,
                         gsum.data_ptr<float>(), hsum.data_ptr<float>(),
                         val_t, feat_t, bl_lo, NN, NN);
      HIP_CHECK(hipGetLastError());
    }
    vals.mul_(1.0 / (double)T);
    return {feats, thrs, vals};
  }

  auto node_id = torch::zeros({nt}, optI);
  auto hist = torch::empty({ccells * KP}, optF);
  auto hist_prev = torch::empty(
      {(long)std::max(1, max_lvl_nodes / 2) * F * 256 * 3 * KP}, optF);
  long pcells = (long)std::max(1, max_lvl_nodes / 2) * F * 256 * 3;
  auto gsum = torch::zeros({NN}, optF);
  auto hsum = torch::zeros({NN}, optF);
  auto ones = torch::ones({nt}, optF);
  auto idx_t = bootstrap ? torch::empty({nt}, optI) : idxmap0;
  auto y_boot = bootstrap ? torch::empty({nt}, optF) : y_tr;
  auto w_boot = (weighted && bootstrap) ? torch::empty({nt}, optF) : sw;
  auto G = (KP > 1) ? torch::empty({(long)KP, nt}, optF)
                    : torch::empty({0}, optF);
  auto y_w = (weighted && KP == 1) ? torch::empty({nt}, optF)
                                   : torch::empty({0}, optF);

  for (int t = 0; t < T; ++t) {
    unsigned st = rf_hash((unsigned)seed ^ (unsigned)(t * 0x9e3779b9u));
    unsigned fs = rf_hash(st ^ 0x85ebca6bu);
    torch::Tensor idx_u = idx_t, y_u = y_boot, w_u = w_boot;
    if (bootstrap) {
      hipLaunchKernelGGL(rf_bootstrap_kernel, dim3(blocks), dim3(256), 0, s,
                         idxmap0.data_ptr<int>(), y_tr.data_ptr<float>(),
                         idx_t.data_ptr<int>(), y_boot.data_ptr<float>(),
                         nt, st,
                         weighted ? sw.data_ptr<float>() : nullptr,
                         weighted ? w_boot.data_ptr<float>() : nullptr);
      // sort the resample by row id: histogram/sum kernels are order-
      // invariant, and sorted gathers coalesce the feature-major bin
      // reads (a random-order resample made every 1-byte load its own
      // 64 B line)
      auto srt = torch::sort(idx_t);
      idx_u = std::get<0>(srt).contiguous();
      auto perm = std::get<1>(srt);
      y_u = y_boot.index_select(0, perm).contiguous();
      if (weighted) w_u = w_boot.index_select(0, perm).contiguous();
    }
    const float* wp_u = weighted ? w_u.data_ptr<float>() : nullptr;
    if (KP > 1)
      hipLaunchKernelGGL(rf_planes_kernel, dim3(blocks), dim3(256), 0, s,
                         y_u.data_ptr<float>(), G.data_ptr<float>(), nt,
                         KP, wp_u);
    if (weighted && KP == 1) y_w.copy_(y_u).mul_(w_u);
    HIP_CHECK(hipMemsetAsync(node_id.data_ptr(), 0, nt * 4, s));
    int* feat_t = feats.data_ptr<int>() + (long)t * KP * NN;
    int* thr_t = thrs.data_ptr<int>() + (long)t * KP * NN;
    float* val_t = vals.data_ptr<float>() + (long)t * KP * NN;
    for (int d = 0; d < (int)max_depth; ++d) {
      int lvl_lo = (1 << d) - 1;
      int lvl_nodes = 1 << d;
      {
        // ONE launch histograms every class plane (rows stay cache-hot
        // across classes inside each block); classification g-planes are
        // 0/1 indicators -> packed single-atomic cells
        const float* gp = (KP > 1)
                              ? G.data_ptr<float>()
                              : (weighted ? y_w.data_ptr<float>()
                                          : y_u.data_ptr<float>());
        launch_hist_level(Xtp, idx_u.data_ptr<int>(),
                          node_id.data_ptr<int>(), gp,
                          weighted ? wp_u : ones.data_ptr<float>(),
                          hist.data_ptr<float>(),
                          nt, n_rows, F, d, weighted ? wmax : 1.f, false,
                          (K != 0) && !weighted, s, KP,
                          nt, ccells);
      }
      if (d > 0) {
        for (int c = 0; c < KP; ++c) {
          int prev_lo = (1 << (d - 1)) - 1;
          long cells = (long)F * 256 * 3;
          unsigned gx = (unsigned)std::min<long>((cells + 255) / 256, 1024);
          hipLaunchKernelGGL(gbt_sibling_kernel,
                             dim3(gx, (unsigned)(lvl_nodes / 2)), dim3(256),
                             0, s,
                             hist_prev.data_ptr<float>() + (long)c * pcells,
                             hist.data_ptr<float>() + (long)c * ccells,
                             feat_t, prev_lo, F, lvl_nodes);
        }
      }
      if (KP > 1) {
        hipLaunchKernelGGL(rf_split_find_multi_kernel, dim3(lvl_nodes),
                           dim3(256), 0, s, hist.data_ptr<float>(), ccells,
                           KP, F, lvl_lo, (int)min_leaf, kfeat, fs,
                           (int)splitter_random, feat_t,
                           thr_t, val_t, (long)NN);
      } else {
        hipLaunchKernelGGL(gbt_split_find_kernel, dim3(lvl_nodes), dim3(256),
                           0, s, hist.data_ptr<float>(), F, lvl_lo, 0.f,
                           -1.f, (int)min_leaf, 0, feat_t, thr_t, val_t,
                           kfeat, fs, (int)splitter_random);
      }
      if (d + 1 < (int)max_depth) {
        long lvlcells = (long)lvl_nodes * F * 256 * 3;
        for (int c = 0; c < KP; ++c)
          hist_prev.narrow(0, (long)c * pcells, lvlcells)
              .copy_(hist.narrow(0, (long)c * ccells, lvlcells),
                     /*non_blocking=*/true);
      }
      hipLaunchKernelGGL(gbt_split_apply_kernel, dim3(blocks), dim3(256),
                         0, s, Xp, idx_u.data_ptr<int>(),
                         node_id.data_ptr<int>(), feat_t, thr_t, nt, F,
                         lvl_lo, lvl_lo + lvl_nodes);
      HIP_CHECK(hipGetLastError());
    }
    for (int c = 0; c < KP; ++c) {
      const float* gp = (KP > 1)
                            ? G.data_ptr<float>() + (long)c * nt
                            : (weighted ? y_w.data_ptr<float>()
                                        : y_u.data_ptr<float>());
      HIP_CHECK(hipMemsetAsync(gsum.data_ptr(), 0, NN * 4, s));
      HIP_CHECK(hipMemsetAsync(hsum.data_ptr(), 0, NN * 4, s));
      hipLaunchKernelGGL(gbt_node_sums_kernel,
                         dim3(blocks,
                              (unsigned)(((NN - bl_lo) + 127) / 128)),
                         dim3(256), 0,
                         s, node_id.data_ptr<int>(), gp,
                         weighted ? wp_u : ones.data_ptr<float>(),
                         gsum.data_ptr<float>(),
                         hsum.data_ptr<float>(), nt, bl_lo, NN, 0.f, 0.f,
                         1.f);
      hipLaunchKernelGGL(gbt_leaf_vals_kernel,
                         dim3(((NN - bl_lo) + 255) / 256), dim3(256), 0, s,
                         gsum.data_ptr<float>(), hsum.data_ptr<float>(),
                         val_t + (long)c * NN, feat_t + (long)c * NN, 0.f,
                         -1.f, bl_lo, NN);
    }
    HIP_CHECK(hipGetLastError());
  }
  vals.mul_(1.0 / (double)T);           // forest average via summing walk
  return {feats, thrs, vals};
}

// ---------------------------------------------------------------------------
// flagship_ablate: time the fwd kernel with pieces removed, to locate the
// wall empirically (guide common-mistake #8: ablate before optimizing).
// bits: 1 = skip Dt store, 2 = trivial epilogue (d = z), 4 = skip X stage,
// 8 = skip W stage, 16 = skip MFMA loop.
// ---------------------------------------------------------------------------
template <int ABL>
__global__ __launch_bounds__(1024)
void fwd_dAB_kernel(const __bf16* __restrict__ X, const float* __restrict__ y,
                    const int* __restrict__ idx, const __bf16* __restrict__ Wt,
                    const float* __restrict__ bias,
                    const int* __restrict__ loss_id,
                    const int* __restrict__ target, __bf16* __restrict__ Dt,
                    float* __restrict__ loss_sum, float* __restrict__ db_sum,
                    int nt, int NTp, int Fp, int Bp, int want_loss) {
  constexpr int NF = 4;
  __shared__ __bf16 sX[2][256 * 64];
  __shared__ __bf16 sW[2][256 * 64];
  __shared__ float sLoss[256];
  __shared__ float sDb[256];
  __shared__ int sIdx[256];
  __shared__ float sY[256];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int cwave = wave & 3;
  const int rquad = wave >> 2;
  const int rt = blockIdx.x;
  const int g = lane >> 4;
  const int rl8 = lane >> 3;
  const int slot = lane & 7;

  if (tid < 256) {
    int gi = idx[rt * 256 + tid];
    sIdx[tid] = gi;
    sY[tid] = y[gi];
    sLoss[tid] = 0.f;
    sDb[tid] = 0.f;
  }
  __syncthreads();

  auto stage = [&](int b, int kc) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int rbase = q * 128 + wave * 8;
      int r = rbase + rl8;
      int ksw = kc + ((slot ^ (r & 7)) << 3);
      if (!(ABL & 4))
        gload_lds16(X + (long)sIdx[r] * Fp + ksw, &sX[b][rbase * 64]);
      if (!(ABL & 8))
        gload_lds16(Wt + (long)r * Fp + ksw, &sW[b][rbase * 64]);
    }
  };

  f32x4 acc[4][NF];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int nkc = Fp >> 6;
  for (int kc = 0; kc < nkc; ++kc) {
    int b = kc & 1;
    if (kc + 1 < nkc) stage(b ^ 1, (kc + 1) << 6);
    if (!(ABL & 16)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 a[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          int r = rquad * 64 + m * 16 + (lane & 15);
          a[m] = frag12(sX[b], r, h * 4 + g);
        }
#pragma unroll
        for (int fn = 0; fn < NF; ++fn) {
          int c = cwave * 64 + fn * 16 + (lane & 15);
          bf16x8 bb = frag12(sW[b], c, h * 4 + g);
#pragma unroll
          for (int m = 0; m < 4; ++m)
            acc[m][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                a[m], bb, acc[m][fn], 0, 0, 0);
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

#pragma unroll
  for (int fn = 0; fn < NF; ++fn) {
    int col_in = cwave * 64 + fn * 16 + (lane & 15);
    float bia = bias[col_in];
    int lid = loss_id[col_in];
    int tgt = target[col_in];
    float lsum = 0.f, dsum = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      int row_base = rquad * 64 + m * 16 + ((lane >> 4) << 2);
      bf16x4 dpack;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int gr = rt * 256 + row_base + r;
        float z = acc[m][fn][r] + bia;
        float d;
        if (ABL & 2) {
          d = z;
        } else {
          float yv = sY[row_base + r];
          if (lid == LOSS_LOGISTIC) {
            float t = (yv == (float)tgt) ? 1.f : 0.f;
            d = fast_rcp(1.f + __expf(-z)) - t;
          } else if (lid == LOSS_HINGE) {
            float sg = (yv == (float)tgt) ? 1.f : -1.f;
            d = (sg * z < 1.f) ? -sg : 0.f;
          } else {
            d = z - yv;
          }
          if (gr >= nt) d = 0.f;
        }
        dpack[r] = (__bf16)d;
        dsum += d;
      }
      if (ABL & 1) {
        asm volatile("" ::"v"(dpack[0]), "v"(dpack[2]));  // keep live
      } else {
        *reinterpret_cast<bf16x4*>(
            Dt + (long)col_in * NTp + rt * 256 + row_base) = dpack;
      }
    }
    atomicAdd(&sDb[col_in], dsum + lsum);
  }
  __syncthreads();
  if (tid < 256) atomicAdd(&db_sum[tid], sDb[tid]);
}

std::vector<double> flagship_ablate(int64_t rows, int64_t Fp, int64_t iters) {
  TORCH_CHECK(g_layout >= 0, "probe first");
  auto opt = torch::TensorOptions().dtype(torch::kBFloat16).device(torch::kCUDA);
  long NTp = (rows / 256) * 256;
  auto X = torch::randn({NTp, Fp}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA)).to(torch::kBFloat16);
  auto Wt = torch::randn({256, Fp}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA)).to(torch::kBFloat16) * 0.01;
  auto y = torch::ones({NTp}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA));
  auto idx = torch::arange((long)NTp, torch::TensorOptions().dtype(torch::kInt32).device(torch::kCUDA));
  auto bias = torch::zeros({256}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA));
  auto lossi = torch::zeros({256}, torch::TensorOptions().dtype(torch::kInt32).device(torch::kCUDA));
  auto tgt = torch::ones({256}, torch::TensorOptions().dtype(torch::kInt32).device(torch::kCUDA));
  auto Dt = torch::zeros({256L, NTp}, opt);
  auto ls = torch::zeros({256}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA));
  auto db = torch::zeros({256}, torch::TensorOptions().dtype(torch::kFloat32).device(torch::kCUDA));
  hipStream_t s = cur_stream();
  std::vector<double> out;
  auto run = [&](auto kern) {
    // warmup
    for (int i = 0; i < 3; ++i)
      hipLaunchKernelGGL(kern, dim3((unsigned)(NTp / 256)), dim3(1024), 0, s,
                         reinterpret_cast<const __bf16*>(X.data_ptr()),
                         y.data_ptr<float>(), idx.data_ptr<int>(),
                         reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                         bias.data_ptr<float>(), lossi.data_ptr<int>(),
                         tgt.data_ptr<int>(),
                         reinterpret_cast<__bf16*>(Dt.data_ptr()),
                         ls.data_ptr<float>(), db.data_ptr<float>(),
                         (int)NTp, (int)NTp, (int)Fp, 256, 0);
    hipEvent_t e0, e1;
    HIP_CHECK(hipEventCreate(&e0));
    HIP_CHECK(hipEventCreate(&e1));
    HIP_CHECK(hipEventRecord(e0, s));
    for (int i = 0; i < (int)iters; ++i)
      hipLaunchKernelGGL(kern, dim3((unsigned)(NTp / 256)), dim3(1024), 0, s,
                         reinterpret_cast<const __bf16*>(X.data_ptr()),
                         y.data_ptr<float>(), idx.data_ptr<int>(),
                         reinterpret_cast<const __bf16*>(Wt.data_ptr()),
                         bias.data_ptr<float>(), lossi.data_ptr<int>(),
                         tgt.data_ptr<int>(),
                         reinterpret_cast<__bf16*>(Dt.data_ptr()),
                         ls.data_ptr<float>(), db.data_ptr<float>(),
                         (int)NTp, (int)NTp, (int)Fp, 256, 0);
    HIP_CHECK(hipEventRecord(e1, s));
    HIP_CHECK(hipEventSynchronize(e1));
    float ms = 0;
    HIP_CHECK(hipEventElapsedTime(&ms, e0, e1));
    hipEventDestroy(e0);
    hipEventDestroy(e1);
    out.push_back((double)ms / iters);
  };
  run(fwd_dAB_kernel<0>);    // full
  run(fwd_dAB_kernel<1>);    // no Dt store
  run(fwd_dAB_kernel<2>);    // trivial epilogue
  run(fwd_dAB_kernel<3>);    // no store + trivial epilogue
  run(fwd_dAB_kernel<4>);    // no X stage
  run(fwd_dAB_kernel<8>);    // no W stage
  run(fwd_dAB_kernel<16>);   // no MFMA
  run(fwd_dAB_kernel<17>);   // no MFMA + no store
  run(fwd_dAB_kernel<29>);   // stages only (no mfma/store/epilogue... 1|4 off: 16|8|4|1 = X only? 29 = 16+8+4+1: no mfma, no W, no X, no store)
  return out;
}

void bind_grouped(pybind11::module_& m);  // ska_grouped.hip

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  bind_grouped(m);
  m.def("flagship_ablate", &flagship_ablate,
        "ablation timings for the fwd kernel (ms/launch)");
  m.def("gemm_probe", &gemm_probe, "MFMA layout probe (4 combos)");
  m.def("set_layout", &set_layout);
  m.def("get_layout", &get_layout);
  m.def("msq_rows", &msq_rows, "mean squared row norm");
  m.def("linear_fit", &linear_fit, "batched linear fit (device epoch loop)");
  m.def("linear_scores", &linear_scores, "batched per-candidate scores");
  m.def("linear_search_run", &linear_search_run,
        "whole fold x chunk search loop on device (C++ engine core)");
  m.def("kmeans_fit", &kmeans_fit, "batched Lloyd loop (centroid blocks)");
  m.def("kmeans_assign", &kmeans_assign, "assignment/inertia under centers");
  m.def("row_norms", &row_norms, "per-row squared norms");
  m.def("gbt_bin", &gbt_bin, "device quantile binning");
  m.def("gbt_fit", &gbt_fit, "histogram boosting fit (depth-wise trees)");
  m.def("rf_fit", &rf_fit,
        "RandomForest fit (bootstrap + gini/mse splits, feature subsampling)");
  m.def("gbt_predict", &gbt_predict, "tree-walk raw predictions");
  m.def("gbt_predict_multi", &gbt_predict_multi,
        "one-launch all-class tree walk over [T*K][NN] planes");
  m.def("gbt_metric", &gbt_metric, "accuracy/ss_res sums");
  m.def("csr_linear_fit", &csr_linear_fit,
        "CSR-resident batched linear fit (K5)");
  m.def("csr_linear_scores", &csr_linear_scores,
        "CSR-resident per-candidate scores");
  m.def("gbt_fit_multi", &gbt_fit_multi,
        "multiclass softmax boosting (one tree per class per round)");
  m.def("gbt_metric_multi", &gbt_metric_multi,
        "argmax accuracy over class-major raw planes");
}
