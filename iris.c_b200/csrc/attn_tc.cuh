/*
 * Pieces shared by the tensor-core attention kernels: bounded mbarrier waits
 * and the masking and exponentials of a score row held in registers.
 */
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"

namespace iris_b200 {
namespace sm100 {

/* ---------------- bounded waits ---------------- */

struct Ctx {
    uint32_t bars;                  /* shared address of the barrier block */
    volatile uint32_t *abort_flag;  /* generic pointer to the CTA abort word */
    unsigned int *status;
    unsigned long long wait_ns;
};

/* A wait ran out: raise the CTA's abort flag and record the first such event
 * of the launch in the device status word. */
__device__ __forceinline__ void give_up(const Ctx &c, int site, unsigned aux) {
    *c.abort_flag = 1u;
    if (atomicCAS(c.status, 0u, 1u) == 0u) {
        c.status[1] = (unsigned)site;
        c.status[2] = blockIdx.x;
        c.status[3] = aux;
    }
}

/* Bounded wait. Returns false when the CTA is aborting. `site` identifies
 * the caller in the status word. */
__device__ __forceinline__ bool mbar_wait_slow(const Ctx &c, uint32_t bar, uint32_t parity, int site) {
    unsigned long long t0 = global_ns();
    for (uint32_t spin = 0;; spin++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 63u) == 63u) {
            if (*c.abort_flag) return false;
            if (global_ns() - t0 > c.wait_ns || spin > (1u << 26)) {
                give_up(c, site, parity);
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool mbar_wait(const Ctx &c, int idx, uint32_t parity, int site) {
    uint32_t bar = c.bars + idx * 8;
    if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait_slow(c, bar, parity, site);
}

/* Scores of masked / out-of-range keys become -inf. */
__device__ __forceinline__ void mask_chunk(uint32_t *v, uint32_t bits) {
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (!((bits >> i) & 1u)) v[i] = 0xFF800000u;
}

/* Half an S row (64 scores) -> P (bf16 pairs into 32 columns at tP) and the
 * four partial row sums: one fp32 exponential per score. */
__device__ __forceinline__ void exp_half(const uint32_t *s, float sl2, float neg_ref, float *sum4, uint32_t tP) {
#pragma unroll
    for (int ch = 0; ch < 2; ch++) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float x0 = fmaf(__uint_as_float(s[ch * 32 + 2 * i]), sl2, neg_ref);
            float x1 = fmaf(__uint_as_float(s[ch * 32 + 2 * i + 1]), sl2, neg_ref);
            float p0 = ex2(x0);
            float p1 = ex2(x1);
            sum4[(2 * i) & 3] += p0;
            sum4[(2 * i + 1) & 3] += p1;
            pk[i] = cvt_bf16x2(p0, p1);
        }
        tmem_st16(tP + ch * 16, pk);
    }
}

}  // namespace sm100
}  // namespace iris_b200
