// The batched attention's cutting rule (csrc/plans.hpp) as a plain C function, for tests/test_batch_plans.py.
#include "plans.hpp"

extern "C" void attn_batch_plan_c(int B, int GRP, int NKV, int64_t P, int64_t cap, int kv_bf16, int n_cu, int* out) {
    const q35k::AttnBatchPlan p = q35k::attn_batch_plan(B, GRP, NKV, P, cap, kv_bf16 != 0, n_cu);
    out[0] = p.block;
    out[1] = p.nblk;
    out[2] = p.pieces;
    out[3] = p.pkeys;
    out[4] = p.own;
    out[5] = p.okeys;
}
