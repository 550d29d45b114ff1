// The division of a 4-bit linear layer's launch (q4_plan.h), for a test without a GPU.
#include "q4_plan.h"

extern "C" int q4_plan_of(int rows, int n, int k, int group, int type_bytes, int sms, long long* out) {
    rk::Q4Plan p;
    if (!rk::q4_plan(rows, n, k, group, (size_t)type_bytes, sms, p)) return 0;
    const long long v[] = {p.stages, p.accs, p.sub, p.steps, p.smem, (long long)p.pass_bytes, p.grid, p.tmem_cols,
                           (long long)rk::q4_workspace(rows, k, (size_t)type_bytes)};
    for (int i = 0; i < 9; i++) out[i] = v[i];
    return 1;
}
