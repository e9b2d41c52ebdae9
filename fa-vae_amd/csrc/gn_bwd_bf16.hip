// Backward of group norm with an activation, bf16
#include "groupnorm_bwd.h"

int gn_bwd_bf16(const GnP& p, const GnPlan& pl, float* dgamma, float* dbeta, hipStream_t st) {
    return p.q ? gn_bwd<bf16_t, true>(p, pl, dgamma, dbeta, st) : gn_bwd<bf16_t, false>(p, pl, dgamma, dbeta, st);
}
