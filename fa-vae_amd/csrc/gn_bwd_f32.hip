// Backward of group norm with an activation, f32
#include "groupnorm_bwd.h"

int gn_bwd_f32(const GnP& p, const GnPlan& pl, float* dgamma, float* dbeta, hipStream_t st) {
    return p.q ? gn_bwd<float, true>(p, pl, dgamma, dbeta, st) : gn_bwd<float, false>(p, pl, dgamma, dbeta, st);
}
