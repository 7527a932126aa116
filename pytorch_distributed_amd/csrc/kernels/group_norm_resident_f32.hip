// The register-resident group norm kernels of one element type (a file each, so that they compile side by side).
#define GN_INSTANTIATE
#include "group_norm_resident.h"

template int gn_resident_fwd<float>(const GnPlan&, const GnResidentArgs&);
template int gn_resident_bwd<float>(const GnPlan&, const GnResidentArgs&);
