#include "intfa_paged_decode.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_d256) { return launch_paged<256>(p, sel, stream); } }
