#include "intfa_paged_prefill.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_prefill_d256) { return launch_paged_prefill<256>(p, sel, stream); } }
