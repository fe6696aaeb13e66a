#include "intfa_paged_prefill.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_prefill_d64) { return launch_paged_prefill<64>(p, sel, stream); } }
