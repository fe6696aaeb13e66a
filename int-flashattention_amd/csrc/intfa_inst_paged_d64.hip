#include "intfa_paged_decode.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_d64) { return launch_paged<64>(p, sel, stream); } }
