#include "intfa_latent_expanded.h"
namespace intfa { INTFA_DECL_EXPANDED(launch_expanded_n64_f16) { return launch_expanded<64, 32, 64, 0>(p, causal, stream); } }
