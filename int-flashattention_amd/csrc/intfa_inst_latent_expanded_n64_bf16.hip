#include "intfa_latent_expanded.h"
namespace intfa { INTFA_DECL_EXPANDED(launch_expanded_n64_bf16) { return launch_expanded<64, 32, 64, 1>(p, causal, stream); } }
