#include "intfa_latent_attn.h"
namespace intfa { INTFA_DECL_LATENT(launch_latent_c256_r64_bf16) { return launch_latent<256, 64, 1>(p, rows, stream); } }
