#include "intfa_latent_attn.h"
namespace intfa { INTFA_DECL_LATENT(launch_latent_c512_r32_bf16) { return launch_latent<512, 32, 1>(p, rows, stream); } }
