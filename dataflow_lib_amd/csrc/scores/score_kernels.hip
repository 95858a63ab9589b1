/*
 * Single translation unit of the scoring ops' gfx950 code object (a code
 * object of its own, so that a program without these ops does not load it).
 */
#include "token_logprobs.hip"
#include "token_logprobs_bwd.hip"
#include "distillation_loss.hip"
