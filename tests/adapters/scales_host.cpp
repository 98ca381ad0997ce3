// What the scales of an INT8 call belong to, behind a C interface, for tests
// that need no device.
#include "../../go-semantica_b200/csrc/host/adapter_plan.h"

extern "C" const char* sh_scales(int32_t n_absmax, int32_t n_seqs, int32_t captured, int32_t* per_seq) {
  const char* why = sem::lowrank_scales(n_absmax, n_seqs, captured != 0, per_seq);
  return why ? why : "";
}
