// The dense and gated layers of bf16 rows (dense.hpp).
#include "dense_ops.hpp"

template struct arcn::DenseOps<__bf16>;
