// The dense and gated layers of f16 rows (dense.hpp).
#include "dense_ops.hpp"

template struct arcn::DenseOps<_Float16>;
