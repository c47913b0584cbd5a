// The operators for sequences of signals, compiled beside lib.cu and parts.cu (build.py).
#include "sequence.h"
