// The rotation of heads by position, compiled beside lib.cu (build.py).
#include "heads.h"
