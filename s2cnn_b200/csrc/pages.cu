// Rotation of heads by position and kept keys in pages, compiled beside lib.cu and sequence.cu (build.py).
#include "pages.h"
