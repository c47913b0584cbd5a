// Attention over pages, and copying them, compiled beside lib.cu (build.py).
#include "pages.h"
