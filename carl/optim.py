"""Alias of carl_amd.optim."""
import sys as _sys

import carl_amd.optim as _impl

_sys.modules[__name__] = _impl
