"""Alias of carl_amd.ops."""
import sys as _sys

import carl_amd.ops as _impl

_sys.modules[__name__] = _impl
