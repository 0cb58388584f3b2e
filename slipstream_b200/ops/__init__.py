"""Hand-written sm_100a kernels and their Python entry points."""

from .functions import *  # noqa: F401,F403
from .functions import __all__ as _functions
from .int8 import *  # noqa: F401,F403
from .int8 import __all__ as _int8

__all__ = [*_functions, *_int8]
