"""The compiled torch glue, looked up once."""
from __future__ import annotations

import functools


@functools.lru_cache(maxsize=None)
def glue():
    """``nangila._cuda``. Raises with a clear message when it has not been built."""
    from ..parallel.predres_engine import _glue

    return _glue()
