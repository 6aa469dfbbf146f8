"""torch brings a HIP runtime of its own. A process can hold one: whichever of torch
and the engine's library is loaded first, the second has to find that one, which
works only with torch first. Test modules load the library when they are collected."""
try:
    import torch  # noqa: F401
except ImportError:  # the engine's own tests need none
    pass
