"""Shared parameter-version counter (importable without the native library)."""
EPOCH = [0]
# the part of them that no parameter's own counter shows (see ``ops.param_writes``)
UNCOUNTED = [0]
