"""Exception types of the ABI statuses: the reference compiler's own where it is importable.

The kernel ABI (``mgc_cuda.native``, ``mgc_cuda.paged``) needs no reference compiler; without one
the same names are plain exceptions, so a caller's ``except`` clauses read the same.
"""

from __future__ import annotations

try:
    from mgc_cuda import _reference  # noqa: F401
    from ml_graph_compiler.errors import CodegenError, GraphError
except ImportError:

    class CodegenError(Exception):  # type: ignore[no-redef]
        """A library build or an ABI call failed."""

    class GraphError(Exception):  # type: ignore[no-redef]
        """An operand does not fit the operator, or a device index was out of range."""


__all__ = ["CodegenError", "GraphError"]
