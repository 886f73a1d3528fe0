"""`import flash_evict` from a checkout's root: loads the package in flash-evict-prefill_b200/ under its own name."""
import importlib.util
import os
import sys

_package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "flash-evict-prefill_b200", "flash_evict")
_spec = importlib.util.spec_from_file_location(__name__, os.path.join(_package, "__init__.py"), submodule_search_locations=[_package])
_module = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _module  # what the import statement hands out, and where the package's own imports look
_spec.loader.exec_module(_module)
