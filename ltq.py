"""Lets `import ltq` work in a program whose working folder is the root of a checkout: the package lies in
light-tensor_b200/python, this file puts that folder on the path and hands over to it."""
import importlib
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "light-tensor_b200", "python"))
del sys.modules[__name__]
importlib.import_module("ltq")
