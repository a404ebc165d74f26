from .conv import *
from .activations import *
from .normalizations import *
from .experts import *
from . import functional
