from .base import Layer
from .linear import Dense, Dense4Bit, Flatten
from .convolutional import Conv2D
from .pooling import MaxPooling2D, AvgPooling2D
from .normalize import BatchNormalization, RMSNormalization
from .activators import ReLU, Sigmoid, Tanh, Activation, get_activator
from .ops import Input, Add
