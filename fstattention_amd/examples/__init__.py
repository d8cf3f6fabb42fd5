"""Small programs that use the framework's operators together."""
